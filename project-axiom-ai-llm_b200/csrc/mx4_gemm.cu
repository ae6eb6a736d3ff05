// Products of microscaled 4-bit matrices on the tensor cores (tcgen05.mma kind::mxf4, e2m1 codes,
// one power-of-two scale byte per 32 elements of the reduction, fp32 accumulators in tensor
// memory), grouped over the layer's segment table:
//
//   kModeLinear  out[r][n] = sum_k A[r][k] W[e][n][k]                      (fp32 or bf16 rows)
//   kModeGated   h[r][f]   = q4( silu(g) u ),  g = A[r] . Wg[e][f],  u = A[r] . Wu[e][f]
//
// The second keeps the whole gate: both projections run in one accumulator (columns 0..127 gate,
// 128..255 up), the epilogue thread that owns a row multiplies, finds each 32-block's largest
// magnitude in its own registers and writes codes and scale bytes, so the intermediate of the
// expert feed-forward touches memory at 4.25 bits a value and is the next product's A operand as
// it lies.  The bf16 form of the same operator is grouped_ffn_2sm.cu
// (core/src/CUDA/kernel/moe_router.cu:155-190 of the reference engine).
//
// Thread-block clusters of two CTAs, cta_group::2: M = 256 over the pair, N = 256, a stage of 256
// reduction elements = 128 bytes of codes a row.  Each CTA loads its 128 rows of A, 128 of the 256
// weight rows (Gated: the leader the gate rows, the peer the up rows) and the scale bytes of its
// own A rows and of ALL 256 weight rows: 35 KB a stage, six stages.  At the 4-bit rate a stage
// lasts about 520 cycles, so a single CTA's 128 x 256 tile (51 KB a stage) would ask more of L2
// than it gives; the pair form asks 67 bytes a cycle and SM.
// Scale bytes go from shared to tensor memory with tcgen05.cp (32 lanes x 16 bytes, repeated in
// the four lane quarters), in order with the MMAs of the same issuing thread.
//
// Tensor memory: two 256-column accumulators and 24 columns of scales do not fit in 512 columns.
// The accumulators overlap: the first is columns 0..255, the second 232..487, scales 488..511.
// The epilogue takes the 32-column blocks that hold the shared columns first and then lets the
// next tile's MMAs start; everything else of it runs under them.
//
// Measured: 8192 rows 4096 -> 14336 185 us (5.2 PFLOP/s) in a short run, 8 experts 4096 x 14336 over 16384 rows
// gated 720 us, linear 344 us (5.4 and 5.6 PFLOP/s); back to back the power cap holds them to 4.0-4.8.  A stage took
// 630 cycles where its MMAs take 511 (8192 rows, 14336 -> 4096).
#include "gemm_2sm.cuh"
#include "microscale.cuh"

namespace axm {

namespace {

enum { kModeLinear = 0, kModeGated = 1 };

constexpr int kKStage = 256;                          // reduction elements a stage
constexpr int kCodeBytes = 128 * kKStage / 2;         // 16 KiB: 128 rows of A, or of the weights
constexpr int kScaleABytes = 2 * 512;                 // this CTA's 128 rows, two 128-element chunks
constexpr int kScaleBBytes = 4 * 512;                 // 256 weight rows
constexpr int kStageBytes4 = 2 * kCodeBytes + kScaleABytes + kScaleBBytes;
constexpr int kStages4 = 6;
constexpr int kThreads4 = 192;

constexpr uint32_t kAcc1 = 232;   // first column of the second accumulator
constexpr uint32_t kSfA = 488;    // 2 x 4 columns
constexpr uint32_t kSfB = 496;    // 2 x 8 columns

struct __align__(8) Mx4Shared {
  uint64_t full[kStages4];   // used in the leader: bytes of both CTAs land here
  uint64_t empty[kStages4];  // own: the leader's MMA commit arrives in both CTAs
  uint64_t tmem_full[2];     // own
  uint64_t overlap_free;     // used in the leader: 4 epilogue warps of each CTA, once a tile
  uint32_t tmem_base;
  int abort_flag;
  int total_units;
  int num_groups;
  int tile_prefix[kMaxSegments + 1];
  int group_first[kMaxSegments + 1];
  int pair_prefix[kMaxSegments + 1];
  AxmSegment seg[kMaxSegments];
};
constexpr size_t kMx4SmemBytes = 1024 + (size_t)kStages4 * kStageBytes4 + sizeof(Mx4Shared);
static_assert(kMx4SmemBytes <= 227u * 1024u, "shared memory of the 4-bit pair kernel");

struct Mx4Args {
  const AxmSegment* segments;
  int num_segments;
  int n_total;       // Linear: columns of out; Gated: columns of h
  int k_total;
  int rows_total;    // of the operand and of the output; without a segment table: of the one segment
  int seg_base;      // index of segments[0] in the layer's whole table (scale tiles count from there)
  int experts;
  int expert_base;   // expert id of the first weight matrix
  int out_bf16;      // Linear
  int wn_tiles;      // 128-row tiles of one expert's weights
  void* out;         // Linear: rows of n_total; Gated: codes
  uint8_t* out_scales;
  int* status;
};

// Block-scaled kind::mxf4: A and B e2m1 (code 1), scale type ue8m0 (bit 23), M = 256 over the
// pair, N = 256, both operands K-major.  Bits 29..30 and 4..5 pick the byte pair of the scale
// words of A and B: the two 64-element steps of a 128-element chunk.
constexpr uint32_t mx4_instr_desc(uint32_t step) {
  return ((step * 2u) << 4) | (1u << 7) | (1u << 10) | ((256u >> 3) << 17) | (1u << 23) | ((256u >> 4) << 24) |
         ((step * 2u) << 29);
}

__device__ __forceinline__ void tc_mma2_mx4(uint32_t d_tmem, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                            uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
      "}" ::"r"(d_tmem),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 512 bytes of shared memory (32 rows of 16) to four columns of tensor memory, the same in all four
// lane quarters, in both CTAs of the pair.
__device__ __forceinline__ void tc_cp2_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
struct Unit4 {
  int seg, m_tile, n_tile, seg0;
  bool live;  // false: this half of the pair has no rows
};

// Units are ordered like those of the bf16 pair kernel: expert group by expert group, inside a
// group column tile by column tile, and pairs of row tiles innermost, so that CTA pairs that run
// together share a weight tile.
__device__ __forceinline__ Unit4 decode4(const Mx4Shared* sh, int n_tiles, int unit, int rank) {
  int lo = 0, hi = sh->num_groups - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sh->pair_prefix[mid] * n_tiles <= unit) lo = mid; else hi = mid - 1;
  }
  const int s0 = sh->group_first[lo], s1 = sh->group_first[lo + 1];
  const int base = sh->tile_prefix[s0];
  const int mt = sh->tile_prefix[s1] - base;
  const int pairs = sh->pair_prefix[lo + 1] - sh->pair_prefix[lo];
  const int local = unit - sh->pair_prefix[lo] * n_tiles;
  Unit4 u;
  u.n_tile = local / pairs;
  const int p = local - u.n_tile * pairs;
  u.seg0 = s0;
  u.live = 2 * p + rank < mt;
  const int idx = base + 2 * p + (u.live ? rank : 0);
  int a = s0, b = s1 - 1;
  while (a < b) {
    const int mid = (a + b + 1) >> 1;
    if (sh->tile_prefix[mid] <= idx) a = mid; else b = mid - 1;
  }
  u.seg = a;
  u.m_tile = idx - sh->tile_prefix[a];
  return u;
}

// silu(g) u, and the block's codes and scale byte
__device__ __forceinline__ uint4 gate_block(const uint32_t (&g)[32], const uint32_t (&u)[32], uint32_t& byte) {
  float h[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    const float gv = __uint_as_float(g[j]);
    h[j] = __fdividef(gv, 1.0f + __expf(-gv)) * __uint_as_float(u[j]);
  }
  return mx4_quantize_block(h, byte);
}

// The epilogue of one tile by one of four warps: 128 accumulator rows from `acc` on, a row a thread.
// free_shared() (one lane) is called once the columns that both accumulators use have been read.
template <int kMode, typename Free>
__device__ __forceinline__ void drain_tile(const Mx4Args& args, const Unit4& u, const AxmSegment& sg, uint32_t tmem_base,
                                           int acc, int n_tiles, Free free_shared) {
  constexpr bool kGated = kMode == kModeGated;
  constexpr int kCols = kGated ? 128 : 256;
  const int lane = threadIdx.x & 31, quad = (threadIdx.x >> 5) & 3;
  const int row_in_seg = u.m_tile * 128 + quad * 32 + lane;
  const bool row_ok = u.live && row_in_seg < sg.rows;
  const size_t row = (size_t)sg.out_row0 + (row_ok ? row_in_seg : 0);
  const uint32_t t_addr = tmem_base + ((uint32_t)(quad * 32) << 16) + (acc ? kAcc1 : 0u);
  const int n0 = u.n_tile * kCols;
  // blocks of 32 columns; the shared columns are the last 24 of accumulator 0 and the first
  // 24 of accumulator 1
  constexpr int kBlocks = kCols / 32;
  uint32_t sf_word = 0;
#pragma unroll 1
  for (int i = 0; i < kBlocks; ++i) {
    const int jb = acc ? i : kBlocks - 1 - i;
    const int c0 = jb * 32;
    uint32_t v[32];
    __syncwarp();
    tmem_ld32(t_addr + c0, v);
    if constexpr (kGated) {
      uint32_t up[32];
      tmem_ld32(t_addr + 128 + c0, up);
      tmem_ld_wait();
      if (i == 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) free_shared();
      }
      if (u.live && n0 + c0 < args.n_total) {  // n_total is a multiple of 32
        uint32_t byte;
        const uint4 q = gate_block(v, up, byte);
        sf_word |= byte << (8 * jb);
        if (row_ok)
          __stcs(reinterpret_cast<uint4*>(static_cast<uint8_t*>(args.out) + row * (size_t)(args.n_total >> 1) +
                                          ((n0 + c0) >> 1)), q);
      }
    } else {
      tmem_ld_wait();
      if (i == 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) free_shared();
      }
      if (row_ok) {
        if (args.out_bf16) {
          __nv_bfloat16* p = static_cast<__nv_bfloat16*>(args.out) + row * args.n_total + n0 + c0;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (n0 + c0 + q * 8 < args.n_total) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j)
                w[j] = pack_bf16(__uint_as_float(v[8 * q + 2 * j]), __uint_as_float(v[8 * q + 2 * j + 1]));
              __stcs(reinterpret_cast<uint4*>(p + q * 8), make_uint4(w[0], w[1], w[2], w[3]));
            }
        } else {
          float* p = static_cast<float*>(args.out) + row * args.n_total + n0 + c0;
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (n0 + c0 + q * 4 < args.n_total)
              __stcs(reinterpret_cast<uint4*>(p + q * 4), make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]));
        }
      }
    }
  }
  if constexpr (kGated) {
    // one chunk of scale bytes a tile (128 columns); behind the last one of an odd number, zeros
    if (row_ok) {
      const int r = row_in_seg & 127;
      const size_t t = (size_t)(sg.out_row0 / 128 + args.seg_base + u.seg + u.m_tile);
      const int chunks = mx4_chunks(args.n_total);
      uint8_t* p = args.out_scales + (t * chunks + u.n_tile) * 512 + (r & 31) * 16 + (r >> 5) * 4;
      *reinterpret_cast<uint32_t*>(p) = sf_word;
      if (u.n_tile == n_tiles - 1 && n_tiles < chunks) *reinterpret_cast<uint32_t*>(p + 512) = 0u;
    }
  }
}

template <int kMode>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads4, 1)
mx4_gemm_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_a_sf,
                     const __grid_constant__ CUtensorMap tm_b0, const __grid_constant__ CUtensorMap tm_b1,
                     const __grid_constant__ CUtensorMap tm_b0_sf, const __grid_constant__ CUtensorMap tm_b1_sf,
                     Mx4Args args) {
  constexpr bool kGated = kMode == kModeGated;
  constexpr int kCols = kGated ? 128 : 256;  // output columns a tile
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  // all codes first (1024-byte aligned stages of 32 KiB), then the scale bytes, then the control block
  unsigned char* scales_s = tiles + (size_t)kStages4 * 2 * kCodeBytes;
  Mx4Shared* sh = reinterpret_cast<Mx4Shared*>(scales_s + (size_t)kStages4 * (kScaleABytes + kScaleBBytes));

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t peer = rank ^ 1u;
  const int cluster_id = blockIdx.x >> 1;
  const int num_clusters = gridDim.x >> 1;
  const int n_tiles = (args.n_total + kCols - 1) / kCols;
  const int k_blocks = (args.k_total + kKStage - 1) / kKStage;
  const int nseg = args.num_segments;

  for (int s = threadIdx.x; s < nseg; s += kThreads4)
    sh->seg[s] = product_segment(args.segments, s, args.rows_total, args.expert_base, args.experts);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages4; ++i) {
      mbar_init(&sh->full[i], 1);
      mbar_init(&sh->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&sh->tmem_full[i], 1);
    mbar_init(&sh->overlap_free, 8);
    sh->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_a_sf);
    tma_prefetch_desc(&tm_b0);
    tma_prefetch_desc(&tm_b0_sf);
    if (kGated) {
      tma_prefetch_desc(&tm_b1);
      tma_prefetch_desc(&tm_b1_sf);
    }
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tmem_alloc2(&sh->tmem_base, kTmemCols);
    tmem_relinquish2();
  }
  if (warp == 0) count_tiles(sh, nseg, n_tiles);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();

  const int total_units = sh->total_units;
  const uint32_t tmem_base = sh->tmem_base;
  volatile int* abort_flag = &sh->abort_flag;
  auto raise_abort = [&]() { st_cluster_u32(map_to_cta(smem_u32(&sh->abort_flag), peer), 1u); };

  if (warp == 0) {
    // ---- TMA producer --------------------------------------------------------------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int unit = cluster_id; ok && unit < total_units; unit += num_clusters) {
        const Unit4 uc = decode4(sh, n_tiles, unit, (int)rank);
        const AxmSegment sg = sh->seg[uc.seg];
        const int e = (sh->seg[uc.seg0].expert & 0xffff) - args.expert_base;
        const int a_row = sg.out_row0 + uc.m_tile * 128;
        const int a_tile = sg.out_row0 / 128 + args.seg_base + uc.seg + uc.m_tile;
        const CUtensorMap* mb = kGated && rank == 1 ? &tm_b1 : &tm_b0;
        const int n_row = uc.n_tile * kCols + (kGated ? 0 : (int)rank * 128);
        const int b_tile = e * args.wn_tiles + (kGated ? uc.n_tile : 2 * uc.n_tile);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&sh->empty[stage], phase ^ 1u, abort_flag)) {
            raise_abort();
            ok = false;
            break;
          }
          unsigned char* sa = tiles + (size_t)stage * 2 * kCodeBytes;
          unsigned char* ssf = scales_s + (size_t)stage * (kScaleABytes + kScaleBBytes);
          if (rank == 0) mbar_expect_tx(&sh->full[stage], 2 * kStageBytes4);
          const uint32_t bar = map_to_cta(smem_u32(&sh->full[stage]), 0);
          tma2_load_3d(sa, &tm_a, bar, kb * (kKStage / 2), a_row, 0);
          tma2_load_3d(sa + kCodeBytes, mb, bar, kb * (kKStage / 2), n_row, e);
          tma2_load_3d(ssf, &tm_a_sf, bar, 0, kb * 2, a_tile);
          if constexpr (kGated) {
            tma2_load_3d(ssf + kScaleABytes, &tm_b0_sf, bar, 0, kb * 2, b_tile);
            tma2_load_3d(ssf + kScaleABytes + 1024, &tm_b1_sf, bar, 0, kb * 2, b_tile);
          } else {
            tma2_load_3d(ssf + kScaleABytes, &tm_b0_sf, bar, 0, kb * 2, b_tile);
            // a weight matrix with an odd number of tiles: the next expert's bytes, or the fill
            // value behind the last one; they scale columns that are not stored
            tma2_load_3d(ssf + kScaleABytes + 1024, &tm_b0_sf, bar, 0, kb * 2, b_tile + 1);
          }
          if (++stage == kStages4) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issuer: the leader CTA only -----------------------------------------------------
    // The whole warp runs the loop, one elected lane issues (see elect_one): with one lane running it,
    // issuing a stage's ten tcgen05 instructions took about 900 cycles, the MMAs themselves 520.
    if (rank == 0) {
      const uint64_t codes0 = make_smem_desc(smem_u32(tiles), 16, 1024);
      const uint64_t scales0 = scale_desc(smem_u32(scales_s));
      int stage = 0;
      uint32_t phase = 0;
      int tile = 0;
      bool ok = true;
      for (int unit = cluster_id; ok && unit < total_units; unit += num_clusters, ++tile) {
        // the previous tile's epilogue has taken the columns both accumulators share (and, as it
        // works tile by tile, has finished the tile before)
        if (!__all_sync(0xffffffffu, mbar_wait(&sh->overlap_free, (uint32_t)(tile & 1) ^ 1u, abort_flag))) {
          if (lane == 0) raise_abort();
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + ((tile & 1) ? kAcc1 : 0u);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait(&sh->full[stage], phase, abort_flag))) {
            if (lane == 0) raise_abort();
            ok = false;
            break;
          }
          tc_fence_after();
          // descriptors count in 16-byte units
          const uint64_t da = codes0 + (uint64_t)(stage * (2 * kCodeBytes / 16));
          const uint64_t db = da + kCodeBytes / 16;
          const uint64_t sf = scales0 + (uint64_t)(stage * ((kScaleABytes + kScaleBBytes) / 16));
          if (elect_one()) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              tc_cp2_scales(tmem_base + kSfA + 4 * c, sf + 32 * c);
              tc_cp2_scales(tmem_base + kSfB + 8 * c, sf + kScaleABytes / 16 + 32 * c);
              tc_cp2_scales(tmem_base + kSfB + 8 * c + 4, sf + (kScaleABytes + 1024) / 16 + 32 * c);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)  // 64 elements = 32 bytes a step
              tc_mma2_mx4(d_tmem, da + (uint64_t)(j * 2), db + (uint64_t)(j * 2), mx4_instr_desc(j & 1),
                          tmem_base + kSfA + 4 * (j >> 1), tmem_base + kSfB + 8 * (j >> 1), (kb > 0 || j > 0) ? 1u : 0u);
            tc_commit2_both(smem_u32(&sh->empty[stage]));
          }
          __syncwarp();
          if (++stage == kStages4) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (elect_one()) {
          tc_commit2_both(smem_u32(&sh->tmem_full[tile & 1]));
        }
        __syncwarp();
      }
    }
  } else {
    // ---- epilogue: every CTA drains its own 128 accumulator rows --------------------------------
    const uint32_t leader_free = map_to_cta(smem_u32(&sh->overlap_free), 0);
    int tile = 0;
    for (int unit = cluster_id; unit < total_units; unit += num_clusters, ++tile) {
      const Unit4 uc = decode4(sh, n_tiles, unit, (int)rank);
      if (!__all_sync(0xffffffffu, mbar_wait(&sh->tmem_full[tile & 1], (uint32_t)((tile >> 1) & 1), abort_flag))) break;
      tc_fence_after();
      drain_tile<kMode>(args, uc, sh->seg[uc.seg], tmem_base, tile & 1, n_tiles, [&] { mbar_arrive_cluster(leader_free); });
    }
  }

  // ---- drain: nobody leaves while the peer may still touch its shared memory or TMEM -----------
  tc_fence_before();
  __syncthreads();
  if (sh->abort_flag != 0) {
    long long t0 = clock64();
    while (clock64() - t0 < 4000000LL) {
    }
    if (threadIdx.x == 0 && args.status != nullptr) atomicExch(args.status, kGated ? 11 : 12);
  }
  cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc2(tmem_base, kTmemCols);
  }
}

// ---- the same tile on one CTA -----------------------------------------------------------------
// For segments of up to about a hundred rows, whose time is the weights' way in: a pair's second CTA would
// have no rows of its own there; and for all segments where pairs are not wanted or cannot be scheduled.
// M = 128 rows, N = 256 weight rows, all of them staged by the CTA itself: 51 KB a stage, four stages.  The
// first ring of weights is asked for before the kernel before this one has finished (the weights do not
// depend on it).
constexpr int kStages1 = 4;
constexpr int kStageCodes1 = 3 * kCodeBytes;
constexpr int kStageScales1 = kScaleABytes + kScaleBBytes;
constexpr int kStageBytes1 = kStageCodes1 + kStageScales1;
static_assert(kStages1 <= kStages4, "the control block is the pair kernel's");
constexpr size_t kMx4SmemBytes1 = 1024 + (size_t)kStages1 * kStageBytes1 + sizeof(Mx4Shared);
static_assert(kMx4SmemBytes1 <= 227u * 1024u, "shared memory of the 4-bit one-CTA kernel");

constexpr uint32_t mx4_instr_desc1(uint32_t step) {  // M = 128 of one CTA
  return (mx4_instr_desc(step) & ~(0x1fu << 24)) | ((128u >> 4) << 24);
}
// Units: expert group by expert group, column tile by column tile, row tiles innermost.
__device__ __forceinline__ Unit4 decode1(const Mx4Shared* sh, int n_tiles, int unit) {
  int lo = 0, hi = sh->num_groups - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sh->tile_prefix[sh->group_first[mid]] * n_tiles <= unit) lo = mid; else hi = mid - 1;
  }
  const int s0 = sh->group_first[lo], s1 = sh->group_first[lo + 1];
  const int base = sh->tile_prefix[s0];
  const int mt = sh->tile_prefix[s1] - base;
  const int local = unit - base * n_tiles;
  Unit4 u;
  u.seg0 = s0;
  u.live = true;
  u.n_tile = local / mt;
  const int idx = base + local - u.n_tile * mt;
  int a = s0, b = s1 - 1;
  while (a < b) {
    const int mid = (a + b + 1) >> 1;
    if (sh->tile_prefix[mid] <= idx) a = mid; else b = mid - 1;
  }
  u.seg = a;
  u.m_tile = idx - sh->tile_prefix[a];
  return u;
}

template <int kMode>
__global__ void __launch_bounds__(kThreads4, 1)
mx4_gemm_single_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_a_sf,
                       const __grid_constant__ CUtensorMap tm_b0, const __grid_constant__ CUtensorMap tm_b1,
                       const __grid_constant__ CUtensorMap tm_b0_sf, const __grid_constant__ CUtensorMap tm_b1_sf,
                       Mx4Args args) {
  constexpr bool kGated = kMode == kModeGated;
  constexpr int kCols = kGated ? 128 : 256;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* scales_s = tiles + (size_t)kStages1 * kStageCodes1;
  Mx4Shared* sh = reinterpret_cast<Mx4Shared*>(scales_s + (size_t)kStages1 * kStageScales1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int n_tiles = (args.n_total + kCols - 1) / kCols;
  const int k_blocks = (args.k_total + kKStage - 1) / kKStage;
  const int nseg = args.num_segments;

  launch_dependents();
  // the segment table is older than the kernel before this one, which has waited for everything before
  // itself
  for (int s = threadIdx.x; s < nseg; s += kThreads4)
    sh->seg[s] = product_segment(args.segments, s, args.rows_total, args.expert_base, args.experts);
  if (threadIdx.x == 32) {
    for (int i = 0; i < kStages1; ++i) {
      mbar_init(&sh->full[i], 1);
      mbar_init(&sh->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&sh->tmem_full[i], 1);
    mbar_init(&sh->overlap_free, 4);
    sh->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_b0);
    tma_prefetch_desc(&tm_b0_sf);
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_a_sf);
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(&sh->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  __syncthreads();
  if (warp == 0) count_tiles(sh, nseg, n_tiles);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  const int total_units = sh->tile_prefix[nseg] * n_tiles;
  const uint32_t tmem_base = sh->tmem_base;
  volatile int* abort_flag = &sh->abort_flag;
  const int first = blockIdx.x, step = gridDim.x;

  if (warp == 0) {
    // ---- TMA producer --------------------------------------------------------------------
    if (lane == 0) {
      auto weights = [&](int stage, const Unit4& u, int kb) {
        const int e = (sh->seg[u.seg0].expert & 0xffff) - args.expert_base;
        unsigned char* sb = tiles + (size_t)stage * kStageCodes1 + kCodeBytes;
        unsigned char* sf = scales_s + (size_t)stage * kStageScales1 + kScaleABytes;
        uint64_t* bar = &sh->full[stage];
        const int row = u.n_tile * kCols, tile = e * args.wn_tiles + (kGated ? u.n_tile : 2 * u.n_tile);
        mbar_expect_tx(bar, kStageBytes1);
        tma_load_3d(sb, &tm_b0, bar, kb * (kKStage / 2), row, e);
        tma_load_3d(sb + kCodeBytes, kGated ? &tm_b1 : &tm_b0, bar, kb * (kKStage / 2), kGated ? row : row + 128, e);
        tma_load_3d(sf, &tm_b0_sf, bar, 0, kb * 2, tile);
        // (linear: behind an odd number of tiles the next expert's bytes or the fill value; they scale
        // columns that are not stored)
        tma_load_3d(sf + 1024, kGated ? &tm_b1_sf : &tm_b0_sf, bar, 0, kb * 2, kGated ? tile : tile + 1);
      };
      auto rows = [&](int stage, const Unit4& u, int kb) {
        const AxmSegment sg = sh->seg[u.seg];
        uint64_t* bar = &sh->full[stage];
        tma_load_3d(tiles + (size_t)stage * kStageCodes1, &tm_a, bar, kb * (kKStage / 2), sg.out_row0 + u.m_tile * 128, 0);
        tma_load_3d(scales_s + (size_t)stage * kStageScales1, &tm_a_sf, bar, 0, kb * 2,
                    sg.out_row0 / 128 + args.seg_base + u.seg + u.m_tile);
      };
      // the first ring: weights, then, once the kernel before is done, the rows
      int ahead = 0;
      for (int unit = first; ahead < kStages1 && unit < total_units; unit += step) {
        const Unit4 u = decode1(sh, n_tiles, unit);
        for (int kb = 0; kb < k_blocks && ahead < kStages1; ++kb, ++ahead) weights(ahead, u, kb);
      }
      wait_for_previous();
      int at = 0, stage = 0;  // stages of the first ring that have their rows
      uint32_t phase = 0;
      bool ok = true;
      for (int unit = first; ok && unit < total_units; unit += step) {
        const Unit4 u = decode1(sh, n_tiles, unit);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (at < ahead) {
            ++at;
          } else {
            if (!mbar_wait(&sh->empty[stage], phase ^ 1u, abort_flag)) {
              ok = false;
              break;
            }
            weights(stage, u, kb);
          }
          rows(stage, u, kb);
          if (++stage == kStages1) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issuer (the whole warp, one elected lane issues) -----------------------------------
    const uint64_t codes0 = make_smem_desc(smem_u32(tiles), 16, 1024);
    const uint64_t scales0 = scale_desc(smem_u32(scales_s));
    int stage = 0;
    uint32_t phase = 0;
    int tile = 0;
    bool ok = true;
    for (int unit = first; ok && unit < total_units; unit += step, ++tile) {
      if (!__all_sync(0xffffffffu, mbar_wait(&sh->overlap_free, (uint32_t)(tile & 1) ^ 1u, abort_flag))) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + ((tile & 1) ? kAcc1 : 0u);
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (!__all_sync(0xffffffffu, mbar_wait(&sh->full[stage], phase, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t da = codes0 + (uint64_t)(stage * (kStageCodes1 / 16));
        const uint64_t db = da + kCodeBytes / 16;
        const uint64_t sf = scales0 + (uint64_t)(stage * (kStageScales1 / 16));
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            tc_cp1_scales(tmem_base + kSfA + 4 * c, sf + 32 * c);
            tc_cp1_scales(tmem_base + kSfB + 8 * c, sf + kScaleABytes / 16 + 32 * c);
            tc_cp1_scales(tmem_base + kSfB + 8 * c + 4, sf + (kScaleABytes + 1024) / 16 + 32 * c);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            tc_mma1_mx4(d_tmem, da + (uint64_t)(j * 2), db + (uint64_t)(j * 2), mx4_instr_desc1(j & 1),
                        tmem_base + kSfA + 4 * (j >> 1), tmem_base + kSfB + 8 * (j >> 1), (kb > 0 || j > 0) ? 1u : 0u);
          tc_commit(&sh->empty[stage]);
        }
        __syncwarp();
        if (++stage == kStages1) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      if (elect_one()) tc_commit(&sh->tmem_full[tile & 1]);
      __syncwarp();
    }
  } else {
    // ---- epilogue --------------------------------------------------------------------------------
    wait_for_previous();  // outputs and scratch of the kernels before
    int tile = 0;
    for (int unit = first; unit < total_units; unit += step, ++tile) {
      const Unit4 u = decode1(sh, n_tiles, unit);
      if (!__all_sync(0xffffffffu, mbar_wait(&sh->tmem_full[tile & 1], (uint32_t)((tile >> 1) & 1), abort_flag))) break;
      tc_fence_after();
      drain_tile<kMode>(args, u, sh->seg[u.seg], tmem_base, tile & 1, n_tiles, [&] { mbar_arrive(&sh->overlap_free); });
    }
  }

  tc_fence_before();
  __syncthreads();
  if (sh->abort_flag != 0) {
    long long t0 = clock64();
    while (clock64() - t0 < 4000000LL) {
    }
    if (threadIdx.x == 0 && args.status != nullptr) atomicExch(args.status, kGated ? 15 : 16);
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ---- host side -----------------------------------------------------------------------------

template <int kMode>
int launch_tiles(const CUtensorMap& a, const CUtensorMap& a_sf, const CUtensorMap& b0, const CUtensorMap& b1,
                const CUtensorMap& b0_sf, const CUtensorMap& b1_sf, const Mx4Args& args, bool single, cudaStream_t st) {
  static SmemLimitCache smem = {}, smem1 = {};
  int grid = 0;
  if (!single && use_2sm_kernels()) {
    grid = grid_2sm();
    if (grid < 0) return grid;
  }
  if (grid < 2) {  // few rows a segment, or no pairs: not wanted (AXM_GEMM_2SM=0) or not to be had on this device
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(mx4_gemm_single_kernel<kMode>), kMx4SmemBytes1, &smem1,
                                     "mx4_gemm_single_kernel"))
      return rc;
    return launch_overlapping("mx4_gemm_single_kernel", mx4_gemm_single_kernel<kMode>, sm_count(), kThreads4, kMx4SmemBytes1,
                              st, a, a_sf, b0, b1, b0_sf, b1_sf, args);
  }
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(mx4_gemm_pair_kernel<kMode>), kMx4SmemBytes, &smem,
                                   "mx4_gemm_pair_kernel"))
    return rc;
  mx4_gemm_pair_kernel<kMode><<<grid, kThreads4, kMx4SmemBytes, st>>>(a, a_sf, b0, b1, b0_sf, b1_sf, args);
  return check_launch("mx4_gemm_pair_kernel");
}

}  // namespace

int mx4_map_codes(CUtensorMap* m, const void* base, uint64_t experts, uint64_t rows, uint64_t k, uint32_t box_rows) {
  const uint64_t dims[3] = {k / 2, rows, experts};
  const uint64_t strides[2] = {k / 2, k / 2 * rows};
  const uint32_t box[3] = {128, box_rows, 1};
  return encode_tensor_map_bytes(m, base, 3, dims, strides, box);
}
int mx4_map_scales(CUtensorMap* m, const void* base, uint64_t tiles, int k) {
  const uint64_t dims[3] = {128, (uint64_t)mx4_chunks(k), tiles};
  const uint64_t strides[2] = {512, 512ull * mx4_chunks(k)};
  const uint32_t box[3] = {128, 2, 1};
  return encode_tensor_map_words(m, base, 3, dims, strides, box);
}

// The tables' rows are out_row0 .. of A, of its scale tiles and of the output alike.
static Mx4Args mx4_args(const Mx4Rows& r) {
  Mx4Args ga = {};
  ga.segments = r.segments;
  ga.num_segments = r.segments != nullptr ? r.num_segments : 1;
  ga.rows_total = r.rows;
  ga.seg_base = r.seg_base;
  ga.expert_base = r.expert_base;
  ga.status = r.status;
  return ga;
}

int launch_mx4_linear(const Mx4Rows& r, const void* a_codes, const void* a_scales, const void* w_codes,
                      const void* w_scales, int experts, int k, int n, void* out, bool out_bf16, cudaStream_t st) {
  CUtensorMap a, a_sf, b, b_sf;
  int rc;
  const int wn = (n + 127) / 128;
  if ((rc = mx4_map_codes(&a, a_codes, 1, r.rows, k, 128))) return rc;
  if ((rc = mx4_map_scales(&a_sf, a_scales, mx4_row_tiles(r.rows, r.table_segments), k))) return rc;
  if ((rc = mx4_map_codes(&b, w_codes, experts, n, k, 128))) return rc;
  if ((rc = mx4_map_scales(&b_sf, w_scales, (uint64_t)experts * wn, k))) return rc;
  Mx4Args ga = mx4_args(r);
  ga.experts = experts;
  ga.n_total = n;
  ga.k_total = k;
  ga.out_bf16 = out_bf16 ? 1 : 0;
  ga.wn_tiles = wn;
  ga.out = out;
  return launch_tiles<kModeLinear>(a, a_sf, b, b, b_sf, b_sf, ga, r.kernel == kMx4Single, st);
}

int launch_mx4_gated(const Mx4Rows& r, const void* a_codes, const void* a_scales, const AxmMx4Experts* w, int experts,
                     int d, int f, void* h_codes, void* h_scales, cudaStream_t st) {
  CUtensorMap a, a_sf, g, u, g_sf, u_sf;
  int rc;
  const int wn = (f + 127) / 128;
  if ((rc = mx4_map_codes(&a, a_codes, 1, r.rows, d, 128))) return rc;
  if ((rc = mx4_map_scales(&a_sf, a_scales, mx4_row_tiles(r.rows, r.table_segments), d))) return rc;
  if ((rc = mx4_map_codes(&g, w->gate_codes, experts, f, d, 128))) return rc;
  if ((rc = mx4_map_codes(&u, w->up_codes, experts, f, d, 128))) return rc;
  if ((rc = mx4_map_scales(&g_sf, w->gate_scales, (uint64_t)experts * wn, d))) return rc;
  if ((rc = mx4_map_scales(&u_sf, w->up_scales, (uint64_t)experts * wn, d))) return rc;
  Mx4Args ga = mx4_args(r);
  ga.experts = experts;
  ga.n_total = f;
  ga.k_total = d;
  ga.wn_tiles = wn;
  ga.out = h_codes;
  ga.out_scales = static_cast<uint8_t*>(h_scales);
  return launch_tiles<kModeGated>(a, a_sf, g, u, g_sf, u_sf, ga, r.kernel == kMx4Single, st);
}

}  // namespace axm
