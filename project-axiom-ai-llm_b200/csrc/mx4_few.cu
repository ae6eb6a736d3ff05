// The 4-bit products of calls with few rows a segment (one token, a short batch, many experts): what
// counts is how fast the weights stream in, so the roles are turned around.
//
// 128 weight rows are the M side of the MMA (cta_group::1), the segment's rows its N side (16, 32, 64 or
// 128 of them, a template parameter; a segment may have several such tiles).  The scale tiles of the
// activations are laid out with as many rows, so that each tile's bytes begin in the first column.  A stage is 256
// reduction elements: 16 KiB of codes and 1 KiB of scale bytes for the weights (twice that for gate
// and up), 128 bytes of codes a row for the activations.
//
// A unit is a weight tile (128 features) with a row tile, dealt out round robin.  An SM can pull
// more than its share of the memory's bandwidth, so tiles that do not divide evenly among the SMs cost
// nothing as long as the rest still are many; only where there are few (few_enough) is the reduction of
// each cut into equal ranges, units of their own.  A cut tile is finished by the unit that arrives last
// (a counter, nobody waits): all of them leave their partial sums in the workspace, and the last
// adds them in the order of the reduction, so the result does not depend on who was last.
// Cutting all work into equal pieces regardless (24 or 25 stages a CTA for a wide layer's 224 gate/up
// tiles) was built first and lost what it gained to the partial sums: one token's product 4096 -> 14336
// 17 us, 128 tokens 31 us.
//
// The accumulator has a feature a lane and a row a column.  Linear output is stored straight from
// there (32 neighbouring features of a row).  The gated product's values are turned over through
// shared memory, 32 rows at a time, so that a lane holds a row's 32-block and quantises it
// in registers as the pair kernel does.
//
// The weights do not depend on the kernel before: the producer asks for its first stages' weights
// before it waits for that kernel (programmatic dependent launch), then for the activations.
// Measured: one token 4096 -> 14336 10.9 us with its quantisation; one token through two experts 4096 x 14336
// gated 26.5 us (125 MB), linear 23.0 us (62 MB), overlapping by 8; 16 tokens in all 126 us (742 MB, 5.9 TB/s).
#include "gemm_2sm.cuh"
#include "microscale.cuh"

namespace axm {

namespace {

constexpr int kThreadsF = 192;
constexpr int kWCodeBytes = 128 * 128;  // 128 weight rows x 256 elements
constexpr int kScaleChunk2 = 1024;      // two 512-byte chunks

template <bool kGated, int N>
struct FewCfg {
  static constexpr int kWeights = kGated ? 2 : 1;
  static constexpr int kCodeBytes = kWeights * kWCodeBytes + N * 128;
  static constexpr int kScaleBytes = (kWeights + 1) * kScaleChunk2;
  static constexpr int kStageBytes = kCodeBytes + kScaleBytes;
  static constexpr int kFit = (198 * 1024) / kStageBytes;
  static constexpr int kStages = kFit < 10 ? kFit : 10;
  static constexpr int kAccCols = kWeights * N;
  static constexpr int kAccs = 2 * kAccCols + 48 <= 512 ? 2 : 1;
  static constexpr int kSf = kAccs * kAccCols;  // first scale column
  static constexpr int kSfCols = kWeights * 8 + 8;  // weights (8 each), then rows (8)
  static constexpr int kNeed = kSf + kSfCols;
  static constexpr int kTmem = kNeed <= 64 ? 64 : kNeed <= 128 ? 128 : kNeed <= 256 ? 256 : 512;
  static constexpr int kPartial = kWeights * N * 128;  // floats of one partial tile
};

template <int kStages>
struct __align__(8) FewShared {
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  int is_last;
  int prefix[kMaxSegments + 1];  // row tiles before segment s
  AxmSegment seg[kMaxSegments];
  float turn[4][32 * 33];  // per epilogue warp: 32 rows x 32 features
};

struct FewArgs {
  const AxmSegment* segments;
  int num_segments;
  int rows_total;
  int seg_base;
  int experts;
  int expert_base;
  int n_total;
  int k_total;
  int wn_tiles;
  int out_bf16;
  void* out;
  uint8_t* out_scales;
  float* partial;      // a partial tile a unit
  uint32_t* counters;  // one a tile, zero between launches
  int* status;
};

// Block-scaled kind::mxf4 like the pair kernel's, M = 128 of one CTA.
template <int N>
constexpr uint32_t few_instr_desc(uint32_t step) {
  return ((step * 2u) << 4) | (1u << 7) | (1u << 10) | (((uint32_t)N >> 3) << 17) | (1u << 23) | ((128u >> 4) << 24) |
         ((step * 2u) << 29);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

// Whether all 128 threads of the epilogue say yes.
__device__ __forceinline__ bool epilogue_agree(bool yes) {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.red.and.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}"
      : "=r"(r)
      : "r"((uint32_t)yes)
      : "memory");
  return r != 0;
}

struct FewTile {
  int seg, f_tile, row_tile;
};

// One CTA's units, in order.
struct Units {
  long long at, end, step;
  int splits, k_blocks, k_per;
  __device__ bool next(long long& tile, int& kb0, int& kb1) {
    if (at >= end) return false;
    tile = splits == 1 ? at : at / splits;
    kb0 = (int)(at - tile * splits) * k_per;
    kb1 = kb0 + k_per < k_blocks ? kb0 + k_per : k_blocks;
    at += step;
    return true;
  }
};
// Units below which the reduction is cut: fewer with wide row tiles, whose partial sums cost more.
// A cut call has less than twice as many.  A linear call with its quantisation, weights from HBM, uncut and cut
// by this rule, us:
//                 1 row         24 rows       48 rows       112 rows
//   11008 -> 4096 19.4 -> 12.9  19.6 -> 17.2  19.9 -> 17.1  21.1 -> 22.6
//    8192 -> 2048 15.8 -> 10.6  15.9 -> 13.4  16.3 -> 14.6  17.5 -> 19.0
//    4096 -> 4096 11.0 -> 10.0  11.3 -> 14.4  11.3 -> 13.1  12.5 -> 17.6
//    2048 -> 1024  8.5 ->  7.9   8.9 -> 11.5   9.0 -> 11.9   9.5 -> 14.8
//    1024 -> 4096  6.6 ->  7.3   6.9 ->  8.9   7.2 -> 10.2   8.3 -> 14.2
// So it gains where the reduction is long and the row tile narrow, and loses elsewhere: it does not look at the
// length of the reduction.  (A limit of 148 units: 9.3 and 10.1 for one row 4096 -> 4096 and 8192 -> 2048, but 18.9
// where 24 rows 2048 -> 8192 take 9.3.)
constexpr int few_enough(int n) { return n <= 32 ? 96 : n == 64 ? 64 : 48; }

template <bool kGated, int N>
__global__ void __launch_bounds__(kThreadsF, 1)
mx4_few_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_a_sf,
               const __grid_constant__ CUtensorMap tm_w0, const __grid_constant__ CUtensorMap tm_w1,
               const __grid_constant__ CUtensorMap tm_w0_sf, const __grid_constant__ CUtensorMap tm_w1_sf, FewArgs args) {
  using Cfg = FewCfg<kGated, N>;
  constexpr int kStages = Cfg::kStages;
  using Shared = FewShared<kStages>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* scales_s = tiles + (size_t)kStages * Cfg::kCodeBytes;
  Shared* sh = reinterpret_cast<Shared*>(scales_s + (size_t)kStages * Cfg::kScaleBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int nseg = args.num_segments;
  const int f_tiles = (args.n_total + 127) / 128;
  const int k_blocks = (args.k_total + 255) / 256;

  // the next kernel may start its own preparations; it waits for this one before it reads
  launch_dependents();

  // The segment table is older than the kernel before this one (see the launch), so it may be read
  // at once.
  for (int s = threadIdx.x; s < nseg; s += kThreadsF)
    sh->seg[s] = product_segment(args.segments, s, args.rows_total, args.expert_base, args.experts);
  if (threadIdx.x == 32) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh->full[i], 1);
      mbar_init(&sh->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh->tmem_full[i], 1);
      mbar_init(&sh->tmem_empty[i], 4);
    }
    sh->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tma_prefetch_desc(&tm_w0);
    tma_prefetch_desc(&tm_w0_sf);
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_a_sf);
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(&sh->tmem_base, Cfg::kTmem);
    tmem_relinquish();
  }
  __syncthreads();
  if (warp == 0) {  // row tiles before each segment
    int before = 0;
    for (int s0 = 0; s0 < nseg; s0 += 32) {
      const int s = s0 + lane;
      const int rows = s < nseg ? sh->seg[s].rows : 0;
      const int mine = rows > 0 ? (rows + N - 1) / N : 0;
      int sum = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += v;
      }
      if (s < nseg) sh->prefix[s] = before + sum - mine;
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) sh->prefix[nseg] = before;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  const uint32_t tmem_base = sh->tmem_base;
  volatile int* abort_flag = &sh->abort_flag;
  const long long tiles_n = (long long)sh->prefix[nseg] * f_tiles;
  int k_per = k_blocks;
  if (tiles_n > 0 && tiles_n < few_enough(N)) {
    // the last to arrive reads every range's partial tile: the larger they are, the fewer
    const int want = min(min((int)(few_enough(N) + tiles_n - 1) / (int)tiles_n, k_blocks), 256 / N);
    k_per = (k_blocks + want - 1) / want;
  }
  const int splits = (k_blocks + k_per - 1) / k_per;  // none of the ranges is empty
  const Units mine = {(long long)blockIdx.x, tiles_n * splits, (long long)gridDim.x, splits, k_blocks, k_per};

  // tiles: segment by segment, weight tile by weight tile, row tiles innermost
  auto decode = [&](long long tile) {
    int lo = 0, hi = nseg - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)sh->prefix[mid] * f_tiles <= tile) lo = mid; else hi = mid - 1;
    }
    const int row_tiles = sh->prefix[lo + 1] - sh->prefix[lo];
    const int local = (int)(tile - (long long)sh->prefix[lo] * f_tiles);
    FewTile t;
    t.seg = lo;
    t.f_tile = local / row_tiles;
    t.row_tile = local - t.f_tile * row_tiles;
    return t;
  };

  if (warp == 0) {
    // ---- producer --------------------------------------------------------------------------
    if (lane == 0) {
      auto weights = [&](int stage, const FewTile& t, int kb) {
        const int e = (sh->seg[t.seg].expert & 0xffff) - args.expert_base;
        unsigned char* codes = tiles + (size_t)stage * Cfg::kCodeBytes;
        unsigned char* sf = scales_s + (size_t)stage * Cfg::kScaleBytes;
        uint64_t* bar = &sh->full[stage];
        mbar_expect_tx(bar, Cfg::kStageBytes);
        tma_load_3d(codes, &tm_w0, bar, kb * 128, t.f_tile * 128, e);
        tma_load_3d(sf, &tm_w0_sf, bar, 0, kb * 2, e * args.wn_tiles + t.f_tile);
        if constexpr (kGated) {
          tma_load_3d(codes + kWCodeBytes, &tm_w1, bar, kb * 128, t.f_tile * 128, e);
          tma_load_3d(sf + kScaleChunk2, &tm_w1_sf, bar, 0, kb * 2, e * args.wn_tiles + t.f_tile);
        }
      };
      auto rows = [&](int stage, const FewTile& t, int kb) {
        const AxmSegment sg = sh->seg[t.seg];
        unsigned char* codes = tiles + (size_t)stage * Cfg::kCodeBytes + Cfg::kWeights * kWCodeBytes;
        unsigned char* sf = scales_s + (size_t)stage * Cfg::kScaleBytes + Cfg::kWeights * kScaleChunk2;
        uint64_t* bar = &sh->full[stage];
        tma_load_3d(codes, &tm_a, bar, kb * 128, sg.out_row0 + t.row_tile * N, 0);
        tma_load_3d(sf, &tm_a_sf, bar, 0, kb * 2,
                    sg.out_row0 / N + args.seg_base + t.seg + t.row_tile);
      };
      Units p = mine, q = mine;  // q: the activations of the stages p has asked weights for
      long long tile;
      int kb0, kb1;
      int ahead = 0;
      // the first ring of weights, before the kernel before this one has finished
      bool waited = false;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && p.next(tile, kb0, kb1)) {
        const FewTile t = decode(tile);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!waited && ahead == kStages) {
            wait_for_previous();
            waited = true;
            int n = 0;
            long long t2;
            int b0, b1;
            while (n < ahead && q.next(t2, b0, b1)) {
              const FewTile u = decode(t2);
              for (int b = b0; b < b1 && n < ahead; ++b, ++n) rows(n, u, b);
            }
          }
          if (waited && !mbar_wait(&sh->empty[stage], phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          weights(stage, t, kb);
          if (waited) rows(stage, t, kb); else ++ahead;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!waited) {
        wait_for_previous();
        int n = 0;
        long long t2;
        int b0, b1;
        while (n < ahead && q.next(t2, b0, b1)) {
          const FewTile u = decode(t2);
          for (int b = b0; b < b1 && n < ahead; ++b, ++n) rows(n, u, b);
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issuer (the whole warp, one elected lane issues) -------------------------------------
    {
      const uint64_t codes0 = make_smem_desc(smem_u32(tiles), 16, 1024);
      const uint64_t scales0 = scale_desc(smem_u32(scales_s));
      const uint32_t sf_w = tmem_base + Cfg::kSf, sf_a = sf_w + Cfg::kWeights * 8;
      int stage = 0;
      uint32_t phase = 0;
      Units p = mine;
      long long tile;
      int kb0, kb1;
      bool ok = true;
      for (int i = 0; ok && p.next(tile, kb0, kb1); ++i) {
        const int acc = Cfg::kAccs == 2 ? (i & 1) : 0;
        const uint32_t turn = Cfg::kAccs == 2 ? (uint32_t)(i >> 1) : (uint32_t)i;
        if (!__all_sync(0xffffffffu, mbar_wait(&sh->tmem_empty[acc], (turn & 1u) ^ 1u, abort_flag))) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)acc * Cfg::kAccCols;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait(&sh->full[stage], phase, abort_flag))) {
            ok = false;
            break;
          }
          tc_fence_after();
          // descriptors count in 16-byte units
          const uint64_t dw = codes0 + (uint64_t)(stage * (Cfg::kCodeBytes / 16));
          const uint64_t dr = dw + Cfg::kWeights * kWCodeBytes / 16;
          const uint64_t sf = scales0 + (uint64_t)(stage * (Cfg::kScaleBytes / 16));
          if (elect_one()) {
#pragma unroll
            for (int w = 0; w < Cfg::kWeights + 1; ++w)
#pragma unroll
              for (int c = 0; c < 2; ++c) tc_cp1_scales(sf_w + w * 8 + c * 4, sf + (w * kScaleChunk2 + c * 512) / 16);
#pragma unroll
            for (int w = 0; w < Cfg::kWeights; ++w)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                tc_mma1_mx4(d_tmem + w * N, dw + (uint64_t)(w * (kWCodeBytes / 16) + j * 2), dr + (uint64_t)(j * 2),
                            few_instr_desc<N>(j & 1), sf_w + w * 8 + 4 * (j >> 1), sf_a + 4 * (j >> 1),
                            (kb > kb0 || j > 0) ? 1u : 0u);
            tc_commit(&sh->empty[stage]);
          }
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) {
          if (elect_one()) tc_commit(&sh->tmem_full[acc]);
          __syncwarp();
        }
      }
    }
  } else {
    // ---- epilogue --------------------------------------------------------------------------------
    const int quad = warp & 3;
    float* turn_s = sh->turn[warp - 2];
    const int feature = quad * 32 + lane;
    wait_for_previous();  // outputs and partial sums of earlier launches
    Units p = mine;
    long long tile;
    int kb0, kb1;
    for (int i = 0; p.next(tile, kb0, kb1); ++i) {
      const int acc = Cfg::kAccs == 2 ? (i & 1) : 0;
      const uint32_t turn = Cfg::kAccs == 2 ? (uint32_t)(i >> 1) : (uint32_t)i;
      const FewTile t = decode(tile);
      const AxmSegment sg = sh->seg[t.seg];
      const int rows = min(sg.rows - t.row_tile * N, N);
      // the four warps go on or give up together: they meet at barriers below
      if (!epilogue_agree(mbar_wait(&sh->tmem_full[acc], turn & 1u, abort_flag))) break;
      tc_fence_after();
      const uint32_t t_addr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)acc * Cfg::kAccCols;
      const bool whole = splits == 1;
      bool finish = true;
      if (!whole) {
        // less than 2 few_enough(N) units where tiles are cut
        float* mine_p = args.partial + (size_t)(tile * splits + kb0 / k_per) * Cfg::kPartial;
#pragma unroll 1
        for (int n0 = 0; n0 < rows; n0 += 16) {
#pragma unroll
          for (int w = 0; w < Cfg::kWeights; ++w) {
            uint32_t v[16];
            __syncwarp();
            tmem_ld16(t_addr + w * N + n0, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (n0 + j < rows) __stcg(mine_p + (size_t)(w * N + n0 + j) * 128 + feature, __uint_as_float(v[j]));
          }
        }
        __threadfence();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (threadIdx.x == 64) {
          const uint32_t before = atomicAdd(args.counters + tile, 1u);
          const bool last = before == (uint32_t)(splits - 1);
          if (last) args.counters[tile] = 0u;
          sh->is_last = last ? 1 : 0;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        finish = sh->is_last != 0;
        if (finish) __threadfence();
      }
      if (finish) {
        // sixteen rows at a time: from tensor memory, or the sum of the pieces' partial tiles
        auto fetch = [&](int w, int n0, float (&v)[16]) {
          if (whole) {
            uint32_t r[16];
            __syncwarp();
            tmem_ld16(t_addr + w * N + n0, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = 0.0f;
            const float* q = args.partial + (size_t)(tile * splits) * Cfg::kPartial + (size_t)(w * N + n0) * 128 + feature;
#pragma unroll 2
            for (int z = 0; z < splits; ++z, q += Cfg::kPartial) {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (n0 + j < rows) v[j] += __ldcg(q + j * 128);
            }
          }
        };
        const int f0 = t.f_tile * 128 + quad * 32;  // this warp's 32 features
        const size_t row0 = (size_t)sg.out_row0 + t.row_tile * N;
        if constexpr (kGated) {
          const int chunks = mx4_chunks(args.n_total);
          uint8_t* sf0 = args.out_scales + ((size_t)(sg.out_row0 / N + args.seg_base + t.seg + t.row_tile) * chunks + t.f_tile) * 512;
#pragma unroll 1
          for (int n0 = 0; n0 < rows; n0 += 32) {
#pragma unroll 1
            for (int half = 0; half < (N < 32 ? 1 : 2); ++half) {
              const int m0 = n0 + 16 * half;
              if (m0 >= rows) break;
              float g[16], u[16];
              fetch(0, m0, g);
              fetch(1, m0, u);
#pragma unroll
              for (int j = 0; j < 16; ++j)
                turn_s[(16 * half + j) * 33 + lane] = __fdividef(g[j], 1.0f + __expf(-g[j])) * u[j];
            }
            __syncwarp();
            // lane j: row n0 + j, its 32 features a block (n_total is a multiple of 32); scale bytes of
            // blocks behind F are 0, as are those of the chunk behind an odd number of them
            if (n0 + lane < rows) {
              const int r = n0 + lane;
              uint8_t* sf = sf0 + (r & 31) * 16 + (r >> 5) * 4;
              uint32_t byte = 0;
              if (f0 < args.n_total) {
                float h[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) h[j] = turn_s[lane * 33 + j];
                *reinterpret_cast<uint4*>(static_cast<uint8_t*>(args.out) +
                                          (row0 + n0 + lane) * (size_t)(args.n_total >> 1) + (f0 >> 1)) =
                    mx4_quantize_block(h, byte);
              }
              sf[quad] = (uint8_t)byte;
              if (quad == 0 && t.f_tile == f_tiles - 1 && f_tiles < chunks) *reinterpret_cast<uint32_t*>(sf + 512) = 0u;
            }
            __syncwarp();
          }
        } else {
          const size_t step = args.n_total;
          size_t el = row0 * step + f0 + lane;
#pragma unroll 1
          for (int n0 = 0; n0 < rows; n0 += 16, el += 16 * step) {
            float v[16];
            fetch(0, n0, v);
            if (f0 + lane < args.n_total) {
              if (args.out_bf16) {
                __nv_bfloat16* to = static_cast<__nv_bfloat16*>(args.out) + el;
#pragma unroll
                for (int j = 0; j < 16; ++j, to += step)
                  if (n0 + j < rows) *to = __float2bfloat16_rn(v[j]);
              } else {
                float* to = static_cast<float*>(args.out) + el;
#pragma unroll
                for (int j = 0; j < 16; ++j, to += step)
                  if (n0 + j < rows) *to = v[j];
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->tmem_empty[acc]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (sh->abort_flag != 0) {
    long long t0 = clock64();
    while (clock64() - t0 < 4000000LL) {
    }
    if (threadIdx.x == 0 && args.status != nullptr) atomicExch(args.status, kGated ? 13 : 14);
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::kTmem);
  }
}

template <bool kGated, int N>
int launch_few(const Mx4Rows& r, const void* a_codes, const void* a_scales, const void* const (&w)[4], int experts, int k,
               int n, FewArgs ga, cudaStream_t st) {
  using Cfg = FewCfg<kGated, N>;
  constexpr size_t smem_bytes = 1024 + (size_t)Cfg::kStages * Cfg::kStageBytes + sizeof(FewShared<Cfg::kStages>);
  static_assert(smem_bytes <= 227u * 1024u, "shared memory of the few-rows kernel");
  static SmemLimitCache smem = {};
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(mx4_few_kernel<kGated, N>), smem_bytes, &smem, "mx4_few_kernel"))
    return rc;
  CUtensorMap a, a_sf, w0, w1, w0_sf, w1_sf;
  int rc;
  const int wn = (n + 127) / 128;
  if ((rc = mx4_map_codes(&a, a_codes, 1, r.rows, k, N))) return rc;
  if ((rc = mx4_map_scales(&a_sf, a_scales, mx4_row_tiles(r.rows, r.table_segments, N), k))) return rc;
  if ((rc = mx4_map_codes(&w0, w[0], experts, n, k, 128))) return rc;
  if ((rc = mx4_map_scales(&w0_sf, w[1], (uint64_t)experts * wn, k))) return rc;
  if constexpr (kGated) {
    if ((rc = mx4_map_codes(&w1, w[2], experts, n, k, 128))) return rc;
    if ((rc = mx4_map_scales(&w1_sf, w[3], (uint64_t)experts * wn, k))) return rc;
  } else {
    w1 = w0;
    w1_sf = w0_sf;
  }
  ga.segments = r.segments;
  ga.num_segments = r.segments != nullptr ? r.num_segments : 1;
  ga.rows_total = r.rows;
  ga.seg_base = r.seg_base;
  ga.experts = experts;
  ga.expert_base = r.expert_base;
  ga.status = r.status;
  ga.n_total = n;
  ga.k_total = k;
  ga.wn_tiles = wn;
  ga.partial = r.few_partial;
  ga.counters = r.few_counters;
  // Starts while the kernel before it drains.  That kernel has waited for everything before itself,
  // so what is older (weights, segment table) may be read without waiting.
  return launch_overlapping("mx4_few_kernel", mx4_few_kernel<kGated, N>, sm_count(), kThreadsF, smem_bytes, st, a, a_sf, w0, w1,
                            w0_sf, w1_sf, ga);
}

template <bool kGated>
int launch_few_n(const Mx4Rows& r, const void* a_codes, const void* a_scales, const void* const (&w)[4], int experts,
                 int k, int n, const FewArgs& ga, cudaStream_t st) {
  switch (r.tile_rows) {
    case 16: return launch_few<kGated, 16>(r, a_codes, a_scales, w, experts, k, n, ga, st);
    case 32: return launch_few<kGated, 32>(r, a_codes, a_scales, w, experts, k, n, ga, st);
    case 64: return launch_few<kGated, 64>(r, a_codes, a_scales, w, experts, k, n, ga, st);
    default: return launch_few<kGated, 128>(r, a_codes, a_scales, w, experts, k, n, ga, st);
  }
}

}  // namespace

// What decides is the rows a segment has on average.  Few-rows kernels, one CTA a tile, pairs, in us
// (experts of a top-k layer; one matrix):
//   64 experts 2048 x 1408, top 6   64 tokens (6 rows)   60   65   97      256 (24)   66   68  100
//                                  515 (48)              82   73  105     1030 (97)   87   82  110   2060 (193)  148  133  122
//   8 experts 4096 x 14336, top 2  128 (32)             133  140  180      256 (64)  164  145  195    512 (128)  234  202  199
//   one matrix 4096 -> 14336        64                   12   14   15      128        14   16   17    256         20   17   18
//              14336 -> 4096        64                   20   29   28 (few column tiles: the few-rows kernels cut the reduction)
// Weights of other shapes, us of a feed-forward (rows a segment: few / one CTA / pairs) and of a linear call:
//   16 experts 1024 x 512    24: 19 / 15 / 21     56: 17 / 15 / 22    144: 24 / 19 / 24    256: 30 / 24 / 30
//    8 experts 2048 x 5632   24: 35 / 38 / 49     56: 44 / 40 / 50    144: 68 / 48 / 53    256: 86 / 65 / 72
//   32 experts 512 x 2048    24: 25 / 26 / 42     56: 30 / 28 / 43    144: 55 / 39 / 46    256: 70 / 50 / 64
//   128 experts 2048 x 768   24: 78 / 72 / 114    56: 92 / 80 / 123   144: 194 / 134 / 157  256: 235 / 174 / 220
//   16 experts 5120 x 1536   24: 50 / 52 / 62     56: 58 / 55 / 67    144: 87 / 81 / 84    256: 109 / 101 / 107
//   2048 -> 2048             64: 13.9 / 9.1 / 10.6    128: 16.0 / 10.5 / 12.3    512: 10.8 / 11.2 / 13.3
//   5120 -> 5120             64: 14.7 / 15.4 / 16.9   128: 20.2 / 17.9 / 19.4    512: 21.9 / 19.4 / 21.0
//   8192 -> 10240            64: 17.3 / 20.7 / 21.6   128: 19.2 / 23.8 / 24.5    512: 41.4 / 41.7 / 37.5
//   1024 -> 16384            64:  8.1 / 8.3 / 11.3    128:  9.3 / 9.4 / 12.6     512: 17.6 / 13.6 / 16.2
// The limit at 40 rows holds within a few per cent but for the smallest experts (24 rows: a fifth lost).  The one
// at 128 is the wide layer's: all five of these would gain 5 to 24 % from the one-CTA kernel at 144 to 384 rows, and
// small single matrices up to a third at 64 to 512; the rule does not look at K and N.
// The few-rows kernels' row tiles are as wide as a segment has rows at most, or on average with room to
// spare: a wider tile costs epilogue and tensor time, a narrower one reads the weights again (from
// L2) for every further tile.
int mx4_choose(int rows, int num_segments, int max_rows, int* tile_rows) {
  const int average = (rows + num_segments - 1) / num_segments;
  *tile_rows = 128;
  if (average > 128) return kMx4Pair;
  if (num_segments > 1 && average > 40) return kMx4Single;
  for (int n = 16; n <= 64; n *= 2)
    if ((max_rows <= n || average <= n * 3 / 4) && rows / n + num_segments <= mx4_row_tiles_most(rows, num_segments)) {
      *tile_rows = n;
      break;
    }
  return kMx4Few;
}

int mx4_few_counters() { return few_enough(16); }

// The same for every width, so that a workspace made for many rows serves few.
size_t mx4_few_partial_bytes(bool gated) {
  size_t most = 0;
  for (int n = 16; n <= 128; n *= 2) {
    const size_t floats = (size_t)2 * few_enough(n) * (gated ? 2 : 1) * n * 128;
    most = floats > most ? floats : most;
  }
  return most * sizeof(float);
}

int launch_mx4_linear_few(const Mx4Rows& r, const void* a_codes, const void* a_scales, const void* w_codes,
                          const void* w_scales, int experts, int k, int n, void* out, bool out_bf16, cudaStream_t st) {
  FewArgs ga = {};
  ga.out = out;
  ga.out_bf16 = out_bf16 ? 1 : 0;
  const void* const w[4] = {w_codes, w_scales, nullptr, nullptr};
  return launch_few_n<false>(r, a_codes, a_scales, w, experts, k, n, ga, st);
}

int launch_mx4_gated_few(const Mx4Rows& r, const void* a_codes, const void* a_scales, const AxmMx4Experts* x, int experts,
                         int d, int f, void* h_codes, void* h_scales, cudaStream_t st) {
  FewArgs ga = {};
  ga.out = h_codes;
  ga.out_scales = static_cast<uint8_t*>(h_scales);
  const void* const w[4] = {x->gate_codes, x->gate_scales, x->up_codes, x->up_scales};
  return launch_few_n<true>(r, a_codes, a_scales, w, experts, d, f, ga, st);
}

}  // namespace axm
