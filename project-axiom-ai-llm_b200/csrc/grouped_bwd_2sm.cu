// Weight gradients of the expert FFN on CTA pairs (tcgen05.mma.cta_group::2):
//   dW[e][m, n] = sum over the expert's rows r of A[r, m] * B[r, n]
// used for dWd = h^T dO, dWg = x^T dG, dWu = x^T dU.  Both operands are MN-major (the rows
// are the reduction index), the output is fp32 in the weight's own [in][out] layout, as the
// reference engine's dense backward produces for its FFN weights
// (core/src/CUDA/kernel/backward_pass.cu:1013-1048; the engine has no MoE backward).
//
// Same product as kWGRAD of grouped_bwd.cu, which stays as the fallback.  There a CTA
// fills 48 KB of operands per k-block; here the two CTAs of a pair compute a 256 x 256
// tile together, each staging its own 128 rows of A^T and only half of B's columns:
// 32 KB per k-block and CTA, six stages instead of four.  A unit is (expert, n-tile,
// pair of m-tiles); with an odd number of m-tiles the last pair's second half idles.
// Segments must be padded to a multiple of 64 rows with zero rows (training layout).
// The fp32 tile leaves through a per-warp staging block and TMA stores, which clip at the
// matrix edge.  All waits are bounded; a wait that gives up winds both CTAs down and sets
// the status word to 9.
#include "gemm_2sm.cuh"
#include "microscale.cuh"

namespace axm {

namespace {

struct __align__(8) WgradShared2 {
  uint64_t full[kStages2];    // used in the leader: bytes of both CTAs land here
  uint64_t empty[kStages2];   // own: the leader's MMA commit arrives in both CTAs
  uint64_t tmem_full[2];      // own
  uint64_t tmem_empty[2];     // used in the leader: 4 epilogue warps of each CTA
  uint32_t tmem_base;
  int abort_flag;
  AxmSegment seg[kMaxSegments];
};

constexpr int kWgradStagingBytes = 4 * 4096;  // one 32 x 32 fp32 block per epilogue warp
constexpr size_t kWgrad2SmemBytes =
    1024 + (size_t)kStages2 * kStageBytes2 + kWgradStagingBytes + sizeof(WgradShared2);
static_assert(kWgrad2SmemBytes <= 227u * 1024u, "shared memory of the pair weight-gradient kernel");

constexpr int kWgradProblems = 3;
struct Wgrad2Args {
  const AxmSegment* segments;
  int num_segments;
  int num_problems;
  int m_total[kWgradProblems];  // rows of one expert's gradient
  int n_total[kWgradProblems];  // columns
  int units_before[kWgradProblems + 1];
  int* status;
  int overlap;  // see launch_overlapping
  int rows_checked;  // training step with 8-bit checkpoints: as in the other products' arguments
  int experts;
};
// The maps of a launch's problems: A, B and the gradient.
struct Wgrad2Maps {
  CUtensorMap a[kWgradProblems], b[kWgradProblems], out[kWgradProblems];
};

// fp32 accumulate, bf16 A and B both MN-major, N = 256, M = 256 over the pair
constexpr uint32_t kInstrDescWgrad2 = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) |
                                      ((uint32_t)(UMMA_N >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);

struct WgradUnit {
  int problem, seg, n_tile, m_tile, a_m_tile;
  bool live;  // false: this half of the pair has no tile (odd number of m-tiles)
};

__device__ __forceinline__ WgradUnit decode_wgrad(const Wgrad2Args& args, int unit, int rank) {
  WgradUnit u;
  u.problem = 0;
  while (u.problem + 1 < args.num_problems && unit >= args.units_before[u.problem + 1]) ++u.problem;
  unit -= args.units_before[u.problem];
  const int n_tiles = (args.n_total[u.problem] + UMMA_N - 1) / UMMA_N;
  const int m_tiles = (args.m_total[u.problem] + BM - 1) / BM;
  const int pairs_w = (m_tiles + 1) / 2;
  const int per = pairs_w * n_tiles;
  u.seg = unit / per;
  const int local = unit - u.seg * per;
  u.n_tile = local / pairs_w;
  const int p = local - u.n_tile * pairs_w;
  u.m_tile = 2 * p + rank;
  u.live = u.m_tile < m_tiles;
  u.a_m_tile = u.live ? u.m_tile : 2 * p;  // an idle half still stages (the leader's) rows
  return u;
}

// kBf16: the gradient leaves as bf16 (rounded once from the fp32 accumulator): half the bytes of
// the largest outputs of a training step.
template <bool kBf16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
grouped_wgrad_2sm_kernel(const __grid_constant__ Wgrad2Maps maps, const __grid_constant__ Wgrad2Args args) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* staging = tiles + (size_t)kStages2 * kStageBytes2;  // 1024-byte aligned
  WgradShared2* sh = reinterpret_cast<WgradShared2*>(staging + kWgradStagingBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();  // 0 = leader
  const uint32_t peer = rank ^ 1u;
  const int cluster_id = blockIdx.x >> 1;
  const int num_clusters = gridDim.x >> 1;
  const int nseg = args.num_segments;
  const int total_units = args.units_before[args.num_problems];

  if (args.overlap) launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages2; ++i) {
      mbar_init(&sh->full[i], 1);
      mbar_init(&sh->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh->tmem_full[i], 1);
      mbar_init(&sh->tmem_empty[i], 8);
    }
    sh->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&maps.a[0]);
    tma_prefetch_desc(&maps.b[0]);
    tma_prefetch_desc(&maps.out[0]);
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc2(&sh->tmem_base, kTmemCols);
    tmem_relinquish2();
  }
  if (args.overlap) wait_for_previous();
  for (int s = threadIdx.x; s < nseg; s += kGemmThreads) {
    const AxmSegment sg = args.segments[s];
    sh->seg[s] = args.rows_checked > 0 ? kept_inside(sg, args.rows_checked, 0, args.experts) : sg;
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // barriers of both CTAs are initialised before anyone signals across
  tc_fence_after();

  const uint32_t tmem_base = sh->tmem_base;
  volatile int* abort_flag = &sh->abort_flag;
  auto raise_abort = [&]() {  // tell the peer too, so that the pair winds down together
    st_cluster_u32(map_to_cta(smem_u32(&sh->abort_flag), peer), 1u);
  };

  if (warp == 0) {
    // ---- TMA producer: own 128 columns of A^T, own half of B ---------------------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int unit = cluster_id; ok && unit < total_units; unit += num_clusters) {
        const WgradUnit u = decode_wgrad(args, unit, (int)rank);
        const AxmSegment sg = sh->seg[u.seg];
        const int k_blocks = (sg.rows + BK - 1) / BK;
        const int a_col = u.a_m_tile * BM;
        const int b_col = u.n_tile * UMMA_N + (int)rank * 128;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&sh->empty[stage], phase ^ 1u, abort_flag)) {
            raise_abort();
            ok = false;
            break;
          }
          unsigned char* sa = tiles + (size_t)stage * kStageBytes2;
          unsigned char* sb = sa + kABytes;
          if (rank == 0) mbar_expect_tx(&sh->full[stage], 2 * kStageBytes2);
          const uint32_t bar = map_to_cta(smem_u32(&sh->full[stage]), 0);
          const int row = sg.a_row0 + kb * BK;
#pragma unroll
          for (int c = 0; c < 2; ++c) tma2_load_2d(sa + c * kBChunkBytes, &maps.a[u.problem], bar, a_col + c * 64, row);
#pragma unroll
          for (int c = 0; c < 2; ++c) tma2_load_2d(sb + c * kBChunkBytes, &maps.b[u.problem], bar, b_col + c * 64, row);
          if (++stage == kStages2) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issuer: the leader CTA only (the whole warp, one elected lane issues) ------
    if (rank == 0) {
      const uint64_t tiles_desc = make_smem_desc(smem_u32(tiles), kBChunkBytes, 1024);
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int unit = cluster_id; ok && unit < total_units; unit += num_clusters) {
        const WgradUnit u = decode_wgrad(args, unit, 0);
        const int k_blocks = (sh->seg[u.seg].rows + BK - 1) / BK;
        if (!__all_sync(0xffffffffu, mbar_wait(&sh->tmem_empty[acc], acc_phase ^ 1u, abort_flag))) {
          if (lane == 0) raise_abort();
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)acc * UMMA_N;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait(&sh->full[stage], phase, abort_flag))) {
            if (lane == 0) raise_abort();
            ok = false;
            break;
          }
          tc_fence_after();
          // MN-major operands: 64-wide chunks 8192 B apart, 8-k groups 1024 B apart, +2048 B per 16 k;
          // descriptors count in 16-byte units
          const uint64_t da = tiles_desc + (uint64_t)(stage * (kStageBytes2 / 16));
          const uint64_t db = da + kABytes / 16;
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < BK / UMMA_K; ++j)
              tc_mma2_bf16(d_tmem, da + (uint64_t)(j * 128), db + (uint64_t)(j * 128), kInstrDescWgrad2,
                           (kb > 0 || j > 0) ? 1u : 0u);
            tc_commit2_both(smem_u32(&sh->empty[stage]));
          }
          __syncwarp();
          if (++stage == kStages2) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        // with no rows nothing was issued and the commits arrive at once; the epilogue writes zeros
        if (elect_one()) tc_commit2_both(smem_u32(&sh->tmem_full[acc]));
        __syncwarp();
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
  } else {
    // ---- epilogue: every CTA drains its own 128 accumulator rows -----------------------
    const int quad = warp & 3;
    unsigned char* stage_w = staging + (size_t)((warp - 2) & 3) * 4096;
    int acc = 0;
    uint32_t acc_phase = 0;
    const uint32_t leader_tmem_empty0 = map_to_cta(smem_u32(&sh->tmem_empty[0]), 0);
    const uint32_t leader_tmem_empty1 = map_to_cta(smem_u32(&sh->tmem_empty[1]), 0);
    for (int unit = cluster_id; unit < total_units; unit += num_clusters) {
      const WgradUnit u = decode_wgrad(args, unit, (int)rank);
      const AxmSegment sg = sh->seg[u.seg];
      const int k_blocks = (sg.rows + BK - 1) / BK;
      if (!__all_sync(0xffffffffu, mbar_wait(&sh->tmem_full[acc], acc_phase, abort_flag))) break;
      tc_fence_after();
      const int n0 = u.n_tile * UMMA_N;
      const int block_row0 = u.m_tile * BM + quad * 32;
      const uint32_t t_addr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)acc * UMMA_N;
      if (u.live) {
#pragma unroll 1
        for (int c0 = 0; c0 < UMMA_N; c0 += 32) {
          uint32_t v[32];
          __syncwarp();
          tmem_ld32(t_addr + c0, v);
          tmem_ld_wait();
          if (k_blocks == 0) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0u;
          }
          // Lane = row of the 32 x 32 block; piece q of row r sits at q ^ (r & 7), the 128-byte
          // swizzle of the output map (and free of bank conflicts); one TMA store per block.
          if (lane == 0) bulk_wait_read();  // the previous block's store has read the buffer
          __syncwarp();
          if (n0 + c0 < args.n_total[u.problem] && block_row0 < args.m_total[u.problem] && (sg.expert & 0xffff) < args.experts) {
            if constexpr (kBf16) {  // rows of 64 bytes, the 64-byte swizzle of the bf16 output map
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                uint32_t w4[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  w4[j] = pack_bf16(__uint_as_float(v[8 * q + 2 * j]), __uint_as_float(v[8 * q + 2 * j + 1]));
                *reinterpret_cast<uint4*>(stage_w + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) =
                    make_uint4(w4[0], w4[1], w4[2], w4[3]);
              }
            } else {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                *reinterpret_cast<uint4*>(stage_w + lane * 128 + ((q ^ (lane & 7)) << 4)) =
                    make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&maps.out[u.problem], stage_w, n0 + c0, block_row0, sg.expert & 0xffff);
              bulk_commit_group();
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc == 0 ? leader_tmem_empty0 : leader_tmem_empty1);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
    if (lane == 0) bulk_wait_all();
  }

  // ---- drain: nobody leaves while the peer may still touch its shared memory or TMEM -----
  tc_fence_before();
  __syncthreads();
  if (sh->abort_flag != 0) {
    long long t0 = clock64();
    while (clock64() - t0 < 4000000LL) {
    }
    if (threadIdx.x == 0 && args.status != nullptr) atomicExch(args.status, 9);
  }
  cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc2(tmem_base, kTmemCols);
  }
}

// Row-major bf16 matrix [rows][cols]; box = 64 columns x 64 rows (rows = reduction index).
int map_kbox(CUtensorMap* m, const void* base, uint64_t rows, uint64_t cols) {
  const uint64_t dims[2] = {cols, rows};
  const uint64_t strides[1] = {cols * 2};
  const uint32_t box[2] = {64, 64};
  return encode_tensor_map(m, base, 2, dims, strides, box);
}

}  // namespace

template <bool kBf16>
static int launch_wgrad_as(const AxmSegment* segments, int32_t num_segments, int32_t rows_total, int32_t experts,
                           const WgradProblem* problems, int32_t num_problems, int32_t* status, cudaStream_t st,
                           bool overlap) {
  static SmemLimitCache smem = {};
  if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(grouped_wgrad_2sm_kernel<kBf16>), kWgrad2SmemBytes,
                                   &smem, "grouped_wgrad_2sm_kernel"))
    return rc;
  const int grid = grid_2sm();
  if (grid < 0) return grid;
  if (grid < 2) return fail(AXM_ERR_DEVICE, "two-SM clusters cannot be scheduled on this device");
  Wgrad2Maps maps;
  Wgrad2Args wa = {};
  wa.segments = segments;
  wa.num_segments = num_segments;
  wa.num_problems = num_problems;
  wa.status = status;
  wa.overlap = overlap ? 1 : 0;
  wa.rows_checked = overlap ? rows_total : 0;
  wa.experts = experts;
  for (int p = 0; p < num_problems; ++p) {
    const WgradProblem& w = problems[p];
    int rc;
    if ((rc = map_kbox(&maps.a[p], w.a, (uint64_t)rows_total, (uint64_t)w.m))) return rc;
    if ((rc = map_kbox(&maps.b[p], w.b, (uint64_t)rows_total, (uint64_t)w.n))) return rc;
    const uint64_t dims[3] = {(uint64_t)w.n, (uint64_t)w.m, (uint64_t)experts};
    const uint64_t size = kBf16 ? 2 : 4;
    const uint64_t strides[2] = {(uint64_t)w.n * size, (uint64_t)w.n * (uint64_t)w.m * size};
    const uint32_t box[3] = {32, 32, 1};
    if constexpr (kBf16) {
      if ((rc = encode_tensor_map_sw64(&maps.out[p], w.d_w, 3, dims, strides, box))) return rc;
    } else {
      if ((rc = encode_tensor_map_f32(&maps.out[p], w.d_w, 3, dims, strides, box))) return rc;
    }
    wa.m_total[p] = w.m;
    wa.n_total[p] = w.n;
    const int pairs_w = ((w.m + BM - 1) / BM + 1) / 2, n_tiles = (w.n + UMMA_N - 1) / UMMA_N;
    wa.units_before[p + 1] = wa.units_before[p] + num_segments * pairs_w * n_tiles;
  }
  for (int p = num_problems; p < kWgradProblems; ++p) {
    maps.a[p] = maps.a[0];
    maps.b[p] = maps.b[0];
    maps.out[p] = maps.out[0];
  }
  if (overlap)
    return launch_overlapping("grouped_wgrad_2sm_kernel", grouped_wgrad_2sm_kernel<kBf16>, grid, kGemmThreads,
                              kWgrad2SmemBytes, st, maps, wa);
  grouped_wgrad_2sm_kernel<kBf16><<<grid, kGemmThreads, kWgrad2SmemBytes, st>>>(maps, wa);
  return check_launch("grouped_wgrad_2sm_kernel");
}

// dW[e] = A^T . B over each segment's rows: A [rows_total][m], B [rows_total][n] (bf16), dW
// [experts][m][n] fp32 or bf16, for each of the problems.  AXM_ERR_DEVICE when pairs cannot be
// scheduled, so that the caller can fall back to the one-SM kernel.
int launch_wgrad_2sm(const AxmSegment* segments, int32_t num_segments, int32_t rows_total, int32_t experts,
                     const WgradProblem* problems, int32_t num_problems, int32_t* status, cudaStream_t st, bool out_bf16,
                     bool overlap) {
  if (num_problems < 1 || num_problems > kWgradProblems)
    return fail(AXM_ERR_ARGUMENT, "launch_wgrad_2sm: %d problems", num_problems);
  return out_bf16 ? launch_wgrad_as<true>(segments, num_segments, rows_total, experts, problems, num_problems, status, st, overlap)
                  : launch_wgrad_as<false>(segments, num_segments, rows_total, experts, problems, num_problems, status, st, overlap);
}

}  // namespace axm
