// Quantising to microscaled blocks and reading them back (formats: microscale.cuh).  The engine
// has no low-bit formats; its bf16 weights and their fp32 master copies
// (core/src/CUDA/util/gpu_types.cuh:148-168) are what these kernels read.
//
// All four are bound by memory: every value is read once and written once.
#include "microscale.cuh"

namespace axm {

namespace {

// Eight neighbouring values of a row as fp32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = bf16_lo(w[j]);
    v[2 * j + 1] = bf16_hi(w[j]);
  }
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]);
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// One warp per 256 neighbouring elements of a row: a lane holds eight of them (a 16-byte load of
// bf16), four lanes a block.  kBits = 4: scale bytes in tile order, the row's last, partial run
// padded with zero bytes.  kBits = 8: codes [rows][K], scale bytes [rows][K / 32].
// `from` says which source row a row comes from; row_src[r] < 0: zeros.
template <int kBits, typename T>
__global__ void __launch_bounds__(256)
mx_quantize_rows_kernel(const T* __restrict__ x, long long ld, Mx4Gather from, int rows, int k,
                        const AxmSegment* __restrict__ segments, int num_segments,
                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int32_t* status) {
  if (status != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *status = 0;
  const int lane = threadIdx.x & 31;
  const int runs = (k + 255) / 256;
  const long long items = (long long)rows * runs;
  const long long step = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < items; item += step) {
    const int row = (int)(item / runs);
    const int run = (int)(item - (long long)row * runs);
    const int k0 = run * 256 + lane * 8;
    long long src = row;
    if (row >= from.tail_row0) {
      src = (row - from.tail_row0) % from.tail_mod;
    } else if (from.row_src != nullptr) {
      const int s = __ldg(from.row_src + row);
      src = s < 0 ? -1 : s / from.row_div;
    }
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k0 < k && src >= 0) load8<T>(x + src * ld + k0, v);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t s = mx_scale_byte<kBits == 4 ? 2 : 8>(top);
    const float inv = mx_inverse_scale(s);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= inv;
    if constexpr (kBits == 4) {
      if (k0 < k) *reinterpret_cast<uint32_t*>(codes + (size_t)row * (k >> 1) + (k0 >> 1)) = mx4_pack8(v);
      int seg = 0, tile_row = row;
      if (segments != nullptr) {
        seg = segment_of_row(segments, num_segments, row);
        if (seg < 0) continue;  // a row behind its segment's end has no place among the tiles
        tile_row = row - __ldg(&segments[seg].out_row0);
      }
      // the four bytes of a 128-element chunk gathered into one word by the chunk's first lane
      uint32_t word = s << (8 * ((lane >> 2) & 3));
      word |= __shfl_xor_sync(0xffffffffu, word, 4);
      word |= __shfl_xor_sync(0xffffffffu, word, 8);
      if ((lane & 15) == 0) {
        const int first = segments != nullptr ? __ldg(&segments[seg].out_row0) : 0;
        const size_t tile = (size_t)(first / 128 + seg + tile_row / 128);
        const int r = tile_row & 127;
        uint8_t* chunk = scales + (tile * mx4_chunks(k) + run * 2 + (lane >> 4)) * 512;
        *reinterpret_cast<uint32_t*>(chunk + (r & 31) * 16 + (r >> 5) * 4) = word;
      }
    } else {
      if (k0 < k) {
        *reinterpret_cast<uint2*>(codes + (size_t)row * k + k0) =
            make_uint2(mx8_pack4(v[0], v[1], v[2], v[3]), mx8_pack4(v[4], v[5], v[6], v[7]));
        if ((lane & 3) == 0) scales[(size_t)row * (k >> 5) + (k0 >> 5)] = (uint8_t)s;
      }
    }
  }
}

template <int kBits, typename T>
__global__ void __launch_bounds__(256)
mx_dequantize_rows_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, int k,
                          const AxmSegment* __restrict__ segments, int num_segments, T* __restrict__ out,
                          long long ld) {
  const int lane = threadIdx.x & 31;
  const int runs = (k + 255) / 256;
  const long long items = (long long)rows * runs;
  const long long step = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < items; item += step) {
    const int row = (int)(item / runs);
    const int run = (int)(item - (long long)row * runs);
    const int k0 = run * 256 + lane * 8;
    if (k0 >= k) continue;
    float v[8];
    if constexpr (kBits == 4) {
      int seg = 0, first = 0;
      if (segments != nullptr) {
        seg = segment_of_row(segments, num_segments, row);
        if (seg < 0) continue;
        first = __ldg(&segments[seg].out_row0);
      }
      const int r = row - first;
      const size_t tile = (size_t)(first / 128 + seg + r / 128);
      const uint8_t* chunk = scales + (tile * mx4_chunks(k) + run * 2 + (lane >> 4)) * 512;
      const float s = mx_scale_value(__ldg(chunk + (r & 31) * 16 + ((r & 127) >> 5) * 4 + ((lane >> 2) & 3)));
      const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(codes + (size_t)row * (k >> 1) + (k0 >> 1)));
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = mx4_code_value(c >> (4 * j)) * s;
    } else {
      const float s = mx_scale_value(__ldg(scales + (size_t)row * (k >> 5) + (k0 >> 5)));
      const uint2 c = __ldg(reinterpret_cast<const uint2*>(codes + (size_t)row * k + k0));
      const uint32_t w[4] = {c.x & 0xffffu, c.x >> 16, c.y & 0xffffu, c.y >> 16};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = mx8_unpack2(w[j]);
        v[2 * j] = f.x * s;
        v[2 * j + 1] = f.y * s;
      }
    }
    store8<T>(out + (size_t)row * ld + k0, v);
  }
}

template <typename T>
__device__ __forceinline__ float2 load2(const T* p);
template <>
__device__ __forceinline__ float2 load2<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(p));
  return make_float2(bf16_lo(w), bf16_hi(w));
}
template <>
__device__ __forceinline__ float2 load2<float>(const float* p) {
  return __ldg(reinterpret_cast<const float2*>(p));
}
__device__ __forceinline__ void store2(__nv_bfloat16* p, float a, float b) {
  *reinterpret_cast<uint32_t*>(p) = pack_bf16(a, b);
}
__device__ __forceinline__ void store2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }

// Expert weights [E][K][N] (N contiguous, as the engine stores them) to codes [E][N][K / 2]: a
// block runs down K, so a thread owns two neighbouring columns and walks 32 rows; a warp's loads
// cover 64 columns.  A CTA turns 256 k x 64 n over in shared memory and writes runs of 128 bytes.
constexpr int kWeightsK = 256, kWeightsN = 64;
template <typename T>
__global__ void __launch_bounds__(256)
mx4_quantize_weights_kernel(const T* __restrict__ w, int k, int n, uint8_t* __restrict__ codes,
                            uint8_t* __restrict__ scales) {
  // 16-byte piece p of column c sits at piece p ^ (c % 8): neither the column-wise stores nor the
  // row-wise loads of a warp meet in a bank
  __shared__ uint4 tile[kWeightsN * 8];
  __shared__ uint8_t sc[kWeightsN][8];
  const int e = blockIdx.z, n0 = blockIdx.x * kWeightsN, k0 = blockIdx.y * kWeightsK;
  const int pair = threadIdx.x & 31, blk = threadIdx.x >> 5;
  const int col = n0 + 2 * pair, kk = k0 + blk * kMxBlock;
  float a[32], b[32];
  uint32_t ta = 0, tb = 0;
  if (col < n && kk < k) {
    const T* p = w + ((size_t)e * k + kk) * n + col;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const float2 v = load2<T>(p + (size_t)j * n);
      a[j] = v.x;
      b[j] = v.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) a[j] = b[j] = 0.0f;
  }
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    ta = max(ta, __float_as_uint(a[j]) & 0x7fffffffu);
    tb = max(tb, __float_as_uint(b[j]) & 0x7fffffffu);
  }
  auto put = [&](const float (&v)[32], uint32_t top, int c) {
    const uint32_t s = mx_scale_byte<2>(top);
    const float inv = mx_inverse_scale(s);
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = v[8 * i + j] * inv;
      q[i] = mx4_pack8(t);
    }
    tile[c * 8 + (blk ^ (c & 7))] = make_uint4(q[0], q[1], q[2], q[3]);
    sc[c][blk] = (uint8_t)s;
  };
  put(a, ta, 2 * pair);
  put(b, tb, 2 * pair + 1);
  __syncthreads();
  // codes: eight threads a column, 128 contiguous bytes
  for (int i = threadIdx.x; i < kWeightsN * 8; i += 256) {
    const int c = i >> 3, piece = i & 7;
    if (n0 + c < n && k0 + piece * kMxBlock < k)
      *reinterpret_cast<uint4*>(codes + ((size_t)e * n + n0 + c) * (k >> 1) + (k0 >> 1) + piece * 16) =
          tile[c * 8 + (piece ^ (c & 7))];
  }
  // scale bytes: one word per column and 128-element chunk
  if (threadIdx.x < kWeightsN * 2) {
    const int c = threadIdx.x >> 1, half = threadIdx.x & 1;
    const int col_w = n0 + c;
    if (col_w < n) {
      const uint32_t word = *reinterpret_cast<const uint32_t*>(&sc[c][half * 4]);
      const size_t t = (size_t)e * ((n + 127) / 128) + col_w / 128;
      const int r = col_w & 127;
      *reinterpret_cast<uint32_t*>(scales + (t * mx4_chunks(k) + blockIdx.y * 2 + half) * 512 + (r & 31) * 16 +
                                   (r >> 5) * 4) = word;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
mx4_dequantize_weights_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int k, int n,
                              T* __restrict__ w) {
  __shared__ uint4 tile[kWeightsN * 8];
  const int e = blockIdx.z, n0 = blockIdx.x * kWeightsN, k0 = blockIdx.y * kWeightsK;
  for (int i = threadIdx.x; i < kWeightsN * 8; i += 256) {
    const int c = i >> 3, piece = i & 7;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (n0 + c < n && k0 + piece * kMxBlock < k)
      v = __ldg(reinterpret_cast<const uint4*>(codes + ((size_t)e * n + n0 + c) * (k >> 1) + (k0 >> 1) + piece * 16));
    tile[c * 8 + (piece ^ (c & 7))] = v;
  }
  __syncthreads();
  const int pair = threadIdx.x & 31, blk = threadIdx.x >> 5;
  const int col = n0 + 2 * pair, kk = k0 + blk * kMxBlock;
  if (col >= n || kk >= k) return;
  float s[2];
  uint32_t q[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = 2 * pair + h, cw = col + h;
    const uint4 v = tile[c * 8 + (blk ^ (c & 7))];
    q[h][0] = v.x; q[h][1] = v.y; q[h][2] = v.z; q[h][3] = v.w;
    const size_t t = (size_t)e * ((n + 127) / 128) + cw / 128;
    const int r = cw & 127;
    s[h] = mx_scale_value(__ldg(scales + (t * mx4_chunks(k) + (kk >> 7)) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (blk & 3)));
  }
  T* p = w + ((size_t)e * k + kk) * n + col;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      store2(p + (size_t)(8 * i + j) * n, mx4_code_value(q[0][i] >> (4 * j)) * s[0],
             mx4_code_value(q[1][i] >> (4 * j)) * s[1]);
}

// Scale bytes as checkpoints keep them, [E][N][K / 32], to tile order.
__global__ void __launch_bounds__(256)
mx4_pack_scales_kernel(const uint8_t* __restrict__ plain, int experts, int k, int n, uint8_t* __restrict__ scales) {
  const int chunks = mx4_chunks(k), blocks = k >> 5;
  const long long items = (long long)experts * n * chunks;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < items; i += (long long)gridDim.x * blockDim.x) {
    const int chunk = (int)(i % chunks);
    const long long en = i / chunks;
    const int col = (int)(en % n);
    const int e = (int)(en / n);
    uint32_t word = 0;
    for (int b = 0; b < 4; ++b) {
      const int kb = chunk * 4 + b;
      if (kb < blocks) word |= (uint32_t)__ldg(plain + en * blocks + kb) << (8 * b);
    }
    const size_t t = (size_t)e * ((n + 127) / 128) + col / 128;
    const int r = col & 127;
    *reinterpret_cast<uint32_t*>(scales + (t * chunks + chunk) * 512 + (r & 31) * 16 + (r >> 5) * 4) = word;
  }
}

int check_dtype(int32_t dtype, const char* what) {
  if (dtype != AXM_DTYPE_BF16 && dtype != AXM_DTYPE_FP32) return fail(AXM_ERR_ARGUMENT, "%s: dtype %d unknown", what, dtype);
  return AXM_OK;
}

int check_rows(int32_t rows, int32_t k, int32_t num_segments, const char* what) {
  if (rows < 0) return fail(AXM_ERR_ARGUMENT, "%s: %d rows", what, rows);
  if (k <= 0 || k % kMxBlock) return fail(AXM_ERR_ARGUMENT, "%s: k %d is not a positive multiple of 32", what, k);
  if (num_segments < 0) return fail(AXM_ERR_ARGUMENT, "%s: num_segments %d negative", what, num_segments);
  return AXM_OK;
}

int check_weights(int32_t experts, int32_t k, int32_t n, const char* what) {
  if (experts <= 0 || experts > 65535) return fail(AXM_ERR_ARGUMENT, "%s: experts %d not in 1..65535", what, experts);
  if (k <= 0 || k % kMxBlock || k > 65535 * kWeightsK)
    return fail(AXM_ERR_ARGUMENT, "%s: k %d is not a positive multiple of 32 up to %d", what, k, 65535 * kWeightsK);
  if (n <= 0 || n % 8) return fail(AXM_ERR_ARGUMENT, "%s: n %d is not a positive multiple of 8", what, n);
  return AXM_OK;
}

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

// Rows of `ld` elements of `dtype` that are read or written in 16-byte pieces.
int check_matrix(const void* p, int32_t dtype, int64_t ld, int32_t k, const char* what) {
  const int64_t piece = dtype == AXM_DTYPE_BF16 ? 8 : 4;
  if (ld < k || ld % piece) return fail(AXM_ERR_ARGUMENT, "%s: row stride %lld for %d columns (a multiple of %lld is needed)", what, (long long)ld, k, (long long)piece);
  if (misaligned(p, 16)) return fail(AXM_ERR_ARGUMENT, "%s: the matrix must be 16-byte aligned", what);
  return AXM_OK;
}

unsigned row_grid(int32_t rows, int32_t k) {
  const long long warps = (long long)rows * ((k + 255) / 256);
  long long blocks = (warps + 7) / 8;
  const long long most = 32LL * sm_count();
  return (unsigned)(blocks < most ? blocks : most);
}

template <int kBits>
int launch_quantize_rows(const void* x, int32_t dtype, int64_t ld, const Mx4Gather& from, int32_t rows, int32_t k,
                         const AxmSegment* segments, int32_t num_segments, void* codes, void* scales,
                         int32_t* status, cudaStream_t st) {
  const unsigned grid = row_grid(rows, k);
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* s = static_cast<uint8_t*>(scales);
  if (dtype == AXM_DTYPE_BF16)
    mx_quantize_rows_kernel<kBits, __nv_bfloat16><<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(x), ld, from,
                                                                       rows, k, segments, num_segments, c, s, status);
  else
    mx_quantize_rows_kernel<kBits, float><<<grid, 256, 0, st>>>(static_cast<const float*>(x), ld, from, rows, k, segments,
                                                                num_segments, c, s, status);
  return check_launch("mx_quantize_rows_kernel");
}

template <int kBits>
int launch_dequantize_rows(const void* codes, const void* scales, int32_t rows, int32_t k, const AxmSegment* segments,
                           int32_t num_segments, void* out, int32_t dtype, int64_t ld, cudaStream_t st) {
  const unsigned grid = row_grid(rows, k);
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  if (dtype == AXM_DTYPE_BF16)
    mx_dequantize_rows_kernel<kBits, __nv_bfloat16><<<grid, 256, 0, st>>>(c, s, rows, k, segments, num_segments,
                                                                         static_cast<__nv_bfloat16*>(out), ld);
  else
    mx_dequantize_rows_kernel<kBits, float><<<grid, 256, 0, st>>>(c, s, rows, k, segments, num_segments,
                                                                  static_cast<float*>(out), ld);
  return check_launch("mx_dequantize_rows_kernel");
}

}  // namespace

int launch_mx4_quantize_rows(const void* x, int32_t dtype, int64_t ld, const Mx4Gather& from, const Mx4Rows& rows, int k,
                             void* codes, void* scales, cudaStream_t st) {
  return launch_quantize_rows<4>(x, dtype, ld, from, rows.rows, k, rows.segments, rows.num_segments, codes, scales,
                                 rows.status, st);
}

int check_mx_matrix(const void* p, int32_t dtype, int64_t ld, int32_t k, const char* what) {
  if (int rc = check_dtype(dtype, what)) return rc;
  return check_matrix(p, dtype, ld, k, what);
}

}  // namespace axm

using namespace axm;

extern "C" int axm_mx4_rows_bytes(int32_t rows, int32_t num_segments, int32_t k, size_t* code_bytes, size_t* scale_bytes) {
  if (int rc = check_rows(rows, k, num_segments, "axm_mx4_rows_bytes")) return rc;
  if (!code_bytes || !scale_bytes) return fail(AXM_ERR_ARGUMENT, "axm_mx4_rows_bytes: null pointer");
  *code_bytes = (size_t)rows * (k / 2);
  *scale_bytes = (size_t)mx4_row_tiles(rows, num_segments > 0 ? num_segments : 1) * mx4_chunks(k) * 512;
  return AXM_OK;
}

extern "C" int axm_mx4_weights_bytes(int32_t experts, int32_t k, int32_t n, size_t* code_bytes, size_t* scale_bytes) {
  if (int rc = check_weights(experts, k, n, "axm_mx4_weights_bytes")) return rc;
  if (!code_bytes || !scale_bytes) return fail(AXM_ERR_ARGUMENT, "axm_mx4_weights_bytes: null pointer");
  *code_bytes = (size_t)experts * n * (k / 2);
  *scale_bytes = (size_t)experts * ((n + 127) / 128) * mx4_chunks(k) * 512;
  return AXM_OK;
}

extern "C" int axm_mx4_quantize_rows(const void* x, int32_t x_dtype, int64_t ld, const int32_t* row_src,
                                     int32_t row_div, int32_t rows, int32_t k, const AxmSegment* segments, int32_t num_segments,
                                     void* codes, void* scales, void* stream) {
  const char* what = "axm_mx4_quantize_rows";
  if (int rc = check_rows(rows, k, num_segments, what)) return rc;
  if (int rc = check_dtype(x_dtype, what)) return rc;
  if (rows == 0) return AXM_OK;  // matrices without rows may have no address
  if (!x || !codes || !scales) return fail(AXM_ERR_ARGUMENT, "%s: null pointer", what);
  if (segments != nullptr && num_segments == 0) return fail(AXM_ERR_ARGUMENT, "%s: an empty segment table", what);
  if (row_src != nullptr && row_div <= 0) return fail(AXM_ERR_ARGUMENT, "%s: row_div %d must be positive", what, row_div);
  if (int rc = check_matrix(x, x_dtype, ld, k, what)) return rc;
  if (misaligned(codes, 16) || misaligned(scales, 16)) return fail(AXM_ERR_ARGUMENT, "%s: codes and scales must be 16-byte aligned", what);
  if (int rc = require_device()) return rc;
  const Mx4Gather from = {row_src, row_div, rows, 1};
  return launch_quantize_rows<4>(x, x_dtype, ld, from, rows, k, segments, num_segments, codes, scales,
                                 nullptr, static_cast<cudaStream_t>(stream));
}

extern "C" int axm_mx4_dequantize_rows(const void* codes, const void* scales, int32_t rows, int32_t k,
                                       const AxmSegment* segments, int32_t num_segments, void* out, int32_t out_dtype,
                                       int64_t ld, void* stream) {
  const char* what = "axm_mx4_dequantize_rows";
  if (int rc = check_rows(rows, k, num_segments, what)) return rc;
  if (int rc = check_dtype(out_dtype, what)) return rc;
  if (rows == 0) return AXM_OK;  // matrices without rows may have no address
  if (!codes || !scales || !out) return fail(AXM_ERR_ARGUMENT, "%s: null pointer", what);
  if (segments != nullptr && num_segments == 0) return fail(AXM_ERR_ARGUMENT, "%s: an empty segment table", what);
  if (int rc = check_matrix(out, out_dtype, ld, k, what)) return rc;
  if (misaligned(codes, 16) || misaligned(scales, 16)) return fail(AXM_ERR_ARGUMENT, "%s: codes and scales must be 16-byte aligned", what);
  if (int rc = require_device()) return rc;
  return launch_dequantize_rows<4>(codes, scales, rows, k, segments, num_segments, out, out_dtype, ld,
                                   static_cast<cudaStream_t>(stream));
}

extern "C" int axm_mx8_quantize_rows(const void* x, int32_t x_dtype, int64_t ld, int32_t rows, int32_t k, void* codes,
                                     void* scales, void* stream) {
  const char* what = "axm_mx8_quantize_rows";
  if (int rc = check_rows(rows, k, 0, what)) return rc;
  if (int rc = check_dtype(x_dtype, what)) return rc;
  if (rows == 0) return AXM_OK;  // matrices without rows may have no address
  if (!x || !codes || !scales) return fail(AXM_ERR_ARGUMENT, "%s: null pointer", what);
  if (int rc = check_matrix(x, x_dtype, ld, k, what)) return rc;
  if (misaligned(codes, 16)) return fail(AXM_ERR_ARGUMENT, "%s: codes must be 16-byte aligned", what);
  if (int rc = require_device()) return rc;
  const Mx4Gather from = {nullptr, 1, rows, 1};
  return launch_quantize_rows<8>(x, x_dtype, ld, from, rows, k, nullptr, 0, codes, scales, nullptr,
                                 static_cast<cudaStream_t>(stream));
}

extern "C" int axm_mx8_dequantize_rows(const void* codes, const void* scales, int32_t rows, int32_t k, void* out,
                                       int32_t out_dtype, int64_t ld, void* stream) {
  const char* what = "axm_mx8_dequantize_rows";
  if (int rc = check_rows(rows, k, 0, what)) return rc;
  if (int rc = check_dtype(out_dtype, what)) return rc;
  if (rows == 0) return AXM_OK;  // matrices without rows may have no address
  if (!codes || !scales || !out) return fail(AXM_ERR_ARGUMENT, "%s: null pointer", what);
  if (int rc = check_matrix(out, out_dtype, ld, k, what)) return rc;
  if (misaligned(codes, 16)) return fail(AXM_ERR_ARGUMENT, "%s: codes must be 16-byte aligned", what);
  if (int rc = require_device()) return rc;
  return launch_dequantize_rows<8>(codes, scales, rows, k, nullptr, 0, out, out_dtype, ld,
                                   static_cast<cudaStream_t>(stream));
}

extern "C" int axm_mx4_quantize_weights(const void* w, int32_t w_dtype, int32_t experts, int32_t k, int32_t n, void* codes,
                                        void* scales, void* stream) {
  const char* what = "axm_mx4_quantize_weights";
  if (int rc = check_weights(experts, k, n, what)) return rc;
  if (int rc = check_dtype(w_dtype, what)) return rc;
  if (!w || !codes || !scales) return fail(AXM_ERR_ARGUMENT, "%s: null pointer", what);
  if (misaligned(w, 16) || misaligned(codes, 16) || misaligned(scales, 16))
    return fail(AXM_ERR_ARGUMENT, "%s: weights, codes and scales must be 16-byte aligned", what);
  if (int rc = require_device()) return rc;
  const dim3 grid((n + kWeightsN - 1) / kWeightsN, (k + kWeightsK - 1) / kWeightsK, experts);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* s = static_cast<uint8_t*>(scales);
  if (w_dtype == AXM_DTYPE_BF16)
    mx4_quantize_weights_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(w), k, n, c, s);
  else
    mx4_quantize_weights_kernel<float><<<grid, 256, 0, st>>>(static_cast<const float*>(w), k, n, c, s);
  return check_launch("mx4_quantize_weights_kernel");
}

extern "C" int axm_mx4_dequantize_weights(const void* codes, const void* scales, int32_t experts, int32_t k, int32_t n,
                                          void* w, int32_t w_dtype, void* stream) {
  const char* what = "axm_mx4_dequantize_weights";
  if (int rc = check_weights(experts, k, n, what)) return rc;
  if (int rc = check_dtype(w_dtype, what)) return rc;
  if (!w || !codes || !scales) return fail(AXM_ERR_ARGUMENT, "%s: null pointer", what);
  if (misaligned(w, 16) || misaligned(codes, 16) || misaligned(scales, 16))
    return fail(AXM_ERR_ARGUMENT, "%s: weights, codes and scales must be 16-byte aligned", what);
  if (int rc = require_device()) return rc;
  const dim3 grid((n + kWeightsN - 1) / kWeightsN, (k + kWeightsK - 1) / kWeightsK, experts);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  if (w_dtype == AXM_DTYPE_BF16)
    mx4_dequantize_weights_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(c, s, k, n, static_cast<__nv_bfloat16*>(w));
  else
    mx4_dequantize_weights_kernel<float><<<grid, 256, 0, st>>>(c, s, k, n, static_cast<float*>(w));
  return check_launch("mx4_dequantize_weights_kernel");
}

extern "C" int axm_mx4_pack_scales(const void* plain, int32_t experts, int32_t k, int32_t n, void* scales, void* stream) {
  const char* what = "axm_mx4_pack_scales";
  if (int rc = check_weights(experts, k, n, what)) return rc;
  if (!plain || !scales) return fail(AXM_ERR_ARGUMENT, "%s: null pointer", what);
  if (misaligned(scales, 16)) return fail(AXM_ERR_ARGUMENT, "%s: scales must be 16-byte aligned", what);
  if (int rc = require_device()) return rc;
  const long long items = (long long)experts * n * mx4_chunks(k);
  long long blocks = (items + 255) / 256;
  if (blocks > 16LL * sm_count()) blocks = 16LL * sm_count();
  mx4_pack_scales_kernel<<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(plain), experts, k, n, static_cast<uint8_t*>(scales));
  return check_launch("mx4_pack_scales_kernel");
}
