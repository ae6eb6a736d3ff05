// Quantising to microscaled blocks and reading them back (formats: microscale.cuh).  The engine
// has no low-bit formats; its bf16 weights and their fp32 master copies
// (core/src/CUDA/util/gpu_types.cuh:148-168) are what these kernels read.
//
// All four are bound by memory: every value is read once and written once.
#include "microscale.cuh"

namespace axm {

namespace {

struct Words8 {
  uint32_t w[8];
};
// 32 bytes in one load or store (the address is a multiple of 16 bytes only where kWide is false).
template <bool kWide>
__device__ __forceinline__ Words8 load32(const void* p) {
  Words8 r;
  if constexpr (kWide) {
    asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
        : "l"(p));
  } else {
    const uint4 a = __ldg(static_cast<const uint4*>(p)), b = __ldg(static_cast<const uint4*>(p) + 1);
    r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
    r.w[4] = b.x; r.w[5] = b.y; r.w[6] = b.z; r.w[7] = b.w;
  }
  return r;
}
template <bool kWide>
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  if constexpr (kWide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    static_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    static_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// Rows are cut into runs of 512 elements, one warp a run: a lane holds sixteen neighbours (32 bytes
// of bf16), two lanes a block.  Of rows of up to 256 (128) elements a warp takes two (four), 2^log_lanes
// lanes each.  A CTA of eight warps gives each row 2^log_wpr of them (as many as
// the row has runs, up to eight; in large calls fewer, so that each has several runs), and a warp
// has up to kAheadOf<T> runs' loads in flight.
// These kernels are bound by their instructions as easily as by memory: a first form with eight
// elements a lane and fp32 arithmetic throughout issued 160 instructions per 256 elements and read
// and wrote 3.9 TB/s.  As it is: 16384 x 4096 bf16 to 8 bits and back 64 us (407 MB, 6.4 TB/s), 8191 x 5632
// fp32 to 4 bits and back 59 us (326 MB, 5.5 TB/s); about half of the issue slots stay empty.
constexpr int kMostAhead = 4;
template <typename T>
constexpr int kAheadOf = sizeof(T) == 2 ? kMostAhead : kMostAhead / 2;  // the same registers

// What the first kernel of a call clears for the ones behind it.
struct MxClear {
  int32_t* status;
  uint32_t* counters;
  int num_counters;
};

// kBits = 4: scale bytes in tile order, the row's last, partial stage padded with zero bytes.
// kBits = 8: codes [rows][K], scale bytes [rows][K / 32].
// kWide: rows start at multiples of 32 bytes.
// `from` says which source row a row comes from; row_src[r] < 0: zeros.
template <int kBits, typename T, bool kWide>
__global__ void __launch_bounds__(256, 4)
mx_quantize_rows_kernel(const T* __restrict__ x, long long ld, Mx4Gather from, int rows, int k, int log_wpr,
                        int log_lanes, const AxmSegment* __restrict__ segments, int num_segments, int tile_rows,
                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, MxClear clear) {
  // a product that is launched to start early may prepare itself now; it waits before it reads
  asm volatile("griddepcontrol.launch_dependents;");
  if (blockIdx.x == 0) {
    if (clear.status != nullptr && threadIdx.x == 0) *clear.status = 0;
    for (int i = threadIdx.x; i < clear.num_counters; i += 256) clear.counters[i] = 0u;
  }
  constexpr bool kBf16 = sizeof(T) == 2;
  constexpr int kAhead = kAheadOf<T>;
  constexpr int kWords = kBf16 ? 1 : 2;  // 32-byte pieces a lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int runs = (k + 511) / 512, wpr = 1 << log_wpr;
  const int log_rpw = 5 - log_lanes;  // rows a warp (more than one only where a row is one run)
  const int group = lane >> log_lanes, in_row = lane & ((1 << log_lanes) - 1);
  const int rows_per_cta = (8 >> log_wpr) << log_rpw;
  for (long long row_at = (long long)blockIdx.x * rows_per_cta + ((warp >> log_wpr) << log_rpw); row_at < rows;
       row_at += (long long)gridDim.x * rows_per_cta) {
    const int row = (int)row_at + group;
    const bool there = row_at + group < rows;
    long long src = there ? row : -1;
    if (there && row >= from.tail_row0) {
      src = (row - from.tail_row0) % from.tail_mod;
    } else if (there && from.row_src != nullptr) {
      const int s = __ldg(from.row_src + row);
      src = s < 0 ? -1 : s / from.row_div;
    }
    const T* in = x + (src < 0 ? 0 : src) * ld;
    Words8 v[kAhead][kWords];
    auto fetch = [&](int run0) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k0 = (run0 + i * wpr) * 512 + in_row * 16;  // k is a multiple of 32: all sixteen or none
        if (k0 < k && src >= 0) {
#pragma unroll
          for (int j = 0; j < kWords; ++j) v[i][j] = load32<kWide>(in + k0 + 8 * j);
        } else {
#pragma unroll
          for (int j = 0; j < kWords; ++j) v[i][j] = Words8{};
        }
      }
    };
    int run0 = warp & (wpr - 1);
    fetch(run0);  // on their way while the row's segment is looked up
    uint8_t* out = codes + (size_t)row * (kBits == 4 ? k >> 1 : k);
    uint8_t* sc = scales;  // this row's scale bytes; kBits 4: in chunk 0
    bool placed = there;   // a row behind its segment's end has no place among the tiles
    if constexpr (kBits == 4) {
      RowSegment at = {0, 0};
      if (segments != nullptr) {
        for (int g = 0; g < (1 << log_rpw); ++g) {
          const RowSegment found = segment_of_row(segments, num_segments, (int)row_at + g);
          if (g == group) at = found;
        }
        placed = there && at.seg >= 0;
      }
      const int r = placed ? row - at.first : 0;
      const int in_tile = r & (tile_rows - 1);
      sc += ((size_t)(at.first / tile_rows + (placed ? at.seg : 0) + r / tile_rows) * mx4_chunks(k)) * 512 +
            (in_tile & 31) * 16 + (in_tile >> 5) * 4;
    } else {
      sc += (size_t)row * (k >> 5);
    }
    for (; run0 < runs; run0 += kAhead * wpr) {
      if (run0 >= kAhead * wpr) fetch(run0);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int run = run0 + i * wpr;
        if (run >= runs) break;
        const int k0 = run * 512 + in_row * 16;
        const bool write = there && k0 < k;
        uint32_t top = 0;
        if constexpr (kBf16) {  // largest magnitude by the bits, two at a time
#pragma unroll
          for (int j = 0; j < 8; ++j) top = __vmaxu2(top, v[i][0].w[j] & 0x7fff7fffu);
          top = max(top & 0xffff0000u, top << 16);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) top = max(top, v[i][j >> 3].w[j & 7] & 0x7fffffffu);
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        const uint32_t s = mx_scale_byte<kBits == 4 ? 2 : 8>(top);
        const float inv = mx_inverse_scale(s);
        auto value = [&](int j) {  // element j of the lane's sixteen, scaled
          if constexpr (kBf16) {
            const uint32_t w = v[i][0].w[j >> 1];
            return ((j & 1) ? bf16_hi(w) : bf16_lo(w)) * inv;
          } else {
            return __uint_as_float(v[i][j >> 3].w[j & 7]) * inv;
          }
        };
        if constexpr (kBits == 4) {
          uint32_t c[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = value(8 * h + j);
            c[h] = mx4_pack8(t);
          }
          if (write) *reinterpret_cast<uint2*>(out + (k0 >> 1)) = make_uint2(c[0], c[1]);
          // the four bytes of a 128-element chunk gathered into one word by the chunk's first lane
          uint32_t word = s << (8 * ((lane >> 1) & 3));
          word |= __shfl_xor_sync(0xffffffffu, word, 2);
          word |= __shfl_xor_sync(0xffffffffu, word, 4);
          const int chunk = run * 4 + (in_row >> 3);
          if (placed && (lane & 7) == 0 && chunk < mx4_chunks(k)) *reinterpret_cast<uint32_t*>(sc + (size_t)chunk * 512) = word;
          // eight lanes hold one chunk; a stage has two
          if (log_lanes == 3 && placed && in_row == 0) *reinterpret_cast<uint32_t*>(sc + 512) = 0u;
        } else if (write) {
          uint32_t c[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) c[h] = mx8_pack4(value(4 * h), value(4 * h + 1), value(4 * h + 2), value(4 * h + 3));
          *reinterpret_cast<uint4*>(out + k0) = make_uint4(c[0], c[1], c[2], c[3]);
          if ((lane & 1) == 0) sc[k0 >> 5] = (uint8_t)s;
        }
      }
    }
  }
}

template <int kBits, typename T, bool kWide>
__global__ void __launch_bounds__(256)
mx_dequantize_rows_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, int k,
                          int log_wpr, int log_lanes, const AxmSegment* __restrict__ segments,
                          int num_segments, T* __restrict__ out, long long ld) {
  constexpr int kAhead = kMostAhead;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int runs = (k + 511) / 512, wpr = 1 << log_wpr;
  const int log_rpw = 5 - log_lanes;
  const int group = lane >> log_lanes, in_row = lane & ((1 << log_lanes) - 1);
  const int rows_per_cta = (8 >> log_wpr) << log_rpw;
  for (long long row_at = (long long)blockIdx.x * rows_per_cta + ((warp >> log_wpr) << log_rpw); row_at < rows;
       row_at += (long long)gridDim.x * rows_per_cta) {
    const int row = (int)row_at + group;
    bool there = row_at + group < rows;
    const uint8_t* in = codes + (size_t)row * (kBits == 4 ? k >> 1 : k);
    const uint8_t* sc = scales;
    T* to = out + (size_t)row * ld;
    if constexpr (kBits == 4) {
      RowSegment at = {0, 0};
      if (segments != nullptr) {
        for (int g = 0; g < (1 << log_rpw); ++g) {
          const RowSegment found = segment_of_row(segments, num_segments, (int)row_at + g);
          if (g == group) at = found;
        }
        there = there && at.seg >= 0;  // others are left as they are
        if (at.seg < 0) at = RowSegment{0, row};
      }
      const int r = row - at.first;
      sc += ((size_t)(at.first / 128 + at.seg + r / 128) * mx4_chunks(k)) * 512 + (r & 31) * 16 + ((r & 127) >> 5) * 4;
    } else {
      sc += (size_t)row * (k >> 5);
    }
    for (int run0 = warp & (wpr - 1); run0 < runs; run0 += kAhead * wpr) {
      uint4 c[kAhead];
      uint32_t s[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int run = run0 + i * wpr, k0 = run * 512 + in_row * 16;
        c[i] = make_uint4(0, 0, 0, 0);
        s[i] = 0;
        if (there && k0 < k) {
          if constexpr (kBits == 4) {
            const uint2 t = __ldg(reinterpret_cast<const uint2*>(in + (k0 >> 1)));
            c[i].x = t.x;
            c[i].y = t.y;
            s[i] = __ldg(sc + (size_t)(run * 4 + (in_row >> 3)) * 512 + ((lane >> 1) & 3));
          } else {
            c[i] = __ldg(reinterpret_cast<const uint4*>(in + k0));
            s[i] = __ldg(sc + (k0 >> 5));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k0 = (run0 + i * wpr) * 512 + in_row * 16;
        if (!there || k0 >= k) break;
        if constexpr (kBits == 8 && sizeof(T) == 4) {
          // one by one: e4m3 under the smallest scales has values (from 2^-136 on) that bf16 has not
          const float f = mx_scale_value(s[i]);
          const uint32_t word[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 two = mx8_unpack2((word[2 * h + (j >> 1)] >> (16 * (j & 1))) & 0xffffu);
              v[2 * j] = __float_as_uint(two.x * f);
              v[2 * j + 1] = __float_as_uint(two.y * f);
            }
            store32<kWide>(to + k0 + 8 * h, v);
          }
          continue;
        }
        const uint32_t f = mx_scale_bf16x2(s[i]);
        uint32_t w[8];
        if constexpr (kBits == 4) {
          uint32_t t[4];
          mx4_decode8(c[i].x, f, t);
          w[0] = t[0]; w[1] = t[1]; w[2] = t[2]; w[3] = t[3];
          mx4_decode8(c[i].y, f, t);
          w[4] = t[0]; w[5] = t[1]; w[6] = t[2]; w[7] = t[3];
        } else {
          mx8_decode4(c[i].x, f, w[0], w[1]);
          mx8_decode4(c[i].y, f, w[2], w[3]);
          mx8_decode4(c[i].z, f, w[4], w[5]);
          mx8_decode4(c[i].w, f, w[6], w[7]);
          const uint32_t word[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
          uint32_t nan = 0;
#pragma unroll
          for (int h = 0; h < 4; ++h) nan |= mx8_nan_codes(word[h]);
          if (nan != 0) {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const uint32_t n = mx8_nan_codes(word[h]);
              w[2 * h] |= ((n & 0x80u) ? 0x7fc0u : 0u) | ((n & 0x8000u) ? 0x7fc00000u : 0u);
              w[2 * h + 1] |= ((n & 0x800000u) ? 0x7fc0u : 0u) | ((n & 0x80000000u) ? 0x7fc00000u : 0u);
            }
          }
        }
        if constexpr (sizeof(T) == 2) {
          store32<kWide>(to + k0, w);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              v[2 * j] = w[4 * h + j] << 16;
              v[2 * j + 1] = w[4 * h + j] & 0xffff0000u;
            }
            store32<kWide>(to + k0 + 8 * h, v);
          }
        }
      }
    }
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
  __shared__ __align__(4) uint8_t sc[kWeightsN][8];  // read back four bytes at a time
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

// 8 x 2048 x 5632 fp32 to codes and back: 109 us (652 MB, 6.0 TB/s).
// Back to [E][K][N]: a thread owns four neighbouring columns of one block of 32 k, and half a warp
// writes 64 columns of a row.
template <typename T>
__global__ void __launch_bounds__(128)
mx4_dequantize_weights_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int k, int n,
                              T* __restrict__ w) {
  __shared__ uint4 tile[kWeightsN * 8];
  const int e = blockIdx.z, n0 = blockIdx.x * kWeightsN, k0 = blockIdx.y * kWeightsK;
  // piece p of column c at p ^ (c / 4 % 8): four columns apart is what the lanes read together
  for (int i = threadIdx.x; i < kWeightsN * 8; i += 128) {
    const int c = i >> 3, piece = i & 7;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (n0 + c < n && k0 + piece * kMxBlock < k)
      v = __ldg(reinterpret_cast<const uint4*>(codes + ((size_t)e * n + n0 + c) * (k >> 1) + (k0 >> 1) + piece * 16));
    tile[c * 8 + (piece ^ ((c >> 2) & 7))] = v;
  }
  __syncthreads();
  const int quad = threadIdx.x & 15, blk = threadIdx.x >> 4;
  const int col = n0 + 4 * quad, kk = k0 + blk * kMxBlock;
  if (col >= n || kk >= k) return;  // n is a multiple of 8: four columns or none
  uint32_t f[4], q[4][4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const uint4 v = tile[(4 * quad + h) * 8 + (blk ^ (quad & 7))];
    q[h][0] = v.x; q[h][1] = v.y; q[h][2] = v.z; q[h][3] = v.w;
  }
  {  // the four columns' scale bytes are 16 bytes apart
    const size_t t = (size_t)e * ((n + 127) / 128) + col / 128;
    const int r = col & 127;
    const uint8_t* p = scales + (t * mx4_chunks(k) + (kk >> 7)) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (blk & 3);
#pragma unroll
    for (int h = 0; h < 4; ++h) f[h] = mx_scale_bf16x2(__ldg(p + 16 * h));
  }
  T* p = w + ((size_t)e * k + kk) * n + col;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t d[4][4];
#pragma unroll
    for (int h = 0; h < 4; ++h) mx4_decode8(q[h][i], f[h], d[h]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t lo, hi;  // columns 0, 1 and 2, 3 of row 8 i + j
      lo = __byte_perm(d[0][j >> 1], d[1][j >> 1], (j & 1) ? 0x7632 : 0x5410);
      hi = __byte_perm(d[2][j >> 1], d[3][j >> 1], (j & 1) ? 0x7632 : 0x5410);
      T* to = p + (size_t)(8 * i + j) * n;
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
      else
        *reinterpret_cast<float4*>(to) = make_float4(bf16_lo(lo), bf16_hi(lo), bf16_lo(hi), bf16_hi(hi));
    }
  }
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

// Warps a row (as a power of two) and CTAs of a row kernel.
struct RowLaunch {
  int log_wpr, log_lanes;
  unsigned grid;
};
RowLaunch row_launch(int32_t rows, int32_t k, int ahead) {
  RowLaunch l = {0, k <= 128 ? 3 : k <= 256 ? 4 : 5, 0};
  const int runs = (k + 511) / 512;
  while (l.log_wpr < 3 && (2 << l.log_wpr) <= runs) ++l.log_wpr;
  // enough rows for every SM's warps: several runs a warp rather than several warps a row (not for
  // fp32 sources, ahead = 1: their runs are twice as long, 8-bit rows 8191 x 5632 58 us against 63)
  while (l.log_wpr > 0 && (runs >> l.log_wpr) < ahead && ((long long)rows << (l.log_wpr - 1)) >= 16LL * sm_count()) --l.log_wpr;
  const long long per = (long long)(8 >> l.log_wpr) << (5 - l.log_lanes);
  const long long blocks = (rows + per - 1) / per, most = 32LL * sm_count();
  l.grid = (unsigned)(blocks < most ? blocks : most);
  return l;
}
// Whether every row of a matrix starts at a multiple of 32 bytes.
bool rows_at_32(const void* p, int64_t ld, int32_t dtype) {
  return !misaligned(p, 32) && ld * (dtype == AXM_DTYPE_BF16 ? 2 : 4) % 32 == 0;
}

template <int kBits, typename T>
int launch_quantize_rows_of(const void* x, bool wide, int64_t ld, const Mx4Gather& from, int32_t rows, int32_t k,
                            const AxmSegment* segments, int32_t num_segments, int tile_rows, void* codes, void* scales,
                            const MxClear& clear, cudaStream_t st) {
  const RowLaunch l = row_launch(rows, k, sizeof(T) == 2 ? kMostAhead : 1);
  auto* kernel = wide ? mx_quantize_rows_kernel<kBits, T, true> : mx_quantize_rows_kernel<kBits, T, false>;
  kernel<<<l.grid, 256, 0, st>>>(static_cast<const T*>(x), ld, from, rows, k, l.log_wpr, l.log_lanes, segments, num_segments, tile_rows,
                                 static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), clear);
  return check_launch("mx_quantize_rows_kernel");
}
template <int kBits>
int launch_quantize_rows(const void* x, int32_t dtype, int64_t ld, const Mx4Gather& from, int32_t rows, int32_t k,
                         const AxmSegment* segments, int32_t num_segments, int tile_rows, void* codes, void* scales,
                         const MxClear& clear, cudaStream_t st) {
  const bool wide = rows_at_32(x, ld, dtype);
  return dtype == AXM_DTYPE_BF16
             ? launch_quantize_rows_of<kBits, __nv_bfloat16>(x, wide, ld, from, rows, k, segments, num_segments, tile_rows, codes, scales, clear, st)
             : launch_quantize_rows_of<kBits, float>(x, wide, ld, from, rows, k, segments, num_segments, tile_rows, codes, scales, clear, st);
}

template <int kBits, typename T>
int launch_dequantize_rows_of(const void* codes, const void* scales, int32_t rows, int32_t k, const AxmSegment* segments,
                              int32_t num_segments, void* out, bool wide, int64_t ld, cudaStream_t st) {
  const RowLaunch l = row_launch(rows, k, kMostAhead);
  auto* kernel = wide ? mx_dequantize_rows_kernel<kBits, T, true> : mx_dequantize_rows_kernel<kBits, T, false>;
  kernel<<<l.grid, 256, 0, st>>>(static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), rows, k,
                                 l.log_wpr, l.log_lanes, segments, num_segments, static_cast<T*>(out), ld);
  return check_launch("mx_dequantize_rows_kernel");
}
template <int kBits>
int launch_dequantize_rows(const void* codes, const void* scales, int32_t rows, int32_t k, const AxmSegment* segments,
                           int32_t num_segments, void* out, int32_t dtype, int64_t ld, cudaStream_t st) {
  const bool wide = rows_at_32(out, ld, dtype);
  return dtype == AXM_DTYPE_BF16
             ? launch_dequantize_rows_of<kBits, __nv_bfloat16>(codes, scales, rows, k, segments, num_segments, out, wide, ld, st)
             : launch_dequantize_rows_of<kBits, float>(codes, scales, rows, k, segments, num_segments, out, wide, ld, st);
}

}  // namespace

int launch_mx4_quantize_rows(const void* x, int32_t dtype, int64_t ld, const Mx4Gather& from, const Mx4Rows& rows, int k,
                             void* codes, void* scales, cudaStream_t st) {
  return launch_quantize_rows<4>(x, dtype, ld, from, rows.rows, k, rows.segments, rows.num_segments, rows.tile_rows, codes, scales,
                                 MxClear{rows.status, rows.few_counters, rows.few_counters ? mx4_few_counters() : 0}, st);
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
  return launch_quantize_rows<4>(x, x_dtype, ld, from, rows, k, segments, num_segments, 128, codes, scales,
                                 MxClear{}, static_cast<cudaStream_t>(stream));
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
  return launch_quantize_rows<8>(x, x_dtype, ld, from, rows, k, nullptr, 0, 128, codes, scales, MxClear{},
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
    mx4_dequantize_weights_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(c, s, k, n, static_cast<__nv_bfloat16*>(w));
  else
    mx4_dequantize_weights_kernel<float><<<grid, 128, 0, st>>>(c, s, k, n, static_cast<float*>(w));
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
