// Microscaled blocks: 32 neighbours along the reduction axis share one power of two.
//
//   scale byte  s = max(exponent field of the block's largest magnitude (as fp32) - emax, 0),
//               i.e. 2^(s - 127) with s - 127 = floor(log2(amax)) - emax, emax = 2 (e2m1) or 8 (e4m3);
//               a block of zeros has s = 0, a block with an infinity or a NaN has s = 255 and
//               stands for NaNs
//   code        x * 2^(127 - s), a product that is exact, rounded to nearest even by the
//               conversion instruction, saturating at 6 (e2m1) or 448 (e4m3)
//
// 4-bit operands of the matrix products (csrc/mx4_gemm.cu): two codes a byte, the lower index in
// the low half; rows of K / 2 bytes.  Their scale bytes are kept in the order in which the tensor
// core wants them in tensor memory: a tile is 128 rows, a chunk of a tile 128 rows x 128 elements
// = 512 bytes with the byte of (row r, block b) at (r % 32) * 16 + (r / 32) * 4 + b.  A tile's
// chunks follow one another, ceil(K / 256) * 2 of them (a pipeline stage is 256 elements); the
// bytes of blocks beyond K are 0, those of rows that do not exist are never written.
// Tiles of activations start at each segment's first row: rows of segment s are in the tiles from
// out_row0 / 128 + s on (never two segments in one tile, whatever their lengths).  Inside a call that
// runs on the few-rows kernels they have 16, 32 or 64 rows instead, in the same places of 512 bytes.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace axm {

constexpr int kMxBlock = 32;

__host__ __device__ constexpr int mx4_chunks(int k) { return (k + 255) / 256 * 2; }
__host__ __device__ constexpr long long mx4_row_tiles(long long rows, int num_segments, int tile_rows = 128) {
  return rows / tile_rows + num_segments;
}
// Room for any tile_rows that mx4_choose settles on, in a workspace made for `rows` or more.
__host__ __device__ constexpr long long mx4_row_tiles_most(long long rows, int num_segments) {
  return rows / 128 + 2LL * num_segments;
}

// The rows of a grouped 4-bit product: a segment table in device memory (its rows are out_row0 ..
// of the operand and of the output; a_row0 is not looked at), or none: one segment of all rows.
enum { kMx4Few = 0, kMx4Single = 1, kMx4Pair = 2 };  // mx4_few.cu; the two of mx4_gemm.cu
struct Mx4Rows {
  const AxmSegment* segments;
  int num_segments;
  int rows;            // of the operand and of the output
  int table_segments;  // segments of the whole table the scale tiles were laid out with
  int seg_base;        // index of segments[0] in that table
  int expert_base;     // expert id of the first weight matrix of this launch
  int tile_rows;       // rows of a scale tile (and of a row tile of the few-rows kernels: 16, 32, 64, 128)
  int kernel;          // kMx4Few, kMx4Single or kMx4Pair
  int32_t* status;
  float* few_partial;      // workspace of the few-rows kernels: partial tiles,
  uint32_t* few_counters;  //   a counter a tile (zero before the first launch of a call)
};

// q4 of the rows of a bf16 or fp32 matrix (microscale.cu).  Row r < tail_row0 comes from source row
// row_src[r] / row_div (row_src null: r), rows from tail_row0 on from (r - tail_row0) % tail_mod.
struct Mx4Gather {
  const int32_t* row_src;
  int row_div;
  int tail_row0;
  int tail_mod;
};
int launch_mx4_quantize_rows(const void* x, int32_t dtype, int64_t ld, const Mx4Gather& from, const Mx4Rows& rows, int k,
                             void* codes, void* scales, cudaStream_t st);
// The products (mx4_gemm.cu).
int launch_mx4_linear(const Mx4Rows& r, const void* a_codes, const void* a_scales, const void* w_codes,
                      const void* w_scales, int experts, int k, int n, void* out, bool out_bf16, cudaStream_t st);
int launch_mx4_gated(const Mx4Rows& r, const void* a_codes, const void* a_scales, const AxmMx4Experts* w, int experts,
                     int d, int f, void* h_codes, void* h_scales, cudaStream_t st);

// The same for few rows a segment (mx4_few.cu), with its workspace.
// The kernel for rows in segments of at most max_rows, and the height of its scale tiles.
int mx4_choose(int rows, int num_segments, int max_rows, int* tile_rows);
int mx4_few_counters();
size_t mx4_few_partial_bytes(bool gated);
int launch_mx4_linear_few(const Mx4Rows& r, const void* a_codes, const void* a_scales, const void* w_codes,
                          const void* w_scales, int experts, int k, int n, void* out, bool out_bf16, cudaStream_t st);
int launch_mx4_gated_few(const Mx4Rows& r, const void* a_codes, const void* a_scales, const AxmMx4Experts* w, int experts,
                         int d, int f, void* h_codes, void* h_scales, cudaStream_t st);

// Tensor maps (mx4_gemm.cu).  Codes: rows of k / 2 bytes, a box of 128 bytes x box_rows rows, 128-byte swizzle.
int mx4_map_codes(CUtensorMap* m, const void* base, uint64_t experts, uint64_t rows, uint64_t k, uint32_t box_rows);
// Scale chunks: words [tiles][chunks][128], a box of two chunks of one tile.
int mx4_map_scales(CUtensorMap* m, const void* base, uint64_t tiles, int k);

#if defined(__CUDACC__)

// Scale byte of a block whose largest magnitude has these fp32 bits (sign cleared).
template <int kEmax>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23);
  if (e == 255) return 255u;
  return e > kEmax ? (uint32_t)(e - kEmax) : 0u;
}
// 2^(127 - s): what a block's values are multiplied with before the conversion.  (s <= 253 for
// finite blocks; for s = 255 the result does not matter, the block reads as NaN.)
__device__ __forceinline__ float mx_inverse_scale(uint32_t s) {
  return __uint_as_float(s >= 254u ? 0x00800000u : (254u - s) << 23);
}
// 2^(s - 127); s = 0 is a subnormal, s = 255 a NaN.
__device__ __forceinline__ float mx_scale_value(uint32_t s) {
  return __uint_as_float(s == 255u ? 0x7fc00000u : (s == 0u ? 0x00400000u : s << 23));
}

// Eight values to eight e2m1 codes, value 0 in the lowest four bits.
__device__ __forceinline__ uint32_t mx4_pack8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t"
      "}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// A row's block of 32 to its codes and scale byte.
__device__ __forceinline__ uint4 mx4_quantize_block(const float (&h)[32], uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) top = max(top, __float_as_uint(h[j]) & 0x7fffffffu);
  byte = mx_scale_byte<2>(top);
  const float inv = mx_inverse_scale(byte);
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = h[8 * i + j] * inv;
    q[i] = mx4_pack8(t);
  }
  return make_uint4(q[0], q[1], q[2], q[3]);
}
// Reading back.  What a block of e2m1 holds is exact in bf16 (two significant bits, 2^-128 the smallest), and
// what a block of e4m3 holds is too but for the smallest codes under the scale bytes 0 to 2 (steps of 2^-136
// to 2^-134), which round once; to fp32 they are decoded one by one (mx8_unpack2).  So codes are decoded two at
// a time: their exponent and mantissa bits moved to bf16's places are the value times 2^-126 (e2m1) or 2^-120
// (e4m3), subnormal codes included, and two packed multiplications by powers of two put that right; the first
// is exact.  Half the instructions of decoding one by one in fp32, which is what bounded the kernels that read
// blocks back.
__device__ __forceinline__ uint32_t mx_scale_bf16x2(uint32_t s) {  // 2^(s - 127), twice
  const uint32_t h = s == 255u ? 0x7fc0u : (s == 0u ? 0x0040u : s << 7);
  return h * 0x10001u;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Eight e2m1 codes to four bf16 pairs.
__device__ __forceinline__ void mx4_decode8(uint32_t codes, uint32_t scale2, uint32_t (&out)[4]) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint32_t c = (codes >> (8 * p)) & 0xffu;
    const uint32_t x = c | (c << 12);  // the two codes at bits 0 and 16
    const uint32_t t = ((x << 6) & 0x01c001c0u) | ((x << 12) & 0x80008000u);
    out[p] = mul_bf16x2(mul_bf16x2(t, 0x7e807e80u), scale2);
  }
}
// Four e4m3 codes to two bf16 pairs.
__device__ __forceinline__ void mx8_decode4(uint32_t codes, uint32_t scale2, uint32_t& lo, uint32_t& hi) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const uint32_t x = __byte_perm(codes, 0, p ? 0x4342 : 0x4140);  // a code in each half
    const uint32_t t = ((x << 4) & 0x07f007f0u) | ((x << 8) & 0x80008000u);
    (p ? hi : lo) = mul_bf16x2(mul_bf16x2(t, 0x7b807b80u), scale2);
  }
}

// Bit 7 of every byte that is e4m3's NaN code (0x7f or 0xff), which mx8_decode4 takes for 480.  The library
// writes none, codes from elsewhere may hold some.
__device__ __forceinline__ uint32_t mx8_nan_codes(uint32_t codes) {
  return ((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// Four values to four e4m3 codes, value 0 in the lowest byte.
__device__ __forceinline__ uint32_t mx8_pack4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t"
      "}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// Two e4m3 codes (low half of the word first) to fp32.
__device__ __forceinline__ float2 mx8_unpack2(uint32_t two) {
  uint32_t h;
  asm("{\n\t"
      ".reg .b16 t;\n\t"
      "cvt.u16.u32 t, %1;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, t;\n\t"
      "}"
      : "=r"(h)
      : "r"(two));
  float2 f;
  asm("{\n\t"
      ".reg .b16 lo, hi;\n\t"
      "mov.b32 {lo, hi}, %2;\n\t"
      "cvt.f32.f16 %0, lo;\n\t"
      "cvt.f32.f16 %1, hi;\n\t"
      "}"
      : "=f"(f.x), "=f"(f.y)
      : "r"(h));
  return f;
}

// The segment that output row `row` belongs to: the last entry with rows that starts at or before it (tables
// are ordered by out_row0; entries without rows may start anywhere, inside another's rows too), and its
// first row.  -1: the row is behind that segment's end.
// By a whole warp: 32 entries at a time, all loads of a round at once (a binary search is a chain of
// dependent loads, 3 us for 64 segments, which every row of a small call waited for).  Loads of four
// bytes: a table is an array of int32 and starts at any multiple of four.
struct RowSegment {
  int seg, first;
};
__device__ __forceinline__ RowSegment segment_of_row(const AxmSegment* segments, int n, int row) {
  const int lane = threadIdx.x & 31;
  RowSegment r = {-1, 0};
  int rows = 0;
  for (int s0 = 0; s0 < n; s0 += 32) {
    const bool there = s0 + lane < n;
    const int start = there ? __ldg(&segments[s0 + lane].out_row0) : 0x7fffffff;
    const int count = there ? __ldg(&segments[s0 + lane].rows) : 0;
    const uint32_t here = __ballot_sync(0xffffffffu, start <= row && count > 0);
    if (here != 0) {
      const int at = 31 - __clz(here);
      r.seg = s0 + at;
      r.first = __shfl_sync(0xffffffffu, start, at);
      rows = __shfl_sync(0xffffffffu, count, at);
    }
    if (__any_sync(0xffffffffu, start > row)) break;  // all further entries start behind the row
  }
  // (a start before the first row would count tiles that the scale buffer does not have)
  if (r.first < 0 || row - r.first >= rows) r.seg = -1;
  return r;
}

// A table's entry, kept inside the buffers whatever it says: rows beyond `rows_total` are dropped, and a
// segment that starts outside or whose expert is not one of this launch's has none (the id is then 0xffff, which
// no launch has: experts are read from 16 bits).
__device__ __forceinline__ AxmSegment kept_inside(AxmSegment sg, int rows_total, int expert_base, int experts) {
  const int e = (sg.expert & ~AXM_SEG_ALT_A) - expert_base;
  const bool known = e >= 0 && e < experts;
  const bool there = known && sg.out_row0 >= 0 && sg.out_row0 < rows_total;
  sg.rows = there ? min(max(sg.rows, 0), rows_total - sg.out_row0) : 0;
  sg.expert = known ? sg.expert : 0xffff;
  return sg;
}
// Entry s of a product's segment table (none: one segment of all rows).
__device__ __forceinline__ AxmSegment product_segment(const AxmSegment* segments, int s, int rows_total, int expert_base,
                                                      int experts) {
  if (segments == nullptr) return AxmSegment{0, 0, rows_total, expert_base};
  return kept_inside(segments[s], rows_total, expert_base, experts);
}

// ---- tcgen05, block-scaled kind::mxf4, one CTA ----
__device__ __forceinline__ void tc_mma1_mx4(uint32_t d_tmem, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                            uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t"
      "}" ::"r"(d_tmem),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_cp1_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Shared-memory descriptor of a 512-byte scale chunk: no swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr >> 4) & 0x3fffu) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

#endif

}  // namespace axm
