// Host side of the calls made of the 4-bit kernels: the linear product, the expert feed-forward
// and the whole layer from 4-bit expert weights.  Like moe_api.cu it validates, carves the
// caller's workspace and enqueues; it allocates nothing and never synchronises.
#include "microscale.cuh"
#include "gemm_common.cuh"
#include "router.cuh"

namespace axm {

int check_mx_matrix(const void* p, int32_t dtype, int64_t ld, int32_t k, const char* what);  // microscale.cu

namespace {

struct Carver {
  char* base;
  size_t off = 0;
  void* take(size_t n) {
    void* p = base ? base + off : nullptr;
    off += (n + 255) & ~static_cast<size_t>(255);
    return p;
  }
};

int check_workspace(const void* ws, size_t have, size_t need) {
  if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 255) != 0)
    return fail(AXM_ERR_WORKSPACE, "workspace is null or not 256-byte aligned");
  if (have < need) return fail(AXM_ERR_WORKSPACE, "workspace has %zu bytes, %zu needed", have, need);
  return AXM_OK;
}

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

int check_experts(const AxmMx4Experts* w, const char* what) {
  if (!w || !w->gate_codes || !w->gate_scales || !w->up_codes || !w->up_scales || !w->down_codes || !w->down_scales)
    return fail(AXM_ERR_ARGUMENT, "%s: null weights", what);
  if (off16(w->gate_codes) || off16(w->gate_scales) || off16(w->up_codes) || off16(w->up_scales) ||
      off16(w->down_codes) || off16(w->down_scales))
    return fail(AXM_ERR_ARGUMENT, "%s: codes and scales must be 16-byte aligned", what);
  return AXM_OK;
}

int check_ffn_desc(const AxmMoeDesc* d, const char* what) {
  if (d == nullptr) return fail(AXM_ERR_ARGUMENT, "desc is null");
  if (d->tokens < 0) return fail(AXM_ERR_ARGUMENT, "%s: tokens %d negative", what, d->tokens);
  if (d->d_model <= 0 || d->d_ff <= 0 || d->d_model % 32 || d->d_ff % 32)
    return fail(AXM_ERR_ARGUMENT, "%s: d_model %d and d_ff %d must be positive multiples of 32", what, d->d_model, d->d_ff);
  if (d->num_experts <= 0 || d->num_experts > 65535)
    return fail(AXM_ERR_ARGUMENT, "%s: num_experts %d not in 1..65535", what, d->num_experts);
  return AXM_OK;
}

// Workspace of the few-rows kernels.  Also where the pair kernels run: a workspace made for many
// rows serves calls with few.
struct FewWs {
  uint32_t* counters;
  float* partial;
};
FewWs carve_few(Carver& c, bool gated) {
  FewWs w;
  w.counters = static_cast<uint32_t*>(c.take(sizeof(uint32_t) * mx4_few_counters()));
  w.partial = static_cast<float*>(c.take(mx4_few_partial_bytes(gated)));
  return w;
}

struct LinearWs {
  int32_t* status;
  void *codes, *scales;
  FewWs few;
  size_t bytes;
};
LinearWs carve_linear(int tokens, int k, void* base) {
  Carver c{static_cast<char*>(base)};
  LinearWs w;
  w.status = static_cast<int32_t*>(c.take(4));
  w.codes = c.take((size_t)tokens * (k / 2));
  w.scales = c.take((size_t)mx4_row_tiles_most(tokens, 1) * mx4_chunks(k) * 512);
  w.few = carve_few(c, false);
  w.bytes = c.off;
  return w;
}

struct FfnWs {
  int32_t* status;
  void *x_codes, *x_scales, *h_codes, *h_scales;
  FewWs few;
  size_t bytes;
};
void carve_ffn(Carver& c, int rows, int num_segments, int d, int f, FfnWs* w) {
  w->few = carve_few(c, true);
  w->x_codes = c.take((size_t)rows * (d / 2));
  w->x_scales = c.take((size_t)mx4_row_tiles_most(rows, num_segments) * mx4_chunks(d) * 512);
  w->h_codes = c.take((size_t)rows * (f / 2));
  w->h_scales = c.take((size_t)mx4_row_tiles_most(rows, num_segments) * mx4_chunks(f) * 512);
}
FfnWs carve_expert_ffn(const AxmMoeDesc* d, int rows, int num_segments, void* base) {
  Carver c{static_cast<char*>(base)};
  FfnWs w;
  w.status = static_cast<int32_t*>(c.take(4));
  carve_ffn(c, rows, num_segments, d->d_model, d->d_ff, &w);
  w.bytes = c.off;
  return w;
}

// Both products of the feed-forward over one range of the table.
int launch_ffn(const Mx4Rows& r, const FfnWs& w, const AxmMx4Experts* experts, int num_experts, int d, int f, void* o,
               bool o_bf16, cudaStream_t st) {
  if (r.kernel == kMx4Few) {
    if (int rc = launch_mx4_gated_few(r, w.x_codes, w.x_scales, experts, num_experts, d, f, w.h_codes, w.h_scales, st)) return rc;
    return launch_mx4_linear_few(r, w.h_codes, w.h_scales, experts->down_codes, experts->down_scales, num_experts, f, d, o,
                                 o_bf16, st);
  }
  if (int rc = launch_mx4_gated(r, w.x_codes, w.x_scales, experts, num_experts, d, f, w.h_codes, w.h_scales, st)) return rc;
  return launch_mx4_linear(r, w.h_codes, w.h_scales, experts->down_codes, experts->down_scales, num_experts, f, d, o,
                           o_bf16, st);
}

struct LayerWs {
  FfnWs ffn;
  float* logits;
  int32_t* topk_idx;
  float* topk_gate;
  int32_t* block_counts;
  int32_t* offsets;
  int32_t* row_src;
  int32_t* slot_dst;
  AxmSegment* segments;
  void* o;
  void* router_scratch;
  size_t router_scratch_bytes;
  size_t bytes;
};
LayerWs carve_layer(const AxmMoeDesc* d, void* base) {
  Carver c{static_cast<char*>(base)};
  LayerWs w;
  const size_t T = d->tokens, E = d->num_experts, k = d->top_k, S = d->num_shared;
  const size_t rows = T * (k + S);
  w.ffn.status = static_cast<int32_t*>(c.take(4));
  w.logits = static_cast<float*>(c.take(4 * T * E));
  w.topk_idx = static_cast<int32_t*>(c.take(4 * T * k));
  w.topk_gate = static_cast<float*>(c.take(4 * T * k));
  w.block_counts = static_cast<int32_t*>(c.take(4 * AXM_ROUTE_BLOCKS * E));
  w.offsets = static_cast<int32_t*>(c.take(4 * (E + 1)));
  w.row_src = static_cast<int32_t*>(c.take(4 * T * k));
  w.slot_dst = static_cast<int32_t*>(c.take(4 * T * k));
  w.segments = static_cast<AxmSegment*>(c.take(sizeof(AxmSegment) * (E + S)));
  carve_ffn(c, (int)rows, (int)(E + S), d->d_model, d->d_ff, &w.ffn);
  w.o = c.take(4 * rows * d->d_model);
  w.router_scratch_bytes = 0;
  axm_moe_router_scratch_bytes(d, &w.router_scratch_bytes);
  w.router_scratch = c.take(w.router_scratch_bytes);
  w.bytes = w.ffn.bytes = c.off;
  return w;
}

int check_layer(const AxmMoeDesc* d) {
  const char* what = "axm_moe_forward_mx4";
  if (int rc = check_ffn_desc(d, what)) return rc;
  size_t ignored;
  return axm_moe_workspace_bytes(d, &ignored);  // the layer's own limits on experts, top_k, shared experts and rows
}

}  // namespace

}  // namespace axm

using namespace axm;

extern "C" int axm_mx4_linear_workspace_bytes(int32_t tokens, int32_t k, int32_t n, size_t* bytes) {
  size_t codes, scales;
  if (int rc = axm_mx4_rows_bytes(tokens, 0, k, &codes, &scales)) return rc;
  if (n <= 0 || n % 8) return fail(AXM_ERR_ARGUMENT, "axm_mx4_linear: n %d is not a positive multiple of 8", n);
  if (bytes == nullptr) return fail(AXM_ERR_ARGUMENT, "bytes is null");
  *bytes = carve_linear(tokens, k, nullptr).bytes;
  return AXM_OK;
}

extern "C" int axm_mx4_linear(const void* x, int32_t x_dtype, int64_t ld, int32_t tokens, int32_t k, int32_t n,
                              const void* w_codes, const void* w_scales, void* out, int32_t out_dtype, void* workspace,
                              size_t workspace_bytes, void* stream) {
  size_t need = 0;
  if (int rc = axm_mx4_linear_workspace_bytes(tokens, k, n, &need)) return rc;
  if (tokens == 0) return AXM_OK;  // matrices without rows may have no address
  if (!x || !w_codes || !w_scales || !out) return fail(AXM_ERR_ARGUMENT, "axm_mx4_linear: null pointer");
  if (int rc = check_mx_matrix(x, x_dtype, ld, k, "axm_mx4_linear: x")) return rc;
  if (out_dtype != AXM_DTYPE_BF16 && out_dtype != AXM_DTYPE_FP32)
    return fail(AXM_ERR_ARGUMENT, "axm_mx4_linear: out_dtype %d unknown", out_dtype);
  if (off16(w_codes) || off16(w_scales) || off16(out))
    return fail(AXM_ERR_ARGUMENT, "axm_mx4_linear: codes, scales and out must be 16-byte aligned");
  if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  if (int rc = require_device()) return rc;
  const LinearWs w = carve_linear(tokens, k, workspace);
  int tile;
  const int kernel = mx4_choose(tokens, 1, tokens, &tile);
  const Mx4Rows rows = {nullptr, 1, tokens, 1, 0, 0, tile, kernel, w.status, w.few.partial, w.few.counters};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Mx4Gather from = {nullptr, 1, tokens, 1};
  if (int rc = launch_mx4_quantize_rows(x, x_dtype, ld, from, rows, k, w.codes, w.scales, st)) return rc;
  return (kernel == kMx4Few ? launch_mx4_linear_few : launch_mx4_linear)(rows, w.codes, w.scales, w_codes, w_scales, 1, k,
                                                                           n, out, out_dtype == AXM_DTYPE_BF16, st);
}

extern "C" int axm_mx4_expert_ffn_workspace_bytes(const AxmMoeDesc* desc, int32_t rows, int32_t num_segments,
                                                  size_t* bytes) {
  const char* what = "axm_mx4_expert_ffn";
  if (int rc = check_ffn_desc(desc, what)) return rc;
  if (rows < 0) return fail(AXM_ERR_ARGUMENT, "%s: %d rows", what, rows);
  if (num_segments < 0 || num_segments > kMaxSegments)
    return fail(AXM_ERR_ARGUMENT, "%s: num_segments %d not in 0..%d", what, num_segments, kMaxSegments);
  if (bytes == nullptr) return fail(AXM_ERR_ARGUMENT, "bytes is null");
  *bytes = carve_expert_ffn(desc, rows, num_segments, nullptr).bytes;
  return AXM_OK;
}

extern "C" int axm_mx4_expert_ffn(const AxmMoeDesc* desc, const void* x, int32_t rows, const AxmSegment* segments,
                                  int32_t num_segments, const AxmMx4Experts* experts, void* o, int32_t o_dtype,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "axm_mx4_expert_ffn";
  size_t need = 0;
  if (int rc = axm_mx4_expert_ffn_workspace_bytes(desc, rows, num_segments, &need)) return rc;
  if (rows == 0 || num_segments == 0) return AXM_OK;  // matrices without rows may have no address
  if (!x || !segments || !o) return fail(AXM_ERR_ARGUMENT, "%s: null pointer", what);
  if (int rc = check_experts(experts, what)) return rc;
  if (o_dtype != AXM_DTYPE_BF16 && o_dtype != AXM_DTYPE_FP32) return fail(AXM_ERR_ARGUMENT, "%s: o_dtype %d unknown", what, o_dtype);
  if (off16(x) || off16(o)) return fail(AXM_ERR_ARGUMENT, "%s: x and o must be 16-byte aligned", what);
  if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  if (int rc = require_device()) return rc;
  const int D = desc->d_model, F = desc->d_ff;
  const FfnWs w = carve_expert_ffn(desc, rows, num_segments, workspace);
  int tile;
  const int kernel = mx4_choose(rows, num_segments, desc->tokens, &tile);
  const Mx4Rows r = {segments, num_segments, rows, num_segments, 0, 0, tile, kernel, w.status, w.few.partial, w.few.counters};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Mx4Gather from = {nullptr, 1, rows, 1};
  if (int rc = launch_mx4_quantize_rows(x, AXM_DTYPE_BF16, D, from, r, D, w.x_codes, w.x_scales, st)) return rc;
  return launch_ffn(r, w, experts, desc->num_experts, D, F, o, o_dtype == AXM_DTYPE_BF16, st);
}

extern "C" int axm_moe_mx4_workspace_bytes(const AxmMoeDesc* desc, size_t* bytes) {
  if (int rc = check_layer(desc)) return rc;
  if (bytes == nullptr) return fail(AXM_ERR_ARGUMENT, "bytes is null");
  *bytes = carve_layer(desc, nullptr).bytes;
  return AXM_OK;
}

extern "C" int axm_moe_forward_mx4(const AxmMoeDesc* desc, const AxmMoeTensors* t, const AxmMx4Experts* experts,
                                   const AxmMx4Experts* shared, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "axm_moe_forward_mx4";
  if (int rc = check_layer(desc)) return rc;
  if (t == nullptr) return fail(AXM_ERR_ARGUMENT, "tensors is null");
  if (desc->tokens == 0) return AXM_OK;
  if (!t->x || !t->router_w || !t->out) return fail(AXM_ERR_ARGUMENT, "%s: x, router_w and out are required", what);
  if (off16(t->x) || off16(t->router_w) || off16(t->out) || off16(t->y))
    return fail(AXM_ERR_ARGUMENT, "%s: x, router_w, out and y must be 16-byte aligned", what);
  if (int rc = check_experts(experts, what)) return rc;
  if (desc->num_shared > 0)
    if (int rc = check_experts(shared, what)) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, carve_layer(desc, nullptr).bytes)) return rc;
  if (int rc = require_device()) return rc;
  const LayerWs w = carve_layer(desc, workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int T = desc->tokens, k = desc->top_k, S = desc->num_shared, E = desc->num_experts, D = desc->d_model,
            F = desc->d_ff;
  float* logits = t->logits ? t->logits : w.logits;
  int32_t* idx = t->topk_idx ? t->topk_idx : w.topk_idx;
  float* gate = t->topk_gate ? t->topk_gate : w.topk_gate;
  int32_t* offsets = t->offsets ? t->offsets : w.offsets;
  int32_t* row_src = t->row_src ? t->row_src : w.row_src;
  int32_t* slot_dst = t->slot_dst ? t->slot_dst : w.slot_dst;
  bool cleared = false;  // the tensor-core router's preparation kernel clears the status word
  int rc;
  if ((rc = launch_router_auto(desc, t->x, t->router_w, t->router_bias, logits, idx, gate, w.block_counts,
                               w.router_scratch, w.router_scratch_bytes, w.ffn.status, stream, &cleared)))
    return rc;
  // placement only: the rows are quantised as they are gathered
  if ((rc = launch_permute(desc, t->x, idx, w.block_counts, t->histogram, offsets, row_src, slot_dst, nullptr,
                           w.segments, cleared ? nullptr : w.ffn.status, st, 1)))
    return rc;
  const int rows = T * (k + S);
  // one kind of kernel and of scale tile for the whole table: the routed experts'
  int tile;
  const int kernel = mx4_choose(rows, E + S, T, &tile);
  Mx4Rows r = {w.segments, E + S, rows, E + S, 0, 0, tile, kernel, nullptr, w.ffn.few.partial, w.ffn.few.counters};
  const Mx4Gather from = {row_src, k, T * k, T};
  if ((rc = launch_mx4_quantize_rows(t->x, AXM_DTYPE_BF16, D, from, r, D, w.ffn.x_codes, w.ffn.x_scales, st))) return rc;
  r.status = w.ffn.status;
  r.num_segments = E;
  if ((rc = launch_ffn(r, w.ffn, experts, E, D, F, w.o, false, st))) return rc;
  if (S > 0) {  // the shared experts: the rest of the table, with weights of their own
    r.segments = w.segments + E;
    r.num_segments = S;
    r.seg_base = E;
    r.expert_base = E;
    if ((rc = launch_ffn(r, w.ffn, shared, S, D, F, w.o, false, st))) return rc;
  }
  const float* o_shared = S > 0 ? static_cast<const float*>(w.o) + (size_t)T * k * D : nullptr;
  return axm_moe_combine(desc, t->x, w.o, o_shared, slot_dst, gate, t->y, t->out, stream);
}
