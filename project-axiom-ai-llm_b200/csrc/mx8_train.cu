// Host side of the expert feed-forward's training step with 8-bit activation checkpoints.  The
// kernels are the pair kernels of grouped_ffn_2sm.cu and grouped_bwd_2sm.cu.
#include <initializer_list>

#include "microscale.cuh"
#include "gemm_common.cuh"

namespace axm {

namespace {

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

int check_call(const AxmMoeDesc* d, int32_t rows, const AxmSegment* segments, int32_t num_segments,
               const AxmMx8Checkpoint* keep, const char* what) {
  if (d == nullptr) return fail(AXM_ERR_ARGUMENT, "desc is null");
  if (d->d_model <= 0 || d->d_ff <= 0 || d->d_model % 8 || d->d_ff % 32)
    return fail(AXM_ERR_ARGUMENT, "%s: d_model %d must be a positive multiple of 8, d_ff %d of 32", what, d->d_model, d->d_ff);
  if (d->num_experts <= 0 || d->num_experts > 65535)
    return fail(AXM_ERR_ARGUMENT, "%s: num_experts %d not in 1..65535", what, d->num_experts);
  if (rows < 0) return fail(AXM_ERR_ARGUMENT, "%s: %d rows", what, rows);
  if (num_segments < 0 || num_segments > kMaxSegments)
    return fail(AXM_ERR_ARGUMENT, "%s: num_segments %d not in 0..%d", what, num_segments, kMaxSegments);
  if (rows == 0 || num_segments == 0) return AXM_OK;  // matrices without rows and empty tables may have no address
  if (!segments || !keep || !keep->gate_codes || !keep->gate_scales || !keep->up_codes || !keep->up_scales)
    return fail(AXM_ERR_ARGUMENT, "%s: null pointer", what);
  if (off16(keep->gate_codes) || off16(keep->up_codes))
    return fail(AXM_ERR_ARGUMENT, "%s: codes must be 16-byte aligned", what);
  return AXM_OK;
}

int check_pointers(std::initializer_list<const void*> all, const char* what) {
  for (const void* p : all) {
    if (p == nullptr) return fail(AXM_ERR_ARGUMENT, "%s: null pointer", what);
    if (off16(p)) return fail(AXM_ERR_ARGUMENT, "%s: matrices must be 16-byte aligned", what);
  }
  return AXM_OK;
}

int check_type(int32_t dtype, const char* what) {
  return dtype == AXM_DTYPE_BF16 || dtype == AXM_DTYPE_FP32 ? AXM_OK
                                                            : fail(AXM_ERR_ARGUMENT, "%s: dtype %d unknown", what, dtype);
}

}  // namespace

}  // namespace axm

using namespace axm;

extern "C" int axm_mx8_checkpoint_bytes(int32_t rows, int32_t d_ff, size_t* code_bytes, size_t* scale_bytes) {
  if (rows < 0 || d_ff <= 0 || d_ff % kMxBlock)
    return fail(AXM_ERR_ARGUMENT, "axm_mx8_checkpoint_bytes: rows %d, d_ff %d (a positive multiple of 32)", rows, d_ff);
  if (!code_bytes || !scale_bytes) return fail(AXM_ERR_ARGUMENT, "axm_mx8_checkpoint_bytes: null pointer");
  *code_bytes = (size_t)rows * d_ff;
  *scale_bytes = (size_t)rows * (d_ff / kMxBlock);
  return AXM_OK;
}

extern "C" int axm_mx8_expert_ffn_train(const AxmMoeDesc* desc, const void* x, int32_t rows, const AxmSegment* segments,
                                        int32_t num_segments, const void* w_gate, const void* w_up, const void* w_down,
                                        const AxmMx8Checkpoint* keep, void* h, void* o, int32_t o_dtype, int32_t* status,
                                        void* stream) {
  const char* what = "axm_mx8_expert_ffn_train";
  if (int rc = check_call(desc, rows, segments, num_segments, keep, what)) return rc;
  if (int rc = check_type(o_dtype, what)) return rc;
  if (rows == 0) return AXM_OK;
  if (int rc = check_pointers({x, w_gate, w_up, w_down, h, o}, what)) return rc;
  if (num_segments == 0) return AXM_OK;
  if (int rc = require_device()) return rc;
  return launch_train8_forward(desc, segments, num_segments, rows, x, w_gate, w_up, w_down, keep, h, o,
                               o_dtype == AXM_DTYPE_BF16, status, static_cast<cudaStream_t>(stream));
}

extern "C" int axm_mx8_expert_ffn_backward(const AxmMoeDesc* desc, const void* x, int32_t rows, const AxmSegment* segments,
                                           int32_t num_segments, const AxmMx8Checkpoint* keep, const void* d_o,
                                           const void* w_gate, const void* w_up, const void* w_down, void* h, void* d_g,
                                           void* d_u, void* d_x, void* d_w_gate, void* d_w_up, void* d_w_down,
                                           int32_t grad_dtype, int32_t* status, void* stream) {
  const char* what = "axm_mx8_expert_ffn_backward";
  if (int rc = check_call(desc, rows, segments, num_segments, keep, what)) return rc;
  if (rows > 0)
    if (int rc = check_pointers({x, d_o, w_gate, w_up, w_down, h, d_g, d_u, d_x}, what)) return rc;
  const bool wgrad = d_w_gate || d_w_up || d_w_down;
  if (wgrad && !(d_w_gate && d_w_up && d_w_down))
    return fail(AXM_ERR_ARGUMENT, "%s: weight gradients: give all three or none", what);
  if (wgrad)
    if (int rc = check_pointers({d_w_gate, d_w_up, d_w_down}, what)) return rc;
  if (int rc = check_type(grad_dtype, what)) return rc;
  if (num_segments == 0) return AXM_OK;
  if (int rc = require_device()) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int D = desc->d_model, F = desc->d_ff, E = desc->num_experts;
  const bool bf16 = grad_dtype == AXM_DTYPE_BF16;
  if (rows == 0) {  // no expert has a row: its gradient is zero
    const size_t bytes = (size_t)E * D * F * (bf16 ? 2 : 4);
    for (void* p : {d_w_gate, d_w_up, d_w_down})
      if (p != nullptr) AXM_CUDA(cudaMemsetAsync(p, 0, bytes, st));
    return AXM_OK;
  }
  int rc;
  if ((rc = launch_train8_dh(desc, segments, num_segments, rows, d_o, w_down, keep, d_g, d_u, h, status, st))) return rc;
  if ((rc = launch_bwd_dx_2sm(desc, segments, num_segments, rows, d_g, d_u, w_gate, w_up, d_x, status, st, bf16, true))) return rc;
  if (!wgrad) return AXM_OK;
  const WgradProblem all[3] = {{h, F, d_o, D, d_w_down}, {x, D, d_g, F, d_w_gate}, {x, D, d_u, F, d_w_up}};
  return launch_wgrad_2sm(segments, num_segments, rows, E, all, 3, status, st, bf16, true);
}
