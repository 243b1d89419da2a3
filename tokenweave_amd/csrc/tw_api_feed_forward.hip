// extern "C" surface of libtokenweave_amd.so, continued: the gated product and its gradients, rows
// to 8-bit codes, the block-scaled product (kernels in tw_gemm.hip, tw_gated.hip and tw_fp8.hip).
#include "tw_common.h"

extern "C" {

int64_t tw_gated_gemm_bf16_nt_workspace(int64_t M, int64_t I, int64_t K) { return tw::gated_gemm_workspace(M, I, K); }

int tw_gated_gemm_bf16_nt(void* out, void* gate_up, const void* a, const void* b, int64_t M, int64_t I, int64_t K,
                          int64_t ldc, int64_t ld_gate_up, int activation, int max_cus, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  return tw::run_gated_gemm_bf16_nt(out, gate_up, a, b, M, I, K, ldc, ld_gate_up, activation, max_cus, workspace,
                                    workspace_bytes, stream);
}

int64_t tw_gated_gemm_bf16_nt_backward_workspace(int64_t M, int64_t I, int64_t K, int want_a, int want_b) {
  return tw::gated_backward_workspace(M, I, K, want_a != 0, want_b != 0);
}

int tw_gated_gemm_bf16_nt_backward(void* grad_a, void* grad_b, const void* grad_out, int64_t ld_grad_out, const void* a,
                                   const void* b, const void* gate_up, int64_t ld_gate_up, int64_t M, int64_t I,
                                   int64_t K, int activation, int max_cus, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
  return tw::run_gated_gemm_bf16_nt_backward(grad_a, grad_b, grad_out, ld_grad_out, a, b, gate_up, ld_gate_up, M, I, K,
                                             activation, max_cus, workspace, workspace_bytes, stream);
}

int tw_quant_fp8_groups(void* out, float* scales, int64_t scale_row_stride, int64_t scale_group_stride,
                        const void* input, int64_t ld_input, int64_t num_rows, int64_t K, int activation, int dtype,
                        void* stream) {
  return tw::run_quant_fp8_groups(out, scales, scale_row_stride, scale_group_stride, input, ld_input, num_rows, K,
                                  activation, dtype, stream);
}

int64_t tw_gemm_fp8_block_nt_workspace(int64_t M, int64_t N, int64_t K) { return tw::gemm_fp8_block_workspace(M, N, K); }

int tw_gemm_fp8_block_nt(void* out, const void* a, const float* a_scales, int64_t scale_row_stride,
                         int64_t scale_block_stride, const void* b, const float* b_scales, int64_t M, int64_t N,
                         int64_t K, int64_t ldc, int dtype, int max_cus, void* workspace, int64_t workspace_bytes,
                         void* stream) {
  return tw::run_gemm_fp8_block_nt(out, a, a_scales, scale_row_stride, scale_block_stride, b, b_scales, M, N, K, ldc,
                                   dtype, max_cus, workspace, workspace_bytes, stream);
}

}  // extern "C"
