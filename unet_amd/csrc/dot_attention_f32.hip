// Dot-product attention, fp32 storage: the entry points.
#include "dot_attention.h"

extern "C" {

int unet_dot_attention_f32(const float *q, int64_t q_ld, const float *k, int64_t k_ld, const float *v, int64_t v_ld,
                           float *out, int64_t out_ld, float *lse, const int32_t *cu_q, const int32_t *cu_k,
                           int num_seqs, int64_t total_q, int64_t total_k, int heads_q, int heads_kv, int head_dim,
                           float scale, int causal, void *workspace, size_t workspace_bytes, unet_stream_t stream) {
  return forward<float>(q, q_ld, k, k_ld, v, v_ld, out, out_ld, lse, cu_q, cu_k, num_seqs, total_q, total_k, heads_q,
                        heads_kv, head_dim, scale, causal, workspace, workspace_bytes, as_stream(stream));
}
int unet_dot_attention_backward_f32(const float *grad_out, int64_t grad_out_ld, const float *q, int64_t q_ld,
                                    const float *k, int64_t k_ld, const float *v, int64_t v_ld, const float *out,
                                    int64_t out_ld, const float *lse, float *grad_q, int64_t grad_q_ld, float *grad_k,
                                    int64_t grad_k_ld, float *grad_v, int64_t grad_v_ld, const int32_t *cu_q,
                                    const int32_t *cu_k, int num_seqs, int64_t total_q, int64_t total_k, int heads_q,
                                    int heads_kv, int head_dim, float scale, int causal, void *workspace,
                                    size_t workspace_bytes, unet_stream_t stream) {
  return backward<float>(grad_out, grad_out_ld, q, q_ld, k, k_ld, v, v_ld, out, out_ld, lse, grad_q, grad_q_ld, grad_k,
                         grad_k_ld, grad_v, grad_v_ld, cu_q, cu_k, num_seqs, total_q, total_k, heads_q, heads_kv, head_dim,
                         scale, causal, workspace, workspace_bytes, as_stream(stream));
}

}  // extern "C"
