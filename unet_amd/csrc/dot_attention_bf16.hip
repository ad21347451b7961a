// Dot-product attention, bf16 storage: the entry points, and the workspaces of both storage types.
#include "dot_attention.h"

extern "C" {

int unet_dot_attention_workspace_bytes(int num_seqs, int64_t total_q, int64_t total_k, int heads_q, int heads_kv,
                                       int head_dim, size_t *bytes_host) {
  UNET_REQUIRE(bytes_host, "dot_attention_workspace_bytes: NULL result");
  TRY(check_shape("dot_attention_workspace_bytes", num_seqs, total_q, total_k, heads_q, heads_kv, head_dim));
  *bytes_host = forward_bytes(most_query_rows(total_q, total_k, heads_q, MOST_SHARES), head_dim);
  return UNET_OK;
}
int unet_dot_attention_backward_workspace_bytes(int num_seqs, int64_t total_q, int64_t total_k, int heads_q,
                                                int heads_kv, int head_dim, size_t *bytes_host) {
  UNET_REQUIRE(bytes_host, "dot_attention_backward_workspace_bytes: NULL result");
  TRY(check_shape("dot_attention_backward_workspace_bytes", num_seqs, total_q, total_k, heads_q, heads_kv, head_dim));
  *bytes_host = rows_bytes(total_q, heads_q) + backward_bytes(most_query_rows(total_q, total_k, heads_q, MOST_DQ_SHARES),
                                                             most_key_rows(total_q, total_k, heads_q, heads_kv), head_dim);
  return UNET_OK;
}

int unet_dot_attention_bf16(const uint16_t *q, int64_t q_ld, const uint16_t *k, int64_t k_ld, const uint16_t *v,
                            int64_t v_ld, uint16_t *out, int64_t out_ld, float *lse, const int32_t *cu_q,
                            const int32_t *cu_k, int num_seqs, int64_t total_q, int64_t total_k, int heads_q,
                            int heads_kv, int head_dim, float scale, int causal, void *workspace,
                            size_t workspace_bytes, unet_stream_t stream) {
  return forward<bf16_t>(q, q_ld, k, k_ld, v, v_ld, out, out_ld, lse, cu_q, cu_k, num_seqs, total_q, total_k, heads_q,
                         heads_kv, head_dim, scale, causal, workspace, workspace_bytes, as_stream(stream));
}
int unet_dot_attention_backward_bf16(const uint16_t *grad_out, int64_t grad_out_ld, const uint16_t *q, int64_t q_ld,
                                     const uint16_t *k, int64_t k_ld, const uint16_t *v, int64_t v_ld,
                                     const uint16_t *out, int64_t out_ld, const float *lse, uint16_t *grad_q,
                                     int64_t grad_q_ld, uint16_t *grad_k, int64_t grad_k_ld, uint16_t *grad_v,
                                     int64_t grad_v_ld, const int32_t *cu_q, const int32_t *cu_k, int num_seqs,
                                     int64_t total_q, int64_t total_k, int heads_q, int heads_kv, int head_dim,
                                     float scale, int causal, void *workspace, size_t workspace_bytes,
                                     unet_stream_t stream) {
  return backward<bf16_t>(grad_out, grad_out_ld, q, q_ld, k, k_ld, v, v_ld, out, out_ld, lse, grad_q, grad_q_ld, grad_k,
                          grad_k_ld, grad_v, grad_v_ld, cu_q, cu_k, num_seqs, total_q, total_k, heads_q, heads_kv, head_dim,
                          scale, causal, workspace, workspace_bytes, as_stream(stream));
}

}  // extern "C"
