// extern "C" surface of libtokenweave_amd.so, continued: rotation, the paged 4-bit cache and
// attention over it (kernels in tw_rotary.hip and tw_attention.hip).
#include "tw_common.h"

extern "C" {

int tw_rotary_positions(const tw_heads* q_out, const tw_heads* q, const tw_heads* k_out, const tw_heads* k,
                        const int64_t* positions, const float* cos_sin, int64_t max_positions,
                        int64_t num_tokens, int head_size, int rotary_dim, int flags, int dtype,
                        void* stream) {
  return tw::run_rotary_positions(q_out, q, k_out, k, positions, cos_sin, max_positions, num_tokens, head_size,
                                  rotary_dim, flags, dtype, stream);
}

int tw_kv4_append(void* pages, int64_t num_pages, int page_size, const tw_heads* k, const tw_heads* v,
                  const int64_t* slots, const tw_heads* q_out, const tw_heads* q,
                  const int64_t* positions, const float* cos_sin, int64_t max_positions,
                  int64_t num_tokens, int head_size, int rotary_dim, int flags, int dtype, void* stream) {
  return tw::run_kv4_append(pages, num_pages, page_size, k, v, slots, q_out, q, positions, cos_sin, max_positions,
                            num_tokens, head_size, rotary_dim, flags, dtype, stream);
}

int tw_kv4_read(const tw_heads* k_out, const tw_heads* v_out, const void* pages, int64_t num_pages, int page_size,
                const int64_t* slots, int64_t num_tokens, int head_size, int dtype, void* stream) {
  return tw::run_kv4_read(k_out, v_out, pages, num_pages, page_size, slots, num_tokens, head_size, dtype, stream);
}

int64_t tw_kv4_attention_workspace(int q_heads, int kv_heads, int head_size, int64_t num_seqs, int64_t num_tokens,
                                   int64_t max_queries, int64_t table_width, int page_size) {
  return tw::kv4_attention_workspace(q_heads, kv_heads, head_size, num_seqs, num_tokens, max_queries, table_width,
                                     page_size);
}

int tw_kv4_attention(const tw_heads* out, const tw_heads* q, const void* pages, int64_t num_pages, int page_size,
                     int kv_heads, const int32_t* block_table, int64_t table_stride, int64_t table_width,
                     const int32_t* seq_lens, const int32_t* query_starts, int64_t num_seqs,
                     int64_t num_tokens, int64_t max_queries, int head_size, float scale, int64_t window,
                     int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  return tw::run_kv4_attention(out, q, pages, num_pages, page_size, kv_heads, block_table, table_stride, table_width,
                               seq_lens, query_starts, num_seqs, num_tokens, max_queries, head_size, scale, window,
                               dtype, workspace, workspace_bytes, stream);
}

}  // extern "C"
