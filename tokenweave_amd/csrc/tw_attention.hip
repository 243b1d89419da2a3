// Attention over the 4-bit paged cache (tw_kv4.h) for gfx950 (wave64).
//
//   o = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m),  s_t = scale * log2(e) * q k_t,  m = max_t s_t
//
// in one pass over the tokens: when a larger s appears, what has been summed is multiplied by
// 2^(m - m').  Scores, m, sums and the output are fp32; the output is rounded once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tw_common.h"
#include "tw_kv4.h"

namespace tw {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

struct AttentionArgs {
  void* out;
  const void* q;
  int64_t out_token, out_head, q_token, q_head;
  Kv4Pages pages;
  int group;  // query heads of a key head
  const int32_t* block_table;
  int64_t table_stride, table_width;
  const int32_t* seq_lens;
  const int32_t* query_starts;  // or null: per_seq each
  int64_t per_seq;
  int64_t num_seqs, num_tokens, max_queries;
  float scale;  // with log2(e)
  int64_t window;
};

// Sequence `s`: its new tokens [first, first + count) and its cached ones.
struct Sequence {
  int64_t first, count, length;
};

__device__ __forceinline__ Sequence sequence(const AttentionArgs& a, int64_t s) {
  Sequence q;
  int64_t end;
  if (a.query_starts) {
    q.first = a.query_starts[s];
    end = a.query_starts[s + 1];
  } else {
    q.first = s * a.per_seq;
    end = q.first + a.per_seq;
  }
  // whatever the arrays hold, only tokens of q and tokens that the table has places for are touched
  q.first = min(max(q.first, (int64_t)0), a.num_tokens);
  q.count = max(min(end, a.num_tokens) - q.first, (int64_t)0);
  q.length = min(max((int64_t)a.seq_lens[s], (int64_t)0), a.table_width << a.pages.page_log2);
  return q;
}

__device__ __forceinline__ const uint8_t* page_of(const AttentionArgs& a, int64_t s, int64_t token, int head) {
  const int64_t page = a.block_table[s * a.table_stride + (token >> a.pages.page_log2)];
  return page < 0 || page >= a.pages.num_pages ? nullptr
                                               : a.pages.data + (page * a.pages.heads + head) * a.pages.head_bytes;
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) x = fmaxf(x, __shfl_xor(x, i));
  return x;
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) x += __shfl_xor(x, i);
  return x;
}

// One wave for one query head of one new token: a lane scores a token, then holds D / 64 channels.
template <typename T, int D>
__global__ __launch_bounds__(64) void attention_row_kernel(AttentionArgs a) {
  using L = Kv4<D>;
  __shared__ float q_row[D];
  const int P = 1 << a.pages.page_log2, lane = threadIdx.x;
  const int64_t s = blockIdx.z;
  const int head = blockIdx.y, kv_head = head / a.group;
  const Sequence seq = sequence(a, s);
  for (int64_t i = blockIdx.x; i < seq.count && i < a.max_queries; i += gridDim.x) {
    const T* q = static_cast<const T*>(a.q) + (seq.first + i) * a.q_token + head * a.q_head;
    __syncthreads();
    for (int c = lane; c < D; c += 64) q_row[c] = (float)q[c];
    __syncthreads();
    const int64_t end = seq.length - seq.count + i + 1;  // tokens before it are seen
    const int64_t begin = a.window > 0 ? max(end - a.window, (int64_t)0) : 0;
    float m = -__builtin_inff(), l = 0.0f, o[D / 64] = {};
    for (int64_t base = begin & ~(int64_t)63; base < end; base += 64) {
      const int64_t t = base + lane;
      const int at = (int)t & (P - 1);
      const uint8_t* page = t >= begin && t < end ? page_of(a, s, t, kv_head) : nullptr;
      float score = -__builtin_inff();
      if (page) {
        score = 0.0f;
        for (int g = 0; g < L::kGroups; ++g) {
          float sum = 0.0f;
          for (int w = 0; w < 4; ++w) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(page + L::key(at) + g * 16 + w * 4);
            for (int c = 0; c < 8; ++c) sum += q_row[g * 32 + w * 8 + c] * e2m1_value(word >> (4 * c));
          }
          score += sum * scale_of(page[L::key_scale(P, at, g)]);
        }
        score *= a.scale;
      }
      const float most = fmaxf(m, wave_max(score));
      const float base_score = most == -__builtin_inff() ? 0.0f : most;
      const float p = __builtin_amdgcn_exp2f(score - base_score), old = __builtin_amdgcn_exp2f(m - base_score);
      l = l * old + wave_sum(p);
      m = most;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) o[c] *= old;
      for (int j = 0; j < 64; ++j) {
        const float pj = __shfl(p, j);
        const uint8_t* pg = reinterpret_cast<const uint8_t*>(__shfl((unsigned long long)page, j));
        if (!pg) continue;
        const int tj = (int)(base + j) & (P - 1);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const int ch = c * 64 + lane, sixteenth = ch / (D / 16), in = ch % (D / 16);
          const uint32_t byte = pg[L::value(P, tj, sixteenth) + in / 2];
          o[c] += pj * e2m1_value(byte >> (4 * (in & 1))) * scale_of(pg[L::value_scale(P, tj, ch / 32)]);
        }
      }
    }
    T* out = static_cast<T*>(a.out) + (seq.first + i) * a.out_token + head * a.out_head;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) out[c * 64 + lane] = (T)(l > 0.0f || l != l ? o[c] / l : 0.0f);
  }
}

template <typename T>
int launch_rows(const AttentionArgs& a, int D, int q_heads, void* stream) {
  const dim3 grid((unsigned)min(a.max_queries, (int64_t)65535), (unsigned)q_heads, (unsigned)a.num_seqs);
  auto kernel = D == 64 ? attention_row_kernel<T, 64> : D == 128 ? attention_row_kernel<T, 128> : attention_row_kernel<T, 256>;
  launch_kernel(kernel, grid, dim3(64), 0, static_cast<hipStream_t>(stream), a);
  return finish_launch("kv4_attention");
}

}  // namespace

int64_t kv4_attention_workspace(int q_heads, int kv_heads, int head_size, int64_t num_seqs, int64_t max_queries,
                                int64_t table_width, int page_size) {
  (void)q_heads, (void)kv_heads, (void)head_size, (void)num_seqs, (void)max_queries, (void)table_width, (void)page_size;
  return 0;
}

int run_kv4_attention(const tw_heads* out, const tw_heads* q, const void* pages, int64_t num_pages, int page_size,
                      int kv_heads, const int32_t* block_table, int64_t table_stride, int64_t table_width,
                      const int32_t* seq_lens, const int32_t* query_starts, int64_t num_seqs, int64_t T,
                      int64_t max_queries, int head_size, float scale, int64_t window, int dtype, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  const char* what = "kv4_attention";
  if (dtype != TW_DTYPE_BF16 && dtype != TW_DTYPE_F16) return set_error(TW_ERR_DTYPE, "%s: unsupported dtype %d", what, dtype);
  if (T < 0 || num_seqs < 0 || max_queries < 0 || window < 0 || table_width < 0 || table_stride < 0)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: a size is negative", what);
  if (T == 0 || num_seqs == 0 || max_queries == 0) return TW_OK;
  AttentionArgs a{};
  if (int rc = check_kv4_pages(what, pages, num_pages, page_size, kv_heads, head_size, &a.pages)) return rc;
  if (!out || !q || !out->data || !q->data) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: out or q is null", what);
  if (q->heads < 1 || q->heads % kv_heads != 0 || q->heads > 65535)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: %lld query heads over %d key heads", what, (long long)q->heads, kv_heads);
  if (out->heads != q->heads) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: out and q have different heads", what);
  if (out->token_stride < 0 || out->head_stride < 0 || q->token_stride < 0 || q->head_stride < 0)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: a stride is negative", what);
  if (!seq_lens || (!block_table && table_width > 0))
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: block_table or seq_lens is null", what);
  if (table_width > ((int64_t)1 << 31) / page_size)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: block_table has room for more than 2^31 tokens", what);
  if (num_seqs > 65535) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: more than 65535 sequences", what);
  if (!query_starts && T % num_seqs != 0)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: %lld tokens are not the same number for each of %lld sequences", what,
                     (long long)T, (long long)num_seqs);
  const int64_t need = kv4_attention_workspace((int)q->heads, kv_heads, head_size, num_seqs, max_queries, table_width, page_size);
  if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: workspace of %lld bytes, need %lld, 16-byte aligned", what,
                     (long long)workspace_bytes, (long long)need);
  a.out = out->data;
  a.q = q->data;
  a.out_token = out->token_stride;
  a.out_head = out->head_stride;
  a.q_token = q->token_stride;
  a.q_head = q->head_stride;
  a.group = (int)(q->heads / kv_heads);
  a.block_table = block_table;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.seq_lens = seq_lens;
  a.query_starts = query_starts;
  a.per_seq = query_starts ? 0 : T / num_seqs;
  a.num_seqs = num_seqs;
  a.num_tokens = T;
  a.max_queries = min(max_queries, T);
  a.scale = scale * kLog2e;
  a.window = window;
  return dtype == TW_DTYPE_BF16 ? launch_rows<__bf16>(a, head_size, (int)q->heads, stream)
                                : launch_rows<_Float16>(a, head_size, (int)q->heads, stream);
}

}  // namespace tw
