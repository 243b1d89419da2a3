// Attention over the 4-bit paged cache (tw_kv4.h) for gfx950 (wave64).
//
//   o = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m),  s_t = scale * log2(e) * q k_t,  m = max_t s_t
//
// in one pass over the tokens: when a larger s appears, what has been summed is multiplied by
// 2^(m - m').  Scores, m, sums and the output are fp32; the output is rounded once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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

// ---------------------------------------------------------------------------
// Few rows: new tokens x query heads of a key head are at most 32.
//
// The keys' codes become fp16 (exact: two significant bits and an exponent within fp16's) and are the
// left operand of 16 x 16 x 32 products with the rows' queries, so that a lane gets the scores of ONE
// row and of tokens 4h .. 4h+3 of 16, h = lane / 16.  The same registers, rounded to fp16, are the right
// operand of the products with the values: which 8 tokens a lane's 8 inner places stand for is free as
// long as both operands agree, so no probability moves between lanes.  The values' codes have to come
// as 8 tokens of one channel; a lane loads 4 tokens x D/16 channels at once (the layout of tw_kv4.h)
// and pairs tokens in registers.
//
// Work is shared by even numbers of 128-token steps over a fixed grid, whatever the sequences'
// lengths: a workgroup finds its steps from the lengths on the device.  What a workgroup holds of a
// sequence that others share goes to the workspace as (m, l, O), and attention_join_kernel joins.
// ---------------------------------------------------------------------------
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4, kWaveTokens = 32, kStep = kWaves * kWaveTokens, kJoinThreads = 256;

// Which unfinished sequence a workgroup began, for the join.
struct SplitHeader {
  int32_t seq, head, last;  // seq < 0: none; last: the workgroup that holds its end
  int32_t unused;
};

struct SplitArgs {
  AttentionArgs a;
  SplitHeader* headers;  // one a workgroup
  float* parts;          // two a workgroup: [rows][D + 2], m and l behind the D channels
  int rows;              // of a part
};

// First token that any new token of the sequence sees, and the 128-token steps from there to its end; a
// sequence with new tokens has one step at least, in which its outputs are written.
__device__ __forceinline__ void steps_of(const AttentionArgs& a, const Sequence& q, int* first, int* count) {
  const int64_t seen = a.window > 0 ? max(q.length - q.count + 1 - a.window, (int64_t)0) : 0;
  *first = (int)(seen / kStep);
  *count = q.count == 0 ? 0 : max((int)((q.length + kStep - 1) / kStep) - *first, 1);
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Sum over the workgroup's threads before this one, and over all.
__device__ __forceinline__ int block_scan(int x, int* total, int* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int sum = x;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    const int y = __shfl_up(sum, i);
    if (lane >= i) sum += y;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int y = lds[w];
    before += w < wave ? y : 0;
    all += y;
  }
  *total = all;
  return before + sum - x;
}

// One wave's 32 tokens of the cache.
template <int D>
struct Tile {
  static constexpr int kWords = D / 32;  // of a lane's share of 16 tokens' keys, and of its four tokens' values
  uint32_t k[2][kWords], v[2][kWords];
  uint32_t ks[2][(D + 127) / 128], vs[2];
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
  if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x;
    w[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4_t x = *reinterpret_cast<const uint4_t*>(p + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[i + j] = x[j];
    }
  }
}

// Offsets of a lane's share within 16 tokens of a page.
template <int D>
struct LaneOffsets {
  int k, v, ks, vs;
  __device__ __forceinline__ explicit LaneOffsets(int P, int lane) {
    using L = Kv4<D>;
    const int n = lane & 15, h = lane >> 4;
    k = n * L::kRow + h * (D / 8);
    v = P * L::kRow + h * (4 * L::kRow) + n * (4 * L::kChunk);
    ks = L::key_scale(P, n, h * D / 128);
    vs = L::value_scale(P, 4 * h, n * (D / 16) / 32);
  }
};

template <int D>
__device__ __forceinline__ void load_tile(Tile<D>& tile, const uint8_t* const (&page)[2], const int (&at)[2],
                                          const LaneOffsets<D>& lane, int P) {
  using L = Kv4<D>;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* p = page[i];
    load_words(tile.k[i], p + (at[i] * L::kRow + lane.k));
    load_words(tile.v[i], p + (at[i] * L::kRow + lane.v));
#pragma unroll
    for (int g = 0; g < (D + 127) / 128; ++g) tile.ks[i][g] = p[at[i] + lane.ks + g * P];
    tile.vs[i] = *reinterpret_cast<const uint32_t*>(p + (at[i] + lane.vs));
  }
}

template <int SEL>
__device__ __forceinline__ half2_t two_values(uint32_t word, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, SEL);
}

__device__ __forceinline__ half8_t eight_values(uint32_t word, float scale) {
  const half2_t a = two_values<0>(word, scale), b = two_values<1>(word, scale), c = two_values<2>(word, scale),
                d = two_values<3>(word, scale);
  return half8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The rows' queries as the right operand: lane (n, h) holds row n's channels h * D/4 .. in steps of 8.
// A row is multiplied by the power of two that brings its largest magnitude to [2^14, 2^15), where
// every bf16 and fp16 value down to 2^-28 of it is exact; the score is multiplied back.
template <typename T, int D>
__device__ __forceinline__ float load_queries(half8_t (&q)[D / 32], const T* row) {
  float x[D / 4], most = 0.0f;
#pragma unroll
  for (int i = 0; i < D / 4; ++i) {
    x[i] = row ? (float)row[i] : 0.0f;
    most = fmaxf(most, __builtin_fabsf(x[i]));
  }
  most = fmaxf(most, __shfl_xor(most, 16));
  most = fmaxf(most, __shfl_xor(most, 32));
  const int e = min(max((int)(__float_as_uint(most) >> 23) - 127, -100), 127);
  const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
#pragma unroll
  for (int i = 0; i < D / 4; ++i) q[i / 8][i % 8] = (_Float16)(x[i] * up);
  return __uint_as_float((uint32_t)(127 - 14 + e) << 23);
}

constexpr float kLift = 14.0f;  // probabilities are held times 2^14: fp16's normal range reaches down to 2^-28 of the largest

template <typename T, int D, int NT>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 1 : 2) void attention_split_kernel(SplitArgs args) {
  const AttentionArgs& a = args.a;
  constexpr int kTiles = D / 16;          // of channels
  constexpr int kRegs = kTiles * 4 + 2;   // what a lane holds of a row: O, m, l
  __shared__ int scan_lds[kWaves];
  __shared__ int found[4];
  __shared__ float merge[2][NT][kRegs][64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, h4 = lane >> 4;
  const int P = 1 << a.pages.page_log2, heads = a.pages.heads, w = blockIdx.x;

  // ---- this workgroup's steps
  int total = 0, first_steps = 0, before = 0;
  const int rounds = (int)((a.num_seqs + 64 * kWaves - 1) / (64 * kWaves));
  for (int r = 0; r < rounds; ++r) {
    const int s = r * 64 * kWaves + threadIdx.x;
    int first, count = 0, sum;
    if (s < a.num_seqs) steps_of(a, sequence(a, s), &first, &count);
    const int at = block_scan(count, &sum, scan_lds);
    if (r == 0) {
      first_steps = count;
      before = at;
    }
    total += sum;
  }
  total *= heads;
  const int share = max((total + (int)gridDim.x - 1) / (int)gridDim.x, 1);
  int pos = w * share;
  const int end = min(pos + share, total);
  if (threadIdx.x == 0) args.headers[w].seq = -1;
  if (pos >= end) return;
  // the sequence that the first step belongs to
  int base = 0;
  for (int r = 0; r < rounds; ++r) {
    const int s = r * 64 * kWaves + threadIdx.x;
    int first, count = first_steps, sum = 0, at = before;
    if (rounds > 1) {
      count = 0;
      if (s < a.num_seqs) steps_of(a, sequence(a, s), &first, &count);
      at = base + block_scan(count, &sum, scan_lds);
    }
    if (count > 0 && at * heads <= pos && pos < (at + count) * heads) {
      found[0] = s;
      found[1] = at * heads;
    }
    base += sum;
  }
  __syncthreads();
  int s = uniform(found[0]), seq_base = uniform(found[1]);

  const LaneOffsets<D> offsets(P, lane);
  while (pos < end) {
    // ---- the next piece: steps [step, step + steps) of key head `head` of sequence s
    const Sequence seq = sequence(a, s);
    int first_step, count;
    steps_of(a, seq, &first_step, &count);
    if (count == 0) {
      ++s;
      continue;
    }
    const int head = (pos - seq_base) / count, inside = (pos - seq_base) - head * count;
    const int steps = min(count - inside, end - pos);
    const int queries = (int)min(seq.count, a.max_queries), rows = queries * a.group;
    const int length = (int)seq.length;
    const int new_from = length - (int)seq.count;  // position of the first new token
    const bool starts = inside == 0, ends = inside + steps == count;

    half8_t q[NT][D / 32];
    float scale[NT], m[NT], l[NT];
    int row_end[NT], row_begin[NT];
    float4_t o[NT][kTiles];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = t * 16 + n, i = row / a.group;
      const T* from = row < rows ? static_cast<const T*>(a.q) + (seq.first + i) * a.q_token +
                                       (int64_t)(head * a.group + row - i * a.group) * a.q_head + h4 * (D / 4)
                                 : nullptr;
      scale[t] = load_queries<T, D>(q[t], from) * a.scale;
      row_end[t] = row < rows ? new_from + i + 1 : 0;
      row_begin[t] = a.window > 0 ? (int)max((int64_t)new_from + i + 1 - a.window, (int64_t)0) : 0;
      m[t] = -__builtin_inff();
      l[t] = 0.0f;
#pragma unroll
      for (int c = 0; c < kTiles; ++c) o[t][c] = float4_t{0, 0, 0, 0};
    }
    // tokens that every row sees need no mask
    const int all_from = a.window > 0 ? (int)max((int64_t)new_from + queries - a.window, (int64_t)0) : 0;
    const int all_to = new_from + 1;
    const int some_from = a.window > 0 ? (int)max((int64_t)new_from + 1 - a.window, (int64_t)0) : 0;
    const int32_t* table = a.block_table + (int64_t)s * a.table_stride;

    const int step0 = first_step + inside;
    auto locate = [&](int step, const uint8_t* (&page)[2], int (&at)[2], bool (&there)[2]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = step * kStep + wave * kWaveTokens + i * 16;
        const int id = t < length ? table[t >> a.pages.page_log2] : -1;
        there[i] = id >= 0 && id < a.pages.num_pages;
        page[i] = a.pages.data + ((int64_t)(there[i] ? id : 0) * heads + head) * a.pages.head_bytes;
        at[i] = t & (P - 1);
      }
    };

    Tile<D> tile;
    const uint8_t* page[2];
    int at[2];
    bool there[2], next_there[2];
    locate(step0, page, at, there);
    load_tile<D>(tile, page, at, offsets, P);
    for (int step = step0; step < step0 + steps; ++step) {
      Tile<D> next = tile;
      next_there[0] = next_there[1] = false;
      if (step + 1 < step0 + steps) {
        locate(step + 1, page, at, next_there);
        load_tile<D>(next, page, at, offsets, P);
      }
      const int t0 = step * kStep + wave * kWaveTokens;
      const bool whole = t0 >= all_from && t0 + kWaveTokens <= all_to && there[0] && there[1];

      // ---- scores: [token][row]
      float4_t sc[NT][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[t][i] = float4_t{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const half8_t k = eight_values(tile.k[i][c], __uint_as_float(tile.ks[i][c / 4] << 23));
#pragma unroll
          for (int t = 0; t < NT; ++t) sc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[t][c], sc[t][i], 0, 0, 0);
        }
      }
      // ---- probabilities
      half8_t p[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[8], most = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = sc[t][i / 4][i % 4] * scale[t];
          if (!whole) {
            const int token = t0 + (i / 4) * 16 + h4 * 4 + i % 4;
            if (token >= row_end[t] || token < row_begin[t] || !there[i / 4]) x[i] = -__builtin_inff();
          }
          most = fmaxf(most, x[i]);
        }
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        if (__builtin_amdgcn_ballot_w64(most > m[t])) {
          const float now = fmaxf(m[t], most);
          const float old = m[t] == now ? 1.0f : __builtin_amdgcn_exp2f(m[t] - now);
          m[t] = now;
          l[t] *= old;
#pragma unroll
          for (int c = 0; c < kTiles; ++c) o[t][c] *= old;
        }
        const float sub = (m[t] == -__builtin_inff() ? 0.0f : m[t]) - kLift;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = __builtin_amdgcn_exp2f(x[i] - sub);
          sum += x[i];
          p[t][i] = (_Float16)x[i];
        }
        l[t] += sum;
      }
      // ---- values: what no row sees may hold anything, and nothing times zero has to be zero
      float vs[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t b = tile.vs[i / 4] >> (8 * (i % 4)) & 255;
        if (!whole) {
          const int token = t0 + (i / 4) * 16 + h4 * 4 + i % 4;
          if (token >= length || token < some_from || !there[i / 4]) b = 127;
        }
        vs[i] = __uint_as_float(b << 23);
      }
      auto channels = [&](auto sel, int word) {  // two channels of the lane's: 2 * sel, 2 * sel + 1 of a word
        constexpr int S = decltype(sel)::value;
        half2_t x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          // four tokens side by side, D/32 bytes each
          const int byte = (i % 4) * (D / 32) + word * 4 + S;
          const uint32_t w32 = tile.v[i / 4][byte / 4];
          x[i] = byte % 4 == 0 ? two_values<0>(w32, vs[i]) : byte % 4 == 1 ? two_values<1>(w32, vs[i])
               : byte % 4 == 2 ? two_values<2>(w32, vs[i]) : two_values<3>(w32, vs[i]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          half8_t v;
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = x[i][j];
#pragma unroll
          for (int t = 0; t < NT; ++t)
            o[t][word * 8 + S * 2 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[t], o[t][word * 8 + S * 2 + j], 0, 0, 0);
        }
      };
#pragma unroll
      for (int word = 0; word < (D + 127) / 128; ++word) {
        channels(std::integral_constant<int, 0>{}, word);
        channels(std::integral_constant<int, 1>{}, word);
        if constexpr (D > 64) {
          channels(std::integral_constant<int, 2>{}, word);
          channels(std::integral_constant<int, 3>{}, word);
        }
      }
      tile = next;
      there[0] = next_there[0];
      there[1] = next_there[1];
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      l[t] += __shfl_xor(l[t], 16);
      l[t] += __shfl_xor(l[t], 32);
    }

    // ---- the waves' parts become one: 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
    for (int half = 2; half >= 1; half >>= 1) {
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float(*to)[64] = merge[wave - half][t];
#pragma unroll
          for (int c = 0; c < kTiles; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) to[c * 4 + i][lane] = o[t][c][i];
          to[kTiles * 4][lane] = m[t];
          to[kTiles * 4 + 1][lane] = l[t];
        }
      }
      __syncthreads();
      if (wave < half) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float(*from)[64] = merge[wave][t];
          const float m2 = from[kTiles * 4][lane], now = fmaxf(m[t], m2);
          const float w1 = m[t] == now ? 1.0f : __builtin_amdgcn_exp2f(m[t] - now);
          const float w2 = m2 == now ? 1.0f : __builtin_amdgcn_exp2f(m2 - now);
          m[t] = now;
          l[t] = l[t] * w1 + from[kTiles * 4 + 1][lane] * w2;
#pragma unroll
          for (int c = 0; c < kTiles; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][c][i] = o[t][c][i] * w1 + from[c * 4 + i][lane] * w2;
        }
      }
    }
    if (wave == 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int row = t * 16 + n, i = row / a.group;
        if (row >= rows) continue;
        // lane (n, h): channels (4h + i) * D/16 + c of row n
        if (starts && ends) {
          T* out = static_cast<T*>(a.out) + (seq.first + i) * a.out_token +
                   (int64_t)(head * a.group + row - i * a.group) * a.out_head + h4 * (D / 4);
          const float inv = l[t] > 0.0f || l[t] != l[t] ? 1.0f / l[t] : 0.0f;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < kTiles; ++c) out[r * kTiles + c] = (T)(o[t][c][r] * inv);
        } else {
          float* part = args.parts + ((int64_t)(2 * w + (starts ? 1 : 0)) * args.rows + row) * (D + 2);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < kTiles; ++c) part[h4 * (D / 4) + r * kTiles + c] = o[t][c][r];
          if (h4 == 0) {
            part[D] = m[t];
            part[D + 1] = l[t];
          }
        }
      }
      if (lane == 0 && starts && !ends) {
        args.headers[w].head = head;
        args.headers[w].last = (pos - inside + count - 1) / share;
        args.headers[w].seq = s;
      }
    }
    pos += steps;
    if (pos == seq_base + heads * count) {
      seq_base = pos;
      ++s;
    }
  }
}

// Joins the parts of one row of a sequence that several workgroups shared: block (w, row).
template <typename T, int D>
__global__ __launch_bounds__(kJoinThreads) void attention_join_kernel(SplitArgs args) {
  const AttentionArgs& a = args.a;
  const int w = blockIdx.x, row = blockIdx.y;
  const SplitHeader header = args.headers[w];
  if (header.seq < 0) return;
  const Sequence seq = sequence(a, header.seq);
  const int i = row / a.group;
  if (i >= seq.count || i >= a.max_queries) return;
  constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes;
  __shared__ float lds[kGroups][D + 1];
  __shared__ float most_of[kJoinThreads / 64];
  const int parts = header.last - w + 1;
  // part 0 is the workgroup's own second place, the others the first place of those behind it
  auto part = [&](int c) {
    return args.parts + ((int64_t)(c == 0 ? 2 * w + 1 : 2 * (w + c)) * args.rows + row) * (D + 2);
  };
  float m = -__builtin_inff();
  for (int c = threadIdx.x; c < parts; c += kJoinThreads) m = fmaxf(m, part(c)[D]);
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) most_of[threadIdx.x >> 6] = m;
  __syncthreads();
  for (int k = 0; k < kJoinThreads / 64; ++k) m = fmaxf(m, most_of[k]);
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  float o[4] = {}, l = 0.0f;
#pragma unroll 4
  for (int c = group; c < parts; c += kGroups) {
    const float* p = part(c);
    const float mc = p[D], weight = mc == m ? 1.0f : __builtin_amdgcn_exp2f(mc - m);
    l += p[D + 1] * weight;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] += p[lane * 4 + k] * weight;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) lds[group][lane * 4 + k] = o[k];
  if (lane == 0) lds[group][D] = l;
  __syncthreads();
  T* out = static_cast<T*>(a.out) + (seq.first + i) * a.out_token +
           (int64_t)(header.head * a.group + row - i * a.group) * a.out_head;
  for (int ch = threadIdx.x; ch < D; ch += kJoinThreads) {
    float sum = 0.0f, all = 0.0f;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
      sum += lds[k][ch];
      all += lds[k][D];
    }
    out[ch] = (T)(all > 0.0f || all != all ? sum / all : 0.0f);
  }
}

// Workgroups of the split kernel: two a compute unit, and no more than there are steps.
int split_grid(int64_t num_seqs, int kv_heads, int64_t table_width, int page_size) {
  const int64_t steps = (table_width * page_size + kStep - 1) / kStep;
  const int cus = device_compute_units();
  return (int)min((int64_t)2 * (cus > 0 ? cus : 256), num_seqs * kv_heads * max(steps, (int64_t)1));
}

constexpr int kMostRows = 32;  // of the split kernel

int64_t split_bytes(int grid, int rows, int head_size) {
  return grid * ((int64_t)sizeof(SplitHeader) + 2 * rows * (head_size + 2) * (int64_t)sizeof(float));
}

template <typename T, int D>
int launch_split(const SplitArgs& args, int grid, void* stream) {
  auto kernel = args.rows <= 16 ? attention_split_kernel<T, D, 1> : attention_split_kernel<T, D, 2>;
  launch_kernel(kernel, dim3((unsigned)grid), dim3(64 * kWaves), 0, static_cast<hipStream_t>(stream), args);
  if (int rc = finish_launch("kv4_attention")) return rc;
  launch_kernel(attention_join_kernel<T, D>, dim3((unsigned)grid, (unsigned)args.rows), dim3(kJoinThreads), 0,
                static_cast<hipStream_t>(stream), args);
  return finish_launch("kv4_attention");
}

template <typename T>
int launch_split(const SplitArgs& args, int D, int grid, void* stream) {
  if (D == 64) return launch_split<T, 64>(args, grid, stream);
  if (D == 128) return launch_split<T, 128>(args, grid, stream);
  return launch_split<T, 256>(args, grid, stream);
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
  if (q_heads < 1 || kv_heads < 1 || num_seqs < 1 || max_queries < 1) return 0;
  const int64_t rows = max_queries * (q_heads / kv_heads);
  return rows > kMostRows ? 0 : split_bytes(split_grid(num_seqs, kv_heads, table_width, page_size), (int)rows, head_size);
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
  if (need > 0) {
    const int grid = split_grid(num_seqs, kv_heads, table_width, page_size);
    // steps are counted in 32 bits
    if ((double)num_seqs * kv_heads * (double)((table_width * page_size + kStep - 1) / kStep + 1) > 2e9)
      return set_error(TW_ERR_INVALID_ARGUMENT, "%s: the sequences have room for too many tokens", what);
    SplitArgs args{a, static_cast<SplitHeader*>(workspace),
                   reinterpret_cast<float*>(static_cast<char*>(workspace) + grid * sizeof(SplitHeader)),
                   (int)(max_queries * a.group)};
    return dtype == TW_DTYPE_BF16 ? launch_split<__bf16>(args, head_size, grid, stream)
                                  : launch_split<_Float16>(args, head_size, grid, stream);
  }
  return dtype == TW_DTYPE_BF16 ? launch_rows<__bf16>(a, head_size, (int)q->heads, stream)
                                : launch_rows<_Float16>(a, head_size, (int)q->heads, stream);
}

}  // namespace tw
