// Attention over the 4-bit paged cache (tw_kv4.h) for gfx950 (wave64).
//
//   o = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m),  s_t = scale * log2(e) * q k_t,  any m near max_t s_t
//
// in one pass over the tokens: when a larger s appears, what has been summed is multiplied by
// 2^(m - m').  Scores, m, sums and the output are fp32; the output is rounded once.  Queries (lifted by a
// power of two) and cached values are exact in fp16, the type of both products.  Probabilities are not:
// they are rounded to it for the second product (2^-11 each) and summed as rounded, so that their
// weights still sum to one.  An fp16 output is then 1.1 to 1.4 times as far from 64 bits as with fp32
// probabilities (2.6e-4 and 2.1e-4 of its size for four drafted tokens), a bf16 one under 1 % farther.
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
  int64_t table_stride;
  int capacity;  // tokens that a row of the table has places for, at most 2^30
  const int32_t* seq_lens;
  const int32_t* query_starts;  // or null: per_seq each
  int per_seq;
  int num_seqs, num_tokens, max_queries;
  float scale;  // with log2(e)
  int window;   // 0: none
  bool q_wide, out_wide;  // every row is 16-byte aligned
};

// A sequence's new tokens [first, first + count) and how many are cached.
struct Sequence {
  int first, count, length;
};

// Reads of what no kernel here writes, at addresses that a wave's lanes share: through the scalar cache.
typedef const __attribute__((address_space(4))) int32_t* ConstInts;
__device__ __forceinline__ ConstInts constant(const int32_t* p) { return (ConstInts)(uintptr_t)p; }

// UNIFORM: s is the same in all lanes.  Whatever the arrays hold, only tokens of q and tokens that the table has
// places for are touched.
template <bool UNIFORM = false>
__device__ __forceinline__ Sequence sequence(const AttentionArgs& a, int s) {
  int first, end;
  if (a.query_starts) {
    first = UNIFORM ? constant(a.query_starts)[s] : a.query_starts[s];
    end = UNIFORM ? constant(a.query_starts)[s + 1] : a.query_starts[s + 1];
  } else {
    first = s * a.per_seq;
    end = first + a.per_seq;
  }
  const int length = UNIFORM ? constant(a.seq_lens)[s] : a.seq_lens[s];
  // New tokens behind q's last belong to a later call: here the sequence ends before them.
  const int later = max(end, a.num_tokens) - a.num_tokens;
  first = min(max(first, 0), a.num_tokens);
  end = min(max(end, 0), a.num_tokens);  // (before the subtraction: it would not fit 32 bits)
  return {first, max(end - first, 0), max(min(max(length, 0), a.capacity) - later, 0)};
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
// A sequence's 128-token steps are cut into even pieces, as many in all as the grid holds workgroups,
// whatever the lengths: a workgroup finds its pieces from the lengths on the device.  The pieces of a
// sequence that has several go to the workspace as (m, l, O), and attention_join_kernel joins them.
//
// What bounds it: the cache's bytes where there are many (256 sequences of 4096 tokens, 8 key heads, D = 128, 1.15 GB:
// 243 us = 4.7 TB/s, where a large copy reaches 5.16), latencies below some 50 MB: lengths, pages' numbers and keys
// wait for each other, and the join is a launch of its own (traced: a sequence of 700 tokens 6.7 + 4.2 us, 64 ragged
// ones of 29.7 MB 14.2 + 3.9).  Of 17 to 32 rows the vector unit as well: 32 sequences of 4096 with four new tokens 22 us
// (D = 256: 46; without the bound on probabilities, kMost, 21.7 and 43.4).  Two tiles of keys and values are under way
// in registers, not LDS: no wave needs another's keys, so none waits at a barrier (those 256 sequences took, step by
// step, 282 us with barriers, 268 without, 239 with two tiles).
// ---------------------------------------------------------------------------
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4, kWaveTokens = 32, kStep = kWaves * kWaveTokens, kJoinThreads = 256;

// Of a sequence and key head: in how many pieces its steps are, and the first one's part in the workspace
// where they are several (the others' follow).
struct PieceHeader {
  int32_t count, slot;
};

struct SplitArgs {
  AttentionArgs a;
  PieceHeader* headers;  // [num_seqs][kv_heads]
  float* parts;    // [slots][rows][D + 4], m and l behind the D channels
  int rows;        // of a part
  int budget;      // pieces that the steps are cut into; at most one more for each sequence and key head
  int group_inv;   // 65536 / group + 1
};

// First token that any new token of the sequence sees, and the 128-token steps from there to its end; a
// sequence with new tokens has one step at least, in which its outputs are written.
__device__ __forceinline__ void steps_of(const AttentionArgs& a, const Sequence& q, int* first, int* count) {
  const int seen = a.window > 0 ? max(q.length - q.count + 1 - a.window, 0) : 0;
  *first = seen / kStep;
  *count = q.count == 0 ? 0 : max((q.length + kStep - 1) / kStep - *first, 1);
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The value of this lane and of the one 32 (16) lanes across, in two registers in either order.
struct Both {
  float a, b;
};
__device__ __forceinline__ Both across32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}
__device__ __forceinline__ Both across16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}
__device__ __forceinline__ float max32(float x) {
  const Both y = across32(x);
  return fmaxf(y.a, y.b);
}
__device__ __forceinline__ float max16(float x) {
  const Both y = across16(x);
  return fmaxf(y.a, y.b);
}

// Sum over the wave's lanes up to this one.
__device__ __forceinline__ int wave_scan(int x) {
#define TW_SCAN_STEP(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false)
  TW_SCAN_STEP(0x111, 0xf);  // from 1, 2, 4, 8 lanes before, within 16
  TW_SCAN_STEP(0x112, 0xf);
  TW_SCAN_STEP(0x114, 0xf);
  TW_SCAN_STEP(0x118, 0xf);
  TW_SCAN_STEP(0x142, 0xa);  // the 16 before, into the second and the fourth 16
  TW_SCAN_STEP(0x143, 0xc);  // the first half, into the second
#undef TW_SCAN_STEP
  return x;
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

// Where a wave's 32 tokens are: two sixteens, each in one page.
struct Place {
  const uint8_t* block[2];
  int at[2];
  bool there[2];
};

template <int D>
__device__ __forceinline__ void load_keys(Tile<D>& tile, const Place& place, const LaneOffsets<D>& lane, int P) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* p = place.block[i];
    load_words(tile.k[i], p + (place.at[i] * Kv4<D>::kRow + lane.k));
#pragma unroll
    for (int g = 0; g < (D + 127) / 128; ++g) tile.ks[i][g] = p[place.at[i] + lane.ks + g * P];
  }
}

template <int D>
__device__ __forceinline__ void load_values(Tile<D>& tile, const Place& place, const LaneOffsets<D>& lane) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* p = place.block[i];
    load_words(tile.v[i], p + (place.at[i] * Kv4<D>::kRow + lane.v));
    tile.vs[i] = *reinterpret_cast<const uint32_t*>(p + (place.at[i] + lane.vs));
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
template <typename T, int N>
__device__ __forceinline__ void load_row(float (&x)[N], const T* row, bool wide) {
  if (wide) {
    typedef T vec_t __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      const vec_t v = *reinterpret_cast<const vec_t*>(row + i);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i + j] = (float)v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)row[i];
  }
}

// What a row is multiplied by before its products, the power of two that brings its largest magnitude to [2^14,
// 2^15) and the sign of `scale`, and what the products are multiplied by: more than zero, so that the largest
// product is the largest score and a product of minus infinity a score of minus infinity.
__device__ __forceinline__ float lift_of(float most, float scale, float* back) {
  const int e = min(max((int)(__float_as_uint(most) >> 23) - 127, -100), 127);
  const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
  *back = scale == 0.0f ? 1.0f : fmaxf(__uint_as_float((uint32_t)(127 - 14 + e) << 23) * __builtin_fabsf(scale), 0x1p-126f);
  return scale == 0.0f ? 0.0f : __builtin_copysignf(up, scale);
}

template <typename T, int D>
struct RawQueries {
  typedef T vec_t __attribute__((ext_vector_type(8)));
  vec_t x[D / 32];
  __device__ __forceinline__ void load(const T* row, bool wide) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      x[i] = vec_t{};
      if (row && wide) x[i] = *reinterpret_cast<const vec_t*>(row + i * 8);
      if (row && !wide) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = row[i * 8 + j];
      }
    }
  }
  // Returns what the products are multiplied by to be scores.
  __device__ __forceinline__ float lift(half8_t (&q)[D / 32], float scale) const {
    float most = 0.0f, back;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) most = fmaxf(most, __builtin_fabsf((float)x[i / 8][i % 8]));
    most = max32(max16(most));
    const float up = lift_of(most, scale, &back);
#pragma unroll
    for (int i = 0; i < D / 4; ++i) q[i / 8][i % 8] = (_Float16)((float)x[i / 8][i % 8] * up);
    return back;
  }
};

// x / d for 0 <= x < 2^24 and d's reciprocal.
__device__ __forceinline__ int divide(int x, int d, float inv) {
  int q = (int)((float)x * inv);
  const int r = x - q * d;
  q += r >= d ? 1 : 0;
  q -= r < 0 ? 1 : 0;
  return q;
}

// Four neighbouring channels of an output row.
template <typename T>
__device__ __forceinline__ void store4(T* out, const float4_t& x, bool wide) {
  typedef T vec_t __attribute__((ext_vector_type(4)));
  const vec_t v = {(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
  if (wide) {
    *reinterpret_cast<vec_t*>(out) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = v[i];
  }
}

// The exponents' base for a maximum: the next 64th.  Neither kLift - m nor the factor from one m to the next is rounded
// then, and the largest probabilities are just below a power of two, where fp16 is finest.
__device__ __forceinline__ float base_of(float most) { return __builtin_ceilf(most * 64.0f) * 0.015625f; }

// From kFar on neighbouring fp32 values are half and more apart, up to far more than the exponents' range: a score's
// product with the scale, which is not rounded where m is subtracted, may be that much above or below the maximum, which
// was.  (From 2^25 on, where scores of 3e7 are, a row's largest probability was infinite or zero.)
constexpr float kFar = 0x1p22f;
__device__ __forceinline__ bool is_far(float m) { return __builtin_fabsf(m) >= kFar && __builtin_fabsf(m) < __builtin_inff(); }

// Rows of tokens that no sequence has, before the first one's and behind the last one's: zeros, by the
// workgroups of a launch that have no second place in the grid (those of a join's first rows).
struct Rest {
  int before, behind;  // [0, before) and [behind, num_tokens)
};
__device__ __forceinline__ Rest rest_of(const AttentionArgs& a) {
  if (!a.query_starts) return {0, a.num_tokens};
  const int first = constant(a.query_starts)[0], last = constant(a.query_starts)[a.num_seqs];
  const int before = min(max(first, 0), a.num_tokens);
  return {before, last < first ? a.num_tokens : min(max(last, 0), a.num_tokens)};  // (in no order: nothing is behind)
}
template <typename T, int D, int THREADS>
__device__ __forceinline__ void clear_rest(const AttentionArgs& a) {
  const Rest rest = rest_of(a);
  const int tokens = rest.before + a.num_tokens - rest.behind;
  if (tokens == 0) return;
  const int64_t heads = a.pages.heads * a.group, columns = D / 4;
  const int64_t block = (int64_t)blockIdx.z * gridDim.x + blockIdx.x, threads = (int64_t)gridDim.x * gridDim.z * THREADS;
  for (int64_t i = block * THREADS + threadIdx.x; i < tokens * heads * columns; i += threads) {
    const int64_t row = i / columns;
    const int at = (int)(row / heads), token = at < rest.before ? at : at - rest.before + rest.behind;
    store4(static_cast<T*>(a.out) + (int64_t)token * a.out_token + (row - at * heads) * a.out_head +
               (i - row * columns) * 4,
           float4_t{0, 0, 0, 0}, a.out_wide);
  }
}

// Few rows: probabilities are held times 2^14, so that fp16's normal range reaches down to 2^-28 of the largest.  A far
// maximum's base is two to four neighbouring values below it: the largest exponent is kLift or more, and what is above
// kMost counts as kMost, so that scores closer than their own rounding errors weigh the same.
// (Four instructions of 32 tokens: 243.3 us instead of 240.5 for 256 sequences of 4096 tokens, 64 + 8 heads of 128; a base
// that is the maximum itself, as of many rows, took three more registers and 245.3.)
constexpr float kLift = 14.0f;
constexpr _Float16 kMost = (_Float16)0x1p15f;
__device__ __forceinline__ float low_base_of(float most) {
  return is_far(most) ? __builtin_fmaf(__builtin_fabsf(most), -0x1p-22f, most) : base_of(most);
}

// Many rows: probabilities are held times 2^(kTileLift - m).  m need not be the maximum so far, only within kSlack of
// it: so they stay within 2^15, fp16's normal range reaches down to 2^-21 of the largest or lower and its subnormals to
// 2^-31, and a row's sums are multiplied anew a few times in all instead of in most units (one of 64 rows has a new
// maximum in most of the first hundred units: 211 us with the maximum itself and 188 us so, before the later steps, for
// 8192 queries of 8 heads).
// A far maximum is the base itself and scores are rounded as it was: the largest is exactly zero below it.
constexpr float kTileLift = 7.0f, kSlack = 8.0f;
__device__ __forceinline__ float tile_base_of(float most) { return is_far(most) ? most : base_of(most); }
__device__ __forceinline__ float below(float x, float scale, float m) {
#pragma clang fp contract(off)
  const float s = x * scale;
  return s - m;
}

template <typename T, int D, int NT>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 1 : 2) void attention_split_kernel(SplitArgs args) {
  const AttentionArgs& a = args.a;
  constexpr int kTiles = D / 16;          // of channels
  __shared__ __align__(16) float merge[kWaves][NT * 16][D + 4];  // a wave's O; four words more: no two rows in one bank
  __shared__ float merge_m[kWaves][NT * 16], merge_l[kWaves][NT * 16];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 15, h4 = lane >> 4;
  const int P = 1 << a.pages.page_log2, heads = a.pages.heads, w = blockIdx.x;

  // ---- every wave counts all sequences' steps and pieces, 64 sequences at a time; the first 256 are kept
  constexpr int kKept = 4;
  Sequence kept[kKept];
  int pieces[kKept];
  const int rounds = (a.num_seqs + 63) / 64;
  auto read = [&](int r) {
    const int s = r * 64 + lane;
    return s < a.num_seqs ? sequence(a, s) : Sequence{0, 0, 0};
  };
  auto steps_in = [&](const Sequence& seq) {
    int first, count;
    steps_of(a, seq, &first, &count);
    return count;
  };
  int total = 0;
#pragma unroll
  for (int r = 0; r < kKept; ++r) kept[r] = read(r);
#pragma unroll
  for (int r = 0; r < kKept; ++r) {
    pieces[r] = steps_in(kept[r]);
    total += pieces[r];
  }
  for (int r = kKept; r < rounds; ++r) total += steps_in(read(r));
  total = __builtin_amdgcn_readlane(wave_scan(total), 63) * heads;
  const int share = max((total + args.budget - 1) / args.budget, 1);
  const float share_inv = 1.0f / (float)share;
  auto pieces_in = [&](int steps) { return divide(steps + share - 1, share, share_inv); };
  auto several = [](int count) { return count > 1 ? count : 0; };
  int all = 0;
#pragma unroll
  for (int r = 0; r < kKept; ++r) {
    pieces[r] = pieces_in(pieces[r]);
    all += pieces[r];
  }
  for (int r = kKept; r < rounds; ++r) {
    all += pieces_in(steps_in(read(r)));
  }
  all = __builtin_amdgcn_readlane(wave_scan(all), 63) * heads;

  const LaneOffsets<D> offsets(P, lane);
  for (int piece = w; piece < all; piece += gridDim.x) {
    // ---- whose piece it is
    int s = 0, inside = 0, count = 1, slot = 0;
    Sequence seq{0, 0, 0};
    {
      bool found = false;
      int base = 0, slot_base = 0;
      auto look = [&](int r, int own, const Sequence& from) {
        const int upto = base + wave_scan(own), slots_upto = slot_base + wave_scan(several(own));
        const uint64_t here = __builtin_amdgcn_ballot_w64(piece < upto * heads);
        if (here) {
          const int at = __builtin_ctzll(here);
          s = r * 64 + at;
          count = __builtin_amdgcn_readlane(own, at);
          inside = piece - (__builtin_amdgcn_readlane(upto, at) - count) * heads;
          slot = (__builtin_amdgcn_readlane(slots_upto, at) - several(count)) * heads + inside;
          seq.first = __builtin_amdgcn_readlane(from.first, at);
          seq.count = __builtin_amdgcn_readlane(from.count, at);
          seq.length = __builtin_amdgcn_readlane(from.length, at);
          found = true;
        }
        base = __builtin_amdgcn_readlane(upto, 63);
        slot_base = __builtin_amdgcn_readlane(slots_upto, 63);
      };
#pragma unroll
      for (int r = 0; r < kKept; ++r)
        if (!found) look(r, pieces[r], kept[r]);
      for (int r = kKept; r < rounds && !found; ++r) {
        const Sequence from = read(r);
        look(r, pieces_in(steps_in(from)), from);
      }
    }
    const int head = inside / count, part = inside - head * count;
    int first_step, seq_steps;
    steps_of(a, seq, &first_step, &seq_steps);
    const int each = seq_steps / count, longer = seq_steps - each * count;
    const int step0 = first_step + part * each + min(part, longer), step_end = step0 + each + (part < longer ? 1 : 0);
    const int queries = min(seq.count, a.max_queries), rows = queries * a.group;
    const int length = seq.length, new_from = length - seq.count;  // position of the first new token

    // Two tiles in registers, worked on in turn: the keys of the tile after next are fetched over those just
    // used, and so are the values; the pages' numbers are fetched one tile earlier still.
    const ConstInts table = constant(a.block_table) + (int64_t)s * a.table_stride;
    auto ids_of = [&](int step, int (&ids)[2]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = step * kStep + wave * kWaveTokens + i * 16;
        ids[i] = step < step_end && t < length ? table[t >> a.pages.page_log2] : -1;
      }
    };
    auto place_of = [&](int step, const int (&ids)[2]) {
      Place place;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        place.there[i] = ids[i] >= 0 && ids[i] < a.pages.num_pages;
        // tokens of a missing page are read from page 0 and masked
        place.block[i] = a.pages.data + ((int64_t)(place.there[i] ? ids[i] : 0) * heads + head) * a.pages.head_bytes;
        place.at[i] = (step * kStep + wave * kWaveTokens + i * 16) & (P - 1);
      }
      return place;
    };
    int ids[2], first_ids[2];
    ids_of(step0, first_ids);
    ids_of(step0 + 1, ids);

    RawQueries<T, D> raw[NT];
    int row_end[NT], row_begin[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = t * 16 + n, i = row * args.group_inv >> 16;
      raw[t].load(row < rows ? static_cast<const T*>(a.q) + (int64_t)(seq.first + i) * a.q_token +
                                   (int64_t)(head * a.group + row - i * a.group) * a.q_head + h4 * (D / 4)
                             : nullptr,
                  a.q_wide);
      row_end[t] = row < rows ? new_from + i + 1 : 0;
      row_begin[t] = a.window > 0 ? max(new_from + i + 1 - a.window, 0) : 0;
    }
    float one = 1.0f;
    asm volatile("" : "+s"(one));  // (not known: a conversion and an addition are one instruction then)
    Tile<D> even, odd;
    Place even_place = place_of(step0, first_ids), odd_place = place_of(step0 + 1, ids);
    load_keys<D>(even, even_place, offsets, P);
    load_values<D>(even, even_place, offsets);
    if (step0 + 1 < step_end) {
      load_keys<D>(odd, odd_place, offsets, P);
      load_values<D>(odd, odd_place, offsets);
    }
    ids_of(step0 + 2, ids);

    half8_t q[NT][D / 32];
    float scale[NT], m[NT], l[NT];
    float4_t o[NT][kTiles];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      scale[t] = raw[t].lift(q[t], a.scale);
      m[t] = -__builtin_inff();
      l[t] = 0.0f;
#pragma unroll
      for (int c = 0; c < kTiles; ++c) o[t][c] = float4_t{0, 0, 0, 0};
    }
    // tokens that every row sees need no mask
    const int all_from = a.window > 0 ? max(new_from + queries - a.window, 0) : 0;
    const int all_to = new_from + 1;
    const int some_from = a.window > 0 ? max(new_from + 1 - a.window, 0) : 0;

    auto work_on = [&](Tile<D>& tile, Place& place, int step) {
      const bool there[2] = {place.there[0], place.there[1]};
      const bool more = step + 2 < step_end;
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
      if (more) {
        place = place_of(step + 2, ids);
        load_keys<D>(tile, place, offsets, P);
        ids_of(step + 3, ids);
      }
      // ---- probabilities
      half8_t p[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[8], most = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = sc[t][i / 4][i % 4];
          if (!whole) {
            const int token = t0 + (i / 4) * 16 + h4 * 4 + i % 4;
            if (token >= row_end[t] || token < row_begin[t] || !there[i / 4]) x[i] = -__builtin_inff();
          }
          most = fmaxf(most, x[i]);
        }
        most = max32(max16(most)) * scale[t];
        if (__builtin_amdgcn_ballot_w64(most > m[t])) {
          const float now = fmaxf(m[t], low_base_of(most));
          const float old = m[t] == now ? 1.0f : __builtin_amdgcn_exp2f(m[t] - now);
          m[t] = now;
          l[t] *= old;
#pragma unroll
          for (int c = 0; c < kTiles; ++c) o[t][c] *= old;
        }
        const float add = kLift - (m[t] == -__builtin_inff() ? 0.0f : m[t]);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) p[t][i] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(x[i], scale[t], add));
        p[t] = __builtin_elementwise_minimum(p[t], half8_t(kMost));  // (what is not a number stays so)
#pragma unroll
        for (int i = 0; i < 8; ++i)  // (as rounded: one token's output is its value, to the bit)
          sum = __builtin_fmaf((float)p[t][i], one, sum);
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
      // Where some rows see a token and others do not, a value that is not a number is kept out of the products (times
      // zero it is not zero) and put into the sums of the rows that see it, which a product of ones and zeros finds.
      if (!whole) {
        bool any = false;
        half8_t odd_ones;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool odd_one = vs[i] == __builtin_inff();
          any = any || odd_one;
          odd_ones[i] = odd_one ? (_Float16)1.0f : (_Float16)0.0f;
        }
        if (__builtin_amdgcn_ballot_w64(any)) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (vs[i] == __builtin_inff()) vs[i] = 1.0f;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            half8_t seen;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int token = t0 + (i / 4) * 16 + h4 * 4 + i % 4;
              seen[i] = token < row_end[t] && token >= row_begin[t] ? (_Float16)1.0f : (_Float16)0.0f;
            }
            const float4_t found = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd_ones, seen, float4_t{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (found[r] > 0.0f) {
#pragma unroll
                for (int c = 0; c < kTiles; ++c) o[t][c][r] = __builtin_nanf("");
              }
          }
        }
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
      if (more) load_values<D>(tile, place, offsets);
    };

    for (int step = step0; step < step_end; step += 2) {
      work_on(even, even_place, step);
      if (step + 1 < step_end) work_on(odd, odd_place, step + 1);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const Both x = across16(l[t]), y = across32(x.a + x.b);
      l[t] = y.a + y.b;
    }

    // ---- the waves' parts become one
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = t * 16 + n;
      if (row >= rows) continue;
      // lane (n, h): channels (4h + r) * D/16 + c of row n
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < kTiles; c += 4)
          *reinterpret_cast<float4_t*>(&merge[wave][row][h4 * (D / 4) + r * kTiles + c]) =
              float4_t{o[t][c][r], o[t][c + 1][r], o[t][c + 2][r], o[t][c + 3][r]};
      if (h4 == 0) {
        merge_m[wave][row] = m[t];
        merge_l[wave][row] = l[t];
      }
    }
    __syncthreads();
    for (int item = threadIdx.x; item < rows * (D / 4); item += 64 * kWaves) {
      const int row = item / (D / 4), ch = item % (D / 4) * 4, i = row * args.group_inv >> 16;
      float most = merge_m[0][row];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) most = fmaxf(most, merge_m[k][row]);
      float4_t sum = {0, 0, 0, 0};
      float all = 0.0f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const float mk = merge_m[k][row], weight = mk == most ? 1.0f : __builtin_amdgcn_exp2f(mk - most);
        all += merge_l[k][row] * weight;
        sum += *reinterpret_cast<const float4_t*>(&merge[k][row][ch]) * weight;
      }
      if (count == 1) {
        T* out = static_cast<T*>(a.out) + (int64_t)(seq.first + i) * a.out_token +
                 (int64_t)(head * a.group + row - i * a.group) * a.out_head + ch;
        store4(out, sum * (all > 0.0f || all != all ? 1.0f / all : 0.0f), a.out_wide);
      } else {
        float* part = args.parts + ((int64_t)slot * args.rows + row) * (D + 4);
        *reinterpret_cast<float4_t*>(part + ch) = sum;
        if (ch == 0) {
          part[D] = most;
          part[D + 1] = all;
        }
      }
    }
    if (threadIdx.x == 0 && part == 0) args.headers[s * heads + head] = PieceHeader{count, slot};
  }
}

// Joins the parts of one row: block (sequence and key head, row, CH channels).  A thread has four channels of
// every kGroups-th part, kAtOnce of them under way at once.
template <typename T, int D, int CH>
__global__ __launch_bounds__(kJoinThreads) void attention_join_kernel(SplitArgs args) {
  const AttentionArgs& a = args.a;
  const int s = blockIdx.x / a.pages.heads, head = blockIdx.x - s * a.pages.heads, row = blockIdx.y, ch0 = blockIdx.z * CH;
  const PieceHeader header = args.headers[blockIdx.x];
  const Sequence seq = sequence<true>(a, s);
  if (blockIdx.y == 0) clear_rest<T, D, kJoinThreads>(a);
  // (a sequence without new tokens has no piece and leaves its header as it was)
  if (row >= min(seq.count, a.max_queries) * a.group || header.count < 2) return;
  constexpr int kLanes = CH / 4, kGroups = kJoinThreads / kLanes, kAtOnce = 8;
  __shared__ __align__(16) float lds[kGroups][CH];
  __shared__ float lds_m[kGroups], lds_l[kGroups];
  const int parts = header.count, lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int64_t part_size = (int64_t)args.rows * (D + 4);
  const float* base = args.parts + header.slot * part_size + (int64_t)row * (D + 4);
  float4_t o = {0, 0, 0, 0};
  float m = -__builtin_inff(), l = 0.0f;
  for (int c0 = group; c0 < parts; c0 += kGroups * kAtOnce) {
    float4_t x[kAtOnce];
    float2 ml[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      // (a part behind the last is the last one again, with no weight)
      const float* p = base + min(c0 + k * kGroups, parts - 1) * part_size;
      x[k] = *reinterpret_cast<const float4_t*>(p + ch0 + lane * 4);
      ml[k] = *reinterpret_cast<const float2*>(p + D);
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (c0 + k * kGroups >= parts) ml[k] = make_float2(-__builtin_inff(), 0.0f);
    float most = m;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) most = fmaxf(most, ml[k].x);
    const float old = m == most ? 1.0f : __builtin_amdgcn_exp2f(m - most);
    m = most;
    l *= old;
    o *= old;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const float weight = c0 + k * kGroups >= parts ? 0.0f
                           : ml[k].x == most        ? 1.0f
                                                    : __builtin_amdgcn_exp2f(ml[k].x - most);
      l += ml[k].y * weight;
      o += x[k] * weight;
    }
  }
  *reinterpret_cast<float4_t*>(&lds[group][lane * 4]) = o;
  if (lane == 0) {
    lds_m[group] = m;
    lds_l[group] = l;
  }
  __syncthreads();
  if (threadIdx.x >= kLanes) return;
  float most = lds_m[0], all = 0.0f;
#pragma unroll
  for (int k = 1; k < kGroups; ++k) most = fmaxf(most, lds_m[k]);
  float4_t sum = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < kGroups; ++k) {
    const float weight = lds_m[k] == most ? 1.0f : __builtin_amdgcn_exp2f(lds_m[k] - most);
    all += lds_l[k] * weight;
    sum += *reinterpret_cast<const float4_t*>(&lds[k][lane * 4]) * weight;
  }
  const int i = row * args.group_inv >> 16;
  T* out = static_cast<T*>(a.out) + (int64_t)(seq.first + i) * a.out_token +
           (int64_t)(head * a.group + row - i * a.group) * a.out_head + ch0 + lane * 4;
  store4(out, sum * (all > 0.0f || all != all ? 1.0f / all : 0.0f), a.out_wide);
}

// Of the split kernel, two operands' width.  One new token of each of 8 sequences of 4096, 8 rows: 10 us, in tiles 23;
// of 300 of 700 with 8 key heads 78 and 232; four new tokens of each of 32 of 4096, 32 rows: 22 and 34.  Up to 16 rows
// one operand is enough (8 sequences 10 us, with two operands 11; 300 sequences 78 and 96).
constexpr int kMostRows = 32;

// Cut of a call's steps.  While there is room, every piece has a workgroup of its own, two a compute unit, which is how
// many of them run at once at D = 128 (their registers allow no third; of D = 256 one runs, the other after it, of D = 64
// a third could); sequences and key heads beyond half of that are cut in four pieces a compute unit on top, which the
// workgroups take in turn.  8 heads over a key head, D = 128: 64 sequences of 1 to 4096 tokens and 8 key heads 45.1 us
// so, 48.5 with two pieces a compute unit and 49.7 with eight, 40 of 16 to 8192 tokens 30.3, 32.0 and 31.2; but 64 that
// are all of 2048 tokens 41.8, 35.8 and 50.6: lengths that differ are taken to be the ordinary case.
struct SplitPlan {
  int grid, budget;
  int64_t header_bytes, bytes;
};

SplitPlan plan_split(int64_t num_seqs, int kv_heads, int64_t table_width, int page_size, int rows, int head_size) {
  const int cus = device_compute_units();
  const int64_t room = 2 * (int64_t)(cus > 0 ? cus : 256), units = num_seqs * kv_heads;
  const int64_t steps = units * max((table_width * page_size + kStep - 1) / kStep, (int64_t)1);
  SplitPlan plan;
  plan.grid = (int)min(room, steps);
  plan.budget = (int)(units <= room / 2 ? room - units : 2 * room);
  // of n > share steps come ceil(n / share) < 2 n / share pieces
  const int64_t parts = min((int64_t)2 * plan.budget, steps);
  plan.header_bytes = (units * (int64_t)sizeof(PieceHeader) + 15) / 16 * 16;
  plan.bytes = plan.header_bytes + parts * rows * (head_size + 4) * (int64_t)sizeof(float);
  return plan;
}

template <typename T, int D>
int launch_split(const SplitArgs& args, int grid, void* stream) {
  auto kernel = args.rows <= 16 ? attention_split_kernel<T, D, 1> : attention_split_kernel<T, D, 2>;
  launch_kernel(kernel, dim3((unsigned)grid), dim3(64 * kWaves), 0, static_cast<hipStream_t>(stream), args);
  if (int rc = finish_launch("kv4_attention")) return rc;
  // Few rows may be in very many pieces: more workgroups then share a row's channels (one sequence of 65536 tokens,
  // 8 rows: 12.3 us so and 13.6 with whole rows; two of 32768 and 8 key heads, 128 rows: 26.1 and 24.4).
  const bool few = (int64_t)args.a.num_seqs * args.a.pages.heads * args.rows <= 32;
  launch_kernel(few ? attention_join_kernel<T, D, 32> : attention_join_kernel<T, D, D>,
                dim3((unsigned)(args.a.num_seqs * args.a.pages.heads), (unsigned)args.rows, few ? D / 32 : 1), dim3(kJoinThreads), 0,
                static_cast<hipStream_t>(stream), args);
  return finish_launch("kv4_attention");
}

template <typename T>
int launch_split(const SplitArgs& args, int D, int grid, void* stream) {
  if (D == 64) return launch_split<T, 64>(args, grid, stream);
  if (D == 128) return launch_split<T, 128>(args, grid, stream);
  return launch_split<T, 256>(args, grid, stream);
}

// ---------------------------------------------------------------------------
// Many rows: a tile of 32 rows a wave, all of one key head.
//
// The workgroup turns 64 tokens at a time (32 where heads have 256 channels) into fp16 in LDS, once for all its
// rows.  A wave works on 32 tokens at once with 32 x 32 x 16 products; as above the scores of a row stay in the
// two lanes that hold the row and go into the second product without moving.  Values lie in LDS by channel, their
// tokens in the order in which the scores' registers hold them: of 16 tokens 0-3, 8-11, 4-7, 12-15.
//
// The matrix and the vector units work side by side: the scores of the next 32 tokens are computed between the
// exponentials of the present ones, whose sums come between the present products with the values.  Two waves a SIMD
// unit with 32 rows each: one wave with 64 rows reads LDS half as often, but nothing runs while it moves data (229
// us against 188 before the later steps, for 8192 queries of 8 heads over one key head, D = 128).  What bounds it:
// neither unit by itself.  Of a wave's 32 tokens the products take 512 cycles, the 16 exponentials a lane 256 and some
// 55 other vector instructions 220; laying out the tile, addresses and the barrier come on top.  The matrix unit is
// busy in 34 % of the kernel's cycles and the vector unit in 38 %: the two waves of a SIMD unit pass the barrier
// together and are in the same phase for much of a tile.  That call takes 170 us with its join of 15, 808 TFLOP/s,
// where a product of 8192 x 8192 x 8192 by the library reaches 1332.
// ---------------------------------------------------------------------------
typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr int kSpan = 64;  // tokens in which tiles are measured and cut

// Of a tile's key head that is worked on in even shares: whose rows they are, and the workgroups from `first` to
// `last` that hold parts of it.
struct TileHeader {
  int32_t seq, row0, head, first, last;
};

struct TileArgs {
  AttentionArgs a;
  // Even shares: one header for each tile and key head, and two parts a workgroup, [rows][D + 4]: of the tile that
  // it ends and of the one that it begins.  Null: a workgroup for each tile and key head.
  TileHeader* headers;
  float* parts;
  int tiles;
};

// Tokens that the rows [row, last] of a sequence see, in spans: [from, to).
struct Span {
  int from, to;
};
__device__ __forceinline__ Span span_of(const AttentionArgs& a, const Sequence& q, int row, int last) {
  const int new_from = q.length - q.count, window = a.window > 0 ? a.window : 1 << 30;
  const int from = max(new_from + row / a.group + 1 - window, 0) / kSpan;
  return {from, max((min(new_from + last / a.group + 1, q.length) + kSpan - 1) / kSpan, from)};
}

constexpr int kMostShared = 4096;  // tiles times key heads that are worked on in even shares (their ends are in LDS)

// Sum over the workgroup's threads before this one, and over all.
template <int THREADS>
__device__ __forceinline__ int block_scan(int x, int* total, int* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sum = wave_scan(x);
  __syncthreads();
  if (lane == 63) lds[wave] = sum;
  __syncthreads();
  int before = sum - x, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const int y = lds[w];
    before += w < wave ? y : 0;
    all += y;
  }
  *total = all;
  return before;
}

__device__ __forceinline__ int tiles_in(const AttentionArgs& a, const Sequence& q, int rows_of_tile) {
  return (min(q.count, a.max_queries) * a.group + rows_of_tile - 1) / rows_of_tile;
}

// Whose tile it is and its place there (uniform); a tile behind the last: seq < 0.
struct FoundTile {
  int seq, place;
};
template <int THREADS>
__device__ __forceinline__ FoundTile find_tile(const AttentionArgs& a, int tile, int rows_of_tile, int* lds) {
  int* const found = lds + THREADS / 64;
  if (threadIdx.x == 0) found[0] = -1;
  int base = 0;
  for (int s0 = 0; s0 < a.num_seqs && base <= tile; s0 += THREADS) {
    const int s = s0 + threadIdx.x, count = s < a.num_seqs ? tiles_in(a, sequence(a, s), rows_of_tile) : 0;
    int all;
    const int before = base + block_scan<THREADS>(count, &all, lds);
    if (tile >= before && tile < before + count) {
      found[0] = s;
      found[1] = tile - before;
    }
    base += all;
  }
  __syncthreads();
  return {uniform(found[0]), uniform(found[1])};
}

template <int D>
struct TileShape {
  // eight waves, two a SIMD unit, share a tile's keys and values; heads of 256 channels leave registers for one
  static constexpr int kWaves = D == 256 ? 4 : 8, kThreads = 64 * kWaves, kRows = 32 * kWaves;
  static constexpr int kTokens = D == 256 ? 32 : 64, kUnits = kTokens / 32;
  static constexpr int kKeyRow = D * 2 + 16, kValueRow = kTokens * 2 + 16;  // 16 bytes more: no two lanes' rows in one bank
  static constexpr int kKeyBytes = kTokens * kKeyRow, kValueBytes = D * kValueRow;
  static constexpr int kKeyBuffers = kUnits + 1;            // of the tiles whose scores are being computed, and the one written
  static constexpr int kKeyChunks = kTokens * (D / 32);     // 32 channels of a token
  static constexpr int kValueChunks = (kTokens / 4) * 16;   // 4 tokens of a sixteenth
  // keys by the first threads, values by the last ones; where there are not threads for both, some do both
  static constexpr bool kApart = kKeyChunks + kValueChunks <= kThreads;
  static constexpr int kValueThread = kThreads - kValueChunks;
  static_assert(kKeyChunks <= kThreads && kValueChunks <= kThreads, "one chunk a thread");
};

// What a thread fetches of a tile.
template <int D>
struct Fetched {
  using S = TileShape<D>;
  uint32_t first[D / 32 > 4 ? D / 32 : 4], first_scale;
  uint32_t second[S::kApart ? 1 : D / 32], second_scale;
  __device__ __forceinline__ uint32_t (&keys())[4] { return reinterpret_cast<uint32_t(&)[4]>(first); }
  __device__ __forceinline__ uint32_t (&values())[D / 32] {
    if constexpr (S::kApart) return reinterpret_cast<uint32_t(&)[D / 32]>(first);
    else return second;
  }
  __device__ __forceinline__ uint32_t& value_scale() {
    if constexpr (S::kApart) return first_scale;
    else return second_scale;
  }
};

// A barrier for what is in LDS alone: loads from memory stay under way.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <typename T, int D>
__global__ __launch_bounds__(TileShape<D>::kThreads, TileShape<D>::kWaves / 4) void attention_tile_kernel(TileArgs args) {
  using S = TileShape<D>;
  using L = Kv4<D>;
  const AttentionArgs& a = args.a;
  __shared__ __align__(16) uint8_t key_buffers[S::kKeyBuffers][S::kKeyBytes];
  __shared__ __align__(16) uint8_t value_buffers[2][S::kValueBytes];
  __shared__ int scan[S::kWaves + 2];
  __shared__ int odd_unit;  // the last unit with values that are not numbers
  __shared__ int first_tile[kMostShared + 1], unit_end[kMostShared];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int P = 1 << a.pages.page_log2, heads = a.pages.heads;
  const int window = a.window > 0 ? a.window : 1 << 30;

  if (blockIdx.y == 0) clear_rest<T, D, S::kThreads>(a);
  if (threadIdx.x == 0) odd_unit = -1;  // (a barrier follows, with the search for the tiles)

  // ---- Which tiles: one, or an even share of all tiles' spans.  In the order of the shares a long tile of a prompt
  // and a short one take turns: the last, the first, the last but one, ...
  const bool shared = args.headers != nullptr;
  int tiles = 0, units = 0, share = 1, unit = 0, at = 0, end = 1;
  if (shared) {
    for (int s0 = 0; s0 < a.num_seqs; s0 += S::kThreads) {
      const int s = s0 + threadIdx.x, count = s < a.num_seqs ? tiles_in(a, sequence(a, s), S::kRows) : 0;
      int all;
      const int before = block_scan<S::kThreads>(count, &all, scan);
      if (s < a.num_seqs) first_tile[s] = tiles + before;
      tiles += all;
    }
    if (threadIdx.x == 0) first_tile[a.num_seqs] = tiles;
    __syncthreads();
    tiles = min(tiles, args.tiles);  // (more only where query_starts does not rise)
    units = tiles * heads;
  }
  auto find = [&](int unit) {  // the tile of a unit of the shares
    const int k = unit / heads, tile = k & 1 ? k >> 1 : tiles - 1 - (k >> 1);
    int low = 0, high = a.num_seqs;  // the last sequence whose first tile is not behind it
    while (high - low > 1) {
      const int middle = (low + high) >> 1;
      if (first_tile[middle] <= tile) low = middle;
      else high = middle;
    }
    return FoundTile{low, tile - first_tile[low]};
  };
  auto span_in = [&](const Sequence& seq, int row0) {
    return span_of(a, seq, row0, min(row0 + S::kRows, min(seq.count, a.max_queries) * a.group) - 1);
  };
  if (shared) {
    int total = 0;
    for (int u0 = 0; u0 < units; u0 += S::kThreads) {
      const int u = u0 + threadIdx.x;
      int count = 0, all;
      if (u < units) {
        const FoundTile own = find(u);
        const Span span = span_in(sequence(a, own.seq), own.place * S::kRows);
        count = max(span.to - span.from, 1);
      }
      const int before = total + block_scan<S::kThreads>(count, &all, scan);
      if (u < units) unit_end[u] = before + count;
      total += all;
    }
    __syncthreads();
    // headers that no tile has
    for (int u = units + blockIdx.x * S::kThreads + threadIdx.x; u < args.tiles * heads; u += gridDim.x * S::kThreads)
      args.headers[u] = TileHeader{0, 0, 0, 0, 0};
    share = max((total + (int)gridDim.x - 1) / (int)gridDim.x, 1);
    at = blockIdx.x * share;
    end = min(at + share, total);
    if (at >= end) return;
    int low = -1, high = units - 1;  // the first unit that ends behind `at`
    while (high - low > 1) {
      const int middle = (low + high) >> 1;
      if (unit_end[middle] > at) high = middle;
      else low = middle;
    }
    unit = uniform(high);
  }

  for (; at < end; ++unit) {
    FoundTile own;
    int head = blockIdx.y;
    if (shared) {
      own = find(unit);
      own = {uniform(own.seq), uniform(own.place)};
      head = unit - unit / heads * heads;
    } else {
      // a prompt's last tiles see the most: they go first
      own = find_tile<S::kThreads>(a, args.tiles - 1 - (int)blockIdx.x, S::kRows, scan);
      if (own.seq < 0) return;
    }
    const Sequence seq = sequence<true>(a, own.seq);
    const int queries = min(seq.count, a.max_queries), rows = queries * a.group, length = seq.length;
    const int new_from = length - seq.count;
    const int row0 = own.place * S::kRows;

    // ---- tokens that the tile's rows see, and this share of them
    auto end_of = [&](int row) { return min(new_from + row / a.group + 1, length); };
    auto begin_of = [&](int row) { return max(new_from + row / a.group + 1 - window, 0); };
    const int some_from = begin_of(row0);
    Span span = span_in(seq, row0);
    bool starts = true, ends = true;
    if (shared) {
      const int count = max(span.to - span.from, 1), unit_from = uniform(unit_end[unit]) - count;
      starts = at == unit_from;
      ends = unit_from + count <= end;
      const int first = at - unit_from, last = min(end - unit_from, count);
      if (starts && threadIdx.x == 0)
        args.headers[unit] = TileHeader{own.seq, row0, head, (int)blockIdx.x, (unit_from + count - 1) / share};
      at = unit_from + last;
      span = {min(span.from + first, span.to), min(span.from + last, span.to)};
    } else {
      at = end;
    }
    const int tile_from = span.from * (kSpan / S::kTokens), tile_to = span.to * (kSpan / S::kTokens);

    // ---- this wave's rows
    const int row = row0 + wave * 32 + n, query = row / a.group, q_head = head * a.group + row - query * a.group;
    const int row_end = row < rows ? end_of(row) : 0, row_begin = row < rows ? begin_of(row) : 0;
    const int wave_row = row0 + wave * 32, wave_last = min(wave_row + 31, rows - 1);
    const bool idle = wave_row >= rows;
    const int wave_to = uniform(idle ? 0 : end_of(wave_last)), wave_from = uniform(idle ? 0 : begin_of(wave_row));
    const int all_to = uniform(idle ? 0 : end_of(wave_row)), all_from = uniform(idle ? 0 : begin_of(wave_last));
    half8_t q[D / 16];
    float scale;
    {
      const T* from = static_cast<const T*>(a.q) + (int64_t)(seq.first + query) * a.q_token + (int64_t)q_head * a.q_head + h * 8;
      float most = 0.0f;
      float x[D / 16][8] = {};
      if (row < rows) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) load_row(x[c], from + c * 16, a.q_wide);
      }
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, __builtin_fabsf(x[c][j]));
      const float up = lift_of(max32(most), a.scale, &scale);
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) q[c][j] = (_Float16)(x[c][j] * up);
    }
    float m = -__builtin_inff(), l[4] = {};  // l: in four strands, so that no addition waits for the last
    float16_t o[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[c][i] = 0.0f;

    // ---- Pages.  A lane holds the number of one sixteen's page, 1024 tokens in a wave; they are asked for tile by
    // tile.  A missing page is -1, its tokens are read from page 0 and masked.
    const int32_t* table = a.block_table + own.seq * a.table_stride;
    constexpr int kSixteens = S::kTokens / 16, kTilesHeld = 64 / kSixteens;
    struct Pages {
      int a, b, c, d;
    };
    int held = -1;
    auto pages_of = [&](int at) {
      if (at % kTilesHeld == 0 || at == tile_from) {
        const int64_t t = ((int64_t)(at / kTilesHeld) * 64 + lane) * 16;
        const int id = t < length && t < (int64_t)tile_to * S::kTokens ? table[t >> a.pages.page_log2] : -1;
        held = id < a.pages.num_pages ? max(id, -1) : -1;  // (used here, so that the wait for it is here too)
      }
      const int i = at % kTilesHeld * kSixteens;
      auto one = [&](int j) { return j < kSixteens ? __builtin_amdgcn_readlane(held, i + j) : -1; };
      return Pages{one(0), one(1), one(2), one(3)};
    };
    auto missing_of = [&](const Pages& p) {  // a bit for each sixteen
      const int first = (p.a < 0 ? 1 : 0) | (p.b < 0 ? 2 : 0);
      return S::kTokens == 32 ? first : first | (p.c < 0 ? 4 : 0) | (p.d < 0 ? 8 : 0);
    };
    auto block_of = [&](int id) { return a.pages.data + ((int64_t)max(id, 0) * heads + head) * a.pages.head_bytes; };
    // Base of the block that holds a thread's sixteen `i` of the tile: the same for all where a page holds the tile.
    auto block_at = [&](const Pages& p, int i) {
      const uint8_t* block = block_of(p.a);
      if (P < S::kTokens) {
        const uint8_t *b = block_of(p.b), *c = block_of(p.c), *d = block_of(p.d);
        block = i == 1 ? b : block;
        block = i == 2 ? c : block;
        block = i == 3 ? d : block;
      }
      return block;
    };

    // ---- this thread's chunks: 32 channels of a token, four tokens of a sixteenth of the channels
    const int key_chunk = threadIdx.x, value_chunk = (int)threadIdx.x - S::kValueThread;
    const bool has_keys = key_chunk < S::kKeyChunks, has_values = value_chunk >= 0;
    const int key_token = key_chunk / (D / 32), key_group = key_chunk % (D / 32);
    // of 32 neighbouring lanes two sixteenths and 16 fours of tokens: their LDS writes cover all banks
    constexpr int kFours = S::kTokens / 4;
    const int sixteenth = (value_chunk & 1) | (value_chunk / (2 * kFours) << 1), four = value_chunk >> 1 & (kFours - 1);
    const int in_page = P - 1, key_at = key_token & in_page, value_at = four * 4 & in_page;
    const int key_offset = L::key(key_at) + key_group * 16, key_scale_offset = L::key_scale(P, key_at, key_group);
    const int value_offset = L::value(P, value_at, sixteenth);
    const int value_scale_offset = L::value_scale(P, value_at, sixteenth * (D / 16) / 32);
    const int key_place = key_token * S::kKeyRow + key_group * 64;
    // fours 0, 1, 2, 3 of 16 tokens lie in the order 0, 2, 1, 3
    const int value_place = sixteenth * (D / 16) * S::kValueRow + ((four & ~3) | (four & 1) << 1 | (four >> 1 & 1)) * 8;

    Fetched<D> next;
    auto fetch_keys = [&](const Pages& p, int at) {
      if (!has_keys) return;
      const uint8_t* block = block_at(p, key_token >> 4);
      const int t = at * S::kTokens & in_page;  // (0 where pages are smaller than the tile)
      load_words(next.keys(), block + (key_offset + t * L::kRow));
      next.first_scale = block[key_scale_offset + t];
    };
    auto fetch_values = [&](const Pages& p, int at, int missing) {
      if (!has_values) return;
      const uint8_t* block = block_at(p, four >> 2);
      const int t0 = at * S::kTokens, t = t0 & in_page;
      load_words(next.values(), block + (value_offset + t * L::kRow));
      next.value_scale() = *reinterpret_cast<const uint32_t*>(block + (value_scale_offset + t));
      // what no row sees may hold anything, and nothing times zero has to be zero
      if (t0 + S::kTokens > length || t0 < some_from || missing) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int token = t0 + four * 4 + j;
          if (token >= length || token < some_from || missing >> (four >> 2) & 1)
            next.value_scale() = (next.value_scale() & ~(255u << (8 * j))) | 127u << (8 * j);
        }
      }
    };
    auto spread_keys = [&](uint8_t* to) {
      if (!has_keys) return;
      const float ks = __uint_as_float(next.first_scale << 23);
#pragma unroll
      for (int w = 0; w < 4; ++w) *reinterpret_cast<half8_t*>(to + key_place + w * 16) = eight_values(next.keys()[w], ks);
    };
    auto spread_values = [&](uint8_t* to) {
      if (!has_values) return;
      // A value that is not a number is kept out of the products, times zero it would not be zero: the sums of the rows
      // that see it get it after the last tile.
      uint32_t& scales = next.value_scale();
      if (((scales & 0x7f7f7f7f) + 0x01010101) & scales & 0x80808080) {
        odd_unit = unit;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if ((scales >> (8 * j) & 255) == 255) scales ^= 128u << (8 * j);
      }
      float vs[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) vs[j] = __uint_as_float((next.value_scale() >> (8 * j) & 255) << 23);
#pragma unroll
      for (int b = 0; b < D / 32; ++b) {  // byte b of each token: two channels
        half2_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int byte = j * (D / 32) + b;
          const uint32_t w = next.values()[byte / 4];
          x[j] = byte % 4 == 0 ? two_values<0>(w, vs[j]) : byte % 4 == 1 ? two_values<1>(w, vs[j])
               : byte % 4 == 2 ? two_values<2>(w, vs[j]) : two_values<3>(w, vs[j]);
        }
        typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int c = 0; c < 2; ++c)
          *reinterpret_cast<half4_t*>(to + value_place + (2 * b + c) * S::kValueRow) = half4_t{x[0][c], x[1][c], x[2][c], x[3][c]};
      }
    };

    // ---- a unit of 32 tokens
    auto key = [&](const uint8_t* keys, int c) {
      return *reinterpret_cast<const half8_t*>(keys + n * S::kKeyRow + h * 16 + c * 32);
    };
    auto scores = [&](float16_t& sc, const uint8_t* keys) {
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[j] = 0.0f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(key(keys, c), q[c], sc, 0, 0, 0);
    };
    auto mask = [&](float16_t& sc, int t0, int missing) {  // missing: of the unit's two sixteens
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int t = t0 + (j / 4) * 8 + h * 4 + j % 4;
        if (t >= row_end || t < row_begin || missing >> (j / 8) & 1) sc[j] = -__builtin_inff();
      }
    };
    // LDS is read kAhead products before the product, the first keys of a unit in the unit before it (two, three or
    // four ahead: the same time; two leave registers).
    constexpr int kProducts = D / 16, kAhead = 2;
    auto value = [&](const uint8_t* values, int z) {
      return *reinterpret_cast<const half8_t*>(values + (z % (D / 32) * 32 + n) * S::kValueRow + h * 16 + z / (D / 32) * 32);
    };
    half8_t ahead[kAhead];
    auto first_keys = [&](const uint8_t* keys) {
#pragma unroll
      for (int z = 0; z < kAhead; ++z) ahead[z] = key(keys, z);
    };
    // The next unit's scores and the present probabilities, product by product: each with its share of the 16
    // exponentials, whose rounding comes one product later.  Returns the largest exponent.
    auto scores_beside_probabilities = [&](float16_t& sc_next, const uint8_t* keys, const uint8_t* values,
                                           half8_t (&p)[2], const float16_t& sc, float add) {
      constexpr int kEach = 16 / kProducts;
#pragma unroll
      for (int j = 0; j < 16; ++j) sc_next[j] = 0.0f;
      float most = -__builtin_inff(), x[16];
#pragma unroll
      for (int z = 0; z <= kProducts; ++z) {
        if (z < kProducts) {
          sc_next = __builtin_amdgcn_mfma_f32_32x32x16_f16(ahead[z % kAhead], q[z], sc_next, 0, 0, 0);
          ahead[z % kAhead] = z + kAhead < kProducts ? key(keys, z + kAhead) : value(values, z + kAhead - kProducts);
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            const float t = __builtin_fmaf(sc[z * kEach + e], scale, add);
            most = fmaxf(most, t);
            x[z * kEach + e] = __builtin_amdgcn_exp2f(t);
          }
        }
        if (z > 0) {
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            const int i = (z - 1) * kEach + e;
            p[i / 8][i % 8] = (_Float16)x[i];
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      return most;
    };
    // The present products with the values, the sums of the probabilities as rounded among them (`one`: as above).
    float one = 1.0f;
    asm volatile("" : "+s"(one));
    auto gather_beside_sums = [&](const half8_t (&p)[2], const uint8_t* values, const uint8_t* keys_after) {
      constexpr int kEach = 16 / kProducts;
#pragma unroll
      for (int z = 0; z < kProducts; ++z) {
        o[z % (D / 32)] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ahead[z % kAhead], p[z / (D / 32)], o[z % (D / 32)], 0, 0, 0);
        ahead[z % kAhead] = z + kAhead < kProducts ? value(values, z + kAhead) : key(keys_after, z + kAhead - kProducts);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int i = z * kEach + e;
          l[i % 4] = __builtin_fmaf((float)p[i / 8][i % 8], one, l[i % 4]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // Of the unit that begins at a token: whether a row of the wave sees some of it, whether all see all of it.
    const int piece_to = tile_to * S::kTokens, see_from = wave_from - 31;
    const uint32_t see_span = max(min(wave_to, piece_to) - see_from, 0);
    const uint32_t all_span = max(min(all_to, piece_to) - 31 - all_from, 0);
    auto sees = [&](int t0) { return (uint32_t)(t0 - see_from) < see_span; };
    auto all_see = [&](int t0, int missing) { return (uint32_t)(t0 - all_from) < all_span && (missing & 3) == 0; };

    // Probabilities are held times 2^(kTileLift - m), where m need not be the maximum so far: it is raised to the
    // maximum where a row sees its first token and where the maximum is kSlack above it (one of kFar and more: in every
    // unit, where the probabilities are computed anew, from scores as far as the base is).
    float add = kTileLift, limit = row < rows ? -__builtin_inff() : __builtin_inff();
    // The unit of tokens t0 .. t0 + 31, whose scores are there; the scores of the next come.
    auto work_on = [&](int t0, float16_t& sc, float16_t& sc_next, const uint8_t* keys_next, const uint8_t* keys_after,
                       const uint8_t* values, int missing_next) {
      const int t1 = t0 + 32;
      const bool mine_next = sees(t1);
      if (!mine_next && !sees(t0)) {
        first_keys(keys_after);
        return;
      }
      half8_t p[2];
      const float most = scores_beside_probabilities(sc_next, keys_next, values, p, sc, add);
      // (the probabilities stay before the branch)
      asm volatile("" : "+v"(p[0]), "+v"(p[1]));
      if (__builtin_amdgcn_ballot_w64(most > limit)) {
        float top = sc[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) top = fmaxf(top, sc[j]);
        const float raised = max32(most) > limit ? fmaxf(m, tile_base_of(max32(top) * scale)) : m;
        const float old = m == raised ? 1.0f : __builtin_amdgcn_exp2f(m - raised);
        m = raised;
        const bool far = is_far(m);
        limit = m == -__builtin_inff() ? limit : far ? -__builtin_inff() : kTileLift + kSlack;
        add = m == -__builtin_inff() ? kTileLift : kTileLift - m;
#pragma unroll
        for (int j = 0; j < 4; ++j) l[j] *= old;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) o[c] *= old;
        if (__builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            p[j / 8][j % 8] = (_Float16)__builtin_amdgcn_exp2f(far ? below(sc[j], scale, m) + kTileLift
                                                                   : __builtin_fmaf(sc[j], scale, add));
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) p[j / 8][j % 8] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(sc[j], scale, add));
        }
      }
      if (!all_see(t1, missing_next)) mask(sc_next, mine_next ? t1 : 1 << 30, missing_next);
      gather_beside_sums(p, values, keys_after);
    };

    // ---- While tile `at` is worked on, its keys and values and the next tile's keys are in LDS.  Keys are laid out
    // two tiles ahead and values one, and fetched one tile before that.
    uint8_t *keys_now = key_buffers[0], *keys_next = key_buffers[1], *keys_later = key_buffers[S::kKeyBuffers - 1];
    float16_t even, odd;
#pragma unroll
    for (int j = 0; j < 16; ++j) even[j] = odd[j] = -__builtin_inff();  // of a unit that the wave does not see
    Pages pages_now = pages_of(tile_from), pages_next = pages_of(tile_from + 1), pages_later = pages_of(tile_from + 2);
    int missing0 = missing_of(pages_now), missing1 = missing_of(pages_next), missing2 = missing_of(pages_later);
    if (tile_from < tile_to) {
      fetch_values(pages_now, tile_from, missing0);
      if constexpr (S::kApart) {
        fetch_keys(pages_now, tile_from);
        spread_keys(keys_now);
        spread_values(value_buffers[0]);
      } else {
        spread_values(value_buffers[0]);
        fetch_keys(pages_now, tile_from);
        spread_keys(keys_now);
      }
      if (tile_from + 1 < tile_to) {
        fetch_keys(pages_next, tile_from + 1);
        spread_keys(keys_next);
        fetch_values(pages_next, tile_from + 1, missing1);
      }
      if (tile_from + 2 < tile_to) fetch_keys(pages_later, tile_from + 2);
      pages_next = pages_later;
      pages_later = pages_of(tile_from + 3);
    }
    lds_barrier();
    if (tile_from < tile_to && sees(tile_from * S::kTokens)) {
      scores(even, keys_now);
      if (!all_see(tile_from * S::kTokens, missing0)) mask(even, tile_from * S::kTokens, missing0);
    }
    // (with two key buffers the first keys are written over from here on)
    if constexpr (S::kKeyBuffers == 2) lds_barrier();
    // Keys of the unit after next, whatever is there where there is none: they are read and not used.
    first_keys(S::kUnits == 2 ? keys_now + 32 * S::kKeyRow : keys_next);
    // (what comes last in a step goes first where both waves of a SIMD unit could: 174.8 us without, 173.2 with it)
    if (S::kApart && wave * 64 >= S::kValueThread) __builtin_amdgcn_s_setprio(1);
    auto advance = [&](int at, float16_t& first, float16_t& second) {
      const int t0 = at * S::kTokens;
      const uint8_t* values = value_buffers[(at - tile_from) & 1];
      auto move_values = [&]() {
        if (at + 1 < tile_to) spread_values(value_buffers[(at - tile_from + 1) & 1]);
        if (at + 2 < tile_to) fetch_values(pages_next, at + 2, missing2);
      };
      // of the two waves of a SIMD unit one lays out values before its products, the other keys after them
      if constexpr (S::kApart) move_values();
      if constexpr (S::kUnits == 2) {
        const uint8_t *second_now = keys_now + 32 * S::kKeyRow, *second_next = keys_next + 32 * S::kKeyRow;
        work_on(t0, first, second, second_now, keys_next, values, missing0 >> 2);
        work_on(t0 + 32, second, first, keys_next, second_next, values + 64, missing1);
      } else {
        // (the keys after next are being written where the present ones were: read behind the barrier)
        work_on(t0, first, second, keys_next, keys_next, values, missing1);
      }
      uint8_t* const write = S::kUnits == 2 ? keys_later : keys_now;
      if (at + 2 < tile_to) spread_keys(write);
      if (at + 3 < tile_to) fetch_keys(pages_later, at + 3);
      if constexpr (!S::kApart) move_values();
      pages_next = pages_later;
      missing0 = missing1;
      missing1 = missing2;
      missing2 = missing_of(pages_later);
      pages_later = pages_of(at + 4);
      keys_later = keys_now;
      keys_now = keys_next;
      keys_next = write;
      lds_barrier();
      if constexpr (S::kUnits == 1) first_keys(keys_next);
    };
    for (int at = tile_from; at < tile_to; at += 3 - S::kUnits) {
      advance(at, even, odd);
      if (S::kUnits == 1 && at + 1 < tile_to) advance(at + 1, odd, even);
    }
    if (S::kApart) __builtin_amdgcn_s_setprio(0);
    if (odd_unit == unit) {
      uint32_t mine = 0;  // a bit for each 32 channels
#pragma unroll 1
      for (int t0 = tile_from * S::kTokens; t0 < tile_to * S::kTokens; t0 += 32) {
        const int t = t0 + n, id = t < length ? table[t >> a.pages.page_log2] : -1;
        const bool there = id >= 0 && id < a.pages.num_pages;
        const uint8_t* scales = block_of(there ? id : 0);
        const int from = min(max(row_begin - t0, 0), 32), to = min(max(row_end - t0, 0), 32);
        const uint32_t seen = from < to ? (uint32_t)(((uint64_t)1 << to) - ((uint64_t)1 << from)) : 0;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const bool odd_one = there && scales[L::value_scale(P, t & in_page, c)] == 255;
          mine |= (uint32_t)__builtin_amdgcn_ballot_w64(odd_one) & seen ? 1u << c : 0;
        }
      }
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (mine >> c & 1) o[c][j] = __builtin_nanf("");
    }
    const Both sums = across32((l[0] + l[1]) + (l[2] + l[3]));
    const float sum = sums.a + sums.b;
    if (row < rows && starts && ends) {
      T* out = static_cast<T*>(a.out) + (int64_t)(seq.first + query) * a.out_token + (int64_t)q_head * a.out_head;
      const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          store4(out + c * 32 + i * 2 + h * 4, float4_t{o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]} * inv, a.out_wide);
    } else if (row < rows) {
      float* part = args.parts + ((int64_t)(2 * blockIdx.x + (starts ? 1 : 0)) * S::kRows + row - row0) * (D + 4);
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4_t*>(part + c * 32 + i * 2 + h * 4) = float4_t{o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]};
      if (h == 0) {
        part[D] = m;
        part[D + 1] = sum;
      }
    }
    lds_barrier();  // (the next tile's keys and values are written over these)
  }
}

// Joins the parts of a tile's rows: a block takes kJoinRows of them, D / 4 lanes a row, and has the first two parts
// of all its rows under way at once.
constexpr int kJoinRows = 32;

template <typename T, int D>
__global__ __launch_bounds__(256) void attention_join_tile_kernel(TileArgs args) {
  using S = TileShape<D>;
  const AttentionArgs& a = args.a;
  const TileHeader header = args.headers[blockIdx.x];
  const int parts = header.last - header.first + 1, row0 = header.row0, head = header.head;
  if (parts == 1) return;
  const Sequence seq = sequence<true>(a, header.seq);
  const int rows = min(seq.count, a.max_queries) * a.group;
  constexpr int kLanes = D / 4, kAtOnce = 256 / kLanes, kTurns = kJoinRows / kAtOnce;
  const int lane = threadIdx.x % kLanes, first = blockIdx.y * kJoinRows + threadIdx.x / kLanes;
  // the second part of the workgroup that begins the tile, the first of those behind it
  auto part = [&](int c, int row) {
    const int place = 2 * (header.first + c) + (c == 0 ? 1 : 0);
    return args.parts + ((int64_t)place * S::kRows + row) * (D + 4);
  };
  float4_t x[kTurns][2];
  float2 ml[kTurns][2];
#pragma unroll
  for (int k = 0; k < kTurns; ++k)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      // (rows behind the last are not written, but they are there)
      const float* p = part(c, first + k * kAtOnce);
      x[k][c] = *reinterpret_cast<const float4_t*>(p + lane * 4);
      ml[k][c] = *reinterpret_cast<const float2*>(p + D);
    }
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    const int in_tile = first + k * kAtOnce, row = row0 + in_tile;
    if (row >= rows) continue;
    float m = fmaxf(ml[k][0].x, ml[k][1].x);
    float w0 = ml[k][0].x == m ? 1.0f : __builtin_amdgcn_exp2f(ml[k][0].x - m);
    float w1 = ml[k][1].x == m ? 1.0f : __builtin_amdgcn_exp2f(ml[k][1].x - m);
    float l = ml[k][0].y * w0 + ml[k][1].y * w1;
    float4_t o = x[k][0] * w0 + x[k][1] * w1;
    for (int c = 2; c < parts; ++c) {
      const float* p = part(c, in_tile);
      const float2 more = *reinterpret_cast<const float2*>(p + D);
      const float higher = fmaxf(m, more.x);
      w0 = m == higher ? 1.0f : __builtin_amdgcn_exp2f(m - higher);
      w1 = more.x == higher ? 1.0f : __builtin_amdgcn_exp2f(more.x - higher);
      m = higher;
      l = l * w0 + more.y * w1;
      o = o * w0 + *reinterpret_cast<const float4_t*>(p + lane * 4) * w1;
    }
    const int query = row / a.group;
    T* out = static_cast<T*>(a.out) + (int64_t)(seq.first + query) * a.out_token +
             (int64_t)(head * a.group + row - query * a.group) * a.out_head + lane * 4;
    store4(out, o * (l > 0.0f || l != l ? 1.0f / l : 0.0f), a.out_wide);
  }
}

// Tiles of a call, and whether they are worked on in even shares: they do not even out among themselves (a prompt's
// tiles reach back differently far, and what is left over of a last round of workgroups counts), and a part more or
// less is little beside a compute unit that waits.  Not where a sequence has room for 256 tokens or less, whose tiles
// about equal and soon done, and not for more tiles than there is LDS for.  In even shares and in a workgroup
// each, 8 heads over one key head, D = 128: a prompt of 8192 tokens 170 and 236 us, eight of them 1094 and 1137, 32 of
// 2048 348 and 461, 64 of 512 93 and 109; 400 of 200 tokens 224 and 198, 500 of 64 72 and 67.
struct TilePlan {
  int tiles, grid;  // grid: of the even shares; 0: none
  int64_t header_bytes, bytes;
};

TilePlan plan_tiles(int64_t T, int group, int kv_heads, int head_size, int64_t num_seqs, int64_t max_queries,
                    int64_t capacity) {
  TilePlan plan;
  const int64_t rows = head_size == 256 ? TileShape<256>::kRows : TileShape<128>::kRows;
  // every sequence may leave one tile that is not full
  const int64_t tiles = min((T * group + rows - 1) / rows + num_seqs, num_seqs * ((max_queries * group + rows - 1) / rows));
  const int cus = device_compute_units();
  plan.tiles = (int)min(tiles, (int64_t)0x7fffffff);
  // (spans are counted in 32 bits)
  const bool few = tiles * kv_heads <= kMostShared && num_seqs <= kMostShared && capacity > 256 &&
                   (double)(tiles * kv_heads) * (double)(capacity / kSpan + 1) < 2e9;
  plan.grid = few ? (cus > 0 ? cus : 256) : 0;
  plan.header_bytes = (tiles * kv_heads * (int64_t)sizeof(TileHeader) + 15) / 16 * 16;
  plan.bytes = plan.grid == 0 ? 0 : plan.header_bytes + 2 * plan.grid * rows * (head_size + 4) * (int64_t)sizeof(float);
  return plan;
}

template <typename T, int D>
int launch_tiles(const TileArgs& args, int grid, void* stream) {
  const unsigned tiles = (unsigned)args.tiles, heads = (unsigned)args.a.pages.heads;
  launch_kernel(attention_tile_kernel<T, D>, grid ? dim3((unsigned)grid) : dim3(tiles, heads), dim3(TileShape<D>::kThreads),
                0, static_cast<hipStream_t>(stream), args);
  int rc = finish_launch("kv4_attention");
  if (rc != TW_OK || grid == 0) return rc;
  launch_kernel(attention_join_tile_kernel<T, D>, dim3(tiles * heads, TileShape<D>::kRows / kJoinRows), dim3(256), 0,
                static_cast<hipStream_t>(stream), args);
  return finish_launch("kv4_attention");
}

template <typename T>
int launch_tiles(const TileArgs& args, int D, int grid, void* stream) {
  if (D == 64) return launch_tiles<T, 64>(args, grid, stream);
  if (D == 128) return launch_tiles<T, 128>(args, grid, stream);
  return launch_tiles<T, 256>(args, grid, stream);
}

// A call without a new token of any sequence: all tokens are padding.
template <typename T, int D>
__global__ __launch_bounds__(kJoinThreads) void attention_clear_kernel(AttentionArgs a) {
  clear_rest<T, D, kJoinThreads>(a);
}

template <typename T>
int launch_clear(const AttentionArgs& a, int D, void* stream) {
  const int64_t items = (int64_t)a.num_tokens * a.pages.heads * a.group * (D / 4);
  const unsigned grid = (unsigned)min((items + kJoinThreads - 1) / kJoinThreads, (int64_t)2048);
  launch_kernel(D == 64 ? attention_clear_kernel<T, 64> : D == 128 ? attention_clear_kernel<T, 128> : attention_clear_kernel<T, 256>,
                dim3(grid), dim3(kJoinThreads), 0, static_cast<hipStream_t>(stream), a);
  return finish_launch("kv4_attention");
}

bool wide_rows(const tw_heads* h) {
  return reinterpret_cast<uintptr_t>(h->data) % 16 == 0 && h->token_stride % 8 == 0 && h->head_stride % 8 == 0;
}

}  // namespace

int64_t kv4_attention_workspace(int q_heads, int kv_heads, int head_size, int64_t num_seqs, int64_t num_tokens,
                                int64_t max_queries, int64_t table_width, int page_size) {
  if (q_heads < 1 || kv_heads < 1 || num_seqs < 1 || num_tokens < 1 || max_queries < 1) return 0;
  const int group = q_heads / kv_heads;
  max_queries = min(max_queries, num_tokens);
  if (max_queries * group <= kMostRows)
    return plan_split(num_seqs, kv_heads, table_width, page_size, (int)max_queries * group, head_size).bytes;
  return plan_tiles(num_tokens, group, kv_heads, head_size, num_seqs, max_queries, table_width * page_size).bytes;
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
  const bool nothing = num_seqs == 0 || max_queries == 0;
  if (T == 0 || (nothing && !query_starts)) return TW_OK;
  AttentionArgs a{};
  if (int rc = check_kv4_pages(what, pages, num_pages, page_size, kv_heads, head_size, &a.pages)) return rc;
  if (!out || !q || !out->data || !q->data) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: out or q is null", what);
  if (q->heads < 1 || q->heads % kv_heads != 0 || q->heads > 65535)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: %lld query heads over %d key heads", what, (long long)q->heads, kv_heads);
  if (out->heads != q->heads) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: out and q have different heads", what);
  if (out->token_stride < 0 || out->head_stride < 0 || q->token_stride < 0 || q->head_stride < 0)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: a stride is negative", what);
  if (int rc = check_rows_apart(what, "out", out, T, head_size)) return rc;
  if (!nothing && (!seq_lens || (!block_table && table_width > 0)))
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: block_table or seq_lens is null", what);
  if (table_width > ((int64_t)1 << 30) / page_size)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: block_table has room for more than 2^30 tokens", what);
  if (num_seqs > 65535 || T > (1 << 30))
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: more than 65535 sequences or 2^30 tokens", what);
  if (!query_starts && T % num_seqs != 0)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: %lld tokens are not the same number for each of %lld sequences", what,
                     (long long)T, (long long)num_seqs);
  const int64_t need = nothing ? 0 : kv4_attention_workspace((int)q->heads, kv_heads, head_size, num_seqs, T, max_queries,
                                               table_width, page_size);
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
  a.capacity = (int)(table_width * page_size);
  a.seq_lens = seq_lens;
  a.query_starts = query_starts;
  a.per_seq = query_starts ? 0 : (int)(T / num_seqs);
  a.num_seqs = (int)num_seqs;
  a.num_tokens = (int)T;
  a.max_queries = (int)min(max_queries, T);
  a.scale = scale * kLog2e;
  a.window = (int)min(window, (int64_t)1 << 30);
  a.q_wide = wide_rows(q);
  a.out_wide = wide_rows(out);
  if (nothing) return dtype == TW_DTYPE_BF16 ? launch_clear<__bf16>(a, head_size, stream) : launch_clear<_Float16>(a, head_size, stream);
  max_queries = a.max_queries;
  if (max_queries * a.group <= kMostRows) {
    // steps are counted in 32 bits
    if ((double)num_seqs * kv_heads * (double)((table_width * page_size + kStep - 1) / kStep + 1) > 2e9)
      return set_error(TW_ERR_INVALID_ARGUMENT, "%s: the sequences have room for too many tokens", what);
    const int rows = (int)(max_queries * a.group);
    const SplitPlan plan = plan_split(num_seqs, kv_heads, table_width, page_size, rows, head_size);
    const SplitArgs args{a, static_cast<PieceHeader*>(workspace),
                         reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.header_bytes), rows, plan.budget,
                         65536 / a.group + 1};
    return dtype == TW_DTYPE_BF16 ? launch_split<__bf16>(args, head_size, plan.grid, stream)
                                  : launch_split<_Float16>(args, head_size, plan.grid, stream);
  }
  const TilePlan plan = plan_tiles(T, a.group, kv_heads, head_size, num_seqs, max_queries, a.capacity);
  if ((double)T * a.group + (double)num_seqs * 256 > 2e9 || kv_heads > 65535)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: too many rows", what);
  TileArgs args{a, nullptr, nullptr, plan.tiles};
  if (plan.grid > 0) {
    args.headers = static_cast<TileHeader*>(workspace);
    args.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.header_bytes);
  }
  return dtype == TW_DTYPE_BF16 ? launch_tiles<__bf16>(args, head_size, plan.grid, stream)
                                : launch_tiles<_Float16>(args, head_size, plan.grid, stream);
}

}  // namespace tw
