// Rotation of queries and keys by their positions, and the writer and reader of the 4-bit
// paged cache (tw_kv4.h), for gfx950 (wave64).
//
// All are memory-bound: 16 bytes of table, 32 bytes in and 32 out for 16 channels and some ten
// operations on them.  What is turned is read once and written once; a token's cosines and
// sines are read by all its heads from the caches.
//   16384 tokens of 64 + 8 heads of 128, bf16, 612 MB: 115 us = 5.3 TB/s (a large copy: 5.16);
//   8192 tokens, 64 query heads turned, 8 key heads turned and written with their values,
//   310 MB: 75 us = 4.1 TB/s (16 bytes a thread come in and 4.25 go out, and the maximum of 32
//   channels goes through four lanes), read back, 42 MB: 13.5 us.
// A column of a head a thread: 16 channels, so that every access is 16 bytes wide in 16-bit
// types.  Where alignment or sizes forbid it, one pair: 8192 tokens of 64 + 8 heads then take 150
// us instead of 64, and 8 heads' keys and values on their way into the cache 35 instead of 16.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tw_common.h"
#include "tw_kv4.h"

namespace tw {

namespace {

struct Heads {
  void* data;
  int64_t token_stride, head_stride;
};

struct Rotary {
  const int64_t* positions;
  const float* cos_sin;
  int64_t max_positions;
  int dim;          // channels that are turned
  bool interleaved;
  bool inverse;
};

template <typename T, int W>
struct __align__(sizeof(T) * W) Vec {
  T v[W];
};

template <typename T, int W>
__device__ __forceinline__ void load(float (&f)[W], const T* p) {
  const Vec<T, W> x = *reinterpret_cast<const Vec<T, W>*>(p);
#pragma unroll
  for (int i = 0; i < W; ++i) f[i] = (float)x.v[i];
}

template <typename T, int W>
__device__ __forceinline__ void store(T* p, const float (&f)[W]) {
  Vec<T, W> x;
#pragma unroll
  for (int i = 0; i < W; ++i) x.v[i] = (T)f[i];
  *reinterpret_cast<Vec<T, W>*>(p) = x;
}

// Turns one pair.  Products and sum are rounded one by one: a key coded on its way into the cache
// has the same bits wherever it is computed.
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
#pragma clang fp contract(off)
  const float x = a * c - b * s;
  const float y = b * c + a * s;
  a = x;
  b = y;
}

// cos and sin of W pairs from `pair` on of a token; NaN for a position that the table does not have.
template <int W>
__device__ __forceinline__ void table_row(float (&c)[W], float (&s)[W], const Rotary& r, int64_t position, int pair) {
  if (position >= 0 && position < r.max_positions) {
    const float* row = r.cos_sin + position * r.dim;
    if constexpr (W == 1) {
      c[0] = row[pair];
      s[0] = row[pair + (r.dim >> 1)];
    } else {
      load(c, row + pair);
      load(s, row + pair + (r.dim >> 1));
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) c[i] = s[i] = __builtin_nanf("");
  }
  if (r.inverse) {
#pragma unroll
    for (int i = 0; i < W; ++i) s[i] = -s[i];
  }
}

// One column of a head: 2W channels, W pairs or, behind the turned ones, channels to be copied.
template <typename T, int W>
__device__ __forceinline__ void rotate_column(T* out, const T* in, const Rotary& r, int64_t position, int column,
                                              int head_size) {
  const int turned = r.dim / (2 * W);
  float a[W], b[W];
  if (column < turned) {
    const int at_a = r.interleaved ? column * 2 * W : column * W;
    const int at_b = r.interleaved ? at_a + W : at_a + (r.dim >> 1);
    float c[W], s[W];
    load(a, in + at_a);
    load(b, in + at_b);
    table_row(c, s, r, position, column * W);
    if (r.interleaved) {
      if constexpr (W == 1) {
        turn(a[0], b[0], c[0], s[0]);
      } else {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          turn(a[2 * i], a[2 * i + 1], c[i], s[i]);
          turn(b[2 * i], b[2 * i + 1], c[W / 2 + i], s[W / 2 + i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) turn(a[i], b[i], c[i], s[i]);
    }
    store(out + at_a, a);
    store(out + at_b, b);
  } else if (out != in) {
    const int at = r.dim + (column - turned) * 2 * W;
    load(a, in + at);
    store(out + at, a);
    if (W > 1 || at + 1 < head_size) {
      load(b, in + at + W);
      store(out + at + W, b);
    }
  }
}

// Queries and keys as one row of heads per token.  A thread takes one column of one head.
struct RotaryArgs {
  Heads q_out, q, k_out, k;
  int q_heads, heads;  // heads: of both
  int columns;         // of a head
  int head_size;
  int64_t items;       // tokens * heads * columns
  Rotary r;
};

template <typename T, int W>
__device__ __forceinline__ void rotary_item(const RotaryArgs& a, int64_t item) {
  int64_t token;
  int head, column;
  if (a.items <= 0x7fffffff) {  // (a division of 64 bits takes longer than the rest)
    const uint32_t row = (uint32_t)item / (uint32_t)a.columns;
    column = (int)((uint32_t)item - row * (uint32_t)a.columns);
    token = row / (uint32_t)a.heads;
    head = (int)(row - (uint32_t)token * (uint32_t)a.heads);
  } else {
    const int64_t row = item / a.columns;
    column = (int)(item - row * a.columns);
    token = row / a.heads;
    head = (int)(row - token * a.heads);
  }
  const bool is_q = head < a.q_heads;
  const Heads& in = is_q ? a.q : a.k;
  const Heads& out = is_q ? a.q_out : a.k_out;
  const int h = is_q ? head : head - a.q_heads;
  rotate_column<T, W>(static_cast<T*>(out.data) + token * out.token_stride + h * out.head_stride,
                      static_cast<const T*>(in.data) + token * in.token_stride + h * in.head_stride, a.r,
                      a.r.positions[token], column, a.head_size);
}

constexpr int kThreads = 256;

template <typename T, int W>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (item < a.items) rotary_item<T, W>(a, item);
}

// ---------------------------------------------------------------------------
// the cache's writer
// ---------------------------------------------------------------------------
struct AppendArgs {
  Kv4Pages pages;
  Heads k, v;
  const int64_t* slots;
  int64_t tokens;
  int blocks;      // of one head's keys or values: tokens * D/8 threads
  int kv_blocks;   // of all heads' keys and values
  bool turned;
  Rotary r;
  RotaryArgs q;    // the queries (no keys); items = 0: none
};

// Codes of 8 values of a block of 32 whose other 24 are in the three neighbouring lanes.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], uint32_t* scale) {
  uint32_t most = 0;  // magnitudes compare as integers, and a NaN is above them all
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
  most = max(most, (uint32_t)__shfl_xor((int)most, 1));
  most = max(most, (uint32_t)__shfl_xor((int)most, 2));
  // the exponent of most / 7, rounded up: 7 = 1.75 * 2^2
  const int e = min(max((int)((most + 0x1fffffu) >> 23) - 129, kMinExponent), kMaxExponent);
  *scale = most >= 0x7f800000u ? kNanScale : (uint32_t)(e + 127);
  // two values an instruction: the nearest magnitude, ties to the even code, no further than the largest
  const float size = __uint_as_float((uint32_t)(e + 127) << 23);
  uint32_t word = 0;
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[0], x[1], size, 0);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[2], x[3], size, 1);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[4], x[5], size, 2);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, x[6], x[7], size, 3);
  return word;
}

// The value of channel `ch` after the turn, from its own and its partner's.
template <typename T>
__device__ __forceinline__ float turned_one(const T* in, const Rotary& r, int64_t position, int ch) {
  const int half = r.dim >> 1;
  const bool second = r.interleaved ? (ch & 1) : ch >= half;
  const int pair = r.interleaved ? ch >> 1 : (second ? ch - half : ch);
  const int other = r.interleaved ? ch ^ 1 : (second ? ch - half : ch + half);
  float c[1], s[1], a = (float)in[ch], b = (float)in[other];
  table_row(c, s, r, position, pair);
  if (second) {
    turn(b, a, c[0], s[0]);
  } else {
    turn(a, b, c[0], s[0]);
  }
  return a;
}

// 8 turned channels from `ch` on, rounded to T.
template <typename T, bool VEC>
__device__ __forceinline__ void turned8(float (&x)[8], const T* in, const Rotary& r, int64_t position, int ch) {
  if (ch >= r.dim) {
    if constexpr (VEC) {
      load(x, in + ch);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)in[ch + i];
    }
    return;
  }
  if constexpr (VEC) {
    load(x, in + ch);
    if (r.interleaved) {
      float c[4], s[4];
      table_row(c, s, r, position, ch >> 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) turn(x[2 * i], x[2 * i + 1], c[i], s[i]);
    } else {
      const int half = r.dim >> 1;
      const bool second = ch >= half;
      float c[8], s[8], y[8];
      load(y, in + (second ? ch - half : ch + half));
      table_row(c, s, r, position, second ? ch - half : ch);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (second) {
          turn(y[i], x[i], c[i], s[i]);
        } else {
          turn(x[i], y[i], c[i], s[i]);
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ch + i < r.dim ? turned_one(in, r, position, ch + i) : (float)in[ch + i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)(T)x[i];
}

template <int D>
__device__ __forceinline__ uint8_t* head_of(const Kv4Pages& p, int64_t slot, int head, int* t) {
  *t = (int)slot & ((1 << p.page_log2) - 1);
  return p.data + ((slot >> p.page_log2) * p.heads + head) * p.head_bytes;
}

__device__ __forceinline__ bool inside(const Kv4Pages& p, int64_t slot) {
  return slot >= 0 && (slot >> p.page_log2) < p.num_pages;
}

// D / 8 threads code a head's keys or values of one token, 8 channels each.  Neighbouring rows are
// neighbouring tokens of one head, whose bytes are neighbours in a page.
template <typename T, int D, bool VEC, int WQ>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
  if ((int)blockIdx.x >= a.kv_blocks) {
    const int64_t item = (int64_t)((int)blockIdx.x - a.kv_blocks) * kThreads + threadIdx.x;
    if (item < a.q.items) rotary_item<T, WQ>(a.q, item);
    return;
  }
  constexpr int kLanes = D / 8;
  const int which = (int)blockIdx.x / a.blocks;  // keys of all heads, then values of all heads
  const int64_t item = (int64_t)((int)blockIdx.x - which * a.blocks) * kThreads + threadIdx.x;
  const int part = (int)item & (kLanes - 1), ch = part * 8;
  const int64_t token = item / kLanes;
  const bool is_key = which < a.pages.heads;
  const int head = is_key ? which : which - a.pages.heads;
  // whole rows end together: the lanes of a block of 32 stay together
  if (token >= a.tokens) return;
  const int64_t slot = a.slots[token];
  if (!inside(a.pages, slot)) return;
  const Heads& h = is_key ? a.k : a.v;
  const T* in = static_cast<const T*>(h.data) + token * h.token_stride + head * h.head_stride;
  float x[8];
  if (is_key && a.turned) {
    turned8<T, VEC>(x, in, a.r, a.r.positions[token], ch);
  } else if constexpr (VEC) {
    load(x, in + ch);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)in[ch + i];
  }
  uint32_t scale;
  const uint32_t word = encode8(x, &scale);
  using L = Kv4<D>;
  const int P = 1 << a.pages.page_log2;
  int t;
  uint8_t* at = head_of<D>(a.pages, slot, head, &t);
  if (is_key) {
    *reinterpret_cast<uint32_t*>(at + L::key(t) + part * 4) = word;
  } else if constexpr (D == 64) {  // 8 channels are two sixteenths
    *reinterpret_cast<uint16_t*>(at + L::value(P, t, 2 * part)) = (uint16_t)word;
    *reinterpret_cast<uint16_t*>(at + L::value(P, t, 2 * part + 1)) = (uint16_t)(word >> 16);
  } else {
    constexpr int kWords = D / 128;
    *reinterpret_cast<uint32_t*>(at + L::value(P, t, part / kWords) + part % kWords * 4) = word;
  }
  if ((part & 3) == 0)
    at[is_key ? L::key_scale(P, t, part >> 2) : L::value_scale(P, t, part >> 2)] = (uint8_t)scale;
}

template <int I>
__device__ __forceinline__ void pair_of(float (&x)[8], uint32_t word, float scale) {
  typedef float float2_t __attribute__((ext_vector_type(2)));
  const float2_t v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, I);
  x[2 * I] = v[0];
  x[2 * I + 1] = v[1];
}

struct ReadArgs {
  Kv4Pages pages;
  Heads k, v;
  const int64_t* slots;
  int64_t tokens;
  int blocks;  // of one head's keys or values
};

template <typename T, int D, bool VEC>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a) {
  constexpr int kLanes = D / 8;
  const int which = (int)blockIdx.x / a.blocks;
  const int64_t item = (int64_t)((int)blockIdx.x - which * a.blocks) * kThreads + threadIdx.x;
  const int part = (int)item & (kLanes - 1);
  const int64_t token = item / kLanes;
  if (token >= a.tokens) return;
  const bool is_key = which < a.pages.heads;
  const int head = is_key ? which : which - a.pages.heads;
  const int64_t slot = a.slots[token];
  uint32_t word = 0;
  float scale = 1.0f;
  if (inside(a.pages, slot)) {
    using L = Kv4<D>;
    const int P = 1 << a.pages.page_log2;
    int t;
    const uint8_t* at = head_of<D>(a.pages, slot, head, &t);
    if (is_key) {
      word = *reinterpret_cast<const uint32_t*>(at + L::key(t) + part * 4);
    } else if constexpr (D == 64) {
      word = *reinterpret_cast<const uint16_t*>(at + L::value(P, t, 2 * part)) |
             (uint32_t) * reinterpret_cast<const uint16_t*>(at + L::value(P, t, 2 * part + 1)) << 16;
    } else {
      constexpr int kWords = D / 128;
      word = *reinterpret_cast<const uint32_t*>(at + L::value(P, t, part / kWords) + part % kWords * 4);
    }
    // (255 is infinity's exponent, and what is scaled by it is no number)
    scale = __uint_as_float((uint32_t)at[is_key ? L::key_scale(P, t, part >> 2) : L::value_scale(P, t, part >> 2)] << 23);
  }
  float x[8];
  pair_of<0>(x, word, scale);
  pair_of<1>(x, word, scale);
  pair_of<2>(x, word, scale);
  pair_of<3>(x, word, scale);
  const Heads& h = is_key ? a.k : a.v;
  T* out = static_cast<T*>(h.data) + token * h.token_stride + head * h.head_stride + part * 8;
  if constexpr (VEC) {
    store(out, x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = (T)x[i];
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
Heads heads_of(const tw_heads* h) {
  return h ? Heads{h->data, h->token_stride, h->head_stride} : Heads{nullptr, 0, 0};
}

// Whether 16 bytes (8 values of 16 bits, two halves of 8 of 32) may be moved at once anywhere.
bool vector_ok(const tw_heads* h, int bytes) {
  return !h || (reinterpret_cast<uintptr_t>(h->data) % 16 == 0 && h->token_stride * bytes % 16 == 0 &&
                h->head_stride * bytes % 16 == 0);
}

int check_heads(const char* what, const char* name, const tw_heads* h) {
  if (!h || !h->data) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: %s is null", what, name);
  if (h->heads < 1 || h->heads > (1 << 20))
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: %s has %lld heads", what, name, (long long)h->heads);
  if (h->token_stride < 0 || h->head_stride < 0)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: %s has a negative stride", what, name);
  return TW_OK;
}

int check_out_heads(const char* what, const char* name, const tw_heads* h, int64_t T, int head_size) {
  const int rc = check_heads(what, name, h);
  return rc ? rc : check_rows_apart(what, name, h, T, head_size);
}

int check_dtype(const char* what, int dtype) {
  if (dtype != TW_DTYPE_BF16 && dtype != TW_DTYPE_F16 && dtype != TW_DTYPE_F32)
    return set_error(TW_ERR_DTYPE, "%s: unknown dtype %d", what, dtype);
  return TW_OK;
}

int check_rotary(const char* what, const int64_t* positions, const float* cos_sin, int64_t max_positions, int head_size,
                 int rotary_dim, int flags) {
  if (!positions || !cos_sin) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: positions or cos_sin is null", what);
  if (max_positions < 1) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: a table of %lld positions", what, (long long)max_positions);
  if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_size)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: rotary_dim %d, must be even and in [2, head_size %d]", what, rotary_dim,
                     head_size);
  if (flags & ~(TW_ROTARY_INTERLEAVED | TW_ROTARY_INVERSE))
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: unknown flags %d", what, flags);
  if (reinterpret_cast<uintptr_t>(cos_sin) % 4 != 0)
    return set_error(TW_ERR_ALIGNMENT, "%s: cos_sin must be 4-byte aligned", what);
  return TW_OK;
}

int grid_of(const char* what, int64_t items, int64_t* blocks) {
  *blocks = (items + kThreads - 1) / kThreads;
  if (*blocks > 0x7fffffff) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: too many tokens", what);
  return TW_OK;
}

// Columns of 2W channels: whole ones for the turned channels and for the rest.
int columns_of(int head_size, int dim, int w) { return dim / (2 * w) + (head_size - dim + 2 * w - 1) / (2 * w); }

bool wide_columns(int head_size, int dim, const float* cos_sin) {
  return dim % 16 == 0 && head_size % 16 == 0 && reinterpret_cast<uintptr_t>(cos_sin) % 16 == 0;
}

template <template <typename> class F, typename... A>
int by_dtype(int dtype, A&&... a) {
  if (dtype == TW_DTYPE_BF16) return F<__bf16>::run(a...);
  if (dtype == TW_DTYPE_F16) return F<_Float16>::run(a...);
  return F<float>::run(a...);
}

template <typename T>
struct RunRotary {
  static int run(const RotaryArgs& a, bool vec, int64_t blocks, void* stream) {
    launch_kernel(vec ? rotary_kernel<T, 8> : rotary_kernel<T, 1>, dim3((unsigned)blocks), dim3(kThreads), 0,
                  static_cast<hipStream_t>(stream), a);
    return finish_launch("rotary_positions");
  }
};

template <typename T>
struct RunAppend {
  template <int D>
  static int with(const AppendArgs& a, bool vec, bool q_vec, int64_t blocks, void* stream) {
    auto kernel = vec ? (q_vec ? append_kernel<T, D, true, 8> : append_kernel<T, D, true, 1>)
                      : (q_vec ? append_kernel<T, D, false, 8> : append_kernel<T, D, false, 1>);
    launch_kernel(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
    return finish_launch("kv4_append");
  }
  static int run(const AppendArgs& a, int D, bool vec, bool q_vec, int64_t blocks, void* stream) {
    if (D == 64) return with<64>(a, vec, q_vec, blocks, stream);
    if (D == 128) return with<128>(a, vec, q_vec, blocks, stream);
    return with<256>(a, vec, q_vec, blocks, stream);
  }
};

template <typename T>
struct RunRead {
  template <int D>
  static int with(const ReadArgs& a, bool vec, int64_t blocks, void* stream) {
    launch_kernel(vec ? read_kernel<T, D, true> : read_kernel<T, D, false>, dim3((unsigned)blocks), dim3(kThreads), 0,
                  static_cast<hipStream_t>(stream), a);
    return finish_launch("kv4_read");
  }
  static int run(const ReadArgs& a, int D, bool vec, int64_t blocks, void* stream) {
    if (D == 64) return with<64>(a, vec, blocks, stream);
    if (D == 128) return with<128>(a, vec, blocks, stream);
    return with<256>(a, vec, blocks, stream);
  }
};

int bytes_of(int dtype) { return dtype == TW_DTYPE_F32 ? 4 : 2; }

}  // namespace

int check_rows_apart(const char* what, const char* name, const tw_heads* h, int64_t T, int head_size) {
  typedef __int128 wide;  // (strides are the caller's)
  const wide a = h->token_stride, b = h->head_stride, D = head_size, tokens = T - 1, heads = h->heads - 1;
  bool apart = (tokens == 0 || a >= D) && (heads == 0 || b >= D);
  // neither a token's heads within a token's stride nor a head's tokens within a head's: head by head, the nearest tokens
  if (apart && tokens > 0 && heads > 0 && heads * b + D > a && tokens * a + D > b) {
    for (wide x = b; x <= heads * b && apart; x += b) {
      const wide k = x / a;
      apart = (k > tokens || x - k * a >= D) && (k + 1 > tokens || (k + 1) * a - x >= D);
    }
  }
  if (!apart)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: rows of %s share memory: %lld tokens, stride %lld, %lld heads, stride %lld",
                     what, name, (long long)T, (long long)h->token_stride, (long long)h->heads, (long long)h->head_stride);
  return TW_OK;
}

int check_kv4_pages(const char* what, const void* pages, int64_t num_pages, int page_size, int64_t heads, int head_size,
                    Kv4Pages* out) {
  if (head_size != 64 && head_size != 128 && head_size != 256)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: head_size %d, must be 64, 128 or 256", what, head_size);
  if (page_size < TW_KV4_MIN_PAGE || page_size > TW_KV4_MAX_PAGE || (page_size & (page_size - 1)))
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: page_size %d, must be a power of two in [%d, %d]", what, page_size,
                     TW_KV4_MIN_PAGE, TW_KV4_MAX_PAGE);
  if (!pages || num_pages < 1) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: the cache has no pages", what);
  if (heads < 1 || heads > (1 << 20)) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: the cache has %lld heads", what, (long long)heads);
  if (reinterpret_cast<uintptr_t>(pages) % 16 != 0)
    return set_error(TW_ERR_ALIGNMENT, "%s: the pages must be 16-byte aligned", what);
  *out = Kv4Pages{static_cast<uint8_t*>(const_cast<void*>(pages)), num_pages, __builtin_ctz(page_size), (int)heads,
                  (int64_t)page_size * (head_size + head_size / 16)};
  return TW_OK;
}

int run_rotary_positions(const tw_heads* q_out, const tw_heads* q, const tw_heads* k_out, const tw_heads* k,
                         const int64_t* positions, const float* cos_sin, int64_t max_positions, int64_t T, int head_size,
                         int rotary_dim, int flags, int dtype, void* stream) {
  const char* what = "rotary_positions";
  if (T < 0 || head_size < 1) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: bad num_tokens or head_size", what);
  if (int rc = check_dtype(what, dtype)) return rc;
  if (T == 0) return TW_OK;
  if (int rc = check_rotary(what, positions, cos_sin, max_positions, head_size, rotary_dim, flags)) return rc;
  if (int rc = check_heads(what, "q", q)) return rc;
  if (int rc = check_out_heads(what, "q_out", q_out, T, head_size)) return rc;
  if (!k != !k_out) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: k and k_out must both be given or both be null", what);
  if (k) {
    if (int rc = check_heads(what, "k", k)) return rc;
    if (int rc = check_out_heads(what, "k_out", k_out, T, head_size)) return rc;
  }
  if (q_out->heads != q->heads || (k && k_out->heads != k->heads))
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: input and output have different heads", what);
  const int size = bytes_of(dtype);
  const bool vec = wide_columns(head_size, rotary_dim, cos_sin) && vector_ok(q, size) && vector_ok(q_out, size) &&
                   vector_ok(k, size) && vector_ok(k_out, size);
  RotaryArgs a{heads_of(q_out), heads_of(q), heads_of(k_out), heads_of(k), (int)q->heads,
               (int)(q->heads + (k ? k->heads : 0)), columns_of(head_size, rotary_dim, vec ? 8 : 1), head_size, 0,
               Rotary{positions, cos_sin, max_positions, rotary_dim, (flags & TW_ROTARY_INTERLEAVED) != 0,
                      (flags & TW_ROTARY_INVERSE) != 0}};
  a.items = T * a.heads * a.columns;
  int64_t blocks;
  if (int rc = grid_of(what, a.items, &blocks)) return rc;
  return by_dtype<RunRotary>(dtype, a, vec, blocks, stream);
}

int run_kv4_append(void* pages, int64_t num_pages, int page_size, const tw_heads* k, const tw_heads* v,
                   const int64_t* slots, const tw_heads* q_out, const tw_heads* q, const int64_t* positions,
                   const float* cos_sin, int64_t max_positions, int64_t T, int head_size, int rotary_dim, int flags,
                   int dtype, void* stream) {
  const char* what = "kv4_append";
  if (T < 0) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: bad num_tokens", what);
  if (int rc = check_dtype(what, dtype)) return rc;
  if (T == 0) return TW_OK;
  if (int rc = check_heads(what, "k", k)) return rc;
  if (int rc = check_heads(what, "v", v)) return rc;
  if (k->heads != v->heads) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: k and v have different heads", what);
  AppendArgs a{};
  if (int rc = check_kv4_pages(what, pages, num_pages, page_size, k->heads, head_size, &a.pages)) return rc;
  if (!slots) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: slots is null", what);
  a.turned = cos_sin != nullptr;
  if (a.turned) {
    if (int rc = check_rotary(what, positions, cos_sin, max_positions, head_size, rotary_dim, flags)) return rc;
  }
  if (!q != !q_out || (q && !a.turned))
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: q and q_out must both be given, with cos_sin, or both be null", what);
  const int size = bytes_of(dtype);
  a.k = heads_of(k);
  a.v = heads_of(v);
  a.slots = slots;
  a.tokens = T;
  a.r = Rotary{positions, cos_sin, max_positions, rotary_dim, (flags & TW_ROTARY_INTERLEAVED) != 0,
               (flags & TW_ROTARY_INVERSE) != 0};
  const bool wide = a.turned && wide_columns(head_size, rotary_dim, cos_sin);
  const bool vec = (!a.turned || wide) && vector_ok(k, size) && vector_ok(v, size);
  bool q_vec = false;
  if (q) {
    if (int rc = check_heads(what, "q", q)) return rc;
    if (int rc = check_out_heads(what, "q_out", q_out, T, head_size)) return rc;
    if (q->heads != q_out->heads) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: q and q_out have different heads", what);
    q_vec = wide && vector_ok(q, size) && vector_ok(q_out, size);
    a.q = RotaryArgs{heads_of(q_out), heads_of(q), Heads{}, Heads{}, (int)q->heads, (int)q->heads,
                     columns_of(head_size, rotary_dim, q_vec ? 8 : 1), head_size, 0, a.r};
    a.q.items = T * a.q.heads * a.q.columns;
  }
  int64_t kv_blocks, q_blocks;
  if (int rc = grid_of(what, T * (head_size / 8), &kv_blocks)) return rc;
  if (int rc = grid_of(what, a.q.items, &q_blocks)) return rc;
  a.blocks = (int)kv_blocks;
  kv_blocks *= 2 * k->heads;
  if (kv_blocks + q_blocks > 0x7fffffff) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: too many tokens", what);
  a.kv_blocks = (int)kv_blocks;
  return by_dtype<RunAppend>(dtype, a, head_size, vec, q_vec, kv_blocks + q_blocks, stream);
}

int run_kv4_read(const tw_heads* k_out, const tw_heads* v_out, const void* pages, int64_t num_pages, int page_size,
                 const int64_t* slots, int64_t T, int head_size, int dtype, void* stream) {
  const char* what = "kv4_read";
  if (T < 0) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: bad num_tokens", what);
  if (int rc = check_dtype(what, dtype)) return rc;
  if (T == 0) return TW_OK;
  if (int rc = check_out_heads(what, "k_out", k_out, T, head_size)) return rc;
  if (int rc = check_out_heads(what, "v_out", v_out, T, head_size)) return rc;
  if (k_out->heads != v_out->heads) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: k_out and v_out have different heads", what);
  ReadArgs a{};
  if (int rc = check_kv4_pages(what, pages, num_pages, page_size, k_out->heads, head_size, &a.pages)) return rc;
  if (!slots) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: slots is null", what);
  a.k = heads_of(k_out);
  a.v = heads_of(v_out);
  a.slots = slots;
  a.tokens = T;
  int64_t blocks;
  if (int rc = grid_of(what, T * (head_size / 8), &blocks)) return rc;
  a.blocks = (int)blocks;
  blocks *= 2 * k_out->heads;
  if (blocks > 0x7fffffff) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: too many tokens", what);
  const bool vec = vector_ok(k_out, bytes_of(dtype)) && vector_ok(v_out, bytes_of(dtype));
  return by_dtype<RunRead>(dtype, a, head_size, vec, blocks, stream);
}

}  // namespace tw
