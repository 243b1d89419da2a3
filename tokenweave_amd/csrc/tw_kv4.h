// The paged 4-bit cache: where a token's bytes are, and the four-bit values.  Shared by the
// kernels that write it (tw_rotary.hip) and read it (tw_attention.hip).
#ifndef TW_KV4_H
#define TW_KV4_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tw {

// Pages of one call.  A (page, head) block holds keys, values, scales of the keys, scales of the
// values, each part of P tokens (P a power of two).
struct Kv4Pages {
  uint8_t* data;
  int64_t num_pages;
  int page_log2;
  int heads;
  int64_t head_bytes;  // of one head in one page: P * (D + D/16)
};

template <int D>
struct Kv4 {
  static constexpr int kRow = D / 2;         // bytes of a token's codes
  static constexpr int kGroups = D / 32;     // scales of a token
  static constexpr int kChunk = D / 32;      // bytes of a sixteenth of the channels of one token
  static __device__ __forceinline__ int key(int t) { return t * kRow; }
  // Four tokens side by side for each sixteenth of the channels: a lane that multiplies values
  // needs several tokens of the same few channels, and gets four of them in one load.
  static __device__ __forceinline__ int value(int P, int t, int sixteenth) {
    return P * kRow + (t >> 2) * (4 * kRow) + sixteenth * (4 * kChunk) + (t & 3) * kChunk;
  }
  static __device__ __forceinline__ int key_scale(int P, int t, int group) { return 2 * P * kRow + group * P + t; }
  static __device__ __forceinline__ int value_scale(int P, int t, int group) {
    return 2 * P * kRow + (kGroups + group) * P + t;
  }
};

constexpr int kMinExponent = -23, kMaxExponent = 13, kNanScale = 255;

}  // namespace tw

#endif
