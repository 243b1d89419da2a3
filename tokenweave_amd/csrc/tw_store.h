// How matrix tiles store rows of 16-bit values: 8 bytes a lane, 16, or 16 that go through the L2 at once.
//
// The last only where rows begin on 64 bytes: a lane's group of four stores 64, and where those lie across two pieces of
// 64 memory gets parts of each, which the L2 puts together if it may keep them.  "NN" product [4352, 64] x [64, 7944]: 66.6
// us through, 19.4 kept (what it still holds then costs the next kernel 12); rows of 8192 go through in 19.7.
#ifndef TW_STORE_H
#define TW_STORE_H

#include <stdint.h>

#include <type_traits>

namespace tw {

[[maybe_unused]] constexpr int kStoreThrough = 19;  // nt sc0 sc1

enum StoreForm { kNarrowStores, kWideStores, kWideThrough };

inline StoreForm store_form(const void* out, int64_t columns, int64_t ldc) {
  const uintptr_t begin = reinterpret_cast<uintptr_t>(out);
  if (columns % 8 != 0 || ldc % 8 != 0 || begin % 16 != 0) return kNarrowStores;
  return ldc % 32 == 0 && begin % 64 == 0 ? kWideThrough : kWideStores;
}

template <typename F>
__device__ __forceinline__ void with_store_form(int form, F&& f) {
  if (form == kWideThrough) f(std::integral_constant<StoreForm, kWideThrough>{});
  else if (form == kWideStores) f(std::integral_constant<StoreForm, kWideStores>{});
  else f(std::integral_constant<StoreForm, kNarrowStores>{});
}

}  // namespace tw

#endif
