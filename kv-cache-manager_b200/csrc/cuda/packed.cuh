// A second face of a C entry point: all arguments as 8-byte slots behind one pointer (addresses and whole numbers as they are, floats
// as doubles), for callers to whom every argument costs (0.1 us each from Python: 24 of them take longer than the launch).
#pragma once
#include <cstddef>
#include <cstdint>
#include <cstring>
#include <type_traits>
#include <utility>

#include "common.cuh"

namespace kvcm {

template <typename T> inline T packed_slot(const void* slots, size_t i) {
  const char* at = static_cast<const char*>(slots) + 8 * i;
  if constexpr (std::is_floating_point_v<T>) {
    double x;
    std::memcpy(&x, at, 8);
    return T(x);
  } else {
    int64_t x;
    std::memcpy(&x, at, 8);
    if constexpr (std::is_pointer_v<T>) return reinterpret_cast<T>(static_cast<uintptr_t>(x));
    else return static_cast<T>(x);
  }
}
template <typename... A, size_t... I> inline int packed_call(int (*f)(A...), const void* slots, std::index_sequence<I...>) {
  return f(packed_slot<A>(slots, I)...);
}
template <typename... A> inline int packed_call(int (*f)(A...), const void* slots) {
  return packed_call(f, slots, std::index_sequence_for<A...>());
}

}  // namespace kvcm

#define KVCM_PACKED(NAME) \
  KVCM_API int NAME##_packed(const void* slots) { return kvcm::packed_call(NAME, slots); }
