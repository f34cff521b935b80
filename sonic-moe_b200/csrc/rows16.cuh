// 16 bytes at a time of rows that start anywhere (on a value).
#pragma once
#include <stdint.h>

namespace smoe {

// w: the 16 bytes of `row` from `at` on (T: the values' type, `at` a multiple of its size); whatever lies there where that is outside
// of the row's `bytes`.  Two aligned loads, shifted together, each of a block that holds a byte of the row: neither leaves the
// row's own 16-byte blocks.
template <class T>
__device__ __forceinline__ void load16_around_row(const char* row, int at, int bytes, uint32_t (&w)[4]) {
  const int s = static_cast<int>(reinterpret_cast<uintptr_t>(row + at) & 15), first = at - s;
  uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
  if (first > -16 && first < bytes) a = *reinterpret_cast<const uint4*>(row + first);
  if (s != 0 && first + 16 > -16 && first + 16 < bytes) b = *reinterpret_cast<const uint4*>(row + first + 16);
  uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (s & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) v[i] = v[i + 2];
  }
  if (s & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) v[i] = v[i + 1];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = sizeof(T) == 4 ? v[i] : __funnelshift_r(v[i], v[i + 1], 8 * (s & 2));
}

// Zeros where that is outside of the row; the values at its ends one by one, which suits rows whose beginning is aligned with `at` (16384
// rows of 1030 fp16 quantised 19.7 us, 20.5 with the form above and masks).
template <class T>
__device__ __forceinline__ void load16_of_row(const char* row, int at, int bytes, uint32_t (&w)[4]) {
  if (at >= 0 && at + 16 <= bytes) {
    const char* p = row + at;
    const int s = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
    const uint4 a = *reinterpret_cast<const uint4*>(p - s);
    uint4 b = make_uint4(0u, 0u, 0u, 0u);
    if (s != 0) b = *reinterpret_cast<const uint4*>(p - s + 16);
    uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (s & 8) {
#pragma unroll
      for (int i = 0; i < 6; ++i) v[i] = v[i + 2];
    }
    if (s & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) v[i] = v[i + 1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = sizeof(T) == 4 ? v[i] : __funnelshift_r(v[i], v[i + 1], 8 * (s & 2));
  } else {
#pragma unroll
    for (auto& x : w) x = 0u;
#pragma unroll
    for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i) {
      const int o = at + i * static_cast<int>(sizeof(T));
      if (o < 0 || o >= bytes) continue;
      if constexpr (sizeof(T) == 4) w[i] = *reinterpret_cast<const uint32_t*>(row + o);
      else w[i / 2] |= static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(row + o)) << (16 * (i & 1));
    }
  }
}

}  // namespace smoe
