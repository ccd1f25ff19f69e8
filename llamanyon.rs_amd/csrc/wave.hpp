// wave.hpp -- reductions over a wave's lanes without LDS: lanes meet through DPP within 16
// (neighbours, pairs, halves, mirrors) and through the swaps of 16 and 32 lanes across.
#pragma once
#include "swamp_common.hpp"

namespace swamp {

#ifdef __HIP_DEVICE_COMPILE__
struct Two {
  uint32_t a, b;
};
// A value of this lane's group of D, and one of the group beside it: the same two in every
// lane of both, once each group of D agrees on its own.
template <int D>
__device__ __forceinline__ Two beside(uint32_t x) {
  if constexpr (D == 16 || D == 32) {
    const auto r = D == 16 ? __builtin_amdgcn_permlane16_swap(x, x, false, false)
                           : __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return Two{r[0], r[1]};
  } else {
    // lane ^ 1, lane ^ 2, 7 - lane of 8, 15 - lane of 16
    constexpr int ctrl = D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 4 ? 0x141 : 0x140;
    return Two{x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), ctrl, 0xF, 0xF, false))};
  }
}
#endif

template <int D>
__device__ __forceinline__ uint32_t pair_max(uint32_t x) {
#ifdef __HIP_DEVICE_COMPILE__
  const Two t = beside<D>(x);
  return max(t.a, t.b);
#else
  return x;
#endif
}
template <int D>
__device__ __forceinline__ float pair_max(float x) {
#ifdef __HIP_DEVICE_COMPILE__
  const Two t = beside<D>(__float_as_uint(x));
  return fmaxf(__uint_as_float(t.a), __uint_as_float(t.b));
#else
  return x;
#endif
}
template <int D>
__device__ __forceinline__ double pair_sum(double x) {
#ifdef __HIP_DEVICE_COMPILE__
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const Two lo = beside<D>(uint32_t(u)), hi = beside<D>(uint32_t(u >> 32));
  return __builtin_bit_cast(double, uint64_t(hi.a) << 32 | lo.a) +
         __builtin_bit_cast(double, uint64_t(hi.b) << 32 | lo.b);
#else
  return x;
#endif
}

// Over the first n lanes of every n (a power of two): the same in each of them.
template <typename T>
__device__ __forceinline__ T group_max(T x, int n) {
  if (n > 1) x = pair_max<1>(x);
  if (n > 2) x = pair_max<2>(x);
  if (n > 4) x = pair_max<4>(x);
  if (n > 8) x = pair_max<8>(x);
  if (n > 16) x = pair_max<16>(x);
  if (n > 32) x = pair_max<32>(x);
  return x;
}
__device__ __forceinline__ double group_sum(double x, int n) {
  if (n > 1) x = pair_sum<1>(x);
  if (n > 2) x = pair_sum<2>(x);
  if (n > 4) x = pair_sum<4>(x);
  if (n > 8) x = pair_sum<8>(x);
  if (n > 16) x = pair_sum<16>(x);
  if (n > 32) x = pair_sum<32>(x);
  return x;
}

// The sum of x over this lane and those before it.
#ifdef __HIP_DEVICE_COMPILE__
template <int kCtrl, int kRows>
__device__ __forceinline__ int64_t shifted(int64_t x) {  // 0 where nothing comes in
  const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(x), kCtrl, kRows, 0xF, false));
  const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(x >> 32), kCtrl, kRows, 0xF, false));
  return int64_t(uint64_t(hi) << 32 | lo);
}
#endif
__device__ __forceinline__ int64_t sum_to_here(int64_t x) {
#ifdef __HIP_DEVICE_COMPILE__
  x += shifted<0x111, 0xF>(x);  // 1, 2, 4, 8 lanes up within 16
  x += shifted<0x112, 0xF>(x);
  x += shifted<0x114, 0xF>(x);
  x += shifted<0x118, 0xF>(x);
  x += shifted<0x142, 0xA>(x);  // lane 15 of 16 to the next 16, the second and the fourth
  x += shifted<0x143, 0xC>(x);  // lane 31 to the upper 32
#endif
  return x;
}

}  // namespace swamp
