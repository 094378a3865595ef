// Storage types of the operators that take more than fp32, and loads / stores of VW neighbours as one access.
#pragma once
#include "common.hpp"

namespace cvae {

enum DType { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };
typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// conversions to the 16-bit types round to nearest even; every value is widened to fp32 before it is used
template <typename T, int VW> struct __attribute__((aligned(sizeof(T) * VW))) Packed {
  T e[VW];
  __device__ __forceinline__ float f(int i) const { return (float)e[i]; }
  __device__ __forceinline__ void set(int i, float x) { e[i] = (T)x; }
};

}  // namespace cvae
