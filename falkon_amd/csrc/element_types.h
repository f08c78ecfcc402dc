// Element types of the operators that also take 16-bit data, and their conversions (gfx950).
#pragma once
#include <hip/hip_runtime.h>

namespace flk {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

// To the type sums are held in, and back with one rounding to nearest even.
template <typename A, typename T> __device__ __forceinline__ A to_acc(T x) { return (A)x; }
template <typename T, typename A> __device__ __forceinline__ T from_acc(A x) { return (T)x; }

}  // namespace flk
