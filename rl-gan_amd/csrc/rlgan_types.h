// Elements of the operators that take fp32, bf16 or fp16 tensors: wide loads and stores of element-aligned rows, conversion to
// and from the 32-bit floats all arithmetic is done in.  gfx950 only.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rlgan {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

enum { TYPE_F32 = 0, TYPE_BF16 = 1, TYPE_F16 = 2 };

// N consecutive elements.  Rows may begin at any element (an odd leading dimension), so the copy assumes no more than the
// element's own alignment; gfx950 loads and stores 16 bytes at any address.
template <typename T, int N>
struct Vec {
  T v[N];
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(v, p, sizeof(v)); }
  __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, v, sizeof(v)); }
  __device__ __forceinline__ float get(int i) const { return (float)v[i]; }
  __device__ __forceinline__ void set(int i, float x) { v[i] = (T)x; }       // to nearest, ties to even
};

// the statements with T standing for the element type of a tensor
#define RLGAN_BY_TYPE(type, T, ...)                                   \
  do {                                                                \
    if ((type) == TYPE_F32) { typedef float T; __VA_ARGS__; }         \
    else if ((type) == TYPE_BF16) { typedef bf16_t T; __VA_ARGS__; }  \
    else { typedef f16_t T; __VA_ARGS__; }                            \
  } while (0)

}  // namespace rlgan
