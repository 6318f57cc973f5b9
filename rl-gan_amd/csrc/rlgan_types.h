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

// N elements kept as the 32-bit words they were loaded as, so that a row waits in registers at its own width: elements are converted
// where they are used, and `pin` between two uses keeps the compiler from holding on to the converted ones.
template <typename T, int N> struct Words {
  static constexpr int PER = 4 / sizeof(T), COUNT = (N + PER - 1) / PER;
  uint32_t w[COUNT];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (N % PER) w[COUNT - 1] = 0;
    __builtin_memcpy(w, p, N * sizeof(T));
  }
  __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, w, N * sizeof(T)); }
  __device__ __forceinline__ T element(int i) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, w[i]);
    else return __builtin_bit_cast(T, (uint16_t)(w[i / 2] >> (16 * (i & 1))));
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (__is_same(T, bf16_t)) return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    else return (float)element(i);
  }
  __device__ __forceinline__ void set_infinite(int i) {                      // -inf
    if constexpr (sizeof(T) == 4) w[i] = 0xFF800000u;
    else {
      const uint32_t inf = __is_same(T, bf16_t) ? 0xFF80u : 0xFC00u;
      w[i / 2] = i & 1 ? (w[i / 2] & 0xFFFFu) | inf << 16 : (w[i / 2] & 0xFFFF0000u) | inf;
    }
  }
  __device__ __forceinline__ void set_all(const float (&v)[N]) {             // to nearest, ties to even
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = __float_as_uint(v[i]);
    } else {
      typedef T pair __attribute__((ext_vector_type(2)));
      typedef float fpair __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int i = 0; i < COUNT; ++i) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((fpair{v[2 * i], 2 * i + 1 < N ? v[2 * i + 1] : 0.f}), pair));
    }
  }
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) asm volatile("" : "+v"(w[i]));
  }
};

// the statements with T standing for the element type of a tensor
#define RLGAN_BY_TYPE(type, T, ...)                                   \
  do {                                                                \
    if ((type) == TYPE_F32) { typedef float T; __VA_ARGS__; }         \
    else if ((type) == TYPE_BF16) { typedef bf16_t T; __VA_ARGS__; }  \
    else { typedef f16_t T; __VA_ARGS__; }                            \
  } while (0)

}  // namespace rlgan
