// AdamW over any number of tensors in one pass, states in 32 or in 8 bits:
//     m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
// The 8-bit state holds m and the root of v as small floats: 64 elements share the exponent E of the block's largest rounded
// magnitude, and a code counts down from the top of that octave, 127 magnitudes 8 an octave with a sign for m, 255 magnitudes 16
// an octave for the root: 16 octaves each, a rounding of at most 2^-4 and 2^-5.  A power of two as the scale costs no precision
// in a floating code and makes decoding exact.  A magnitude under the range becomes 0 in m but the smallest code in the root,
// so that no step divides by eps alone what was small.  gfx950 only.
#include "rlgan_types.h"
#include "rlgan_host.h"

using namespace rlgan;

namespace {

constexpr int BLOCK = 64;                       // elements that share an exponent: 16 lanes of 4
constexpr int CHUNK = RLGAN_ADAMW_CHUNK;        // elements of a workgroup
constexpr int GROUP = 384;                      // tensors of a launch: their gradients' pointers travel as arguments

struct Grads { const void* p[GROUP]; uint8_t type[GROUP]; };

struct Scalars { float lr_t, root_t, keep; int skip; };

__global__ void adamw_begin_kernel(int32_t* step, const float* lr, double beta1, double beta2, double decay, const uint8_t* skip, Scalars* out) {
  const bool no = skip && *skip;
  const int t = *step + (no ? 0 : 1);
  *step = t;
  const double rate = (double)*lr;
  out->lr_t = (float)(rate / (1.0 - pow(beta1, (double)t)));
  out->root_t = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t)));
  out->keep = (float)(1.0 - rate * decay);
  out->skip = no;
}

template <typename T> __device__ __forceinline__ void load4(const void* base, int64_t i, int64_t n, float v[4]) {
  const T* p = (const T*)base + i;
  if (i + 4 <= n) {
    Vec<T, 4> u;
    u.load(p);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = u.get(k);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = i + k < n ? (float)p[k] : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void store4(void* base, int64_t i, int64_t n, const float v[4]) {
  T* p = (T*)base + i;
  if (i + 4 <= n) {
    Vec<T, 4> u;
#pragma unroll
    for (int k = 0; k < 4; ++k) u.set(k, v[k]);
    u.store(p);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) if (i + k < n) p[k] = (T)v[k];
  }
}
__device__ __forceinline__ void load4(int type, const void* base, int64_t i, int64_t n, float v[4]) {
  RLGAN_BY_TYPE(type, T, load4<T>(base, i, n, v));
}

// 8-bit floats: MAN mantissa bits, COUNT magnitudes
template <int MAN, int COUNT> struct Small {
  static constexpr int ONES = (1 << MAN) - 1;
  // a magnitude rounded to MAN bits behind the leading one (ties to even), in units of that bit with a 32-bit float's exponent;
  // 0 under the normal range, at least 255 << MAN for what no float holds
  static __device__ __forceinline__ int rounded(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v) & 0x7FFFFFFFFFFFFFFFull;
    const uint64_t r = (b + ((1ull << (51 - MAN)) - 1) + ((b >> (52 - MAN)) & 1)) >> (52 - MAN);
    const int64_t u = (int64_t)r - ((int64_t)896 << MAN);
    return u < (1 << MAN) ? 0 : u > (255 << MAN) ? 255 << MAN : (int)u;
  }
  static __device__ __forceinline__ int code(int r, int exponent, bool keep) {
    if (r == 0) return 0;
    const int c = r - ((exponent << MAN) | ONES) + COUNT;
    return c < 1 ? (keep ? 1 : 0) : c;
  }
  static __device__ __forceinline__ float value(int c, int exponent) {
    if (exponent == 255) return __builtin_nanf("");
    const int r = ((exponent << MAN) | ONES) - COUNT + c;
    return c > 0 && r > ONES ? __int_as_float(r << (23 - MAN)) : 0.f;
  }
};
typedef Small<3, 127> First;
typedef Small<4, 255> Root;

// largest of 16 neighbouring lanes
__device__ __forceinline__ int block_max(int v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o));
  return v;
}

__device__ __forceinline__ void decode4(uint32_t cm, int em, uint32_t cr, int er, float m[4], float root[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = (cm >> (8 * k)) & 255;
    const float v = First::value(c & 127, em);
    m[k] = c > 127 ? -v : v;
    root[k] = Root::value((cr >> (8 * k)) & 255, er);
  }
}

__device__ __forceinline__ void encode4(const double m[4], const double root[4], uint32_t& cm, int& em, uint32_t& cr, int& er) {
  int rm[4], rr[4], hm = 0, hr = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    rm[k] = First::rounded(m[k]); rr[k] = Root::rounded(root[k]);
    hm = max(hm, rm[k]); hr = max(hr, rr[k]);
  }
  em = block_max(hm) >> 3; er = block_max(hr) >> 4;
  cm = cr = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int c = First::code(rm[k], em, false);
    cm |= (uint32_t)(c | (c && m[k] < 0 ? 128 : 0)) << (8 * k);
    cr |= (uint32_t)Root::code(rr[k], er, true) << (8 * k);
  }
}

template <int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(const rlgan_adamw_tensor_t* tensors, const int32_t* chunks, int64_t chunk0, int tensor0,
                                                    Grads grads, void* first_, void* second_, uint8_t* first_e, uint8_t* second_e,
                                                    double beta1, double beta2, float eps, const float* grad_scale, const Scalars* scalars) {
  const Scalars sc = *scalars;
  if (sc.skip) return;
  const int ti = chunks[2 * (chunk0 + blockIdx.x)], ci = chunks[2 * (chunk0 + blockIdx.x) + 1];
  const rlgan_adamw_tensor_t T = tensors[ti];
  const void* gp = grads.p[ti - tensor0];
  const int gt = grads.type[ti - tensor0];
  const float gs = grad_scale ? *grad_scale : 1.f;
  const int64_t begin = (int64_t)ci * CHUNK, padded = (T.count + BLOCK - 1) / BLOCK * BLOCK;
  for (int64_t i = begin + 4 * threadIdx.x; i < begin + CHUNK && i < padded; i += 1024) {
    float p[4], g[4], m[4], root[4];
    load4(T.type, T.param, i, T.count, p);
    load4(gt, gp, i, T.count, g);
    const int64_t at = T.offset + i;
    if constexpr (BITS == 32) {
      float v[4];
      float* mp = (float*)first_ + at; float* vp = (float*)second_ + at;
      __builtin_memcpy(m, __builtin_assume_aligned(mp, 16), 16);
      __builtin_memcpy(v, __builtin_assume_aligned(vp, 16), 16);
      const float b1 = (float)beta1, c1 = (float)(1.0 - beta1), b2 = (float)beta2, c2 = (float)(1.0 - beta2);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float gk = g[k] * gs;
        m[k] = m[k] * b1 + gk * c1;
        v[k] = v[k] * b2 + gk * c2 * gk;
        root[k] = sqrtf(v[k]);
      }
      __builtin_memcpy(__builtin_assume_aligned(mp, 16), m, 16);
      __builtin_memcpy(__builtin_assume_aligned(vp, 16), v, 16);
    } else {
      // 64 bits up to the codes, without contraction: b1 m + (1 - b1) g of values with so few bits lands on the border between
      // two codes often enough (15 * 0.9 = 13.5), and 32 bits would decide by their own rounding there
#pragma clang fp contract(off)
      uint32_t* mp = (uint32_t*)first_ + at / 4; uint32_t* rp = (uint32_t*)second_ + at / 4;
      uint8_t* me = first_e + at / BLOCK; uint8_t* re = second_e + at / BLOCK;
      decode4(*mp, *me, *rp, *re, m, root);
      double dm[4], dr[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const double gk = (double)g[k] * (double)gs, r = root[k];
        dm[k] = (double)m[k] * beta1 + gk * (1.0 - beta1);
        dr[k] = sqrt(r * r * beta2 + gk * (1.0 - beta2) * gk);
        m[k] = (float)dm[k]; root[k] = (float)dr[k];
      }
      uint32_t cm, cr;
      int em, er;
      encode4(dm, dr, cm, em, cr, er);
      *mp = cm; *rp = cr;
      if ((threadIdx.x & 15) == 0) { *me = (uint8_t)em; *re = (uint8_t)er; }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = p[k] * sc.keep - sc.lr_t * (m[k] / (root[k] * sc.root_t + eps));
    RLGAN_BY_TYPE(T.type, E, store4<E>(T.param, i, T.count, p));
  }
}

// 8-bit states as 32-bit numbers, and back
__global__ __launch_bounds__(256) void adamw_decode_kernel(const uint32_t* first, const uint32_t* second, const uint8_t* first_e,
                                                           const uint8_t* second_e, int64_t n4, float4* m_out, float4* v_out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n4) return;
  float m[4], r[4];
  decode4(first[i], first_e[i / 16], second[i], second_e[i / 16], m, r);
  m_out[i] = make_float4(m[0], m[1], m[2], m[3]);
  v_out[i] = make_float4(r[0] * r[0], r[1] * r[1], r[2] * r[2], r[3] * r[3]);
}
__global__ __launch_bounds__(256) void adamw_encode_kernel(const float4* m_in, const float4* v_in, int64_t n4, uint32_t* first, uint32_t* second,
                                                           uint8_t* first_e, uint8_t* second_e) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n4) return;                              // n4 is a multiple of 16: whole blocks leave together
  const float4 a = m_in[i], b = v_in[i];
  const double m[4] = {a.x, a.y, a.z, a.w}, r[4] = {sqrt((double)b.x), sqrt((double)b.y), sqrt((double)b.z), sqrt((double)b.w)};
  uint32_t cm, cr;
  int em, er;
  encode4(m, r, cm, em, cr, er);
  first[i] = cm; second[i] = cr;
  if ((threadIdx.x & 15) == 0) { first_e[i / 16] = (uint8_t)em; second_e[i / 16] = (uint8_t)er; }
}

inline int check_adamw(const rlgan_adamw_t* a) {
  if (!a || a->n_tensors <= 0 || !a->tensors || !a->chunks || !a->chunk_begin || !a->first || !a->second || !a->lr || !a->step || !a->scalars)
    return RLGAN_E_ARG;
  if (a->state_bits != 8 && a->state_bits != 32) return RLGAN_E_KIND;
  if (a->state_bits == 8 && (!a->first_exp || !a->second_exp)) return RLGAN_E_ARG;
  if (!(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1) || !(a->eps >= 0)) return RLGAN_E_ARG;
  return 0;
}

}  // namespace

extern "C" {

int rlgan_adamw_step(const rlgan_adamw_t* a, const void* const* grads, const uint8_t* grad_types, const float* grad_scale, const uint8_t* skip,
                     void* stream) {
  if (int e = check_adamw(a)) return e;
  if (!grads || !grad_types) return RLGAN_E_ARG;
  for (int i = 0; i < a->n_tensors; ++i) {
    if (grad_types[i] > TYPE_F16) return RLGAN_E_KIND;
    if (a->chunk_begin[i + 1] < a->chunk_begin[i] || a->chunk_begin[i + 1] - a->chunk_begin[0] > INT32_MAX) return RLGAN_E_DIMS;
    if (!grads[i] && a->chunk_begin[i + 1] > a->chunk_begin[i]) return RLGAN_E_ARG;
  }
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(1), 0, st, a->step, a->lr, a->beta1, a->beta2, a->weight_decay, skip, (Scalars*)a->scalars);
  for (int t0 = 0; t0 < a->n_tensors; t0 += GROUP) {
    const int n = a->n_tensors - t0 < GROUP ? a->n_tensors - t0 : GROUP;
    Grads g{};
    for (int i = 0; i < n; ++i) { g.p[i] = grads[t0 + i]; g.type[i] = grad_types[t0 + i]; }
    const int64_t c0 = a->chunk_begin[t0], c1 = a->chunk_begin[t0 + n];
    if (c1 == c0) continue;
    if (a->state_bits == 32)
      hipLaunchKernelGGL(adamw_kernel<32>, dim3((unsigned)(c1 - c0)), dim3(256), 0, st, a->tensors, a->chunks, c0, t0, g, a->first, a->second,
                         a->first_exp, a->second_exp, a->beta1, a->beta2, a->eps, grad_scale, (const Scalars*)a->scalars);
    else
      hipLaunchKernelGGL(adamw_kernel<8>, dim3((unsigned)(c1 - c0)), dim3(256), 0, st, a->tensors, a->chunks, c0, t0, g, a->first, a->second,
                         a->first_exp, a->second_exp, a->beta1, a->beta2, a->eps, grad_scale, (const Scalars*)a->scalars);
  }
  return (int)hipGetLastError();
}

int rlgan_adamw_decode(const uint8_t* first, const uint8_t* second, const uint8_t* first_exp, const uint8_t* second_exp, int64_t n, float* m,
                       float* v, void* stream) {
  if (!first || !second || !first_exp || !second_exp || !m || !v || n <= 0) return RLGAN_E_ARG;
  if (n % BLOCK) return RLGAN_E_ALIGN;
  if (n / 4 > (int64_t)INT32_MAX * 256) return RLGAN_E_DIMS;
  hipLaunchKernelGGL(adamw_decode_kernel, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, (hipStream_t)stream, (const uint32_t*)first,
                     (const uint32_t*)second, first_exp, second_exp, n / 4, (float4*)m, (float4*)v);
  return (int)hipGetLastError();
}

int rlgan_adamw_encode(const float* m, const float* v, int64_t n, uint8_t* first, uint8_t* second, uint8_t* first_exp, uint8_t* second_exp,
                       void* stream) {
  if (!first || !second || !first_exp || !second_exp || !m || !v || n <= 0) return RLGAN_E_ARG;
  if (n % BLOCK) return RLGAN_E_ALIGN;
  if (n / 4 > (int64_t)INT32_MAX * 256) return RLGAN_E_DIMS;
  hipLaunchKernelGGL(adamw_encode_kernel, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, (hipStream_t)stream, (const float4*)m,
                     (const float4*)v, n / 4, (uint32_t*)first, (uint32_t*)second, first_exp, second_exp);
  return (int)hipGetLastError();
}

}  // extern "C"
