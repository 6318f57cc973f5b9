// Gated linear recurrence over time, forward and backward:
//     f_t = sigmoid(z_t),   p_t = 0 where an episode starts at t, else h_{t-1},   h_t = p_t + (1 - f_t) (x_t - p_t)
// Every unit (batch row, channel) is a recurrence of its own.  A step is the affine map h -> a h + b with a = f (or "drop" at a
// start), and maps compose: (a2, b2) after (a1, b1) is (a2 a1, a2 b1 + b2).  gfx950 only.
#include "rlgan_types.h"
#include "rlgan_host.h"

using namespace rlgan;

namespace {

constexpr float LOG2E = 1.44269504088896340736f;

// f = sigmoid(z) and 1 - f, both to a relative rounding: the smaller one from e^-|z|, the larger as its complement.  Written as
// p + (1 - f)(x - p) a step of a long memory (f next to 1) loses a rounding of h only.
__device__ __forceinline__ void gate(float z, float& f, float& take) {
  const float e = __builtin_amdgcn_exp2f(-LOG2E * fabsf(z));
  const float small = e * __builtin_amdgcn_rcpf(1.f + e), large = 1.f - small;
  f = z >= 0.f ? large : small;
  take = z >= 0.f ? small : large;
}

struct Units {
  int batch, length, width;
  const float* state;
  const uint8_t* starts; int64_t starts_b, starts_t;
  const int32_t* lengths;
};

template <typename T> struct Seq { T* p; int64_t b, t; };

// one thread a unit (VEC units), all steps in a row
template <typename T, int VEC, bool MASK>
__global__ __launch_bounds__(256) void scan_serial_fwd(Units u, Seq<const T> z, Seq<const T> x, Seq<T> h, float* state_out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int wv = u.width / VEC;
  if (i >= (int64_t)u.batch * wv) return;
  const int b = (int)(i / wv), d = (int)(i - (int64_t)b * wv) * VEC;
  const int len = MASK && u.lengths ? min(max(u.lengths[b], 0), u.length) : u.length;
  const T* zp = z.p + b * z.b + d; const T* xp = x.p + b * x.b + d; T* hp = h.p + b * h.b + d;
  float s[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) s[k] = u.state ? u.state[(int64_t)b * u.width + d + k] : 0.f;
  for (int t = 0; t < u.length; ++t) {
    Vec<T, VEC> zv, xv, hv;
    if (!MASK || t < len) {
      zv.load(zp + t * z.t); xv.load(xp + t * x.t);
      const bool start = MASK && u.starts && u.starts[b * u.starts_b + t * u.starts_t];
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float f, take;
        gate(zv.get(k), f, take);
        const float p = start ? 0.f : s[k];
        s[k] = p + take * (xv.get(k) - p);
        hv.set(k, s[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) hv.set(k, 0.f);
    }
    hv.store(hp + t * h.t);
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) state_out[(int64_t)b * u.width + d + k] = s[k];
}

template <typename T, int VEC, bool MASK>
__global__ __launch_bounds__(256) void scan_serial_bwd(Units u, Seq<const T> dh, Seq<const T> z, Seq<const T> x, Seq<const T> h,
                                                       const float* dstate, Seq<T> dz, Seq<T> dx, float* dstate_in) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int wv = u.width / VEC;
  if (i >= (int64_t)u.batch * wv) return;
  const int b = (int)(i / wv), d = (int)(i - (int64_t)b * wv) * VEC;
  const int len = MASK && u.lengths ? min(max(u.lengths[b], 0), u.length) : u.length;
  float c[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) c[k] = dstate ? dstate[(int64_t)b * u.width + d + k] : 0.f;
  for (int t = u.length - 1; t >= 0; --t) {
    Vec<T, VEC> gv, zv, xv, hv, oz, ox;
    if (!MASK || t < len) {
      gv.load(dh.p + b * dh.b + t * dh.t + d); zv.load(z.p + b * z.b + t * z.t + d); xv.load(x.p + b * x.b + t * x.t + d);
      const bool start = MASK && u.starts && u.starts[b * u.starts_b + t * u.starts_t];
      if (t > 0) hv.load(h.p + b * h.b + (t - 1) * h.t + d);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float f, take;
        gate(zv.get(k), f, take);
        const float p = start ? 0.f : t > 0 ? hv.get(k) : u.state ? u.state[(int64_t)b * u.width + d + k] : 0.f;
        const float g = c[k] + gv.get(k), gt = g * take;
        ox.set(k, gt);
        oz.set(k, gt * f * (p - xv.get(k)));
        c[k] = start ? 0.f : f * g;
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) { oz.set(k, 0.f); ox.set(k, 0.f); }
    }
    oz.store(dz.p + b * dz.b + t * dz.t + d); ox.store(dx.p + b * dx.b + t * dx.t + d);
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) dstate_in[(int64_t)b * u.width + d + k] = c[k];
}

inline int check_scan(const rlgan_scan_t* s) {
  if (!s || !s->z.p || !s->x.p) return RLGAN_E_ARG;
  if (s->batch <= 0 || s->length <= 0 || s->width <= 0) return RLGAN_E_ARG;
  if (s->type < TYPE_F32 || s->type > TYPE_F16) return RLGAN_E_KIND;
  if ((int64_t)s->batch * s->width > (int64_t)1 << 31) return RLGAN_E_DIMS;
  return 0;
}

template <typename T> inline Seq<const T> in(const rlgan_seq_t& s) { return {(const T*)s.p, s.batch, s.time}; }
template <typename T> inline Seq<T> out(const rlgan_seq_t& s) { return {(T*)s.p, s.batch, s.time}; }
inline Units units(const rlgan_scan_t* s) {
  return {s->batch, s->length, s->width, s->state, s->starts, s->starts_batch, s->starts_time, s->lengths};
}

}  // namespace

extern "C" {

int rlgan_gated_scan_workspace(int batch, int length, int width, int type, int backward, int64_t* bytes) {
  if (!bytes || batch <= 0 || length <= 0 || width <= 0) return RLGAN_E_ARG;
  if (type < TYPE_F32 || type > TYPE_F16) return RLGAN_E_KIND;
  *bytes = 0;
  return 0;
}

int rlgan_gated_scan_forward(const rlgan_scan_t* s, rlgan_seq_t h, float* state_out, void* workspace, void* stream) {
  if (int e = check_scan(s)) return e;
  if (!h.p || !state_out) return RLGAN_E_ARG;
  const Units u = units(s);
  const bool mask = s->starts || s->lengths;
  const dim3 grid((unsigned)(((int64_t)s->batch * s->width + 255) / 256));
  RLGAN_BY_TYPE(s->type, T, {
    if (mask) hipLaunchKernelGGL((scan_serial_fwd<T, 1, true>), grid, dim3(256), 0, (hipStream_t)stream, u, in<T>(s->z), in<T>(s->x), out<T>(h), state_out);
    else hipLaunchKernelGGL((scan_serial_fwd<T, 1, false>), grid, dim3(256), 0, (hipStream_t)stream, u, in<T>(s->z), in<T>(s->x), out<T>(h), state_out);
  });
  return (int)hipGetLastError();
}

int rlgan_gated_scan_backward(const rlgan_scan_t* s, rlgan_seq_t h, rlgan_seq_t dh, const float* dstate, rlgan_seq_t dz, rlgan_seq_t dx,
                              float* dstate_in, void* workspace, void* stream) {
  if (int e = check_scan(s)) return e;
  if (!h.p || !dh.p || !dz.p || !dx.p || !dstate_in) return RLGAN_E_ARG;
  const Units u = units(s);
  const bool mask = s->starts || s->lengths;
  const dim3 grid((unsigned)(((int64_t)s->batch * s->width + 255) / 256));
  RLGAN_BY_TYPE(s->type, T, {
    if (mask) hipLaunchKernelGGL((scan_serial_bwd<T, 1, true>), grid, dim3(256), 0, (hipStream_t)stream, u, in<T>(dh), in<T>(s->z), in<T>(s->x), in<T>(h), dstate, out<T>(dz), out<T>(dx), dstate_in);
    else hipLaunchKernelGGL((scan_serial_bwd<T, 1, false>), grid, dim3(256), 0, (hipStream_t)stream, u, in<T>(dh), in<T>(s->z), in<T>(s->x), in<T>(h), dstate, out<T>(dz), out<T>(dx), dstate_in);
  });
  return (int)hipGetLastError();
}

}  // extern "C"
