// Clipped policy loss over rows of action logits with a KL term to a reference policy and an entropy bonus, and its gradient:
//     x_j = (z_j - max z) / tau,  s = sum e^x_j,  log p_j = x_j - log s,  H = log s - (sum x_j e^x_j) / s
//     r = exp(log p_a - old),  d = ref - log p_a,  k = e^d - d - 1
//     l = -min(r A, clip(r, 1 - low, 1 + high) A) + beta k - eta H,      L = sum_i w_i l_i
//     dL/dz_j = w / tau [ c (1[j = a] - p_j) + eta p_j (log p_j + H) ],  c = -[clip inactive] r A + beta (1 - e^d)
// gfx950 only.
#include "rlgan_types.h"
#include "rlgan_host.h"

using namespace rlgan;

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr double LN2 = 0.69314718055994530942;

struct Policy {
  int64_t rows; int vocab;
  int64_t ld, ld_legal, ld_d;
  const void* actions; int action64;
  const float* old_logp; const float* advantages; const float* weights; const float* ref_logp;
  const uint8_t* legal;
  float scale2;                       // log2(e) / tau: a difference of logits in the exponent of 2
  double inv_tau, low, high, beta, eta, row_weight;
  float* logp; float* entropy; float* kl; double* row_loss;
};

// what the gradient of a row is made of: d_j = e_j (a0 + a1 x2_j) with e_j = 2^(x2_j - log2_s), and `at` more at the action
struct RowGrad { float log2_s, a0, a1, at; int64_t action; };

template <typename T> __device__ __forceinline__ bool in_row(const Policy& P, const T* z, const uint8_t* legal, int j) {
  return !legal || legal[j];
}

// A row's numbers from its maximum, sum and weighted sum (x in units of log 2).  In 64 bits: the terms cancel against each other
// and a batch's rows do too, and one lane of a row does this once.  `writer`: the thread that leaves the row's results.
// Rows left out (action < 0, weight 0, an action that is not allowed): zeros everywhere.  An action >= vocab: NaN everywhere.
template <typename T>
__device__ RowGrad finish_row(const Policy& P, const T* z, int64_t row, float top, float s, float t2, bool writer) {
  const int64_t a = P.action64 ? ((const int64_t*)P.actions)[row] : ((const int32_t*)P.actions)[row];
  const double w = P.weights ? (double)P.weights[row] : P.row_weight;
  RowGrad g{0.f, 0.f, 0.f, 0.f, -1};
  double loss = 0, logp = 0, entropy = 0, kl = 0;
  bool used = a >= 0 && w != 0;
  if (used && a >= P.vocab) {
    used = false;
    const float nan = __builtin_nanf("");
    loss = logp = entropy = kl = nan;
    g.a0 = nan;
  }
  if (used && P.legal && !P.legal[row * P.ld_legal + a]) used = false;
  float za = 0.f;
  if (used) {
    za = (float)z[a];
    if (za == -INFINITY) used = false;
  }
  if (used) {
    const double adv = P.advantages[row], log_s = log((double)s);
    logp = ((double)za - (double)top) * P.inv_tau - log_s;
    entropy = log_s - LN2 * (double)t2 / (double)s;
    const double r = exp(logp - (double)P.old_logp[row]), lo = 1 - P.low, hi = 1 + P.high;
    const double held = (r < lo ? lo : r > hi ? hi : r) * adv, free = r * adv;
    const bool clipped = free > held;                        // a NaN is never clipped away
    double slope = clipped ? 0.0 : -free;
    loss = -(clipped ? held : free) - P.eta * entropy;
    if (P.ref_logp) {
      const double d = (double)P.ref_logp[row] - logp, em = expm1(d);
      kl = em - d;
      loss += P.beta * kl;
      slope -= P.beta * em;
    }
    loss *= w;
    const double k = w * P.inv_tau;
    g.log2_s = (float)(log_s * (double)LOG2E);
    g.a0 = (float)(k * (P.eta * (entropy - log_s) - slope));
    g.a1 = (float)(k * P.eta * LN2);
    g.at = (float)(k * slope);
    g.action = a;
  }
  if (writer) {
    P.logp[row] = (float)logp; P.entropy[row] = (float)entropy; P.kl[row] = (float)kl;
    P.row_loss[row] = loss;
  }
  return g;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { const float u = __shfl_xor(v, o); v = u > v || u != u ? u : v; }
  return v;
}

// a workgroup a row, the row read three times
template <typename T, bool GRAD>
__global__ __launch_bounds__(256) void policy_rows_kernel(Policy P, const T* logits, T* dlogits) {
  __shared__ float sh[8];
  __shared__ RowGrad shared_row;
  const int64_t row = blockIdx.x;
  const T* z = logits + row * P.ld;
  const uint8_t* legal = P.legal ? P.legal + row * P.ld_legal : nullptr;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float top = -INFINITY;
  for (int j = threadIdx.x; j < P.vocab; j += 256) {
    const float v = in_row(P, z, legal, j) ? (float)z[j] : -INFINITY;
    top = v > top || v != v ? v : top;
  }
  top = wave_max(top);
  if (lane == 0) sh[wave] = top;
  __syncthreads();
  top = sh[0];
  for (int w = 1; w < 4; ++w) top = sh[w] > top || sh[w] != sh[w] ? sh[w] : top;
  if (top == -INFINITY) top = 0.f;
  __syncthreads();
  float s = 0.f, t2 = 0.f;
  for (int j = threadIdx.x; j < P.vocab; j += 256) {
    const float v = in_row(P, z, legal, j) ? (float)z[j] : -INFINITY, x2 = (v - top) * P.scale2, e = __builtin_amdgcn_exp2f(x2);
    s += e;
    t2 += fmaxf(x2, -1e4f) * e;
  }
  s = wave_sum(s); t2 = wave_sum(t2);
  if (lane == 0) { sh[wave] = s; sh[4 + wave] = t2; }
  __syncthreads();
  s = sh[0] + sh[1] + sh[2] + sh[3]; t2 = sh[4] + sh[5] + sh[6] + sh[7];
  if (threadIdx.x == 0) shared_row = finish_row(P, z, row, top, s, t2, true);
  __syncthreads();
  if constexpr (GRAD) {
    const RowGrad g = shared_row;
    T* d = dlogits + row * P.ld_d;
    for (int j = threadIdx.x; j < P.vocab; j += 256) {
      float v = g.a0;
      if (g.action >= 0) {
        const float zj = in_row(P, z, legal, j) ? (float)z[j] : -INFINITY, x2 = (zj - top) * P.scale2;
        v = __builtin_amdgcn_exp2f(x2 - g.log2_s) * (g.a0 + g.a1 * fmaxf(x2, -1e4f));
        if (j == g.action) v += g.at;
      }
      d[j] = (T)v;
    }
  }
}

__global__ __launch_bounds__(1024) void policy_sum_kernel(const double* parts, int64_t n, float* loss) {
  __shared__ double sh[1024];
  double s = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += parts[i];
  sh[threadIdx.x] = s;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) *loss = (float)sh[0];
}

}  // namespace

extern "C" {

int rlgan_policy_loss_workspace(int64_t rows, int vocab, int type, int64_t* bytes) {
  if (!bytes || rows <= 0 || vocab <= 0) return RLGAN_E_ARG;
  if (type < TYPE_F32 || type > TYPE_F16) return RLGAN_E_KIND;
  *bytes = rows * 8;
  return 0;
}

int rlgan_policy_loss(const rlgan_policy_t* p, void* workspace, void* stream) {
  if (!p || !p->logits || !p->actions || !p->old_logp || !p->advantages || !p->loss || !p->logp || !p->entropy || !p->kl || !workspace)
    return RLGAN_E_ARG;
  if (p->rows <= 0 || p->vocab <= 0 || p->rows > INT32_MAX) return RLGAN_E_ARG;
  if (p->type < TYPE_F32 || p->type > TYPE_F16 || (p->action_bytes != 4 && p->action_bytes != 8)) return RLGAN_E_KIND;
  if (p->ld < p->vocab || (p->dlogits && p->ld_d < p->vocab) || (p->legal && p->ld_legal < p->vocab)) return RLGAN_E_ALIGN;
  if (!(p->temperature > 0)) return RLGAN_E_ARG;
  Policy P{p->rows, p->vocab, p->ld, p->ld_legal, p->ld_d, p->actions, p->action_bytes == 8, p->old_logp, p->advantages, p->weights, p->ref_logp,
           p->legal, (float)(1.44269504088896340736 / p->temperature), 1.0 / p->temperature, p->clip_low, p->clip_high, p->kl_coef,
           p->entropy_coef, 1.0 / (double)p->rows, p->logp, p->entropy, p->kl, (double*)workspace};
  hipStream_t st = (hipStream_t)stream;
  RLGAN_BY_TYPE(p->type, T, {
    if (p->dlogits) hipLaunchKernelGGL((policy_rows_kernel<T, true>), dim3((unsigned)p->rows), dim3(256), 0, st, P, (const T*)p->logits, (T*)p->dlogits);
    else hipLaunchKernelGGL((policy_rows_kernel<T, false>), dim3((unsigned)p->rows), dim3(256), 0, st, P, (const T*)p->logits, (T*)nullptr);
  });
  hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(1024), 0, st, (const double*)workspace, p->rows, p->loss);
  return (int)hipGetLastError();
}

}  // extern "C"
