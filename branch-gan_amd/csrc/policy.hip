// Clipped policy loss with a KL term over the vocabulary, forward and backward (bg_policy_loss_fwd / _bwd).
//
// Per row, x = logits / T and c = log2(e) / T:  e_j = 2^(c (logit_j - m)), s = sum e_j, lse = m / T + log s;  with reference logits y
// (the same m', s') the KL is  sum_j p_j ((x_j - x_id) - (y_j - y_id)) - ((lse_x - x_id) - (lse_y - y_id)): the differences are taken
// before the sum and against the sampled token's logits, so neither the logits' size nor an offset between the two models' logits
// (which softmax does not see) costs a policy close to its reference any digits.  c is carried in two floats (its rounding would shift every lse the
// same way); lse, the token's log-prob and the row's loss are put together in fp64 - a handful of operations per row.
//
// HBM-bound: forward reads the logits (and reference logits) once, backward reads them again and writes dlogits.
#include "common.h"

namespace bg {

constexpr int PT = 256;      // threads per row

struct PolicyArgs {
  const void* logits;
  const void* ref;
  const int64_t* ids;
  const float* old_logp;
  const float* ref_logp;
  const float* adv;
  const float* weights;
  int64_t rows, V, x_stride, ref_stride;
  double inv_t, clip_low, clip_high, kl_coef;
  float c_hi, c_lo, inv_t32;
  float* out_logp;
  float* out_kl;
  float* stats;              // per row: m, 1 / s, w dloss_row/dlogp, w kl_coef, (lse_x - x0) - (lse_y - y0), kl, w loss_row (a double);  then 1 / N
};

__device__ __forceinline__ float policy_exp(float d, float c_hi, float c_lo) {        // 2^(d c), d <= 0
  return __builtin_amdgcn_exp2f(__builtin_fmaf(d, c_hi, d * c_lo));
}

// running maximum, sum of exponentials and sum of exponentials times the difference to the reference
struct RowSum {
  float m, s, t;
  __device__ __forceinline__ void rescale(float mn, float c_hi, float c_lo) {
    if (mn > m) {
      const float f = m == -INFINITY ? 0.f : policy_exp(m - mn, c_hi, c_lo);
      s *= f;
      t *= f;
      m = mn;
    }
  }
  __device__ __forceinline__ void join(const RowSum& o, float c_hi, float c_lo) {
    const float mn = fmaxf(m, o.m);
    rescale(mn, c_hi, c_lo);
    const float f = o.m == -INFINITY ? (o.s == 0.f ? 0.f : 1.f) : policy_exp(o.m - mn, c_hi, c_lo);
    s += f * o.s;
    t += f * o.t;
  }
};

__device__ __forceinline__ RowSum row_join(RowSum r, RowSum* red, float c_hi, float c_lo) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    RowSum b;
    b.m = __shfl_xor(r.m, o); b.s = __shfl_xor(r.s, o); b.t = __shfl_xor(r.t, o);
    r.join(b, c_hi, c_lo);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = r;
  __syncthreads();
  r = red[0];
  for (int w = 1; w < PT / 64; ++w) r.join(red[w], c_hi, c_lo);
  return r;
}

// what the logits of a row are taken against in differences: the sampled token's (0 if that one is masked or broken)
template <typename T> __device__ __forceinline__ float row_origin(const T* x, int64_t id) {
  const float v = to_f32(x[id]);
  return __builtin_fabsf(v) <= 3.0e38f ? v : 0.f;
}

__device__ __forceinline__ float row_weight(const PolicyArgs& a, int64_t row) {
  const int64_t id = a.ids[row];
  return id >= 0 && id < a.V ? (a.weights ? a.weights[row] : 1.f) : 0.f;
}

template <typename T, bool REF>
__global__ __launch_bounds__(PT) void policy_rows_kernel(PolicyArgs a) {
  __shared__ RowSum red[PT / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  float* st = a.stats + row * BG_POLICY_STATS;
  const float w = row_weight(a, row);
  if (w == 0.f) {
    if (tid < BG_POLICY_STATS) st[tid] = 0.f;
    if (tid == 0) { a.out_logp[row] = 0.f; a.out_kl[row] = 0.f; }
    return;
  }
  const T* x = (const T*)a.logits + row * a.x_stride;
  const T* y = REF ? (const T*)a.ref + row * a.ref_stride : nullptr;
  const int64_t id = a.ids[row];
  const float x0 = REF ? row_origin(x, id) : 0.f, y0 = REF ? row_origin(y, id) : 0.f;
  RowSum rx = {-INFINITY, 0.f, 0.f}, ry = rx;
  for (int64_t j = tid; j < a.V; j += PT) {
    const float v = to_f32(x[j]);
    rx.rescale(v, a.c_hi, a.c_lo);
    const float e = v == -INFINITY ? 0.f : policy_exp(v - rx.m, a.c_hi, a.c_lo);
    rx.s += e;
    if constexpr (REF) {
      const float u = to_f32(y[j]);
      ry.rescale(u, a.c_hi, a.c_lo);
      ry.s += u == -INFINITY ? 0.f : policy_exp(u - ry.m, a.c_hi, a.c_lo);
      if (e != 0.f) rx.t += e * ((v - x0) - (u - y0));
    }
  }
  rx = row_join(rx, red, a.c_hi, a.c_lo);
  if constexpr (REF) ry = row_join(ry, red, a.c_hi, a.c_lo);
  if (tid != 0) return;
  const double ls = log((double)rx.s);
  const double logp = ((double)to_f32(x[id]) - rx.m) * a.inv_t - ls;
  const double ratio = exp(logp - a.old_logp[row]), A = a.adv[row];
  const double plain = -A * ratio;
  const double clipped = -A * fmin(fmax(ratio, 1.0 - a.clip_low), 1.0 + a.clip_high);
  double slope = plain >= clipped || plain != plain ? plain : 0.0;
  double kl = 0.0, gap = 0.0;
  if constexpr (REF) {
    gap = (((double)rx.m - x0) - ((double)ry.m - y0)) * a.inv_t + (ls - log((double)ry.s));
    kl = (double)rx.t / (double)rx.s * a.inv_t - gap;
  } else if (a.ref_logp) {
    const double d = a.ref_logp[row] - logp, e1 = expm1(d);
    kl = e1 - d;
    slope -= a.kl_coef * e1;
  }
  const double pg = plain != plain ? plain : fmax(plain, clipped);
  a.out_logp[row] = (float)logp;
  a.out_kl[row] = (float)kl;
  st[0] = rx.m;
  st[1] = (float)(1.0 / rx.s);
  st[2] = (float)(w * slope);
  st[3] = (float)(w * a.kl_coef);
  st[4] = (float)gap;
  st[5] = (float)kl;
  *(double*)(st + 6) = w * (pg + a.kl_coef * kl);
}

// loss = sum_r w_r (pg + kl_coef kl) / N in a fixed order, fp64; stats[rows * BG_POLICY_STATS] = 1 / N
__global__ __launch_bounds__(1024) void policy_total_kernel(PolicyArgs a, const float* denominator, float* out_loss) {
  __shared__ double red[2][16];
  const int tid = threadIdx.x;
  double sum = 0.0, wsum = 0.0;
  for (int64_t r = tid; r < a.rows; r += 1024) {
    sum += *(const double*)(a.stats + r * BG_POLICY_STATS + 6);
    wsum += row_weight(a, r);
  }
  sum = wave_sum(sum);
  wsum = wave_sum(wsum);
  if ((tid & 63) == 0) { red[0][tid >> 6] = sum; red[1][tid >> 6] = wsum; }
  __syncthreads();
  if (tid == 0) {
    sum = wsum = 0.0;
    for (int i = 0; i < 16; ++i) { sum += red[0][i]; wsum += red[1][i]; }
    const double n = denominator ? (double)denominator[0] : wsum;
    out_loss[0] = n == 0.0 ? 0.f : (float)(sum / n);
    a.stats[a.rows * BG_POLICY_STATS] = n == 0.0 ? 0.f : (float)(1.0 / n);
  }
}

template <typename T, bool REF>
__global__ __launch_bounds__(PT) void policy_grad_kernel(PolicyArgs a, const float* g_loss, T* dlogits) {
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  T* dx = dlogits + row * a.V;
  const float* st = a.stats + row * BG_POLICY_STATS;
  if (st[1] == 0.f) {                       // does not count (a row that does has s >= 1)
    for (int64_t j = tid; j < a.V; j += PT) dx[j] = from_f32<T>(0.f);
    return;
  }
  const T* x = (const T*)a.logits + row * a.x_stride;
  const T* y = REF ? (const T*)a.ref + row * a.ref_stride : nullptr;
  const float f = g_loss[0] * a.stats[a.rows * BG_POLICY_STATS] * a.inv_t32;
  const float m = st[0], inv_s = st[1], cA = f * st[2], cK = f * st[3], off = st[4] + st[5];
  const int64_t id = a.ids[row];
  const float x0 = REF ? row_origin(x, id) : 0.f, y0 = REF ? row_origin(y, id) : 0.f;
  for (int64_t j = tid; j < a.V; j += PT) {
    const float v = to_f32(x[j]);
    const float p = v == -INFINITY ? 0.f : policy_exp(v - m, a.c_hi, a.c_lo) * inv_s;
    float d = cA * ((j == id ? 1.f : 0.f) - p);
    if constexpr (REF)
      if (p != 0.f) d += cK * p * (((v - x0) - (to_f32(y[j]) - y0)) * a.inv_t32 - off);
    dx[j] = from_f32<T>(d);
  }
}

}  // namespace bg

using namespace bg;

static int policy_check(const char* who, const bg_policy_shape* sh, const void* logits, const void* ref, const int64_t* ids, const float* stats) {
  BG_REQUIRE(sh && logits && ids && stats && ((uintptr_t)stats & 7) == 0, "%s: null argument or stats off the 8-byte grid", who);
  BG_REQUIRE(sh->dtype == BG_F32 || sh->dtype == BG_BF16, "%s: dtype %d", who, sh->dtype);
  BG_REQUIRE(sh->rows > 0 && sh->rows < (1ll << 31) && sh->V > 0 && sh->V < (1ll << 31) && sh->x_stride >= sh->V, "%s: rows=%lld V=%lld stride=%lld",
             who, (long long)sh->rows, (long long)sh->V, (long long)sh->x_stride);
  BG_REQUIRE(!ref || sh->ref_stride >= sh->V, "%s: reference stride %lld", who, (long long)sh->ref_stride);
  BG_REQUIRE(sh->temperature > 0.0 && sh->temperature < 1e6 && sh->temperature > 1e-6, "%s: temperature %g", who, sh->temperature);
  BG_REQUIRE(sh->clip_low >= 0.0 && sh->clip_high >= 0.0, "%s: clip range %g, %g", who, sh->clip_low, sh->clip_high);
  return BG_OK;
}

static PolicyArgs policy_args(const bg_policy_shape* sh, const void* logits, const void* ref, const int64_t* ids, float* stats) {
  PolicyArgs a = {};
  a.logits = logits; a.ref = ref; a.ids = ids; a.stats = stats;
  a.rows = sh->rows; a.V = sh->V; a.x_stride = sh->x_stride; a.ref_stride = sh->ref_stride;
  a.inv_t = 1.0 / sh->temperature;
  a.clip_low = sh->clip_low; a.clip_high = sh->clip_high; a.kl_coef = sh->kl_coef;
  const double c = 1.4426950408889634 / sh->temperature;
  a.c_hi = (float)c;
  a.c_lo = (float)(c - (double)a.c_hi);
  a.inv_t32 = (float)a.inv_t;
  return a;
}

extern "C" int bg_policy_loss_fwd(const bg_policy_shape* sh, const void* logits, const void* ref_logits, const int64_t* ids,
                                  const float* old_logp, const float* ref_logp, const float* advantages, const float* weights,
                                  const float* denominator, float* out_loss, float* out_logp, float* out_kl, float* stats, void* stream) {
  if (int rc = policy_check("bg_policy_loss_fwd", sh, logits, ref_logits, ids, stats)) return rc;
  BG_REQUIRE(old_logp && advantages && out_loss && out_logp && out_kl, "bg_policy_loss_fwd: null argument");
  BG_REQUIRE(!(ref_logits && ref_logp), "bg_policy_loss_fwd: ref_logits and ref_logp exclude each other");
  PolicyArgs a = policy_args(sh, logits, ref_logits, ids, stats);
  a.old_logp = old_logp; a.ref_logp = ref_logp; a.adv = advantages; a.weights = weights;
  a.out_logp = out_logp; a.out_kl = out_kl;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)sh->rows), block(PT);
  if (sh->dtype == BG_F32) {
    if (ref_logits) hipLaunchKernelGGL((policy_rows_kernel<float, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((policy_rows_kernel<float, false>), grid, block, 0, st, a);
  } else {
    if (ref_logits) hipLaunchKernelGGL((policy_rows_kernel<bf16_t, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((policy_rows_kernel<bf16_t, false>), grid, block, 0, st, a);
  }
  hipLaunchKernelGGL(policy_total_kernel, dim3(1), dim3(1024), 0, st, a, denominator, out_loss);
  BG_CHECK_LAUNCH("bg_policy_loss_fwd");
  return BG_OK;
}

extern "C" int bg_policy_loss_bwd(const bg_policy_shape* sh, const void* logits, const void* ref_logits, const int64_t* ids,
                                  const float* stats, const float* g_loss, void* dlogits, void* stream) {
  if (int rc = policy_check("bg_policy_loss_bwd", sh, logits, ref_logits, ids, stats)) return rc;
  BG_REQUIRE(g_loss && dlogits, "bg_policy_loss_bwd: null argument");
  const PolicyArgs a = policy_args(sh, logits, ref_logits, ids, (float*)stats);
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)sh->rows), block(PT);
  if (sh->dtype == BG_F32) {
    if (ref_logits) hipLaunchKernelGGL((policy_grad_kernel<float, true>), grid, block, 0, st, a, g_loss, (float*)dlogits);
    else hipLaunchKernelGGL((policy_grad_kernel<float, false>), grid, block, 0, st, a, g_loss, (float*)dlogits);
  } else {
    if (ref_logits) hipLaunchKernelGGL((policy_grad_kernel<bf16_t, true>), grid, block, 0, st, a, g_loss, (bf16_t*)dlogits);
    else hipLaunchKernelGGL((policy_grad_kernel<bf16_t, false>), grid, block, 0, st, a, g_loss, (bf16_t*)dlogits);
  }
  BG_CHECK_LAUNCH("bg_policy_loss_bwd");
  return BG_OK;
}
