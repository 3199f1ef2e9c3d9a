// Clipped policy loss with a KL term over the vocabulary, forward and backward (bg_policy_loss_fwd / _bwd).
//
// Per row, c = log2(e) / T and m the largest logit:  e_j = 2^(c (logit_j - m)), s = sum e_j, lse = m / T + log s;  with reference
// logits (m', s') the KL is  sum_j p_j ((logit_j - m) - (ref_j - m')) / T - (log s - log s'): the differences are taken against the
// maxima and before the sum, so neither the logits' size nor an offset between the two models' logits (which softmax does not
// see) costs a policy close to its reference any digits.  c is carried in two floats (its rounding would shift every lse the same
// way); the token's log-prob and the loss are put together in fp64 - a handful of operations per row.
//
// HBM-bound.  policy_row_kernel holds a row (and the reference's) in registers from its one reading to the gradient's writing: the
// whole of value and gradient is logits in, dlogits out.  The gradient is the one for g_loss = 1; bg_policy_loss_bwd does it over
// when the loss was scaled after all.  Rows too long for the registers take policy_rows_kernel (forward) and policy_grad_kernel
// (backward), one more reading of the logits.
// Measured, bf16 with the gradient: 2047 rows of 50257 in 85 us (4.8 TB/s), 8184 rows of 50304 with a reference in 609 - 620 us
// (4.0 TB/s; a copy reaches 4.8); the weights' sum and the total, one workgroup each, take 3 and 5 us at 2047 rows, 5 and 13 at 8184, a
// backward call with nothing to do 4.  A loss that was scaled: 118 -> 174 us and 622 -> 1118 us a call.
// A thread works through all NV vectors of its kernel, whatever V is: 2047 rows of 32000 take as long as of 50257.  With a reference
// the kernels of 13 vectors spill 37 (512 threads) and 84 registers (1024: fp32 from V = 26624, bf16 from 53248): 2047 rows of 50257 in
// fp32 421 us (257 at the copy's rate), of 65536 in bf16 368 us (168).
#include "common.h"

namespace bg {

constexpr int PT = 256;      // threads per row of the streaming kernels
constexpr int64_t MAX_ROWS = 1 << 22;      // a launch has fewer than 2^32 threads, a row up to 1024

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  typedef f32x4 type;
};
template <> struct Vec<bf16_t> {
  static constexpr int N = 8;
  typedef bf16x8 type;
};

constexpr int64_t NORM_ROWS = 1024;      // up to here the workgroups of short rows sum the weights themselves (12 KB from L2): a launch less

struct PolicyArgs {
  const void* logits;
  const void* ref;
  const int64_t* ids;
  const float* old_logp;
  const float* ref_logp;
  const float* adv;
  const float* weights;
  int64_t rows, V, x_stride, ref_stride, x_outer, ref_outer, d_outer;
  uint32_t inner;            // rows per group
  double inv_t, clip_low, clip_high, kl_coef;
  float c_hi, c_lo, inv_t32;
  float* out_logp;
  float* out_kl;
  float* stats;              // per row: m, 1 / s, w dloss_row/dlogp, w kl_coef, log s - log s' + kl, m', w loss_row (a double);  then 1 / N
};

// where a row starts: rows of a group lie one stride apart, groups one outer stride
__device__ __forceinline__ int64_t row_at(const PolicyArgs& a, int64_t row, int64_t stride, int64_t outer) {
  const uint32_t group = (uint32_t)row / a.inner;
  return group * outer + ((uint32_t)row - group * a.inner) * stride;
}

// 2^(d c), d <= 0.  c_hi < c, so that c_lo > 0 and d = -inf gives 0, not a NaN.
__device__ __forceinline__ float policy_exp(float d, float c_hi, float c_lo) {
  return __builtin_amdgcn_exp2f(__builtin_fmaf(d, c_hi, d * c_lo));
}

// a row's vectors lie on the 16-byte grid: vector i holds the elements [i N - mis, i N - mis + N), the first and last in part
template <typename T> __device__ __forceinline__ int misalignment(const void* p) { return (int)(((uintptr_t)p & 15) / sizeof(T)); }

// vector at element e0 of a row; elements outside [0, V) are -inf.  aligned: p + e0 is on the grid.
template <typename T> __device__ __forceinline__ typename Vec<T>::type row_vector(const T* p, int64_t e0, int64_t V, bool aligned) {
  typename Vec<T>::type r;
  if (aligned && e0 >= 0 && e0 + Vec<T>::N <= V) return *(const typename Vec<T>::type*)(p + e0);
#pragma unroll
  for (int k = 0; k < Vec<T>::N; ++k) r[k] = e0 + k >= 0 && e0 + k < V ? p[e0 + k] : from_f32<T>(-INFINITY);
  return r;
}
template <typename T> __device__ __forceinline__ void store_row_vector(T* p, int64_t e0, int64_t V, bool aligned, const float (&x)[Vec<T>::N]) {
  if (aligned && e0 >= 0 && e0 + Vec<T>::N <= V) {
    typename Vec<T>::type r;
#pragma unroll
    for (int k = 0; k < Vec<T>::N; ++k) r[k] = from_f32<T>(x[k]);
    *(typename Vec<T>::type*)(p + e0) = r;
  } else {
#pragma unroll
    for (int k = 0; k < Vec<T>::N; ++k)
      if (e0 + k >= 0 && e0 + k < V) p[e0 + k] = from_f32<T>(x[k]);
  }
}

// over the workgroup's NW waves, the result in every thread
template <int NW> __device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) v = fmaxf(v, red[w]);
  return v;
}

// Ends the compiler's knowledge of a register's value: the row is kept as it was read and unpacked anew by each pass over it (left to
// itself the compiler keeps the unpacked floats of bf16 rows from one pass to the next, twice the registers).
template <typename V> __device__ __forceinline__ void forget(V& v) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  u32x4 u = __builtin_bit_cast(u32x4, v);
  asm volatile("" : "+v"(u));
  v = __builtin_bit_cast(V, u);
}

struct RowResult {          // what the gradient of a row needs
  float m, inv_s, slope, w_kl, off, my;
};

__device__ __forceinline__ float inverse(double n) { return n == 0.0 ? 0.f : (float)(1.0 / n); }

// a row's weight, 0 if its id is outside the vocabulary.  The weight is requested beside the id, not after it.
__device__ __forceinline__ float row_weight(const PolicyArgs& a, int64_t row, int64_t& id) {
  id = a.ids[row];
  const float w = *(a.weights ? a.weights + row : (const float*)(a.ids + row));
  return id >= 0 && id < a.V ? (a.weights ? w : 1.f) : 0.f;
}
__device__ __forceinline__ float row_weight(const PolicyArgs& a, int64_t row) {
  int64_t id;
  return row_weight(a, row, id);
}

// log of a sum to ~1e-11, in few registers (the row sits in them meanwhile): s = 2^e f with f in [0.7, 1.42), log f = 2 atanh(z),
// z = (f - 1) / (f + 1), by its series (|z| < 0.176: the first term left out is below 2 z^17 / 17 < 2e-14).
__device__ __forceinline__ double log_sum(double s) {
  if (!(s > 0.0 && s < 1e300)) return s == 0.0 ? -(double)INFINITY : s;          // an empty row; a broken one stays NaN
  int e;
  double f = frexp(s, &e);
  if (f < 0.7071067811865476) { f += f; e -= 1; }
  const double z = (f - 1.0) / (f + 1.0), z2 = z * z;
  double q = 1.0 / 15.0;
  q = fma(q, z2, 1.0 / 13.0); q = fma(q, z2, 1.0 / 11.0); q = fma(q, z2, 1.0 / 9.0);
  q = fma(q, z2, 1.0 / 7.0); q = fma(q, z2, 1.0 / 5.0); q = fma(q, z2, 1.0 / 3.0);
  return fma((double)e, 0.6931471805599453, 2.0 * fma(z * z2, q, z));
}

struct RowInput {           // a row's numbers, requested ahead of the row itself: finish_row is one thread's work that the rest waits for
  float w, old_logp, adv, ref_logp;
  int64_t id;
};

__device__ __forceinline__ RowInput row_input(const PolicyArgs& a, int64_t row) {
  RowInput in;
  in.old_logp = a.old_logp[row];
  in.adv = a.adv[row];
  in.ref_logp = *(a.ref_logp ? a.ref_logp + row : a.old_logp + row);
  in.w = row_weight(a, row, in.id);
  return in;
}

// One thread: the row's statistics to its log-prob, KL, loss term and gradient factors.  ls, lsy: logs of the sums s and of the reference's.
template <bool REF>
__device__ RowResult finish_row(const PolicyArgs& a, int64_t row, const RowInput& in, float m, double s, double ls, float my, double lsy, double t,
                                float x_id) {
  const float w = in.w;
  const double logp = ((double)x_id - m) * a.inv_t - ls;
  const float ratio = expf((float)(logp - in.old_logp)), A = in.adv;
  const float lo = (float)(1.0 - a.clip_low), hi = (float)(1.0 + a.clip_high);
  const float plain = -A * ratio, clipped = -A * fminf(fmaxf(ratio, lo), hi);
  const float pg = plain != plain ? plain : fmaxf(plain, clipped);
  RowResult r;
  r.m = m;
  r.inv_s = 1.f / (float)s;
  float slope = plain >= clipped || plain != plain ? plain : 0.f;
  double gap = 0.0;
  float kl = 0.f;
  if constexpr (REF) {
    gap = ls - lsy;
    kl = (float)(t / s * a.inv_t - gap);
  } else if (a.ref_logp) {
    const float d = (float)((double)in.ref_logp - logp);
    float e1;                                                        // exp(d) - 1
    if (__builtin_fabsf(d) < 0.5f) {                                 // exp(d) - 1 - d by its series: d^11 / 11! < 2^-24 of it
      float q = 1.f / 10.f;
#pragma unroll
      for (int i = 9; i >= 3; --i) q = __builtin_fmaf(d, q, 1.f) / (float)i;
      kl = 0.5f * d * d * __builtin_fmaf(d, q, 1.f);
      e1 = kl + d;
    } else {
      e1 = expf(d) - 1.f;                                           // |d| >= 1/2: no digits to lose
      kl = e1 - d;
    }
    if (a.kl_coef != 0.0) slope -= (float)a.kl_coef * e1;             // a KL that is reported only may be infinite
  }
  r.slope = w * slope;
  r.w_kl = (float)(w * a.kl_coef);
  r.off = (float)gap + kl;
  r.my = my;
  a.out_logp[row] = (float)logp;
  a.out_kl[row] = kl;
  float* st = a.stats + row * BG_POLICY_STATS;
  st[0] = r.m; st[1] = r.inv_s; st[2] = r.slope; st[3] = r.w_kl; st[4] = r.off; st[5] = r.my;
  *(double*)(st + 6) = (double)w * (a.kl_coef != 0.0 ? pg + a.kl_coef * kl : pg);
  return r;
}

__device__ __forceinline__ void skip_row(const PolicyArgs& a, int64_t row) {     // it does not count
  if (threadIdx.x < BG_POLICY_STATS) a.stats[row * BG_POLICY_STATS + threadIdx.x] = 0.f;
  if (threadIdx.x == 0) { a.out_logp[row] = 0.f; a.out_kl[row] = 0.f; }
}

// d loss / d logit of one element from its p and, with a reference, the difference of the two logits
template <bool REF>
__device__ __forceinline__ float grad_of(float p, float diff, float slope, float w_kl, float off, float inv_t) {
  float d = -slope * p;
  if constexpr (REF) {
    const float pk = w_kl * p, k = pk * __builtin_fmaf(diff, inv_t, -off);
    d += pk != 0.f ? k : 0.f;                                        // a masked entry, or a KL that is reported only: the difference may be infinite
  }
  return d;
}

// N = the sum of the weights that count; 1 / N -> stats[rows * BG_POLICY_STATS], before the rows' gradients need it (many rows)
__global__ __launch_bounds__(1024) void policy_norm_kernel(PolicyArgs a) {
  __shared__ double red[16];
  double n = 0.0;
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < a.rows; r += 1024) n += row_weight(a, r);
  n = wave_sum(n);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
  __syncthreads();
  n = 0.0;
  for (int i = 0; i < 16; ++i) n += red[i];
  if (threadIdx.x == 0) a.stats[a.rows * BG_POLICY_STATS] = inverse(n);
}

// loss = sum of the rows' terms / N, in a fixed order, fp64; leaves 1 / N for the backward call
__global__ __launch_bounds__(1024) void policy_total_kernel(PolicyArgs a, const float* denominator, float* out_loss) {
  __shared__ double red[2][16];
  double sum = 0.0, n = 0.0;
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < a.rows; r += 1024) {
    sum += *(const double*)(a.stats + r * BG_POLICY_STATS + 6);
    if (!denominator) n += row_weight(a, r);
  }
  sum = wave_sum(sum);
  n = wave_sum(n);
  if ((threadIdx.x & 63) == 0) { red[0][threadIdx.x >> 6] = sum; red[1][threadIdx.x >> 6] = n; }
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = n = 0.0;
    for (int i = 0; i < 16; ++i) { sum += red[0][i]; n += red[1][i]; }
    if (denominator) n = denominator[0];
    a.stats[a.rows * BG_POLICY_STATS] = inverse(n);
    out_loss[0] = n == 0.0 ? 0.f : (float)(sum / n);
  }
}

// Value and (dlogits != NULL) gradient of a row of at most NT * NV whole vectors, read once.  Its interior - the vectors that lie
// wholly inside - is loaded without branches (indices clamped, what is outside set to -inf), so that all loads of a thread are under
// way together; the fewer than 2 N elements before and after it go one each to the first threads.  Sums: fp32 per thread, fp64
// across them.
template <typename T, bool REF, int NT, int NV>
__global__ __launch_bounds__(NT, 4) void policy_row_kernel(PolicyArgs a, const float* denominator, T* dlogits) {
  constexpr int N = Vec<T>::N, NW = NT / 64;
  typedef typename Vec<T>::type V_t;
  __shared__ float red_m[2][NW];
  __shared__ double red[NW][4];
  __shared__ RowResult sh_row;
  __shared__ float sh_inv_n;
  const uint32_t group = blockIdx.y, at = blockIdx.x;                  // (a division to get them costs a row 2 us: 8184 rows of 50304 with a reference 626 -> 662 us)
  const int64_t row = (int64_t)group * a.inner + at;
  const int tid = threadIdx.x;
  const T* x = (const T*)a.logits + (at * a.x_stride + group * a.x_outer);
  const T* y = REF ? (const T*)a.ref + (at * a.ref_stride + group * a.ref_outer) : nullptr;
  T* dx = dlogits ? dlogits + (at * a.V + group * a.d_outer) : nullptr;
  const int V = (int)a.V, mis = misalignment<T>(x);
  RowInput in = row_input(a, row);
  if (in.w == 0.f) {
    skip_row(a, row);
    const float zero[N] = {};
    if (dlogits)
      for (int i = tid; i * N - mis < V; i += NT) store_row_vector<T>(dx, i * N - mis, V, true, zero);
    return;
  }
  const int lo = mis ? 1 : 0, hi = (V + mis) / N;                      // interior vectors (at least one: V >= 2 N)
  const int head = lo * N - mis > 0 ? lo * N - mis : 0, tail = hi * N - mis;
  const int extra = tid < head ? tid : tail + tid - head;              // the single element of this thread, if below V
  const bool has_extra = extra < V;
  V_t vx[NV], vy[REF ? NV : 1];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = min(max(tid + k * NT, lo), hi - 1);
    vx[k] = *(const V_t*)(x + (i * N - mis));
    if constexpr (REF) vy[k] = *(const V_t*)(y + (i * N - mis));
  }
  const float ex = has_extra ? to_f32(x[extra]) : -INFINITY, ey = REF && has_extra ? to_f32(y[extra]) : -INFINITY;
  const int id = (int)in.id;
  const float x_id = to_f32(x[id]);
  constexpr bool SUM_N = NT == 256;                                    // see NORM_ROWS
  float n32 = denominator || (SUM_N && a.rows <= NORM_ROWS) ? 0.f : a.stats[a.rows * BG_POLICY_STATS];
  if (denominator) n32 = denominator[0];
  asm volatile("" ::"s"(in.old_logp), "s"(in.adv), "s"(in.ref_logp), "s"(n32));          // requested here, not where one thread needs them
  double n64 = 0.0;
  if (SUM_N && a.rows <= NORM_ROWS && !denominator)
    for (int64_t r = tid; r < a.rows; r += NT) n64 += row_weight(a, r);
  V_t none;
#pragma unroll
  for (int j = 0; j < N; ++j) none[j] = from_f32<T>(-INFINITY);
  float m = ex, my = ey;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = tid + k * NT;
    if (k == 0 || (k + 1) * NT > hi) {
      const bool in = i >= lo && i < hi;
      vx[k] = in ? vx[k] : none;
      if constexpr (REF) vy[k] = in ? vy[k] : none;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      m = fmaxf(m, (float)vx[k][j]);
      if constexpr (REF) my = fmaxf(my, (float)vy[k][j]);
    }
  }
  m = block_max<NW>(m, red_m[0]);
  if constexpr (REF) my = block_max<NW>(my, red_m[1]);
  const float ms = m == -INFINITY ? 0.f : m, mys = my == -INFINITY ? 0.f : my;
  float s = 0.f, sy = 0.f, t = 0.f;
  auto add = [&](float v, float u) __attribute__((always_inline)) {
    const float dv = v - ms, e = policy_exp(dv, a.c_hi, a.c_lo);
    s += e;
    if constexpr (REF) {
      const float du = u - mys, d = e * (dv - du);
      sy += policy_exp(du, a.c_hi, a.c_lo);
      t += e != 0.f ? d : 0.f;                                         // a masked entry: its difference may be infinite
    }
  };
  add(ex, ey);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    forget(vx[k]);
    if constexpr (REF) forget(vy[k]);
#pragma unroll
    for (int j = 0; j < N; ++j) add((float)vx[k][j], REF ? (float)vy[REF ? k : 0][j] : 0.f);
  }
  const double s64 = wave_sum((double)s), t64 = REF ? wave_sum((double)t) : 0.0, sy64 = REF ? wave_sum((double)sy) : 0.0;
  if constexpr (SUM_N) n64 = wave_sum(n64);
  if ((tid & 63) == 0) { red[tid >> 6][0] = s64; red[tid >> 6][1] = t64; red[tid >> 6][2] = sy64; red[tid >> 6][3] = n64; }
  __syncthreads();
  if (tid < 64) {
    double S = 0.0, Tt = 0.0, Sy = 0.0, Nw = 0.0;
    for (int i = 0; i < NW; ++i) { S += red[i][0]; Tt += red[i][1]; Sy += red[i][2]; Nw += red[i][3]; }
    const double lg = log_sum(REF && tid == 1 ? Sy : S);
    const double ls = __shfl(lg, 0), lsy = REF ? __shfl(lg, 1) : 0.0;
    if (tid == 0) {
      sh_inv_n = denominator ? inverse(n32) : SUM_N && a.rows <= NORM_ROWS ? inverse(Nw) : n32;
      sh_row = finish_row<REF>(a, row, in, ms, S, ls, mys, lsy, Tt, x_id);
    }
  }
  if (!dlogits) return;
  __syncthreads();
  const RowResult r = sh_row;
  const float f = sh_inv_n * a.inv_t32, slope = f * r.slope, w_kl = f * r.w_kl, off = r.off;
  auto grad = [&](float v, float u) __attribute__((always_inline)) {
    const float dv = v - ms, p = policy_exp(dv, a.c_hi, a.c_lo) * r.inv_s;
    return grad_of<REF>(p, REF ? dv - (u - mys) : 0.f, slope, w_kl, off, a.inv_t32);
  };
  if (has_extra) dx[extra] = from_f32<T>(grad(ex, ey) + (extra == id ? slope : 0.f));
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int i = tid + k * NT;
    if (i >= lo && i < hi) {
      forget(vx[k]);
      if constexpr (REF) forget(vy[k]);
      float d[N];
#pragma unroll
      for (int j = 0; j < N; ++j) d[j] = grad((float)vx[k][j], REF ? (float)vy[REF ? k : 0][j] : 0.f);
      const int hit = id - (i * N - mis);
      if (hit >= 0 && hit < N) {
#pragma unroll
        for (int j = 0; j < N; ++j) d[j] += hit == j ? slope : 0.f;
      }
      V_t o;
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = from_f32<T>(d[j]);
      *(V_t*)(dx + (i * N - mis)) = o;
    }
  }
}

// Streaming forward for rows of any length: the maximum in one reading, the sums in a second.
template <typename T, bool REF>
__global__ __launch_bounds__(PT) void policy_rows_kernel(PolicyArgs a) {
  constexpr int N = Vec<T>::N, NW = PT / 64;
  __shared__ float red_m[2][NW];
  __shared__ double red[NW][3];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const RowInput in = row_input(a, row);
  if (in.w == 0.f) {
    skip_row(a, row);
    return;
  }
  const T* x = (const T*)a.logits + row_at(a, row, a.x_stride, a.x_outer);
  const T* y = REF ? (const T*)a.ref + row_at(a, row, a.ref_stride, a.ref_outer) : nullptr;
  const int mis = misalignment<T>(x);
  const bool y_on = !REF || misalignment<T>(y) == mis;
  float m = -INFINITY, my = -INFINITY;
  for (int64_t e0 = (int64_t)tid * N - mis; e0 < a.V; e0 += PT * N) {
    const typename Vec<T>::type vx = row_vector<T>(x, e0, a.V, true);
    typename Vec<T>::type vy;
    if constexpr (REF) vy = row_vector<T>(y, e0, a.V, y_on);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      m = fmaxf(m, (float)vx[j]);
      if constexpr (REF) my = fmaxf(my, (float)vy[j]);
    }
  }
  m = block_max<NW>(m, red_m[0]);
  if constexpr (REF) my = block_max<NW>(my, red_m[1]);
  const float ms = m == -INFINITY ? 0.f : m, mys = my == -INFINITY ? 0.f : my;
  double s64 = 0.0, sy64 = 0.0, t64 = 0.0;
  for (int64_t e0 = (int64_t)tid * N - mis; e0 < a.V; e0 += PT * N) {
    const typename Vec<T>::type vx = row_vector<T>(x, e0, a.V, true);
    typename Vec<T>::type vy;
    if constexpr (REF) vy = row_vector<T>(y, e0, a.V, y_on);
    float s = 0.f, sy = 0.f, t = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float dv = (float)vx[j] - ms, e = policy_exp(dv, a.c_hi, a.c_lo);
      s += e;
      if constexpr (REF) {
        const float du = (float)vy[j] - mys, d = e * (dv - du);
        sy += policy_exp(du, a.c_hi, a.c_lo);
        t += e != 0.f ? d : 0.f;
      }
    }
    s64 += s; sy64 += sy; t64 += t;
  }
  s64 = wave_sum(s64); t64 = wave_sum(t64); sy64 = wave_sum(sy64);
  if ((tid & 63) == 0) { red[tid >> 6][0] = s64; red[tid >> 6][1] = t64; red[tid >> 6][2] = sy64; }
  __syncthreads();
  if (tid == 0) {
    double S = 0.0, Tt = 0.0, Sy = 0.0;
    for (int i = 0; i < NW; ++i) { S += red[i][0]; Tt += red[i][1]; Sy += red[i][2]; }
    finish_row<REF>(a, row, in, ms, S, log_sum(S), mys, REF ? log_sum(Sy) : 0.0, Tt, to_f32(x[in.id]));
  }
}

// Streaming gradient from the rows' statistics.  unless_one: dlogits holds the gradient for g_loss = 1 already, so that value ends it.
template <typename T, bool REF>
__global__ __launch_bounds__(PT) void policy_grad_kernel(PolicyArgs a, const float* g_loss, T* dlogits, int unless_one) {
  constexpr int N = Vec<T>::N;
  const float g = g_loss[0];
  if (unless_one && g == 1.f) return;
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    T* dx = dlogits + row_at(a, row, a.V, a.d_outer);
    const T* x = (const T*)a.logits + row_at(a, row, a.x_stride, a.x_outer);
    const T* y = REF ? (const T*)a.ref + row_at(a, row, a.ref_stride, a.ref_outer) : nullptr;
    const int mis = misalignment<T>(x);
    const bool y_on = !REF || misalignment<T>(y) == mis, d_on = misalignment<T>(dx) == mis;
    const float* st = a.stats + row * BG_POLICY_STATS;
    const float ms = st[0], inv_s = st[1], off = st[4], mys = st[5];
    const bool counts = inv_s != 0.f;                                  // a row that counts has a finite (or NaN) sum
    const float f = g * a.stats[a.rows * BG_POLICY_STATS] * a.inv_t32, slope = f * st[2], w_kl = f * st[3];
    const int64_t id = a.ids[row];
    for (int64_t e0 = (int64_t)tid * N - mis; e0 < a.V; e0 += PT * N) {
      float d[N] = {};
      if (counts) {
        const typename Vec<T>::type vx = row_vector<T>(x, e0, a.V, true);
        typename Vec<T>::type vy;
        if constexpr (REF) vy = row_vector<T>(y, e0, a.V, y_on);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float dv = (float)vx[j] - ms, p = policy_exp(dv, a.c_hi, a.c_lo) * inv_s;
          d[j] = grad_of<REF>(p, REF ? dv - ((float)vy[j] - mys) : 0.f, slope, w_kl, off, a.inv_t32);
          if (e0 + j == id) d[j] += slope;
        }
      }
      store_row_vector<T>(dx, e0, a.V, d_on, d);
    }
  }
}

}  // namespace bg

using namespace bg;

static int policy_check(const char* who, const bg_policy_shape* sh, const void* logits, const void* ref, const int64_t* ids, const float* stats) {
  BG_REQUIRE(sh && logits && ids && stats && ((uintptr_t)stats & 7) == 0, "%s: null argument or stats off the 8-byte grid", who);
  BG_REQUIRE(sh->dtype == BG_F32 || sh->dtype == BG_BF16, "%s: dtype %d", who, sh->dtype);
  BG_REQUIRE(sh->rows > 0 && sh->rows < MAX_ROWS && sh->V > 0 && sh->V < (1ll << 31) && sh->x_stride >= sh->V, "%s: rows=%lld V=%lld stride=%lld",
             who, (long long)sh->rows, (long long)sh->V, (long long)sh->x_stride);
  BG_REQUIRE(!ref || sh->ref_stride >= sh->V, "%s: reference stride %lld", who, (long long)sh->ref_stride);
  BG_REQUIRE(sh->inner >= 0 && (sh->inner == 0 || sh->rows % sh->inner == 0), "%s: groups of %lld of %lld rows", who, (long long)sh->inner,
             (long long)sh->rows);
  if (sh->inner > 0 && sh->inner < sh->rows)
    BG_REQUIRE(sh->x_outer >= 0 && (!ref || sh->ref_outer >= 0) && sh->d_outer >= sh->inner * sh->V, "%s: group strides %lld, %lld, %lld", who,
               (long long)sh->x_outer, (long long)sh->ref_outer, (long long)sh->d_outer);
  BG_REQUIRE(sh->temperature > 0.0 && sh->temperature < 1e6 && sh->temperature > 1e-6, "%s: temperature %g", who, sh->temperature);
  BG_REQUIRE(sh->clip_low >= 0.0 && sh->clip_high >= 0.0, "%s: clip range %g, %g", who, sh->clip_low, sh->clip_high);
  return BG_OK;
}

static PolicyArgs policy_args(const bg_policy_shape* sh, const void* logits, const void* ref, const int64_t* ids, float* stats) {
  PolicyArgs a = {};
  a.logits = logits; a.ref = ref; a.ids = ids; a.stats = stats;
  a.rows = sh->rows; a.V = sh->V; a.x_stride = sh->x_stride; a.ref_stride = sh->ref_stride;
  a.inner = (uint32_t)(sh->inner ? sh->inner : sh->rows);
  if (a.inner < a.rows) { a.x_outer = sh->x_outer; a.ref_outer = sh->ref_outer; a.d_outer = sh->d_outer; }
  a.inv_t = 1.0 / sh->temperature;
  a.clip_low = sh->clip_low; a.clip_high = sh->clip_high; a.kl_coef = sh->kl_coef;
  const double c = 1.4426950408889634 / sh->temperature;
  a.c_hi = __builtin_nextafterf((float)c, 0.f);
  a.c_lo = (float)(c - (double)a.c_hi);
  a.inv_t32 = (float)a.inv_t;
  return a;
}

// Rows of at most NT * NV vectors.  Few threads for short rows; for the usual vocabularies 512, so that two rows share a CU and one's
// loads cover the other's exponentials (with a reference its two rows spill a part of themselves at 128 registers; 1024 x 7 vectors,
// 768 x 9, 256 x 26 and fewer waves with more registers were all slower).
template <typename T, bool REF> static bool policy_row_launch(const PolicyArgs& a, const float* denominator, T* dlogits, hipStream_t st) {
  const int64_t nvec = a.V / Vec<T>::N + 1;
  if (a.V < 2 * Vec<T>::N) return false;
  // reference or gradient rows that lie elsewhere on the 16-byte grid than the logits': the streaming kernels
  const auto same_grid = [&](const void* p, int64_t stride, int64_t outer) {
    return (((uintptr_t)a.logits ^ (uintptr_t)p) & 15) == 0 && (a.x_stride - stride) * (int64_t)sizeof(T) % 16 == 0 &&
           (a.x_outer - outer) * (int64_t)sizeof(T) % 16 == 0;
  };
  if (REF && !same_grid(a.ref, a.ref_stride, a.ref_outer)) return false;
  if (dlogits && !same_grid(dlogits, a.V, a.d_outer)) return false;
  const int64_t groups = a.rows / a.inner;
  if (groups > 65535) return false;
  const dim3 grid(a.inner, (unsigned)groups);
  if (nvec <= 256 * 2) hipLaunchKernelGGL((policy_row_kernel<T, REF, 256, 2>), grid, dim3(256), 0, st, a, denominator, dlogits);
  else if (nvec <= 256 * 8) hipLaunchKernelGGL((policy_row_kernel<T, REF, 256, 8>), grid, dim3(256), 0, st, a, denominator, dlogits);
  else if (nvec <= 512 * 13) hipLaunchKernelGGL((policy_row_kernel<T, REF, 512, 13>), grid, dim3(512), 0, st, a, denominator, dlogits);
  else if (nvec <= 1024 * 13) hipLaunchKernelGGL((policy_row_kernel<T, REF, 1024, 13>), grid, dim3(1024), 0, st, a, denominator, dlogits);
  else return false;
  return true;
}

template <typename T, bool REF>
static void policy_grad_launch(const PolicyArgs& a, const float* g_loss, T* dlogits, int unless_one, hipStream_t st) {
  const int64_t most = unless_one ? 2048 : a.rows;                     // a launch that may have nothing to do: few workgroups
  hipLaunchKernelGGL((policy_grad_kernel<T, REF>), dim3((unsigned)(a.rows < most ? a.rows : most)), dim3(PT), 0, st, a, g_loss, dlogits, unless_one);
}

template <typename T, bool REF> static int policy_fwd(const PolicyArgs& a, const float* denominator, T* dlogits, hipStream_t st) {
  if (dlogits && !denominator && (a.rows > NORM_ROWS || a.V / Vec<T>::N + 1 > 256 * 8)) hipLaunchKernelGGL(policy_norm_kernel, dim3(1), dim3(1024), 0, st, a);
  if (policy_row_launch<T, REF>(a, denominator, dlogits, st)) return dlogits ? 1 : 0;
  hipLaunchKernelGGL((policy_rows_kernel<T, REF>), dim3((unsigned)a.rows), dim3(PT), 0, st, a);
  return 0;
}

extern "C" int bg_policy_loss_fwd(const bg_policy_shape* sh, const void* logits, const void* ref_logits, const int64_t* ids,
                                  const float* old_logp, const float* ref_logp, const float* advantages, const float* weights,
                                  const float* denominator, float* out_loss, float* out_logp, float* out_kl, float* stats, void* dlogits,
                                  int* has_gradient, void* stream) {
  if (int rc = policy_check("bg_policy_loss_fwd", sh, logits, ref_logits, ids, stats)) return rc;
  BG_REQUIRE(old_logp && advantages && out_loss && out_logp && out_kl, "bg_policy_loss_fwd: null argument");
  BG_REQUIRE(!(ref_logits && ref_logp), "bg_policy_loss_fwd: ref_logits and ref_logp exclude each other");
  BG_REQUIRE(!dlogits || has_gradient, "bg_policy_loss_fwd: dlogits without has_gradient");
  PolicyArgs a = policy_args(sh, logits, ref_logits, ids, stats);
  a.old_logp = old_logp; a.ref_logp = ref_logp; a.adv = advantages; a.weights = weights;
  a.out_logp = out_logp; a.out_kl = out_kl;
  hipStream_t st = (hipStream_t)stream;
  int wrote;
  if (sh->dtype == BG_F32)
    wrote = ref_logits ? policy_fwd<float, true>(a, denominator, (float*)dlogits, st) : policy_fwd<float, false>(a, denominator, (float*)dlogits, st);
  else
    wrote = ref_logits ? policy_fwd<bf16_t, true>(a, denominator, (bf16_t*)dlogits, st) : policy_fwd<bf16_t, false>(a, denominator, (bf16_t*)dlogits, st);
  if (has_gradient) *has_gradient = wrote;
  hipLaunchKernelGGL(policy_total_kernel, dim3(1), dim3(1024), 0, st, a, denominator, out_loss);
  BG_CHECK_LAUNCH("bg_policy_loss_fwd");
  return BG_OK;
}

extern "C" int bg_policy_loss_bwd(const bg_policy_shape* sh, const void* logits, const void* ref_logits, const int64_t* ids,
                                  const float* stats, const float* g_loss, void* dlogits, int has_gradient, void* stream) {
  if (int rc = policy_check("bg_policy_loss_bwd", sh, logits, ref_logits, ids, stats)) return rc;
  BG_REQUIRE(g_loss && dlogits, "bg_policy_loss_bwd: null argument");
  const PolicyArgs a = policy_args(sh, logits, ref_logits, ids, (float*)stats);
  hipStream_t st = (hipStream_t)stream;
  if (sh->dtype == BG_F32) {
    if (ref_logits) policy_grad_launch<float, true>(a, g_loss, (float*)dlogits, has_gradient, st);
    else policy_grad_launch<float, false>(a, g_loss, (float*)dlogits, has_gradient, st);
  } else {
    if (ref_logits) policy_grad_launch<bf16_t, true>(a, g_loss, (bf16_t*)dlogits, has_gradient, st);
    else policy_grad_launch<bf16_t, false>(a, g_loss, (bf16_t*)dlogits, has_gradient, st);
  }
  BG_CHECK_LAUNCH("bg_policy_loss_bwd");
  return BG_OK;
}
