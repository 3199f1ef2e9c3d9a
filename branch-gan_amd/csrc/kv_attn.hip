// Attention over the quantised key / value cache (bg_kv_cache_attn_fwd).
//
// One workgroup per (query row, batch): its four waves take every fourth tile of 32 keys.  A lane scores one key (half of its
// channels), the tile's probabilities go through LDS, and a lane then owns output channels.  Running maximum and sum per wave, the
// four states joined at the end.  All sums in fp32; the held values are exact in fp32.
#include "kv_cache.h"

namespace bg {

template <typename T, int BITS, int DH>
__global__ __launch_bounds__(256) void kv_attn_kernel(KvArgs a, const T* q, int G, int64_t q_sb, int64_t q_sh, int64_t q_st, int max_keys,
                                                      float scale, T* out, int64_t o_sb, int64_t o_sh, int64_t o_st, float* lse) {
  using L = KvTile<BITS, DH>;
  constexpr int PER = DH > 64 ? DH / 64 : 1;
  __shared__ float sh_q[DH], sh_p[4][KV_TILE], sh_m[4], sh_l[4], sh_o[4][DH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int Hq = a.H * G;
  const int t = blockIdx.x / Hq, hq = blockIdx.x % Hq, b = blockIdx.y, h = hq / G;
  for (int i = tid; i < DH; i += 256) sh_q[i] = to_f32(q[b * q_sb + hq * q_sh + t * q_st + i]) * scale;
  __syncthreads();
  const int n = min(a.visible(b, t), max_keys);
  const uint8_t* base = a.data + b * a.c_sb + h * a.c_sh;
  float m = -INFINITY, l = 0.f, o[PER] = {};
  const int key = lane & 31, half = lane >> 5;
  for (int t0 = wave * KV_TILE; t0 < n; t0 += 4 * KV_TILE) {
    const uint8_t* tile = base + (int64_t)(t0 / KV_TILE) * L::BYTES;
    float s = 0.f;
    for (int g = 0; g < L::NG; ++g) {
      float d = 0.f;
      for (int kk = 0; kk < 2; ++kk) {
        const int kg = 2 * half + kk;
        const uint32_t* w = (const uint32_t*)(tile + key * L::KROW + (kg * L::NG + g) * L::WORD);
        for (int e = 0; e < 8; ++e) {
          const int code = BITS == 4 ? (int)((w[0] >> (4 * kv_nibble(e))) & 15u) : (int)((w[e / 4] >> (8 * (e % 4))) & 255u);
          d += sh_q[32 * g + 8 * kg + e] * (float)(code - L::OFF);
        }
      }
      s += d * bf16_bits_to_f32(*(const uint16_t*)(tile + L::KS + L::scale_at(key, g)));
    }
    s += __shfl_xor(s, 32);
    const bool seen = t0 + key < n;
    s = seen ? s : -INFINITY;
    const float mn = fmaxf(m, wave_max(s)), ms = mn == -INFINITY ? 0.f : mn;
    const float p = seen ? expf(s - ms) : 0.f, keep = expf(m - ms);
    l = l * keep + 0.5f * wave_sum(p);                         // both halves of the wave hold the 32 keys
    m = mn;
    if (half == 0) sh_p[wave][key] = p;
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int c = lane + 64 * j;
      if (c < DH) {
        float acc = 0.f;
        const uint32_t* w = (const uint32_t*)(tile + L::V + c * L::VROW);
        for (int k = 0; k < KV_TILE && t0 + k < n; ++k) {
          const int code = BITS == 4 ? (int)((w[k / 8] >> (4 * kv_nibble(k % 8))) & 15u) : (int)((w[k / 4] >> (8 * (k % 4))) & 255u);
          acc += sh_p[wave][k] * (bf16_bits_to_f32(*(const uint16_t*)(tile + L::VS + L::scale_at(k, c / KV_GROUP))) * (float)(code - L::OFF));
        }
        o[j] = o[j] * keep + acc;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  if (lane == 0) { sh_m[wave] = m; sh_l[wave] = l; }
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (lane + 64 * j < DH) sh_o[wave][lane + 64 * j] = o[j];
  __syncthreads();
  float M = -INFINITY, S = 0.f;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, sh_m[w]);
  const float Ms = M == -INFINITY ? 0.f : M;
  float f[4];
  for (int w = 0; w < 4; ++w) { f[w] = expf(sh_m[w] - Ms); S += f[w] * sh_l[w]; }
  for (int c = tid; c < DH; c += 256) {
    float acc = 0.f;
    for (int w = 0; w < 4; ++w) acc += f[w] * sh_o[w][c];
    out[b * o_sb + hq * o_sh + t * o_st + c] = from_f32<T>(n > 0 ? acc / S : 0.f);
  }
  if (lse && tid == 0) lse[((int64_t)b * Hq + hq) * a.T + t] = n > 0 ? M + logf(S) : -INFINITY;
}

}  // namespace bg

using namespace bg;

extern "C" size_t bg_kv_cache_attn_workspace_bytes(const bg_kv_cache*, int, int, int) { return 0; }

extern "C" int bg_kv_cache_attn_fwd(const bg_kv_cache* cache, const void* data, const void* q, int dtype, int Hq, int T, int64_t q_sb,
                                    int64_t q_sh, int64_t q_st, const int32_t* start, const int32_t* counts, int max_keys, float scale,
                                    void* out, int64_t o_sb, int64_t o_sh, int64_t o_st, float* lse, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  if (int rc = kv_check("bg_kv_cache_attn_fwd", cache, data, dtype, T)) return rc;
  BG_REQUIRE(q && out, "bg_kv_cache_attn_fwd: null q / out");
  BG_REQUIRE(Hq > 0 && Hq % cache->H == 0, "bg_kv_cache_attn_fwd: Hq=%d query heads over %d cache heads", Hq, cache->H);
  BG_REQUIRE(max_keys > 0 && max_keys <= cache->capacity, "bg_kv_cache_attn_fwd: max_keys=%d of capacity %d", max_keys, cache->capacity);
  BG_REQUIRE((int64_t)T * Hq < (1ll << 31) && cache->B <= 65535, "bg_kv_cache_attn_fwd: T=%d Hq=%d B=%d", T, Hq, cache->B);
  (void)workspace; (void)workspace_bytes;
  KvArgs a;
  a.data = (uint8_t*)data;
  a.B = cache->B; a.H = cache->H; a.capacity = cache->capacity;
  a.c_sb = cache->c_sb; a.c_sh = cache->c_sh;
  a.start = start; a.counts = counts; a.T = T;
  const int G = Hq / cache->H;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(T * Hq), (unsigned)cache->B);
#define BG_GO(BITS, DH)                                                                                                              \
  if (dtype == BG_F32)                                                                                                               \
    hipLaunchKernelGGL((kv_attn_kernel<float, BITS, DH>), grid, dim3(256), 0, st, a, (const float*)q, G, q_sb, q_sh, q_st, max_keys, \
                       scale, (float*)out, o_sb, o_sh, o_st, lse);                                                                   \
  else                                                                                                                               \
    hipLaunchKernelGGL((kv_attn_kernel<bf16_t, BITS, DH>), grid, dim3(256), 0, st, a, (const bf16_t*)q, G, q_sb, q_sh, q_st,         \
                       max_keys, scale, (bf16_t*)out, o_sb, o_sh, o_st, lse)
  BG_KV_DISPATCH(cache->bits, cache->Dh, BG_GO)
#undef BG_GO
  BG_CHECK_LAUNCH("bg_kv_cache_attn_fwd");
  return BG_OK;
}
