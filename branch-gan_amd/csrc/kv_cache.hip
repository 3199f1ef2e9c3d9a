// The quantised key / value cache: bg_kv_cache_append writes new tokens into it, bg_kv_cache_read gives back the values it holds.
//
// Per (token, head, 32 channels), a = the largest magnitude, L = 7 or 127:
//   s = bf16(a * fp32(1 / L)) (an fp32 product),  c = clamp(round-half-even(x / s), -L, L),  the value held is s * c (exact in fp32: 8 + 7
// bits at most)
// The product is what a tensor divided by a number is on this device (compared for all of [1, 2)), so elementary tensor code
// gives the same cache bit for bit.  bf16(fp32(a / L)) is the other neighbour for 70 (4 bits) and 1 (8 bits) of the 2^23 fp32
// mantissas, where a / L lies halfway between two bf16 numbers to the last bit of fp32 and either is as near; never for bf16 a.
// s is 0 (the group reads as zeros) when it would be subnormal; a group with a NaN, an infinity or a magnitude above 2^127 gets
// s = NaN and reads as NaN, so a broken activation shows instead of turning into a large finite number.
// The code is that of the REAL quotient x / s, not of a rounded one: with r = 1 / s correctly rounded, q0 = x r, q = q0 + (x - q0 s) r
// is the correctly rounded quotient (Markstein).  For bf16 x it lands on k + 1/2 only if the real quotient does (both have 8
// significant bits); for fp32 x the sign of x - q s decides there.  No code needs clamping: s is within 2^-9 of a / L, so |x / s| <
// L + 1/2.  Adding 1.5 * 2^23 + offset rounds q to an integer, half to even, in the float's low bits, where packing takes it from.
//
// Bound by HBM for prompts (bytes in + 0.56 or 1.06 bytes per value out): 16 sequences of up to 2017 tokens, 8 heads of 256, bf16 to
// 4 bits, 289 MB: written in 76 us (3.8 TB/s), read back in 62 (4.7; a copy reaches 4.8).  By launch and latency for one token: 64
// sequences of 16 heads of 64 in 3.4 us, read back in 3.8.
#include "kv_cache.h"

namespace bg {

__device__ __forceinline__ uint16_t f32_to_bf16_bits(float x) {          // round to nearest even, finite x
  const uint32_t u = __float_as_uint(x);
  return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true));
}

// Scale bits of a group from the bits of its largest magnitude (ordered as integers: finite < inf < NaN); rs = 1 / s or 0.
template <int TOP> __device__ __forceinline__ uint16_t group_scale(uint32_t amax_bits, float& s, float& rs) {
  const float a = __uint_as_float(amax_bits);
  uint32_t b = f32_to_bf16_bits(a * (1.0f / TOP));
  if (b < 0x0080u) b = 0;
  const bool broken = amax_bits > 0x7F000000u;
  s = broken ? 0.f : bf16_bits_to_f32(b);
  const float r0 = __builtin_amdgcn_rcpf(s);                    // one step makes it the rounded reciprocal: 1 / s of an 8-bit s stays
  const float r = __builtin_fmaf(__builtin_fmaf(-s, r0, 1.f), r0, r0);      // 2^-33 clear of a tie
  rs = b == 0 || broken ? 0.f : r;
  return broken ? 0x7FC0 : (uint16_t)b;
}

constexpr float KV_MAGIC = 12582912.f;          // 1.5 * 2^23

// The code of x plus OFFSET (0 when rs is 0: x may be anything) in the low bits of KV_MAGIC's integer part: the rest are KV_MAGIC's own bits.
template <typename T, int OFFSET> __device__ __forceinline__ uint32_t code_bits(float x, float s, float rs) {
  const float q0 = x * rs;
  const float e0 = __builtin_fmaf(-q0, s, x);
  float q = __builtin_fmaf(e0, rs, q0);
  if constexpr (sizeof(T) == 4) {
    const float half = q - __builtin_rintf(q);
    if (__builtin_fabsf(half) == 0.5f) {                         // is x on, below or above the border q s ?
      const float e = __builtin_fmaf(-q, s, x);
      if (e != 0.f) q += e > 0.f ? 0.25f : -0.25f;
    }
  }
  return __float_as_uint(q + (KV_MAGIC + (float)OFFSET));
}

// One token per sequence: a thread per (K or V, batch, head, channel).  The 32 lanes of a group share its scale through shuffles;
// K words are put together by 8 lanes, a V code is one nibble of its channel's byte (read, changed, written by its one owner).
template <typename T, int BITS, int DH>
__global__ __launch_bounds__(256) void kv_append_token_kernel(KvArgs a, const T* k, const T* v, int64_t k_sb, int64_t k_sh, int64_t v_sb,
                                                              int64_t v_sh) {
  using L = KvTile<BITS, DH>;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t per = (int64_t)a.B * a.H * DH;
  if (id >= 2 * per) return;                                   // whole groups of 32 lanes (DH is a multiple of 32)
  const bool is_v = id >= per;
  const int64_t j = is_v ? id - per : id;
  const int c = (int)(j % DH), h = (int)((j / DH) % a.H), b = (int)(j / DH / a.H);
  const int pos = a.first(b);
  if (a.count(b) < 1 || pos < 0 || pos >= a.capacity) return;
  const float x = to_f32(is_v ? v[b * v_sb + h * v_sh + c] : k[b * k_sb + h * k_sh + c]);
  uint32_t m = __float_as_uint(x) & 0x7FFFFFFFu;
  m = dpp_max<0xB1>(m);                                        // 1, 2, 4, 8: quad_perm, half row, row mirrors
  m = dpp_max<0x4E>(m);
  m = dpp_max<0x141>(m);
  m = dpp_max<0x140>(m);
  m = max(m, (uint32_t)__shfl_xor((int)m, 16));
  float s, rs;
  const uint16_t sb = group_scale<L::TOP>(m, s, rs);
  const uint32_t code = rs == 0.f ? (uint32_t)L::OFF : code_bits<T, L::OFF>(x, s, rs) & (BITS == 4 ? 15u : 255u);
  uint8_t* tile = a.data + b * a.c_sb + h * a.c_sh + (int64_t)(pos / KV_TILE) * L::BYTES;
  const int key = pos % KV_TILE, g = c / KV_GROUP, kg = (c / 8) % 4;
  if ((c & 31) == 0) *(uint16_t*)(tile + (is_v ? L::VS : L::KS) + L::scale_at(key, g)) = sb;
  if (!is_v) {
    if constexpr (BITS == 4) {
      uint32_t w = code << (4 * kv_nibble(c & 7));
      w |= __shfl_xor(w, 1);
      w |= __shfl_xor(w, 2);
      w |= __shfl_xor(w, 4);
      if ((c & 7) == 0) *(uint32_t*)(tile + key * L::KROW + (kg * L::NG + g) * 4) = w;
    } else {
      tile[key * L::KROW + (kg * L::NG + g) * 8 + (c & 7)] = (uint8_t)code;
    }
  } else {
    uint8_t* word = tile + L::v_word(key >> 3, c);
    if constexpr (BITS == 4) {
      const int nib = kv_nibble(key & 7);
      uint8_t* p = word + (nib >> 1);
      const int sh = 4 * (nib & 1);
      *p = (uint8_t)((*p & ~(15u << sh)) | (code << sh));
    } else {
      word[key & 7] = (uint8_t)code;
    }
  }
}

// Bits of the largest magnitude among 8 numbers; bf16 pairs are compared as packed 16-bit integers.
__device__ __forceinline__ uint32_t max_magnitude(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7FFFFFFFu);
  return m;
}
__device__ __forceinline__ uint32_t max_magnitude(const bf16x8& x) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 u = __builtin_bit_cast(u32x4, x) & 0x7FFF7FFFu;
  // (the casts: a bit cast of a vector element itself reads the first one)
  const u16x2 a = __builtin_elementwise_max(__builtin_bit_cast(u16x2, (uint32_t)u[0]), __builtin_bit_cast(u16x2, (uint32_t)u[1]));
  const u16x2 b = __builtin_elementwise_max(__builtin_bit_cast(u16x2, (uint32_t)u[2]), __builtin_bit_cast(u16x2, (uint32_t)u[3]));
  const uint32_t m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(a, b));
  return max(m << 16, m & 0xFFFF0000u);
}

// 8 neighbouring channels as they come from memory: bf16x8, or float[8]
template <typename T> struct Octet { typedef bf16x8 type; };
template <> struct Octet<float> { struct type { float x[8]; __device__ __forceinline__ float operator[](int i) const { return x[i]; } }; };
__device__ __forceinline__ uint32_t max_magnitude(const Octet<float>::type& x) { return max_magnitude(x.x); }
template <typename T, bool VEC> __device__ __forceinline__ typename Octet<T>::type load_octet(const T* p) {
  typename Octet<T>::type r;
  if constexpr (sizeof(T) == 2) {
    if constexpr (VEC) {
      r = *(const bf16x8*)p;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = p[j];
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 v;
      if constexpr (VEC) v = *(const f32x4*)(p + 4 * h);
      else v = f32x4{p[4 * h], p[4 * h + 1], p[4 * h + 2], p[4 * h + 3]};
#pragma unroll
      for (int j = 0; j < 4; ++j) r.x[4 * h + j] = v[j];
    }
  }
  return r;
}

template <typename T, bool VEC> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = from_f32<T>(x[j]);
  } else if constexpr (sizeof(T) == 2) {
    bf16x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (bf16_t)x[j];
    *(bf16x8*)p = r;
  } else {
    f32x4 r0, r1;
#pragma unroll
    for (int j = 0; j < 4; ++j) { r0[j] = x[j]; r1[j] = x[4 + j]; }
    *(f32x4*)p = r0;
    *(f32x4*)(p + 4) = r1;
  }
}

// Several tokens: 128 threads take the keys, or (the other half of the grid) the values, of 256 / DH tiles; a thread the 8 keys x 8
// channels of one word column (so that the transposition of V stays in its registers).  A tile's part is put together in LDS and
// leaves as whole 16-byte rows; a tile that the new tokens cover only in part is read first, and the codes and scales of its other
// keys go back as they were.  (Keys and values apart: twice the workgroups of half the registers; 8 x 777 tokens of 12 heads of 64
// in fp32 17.9 -> 15.8 us.)
template <typename T, int BITS, int DH, bool VEC, int KV>
__device__ __forceinline__ void append_tiles(const KvArgs& a, const T* src0, int64_t sb, int64_t sh, int64_t st, int blk, int blocks_per_head,
                                             uint8_t* image) {
  using L = KvTile<BITS, DH>;
  constexpr int TPW = 256 / DH, NTH = DH / 2, U = DH / 8;
  constexpr int CODES = KV ? L::V : 0, CODE_BYTES = L::V, SCALES = KV ? L::VS : L::KS, SCALE_BYTES = L::VS - L::KS;
  constexpr int PART = CODE_BYTES + SCALE_BYTES;                // this part of a tile, codes then scales
  const int tid = threadIdx.x, lt = tid / NTH, ti = tid % NTH, u = ti % U, oct = ti / U;
  const int bh = blk / blocks_per_head, b = bh / a.H, h = bh % a.H;
  const int start = a.first(b), count = a.count(b);
  // new tokens that fit: positions lo .. hi - 1
  const int64_t hi64 = (int64_t)start + count;
  const int lo = start < 0 ? 0 : min(start, a.capacity), hi = (int)(hi64 < 0 ? 0 : (hi64 > a.capacity ? a.capacity : hi64));
  const int tile = lo / KV_TILE + (blk % blocks_per_head) * TPW + lt;
  const bool any = (int64_t)tile * KV_TILE < hi && lo < hi;    // tiles past the last token: nothing to do
  const int k0 = any ? tile * KV_TILE : 0;
  const bool whole = k0 >= lo && k0 + KV_TILE <= hi;
  uint8_t* out = a.data + b * a.c_sb + h * a.c_sh + (int64_t)tile * L::BYTES;
  uint8_t* img = image + lt * PART;
  const auto at = [](int i) { return 16 * i < CODE_BYTES ? CODES + 16 * i : SCALES + 16 * i - CODE_BYTES; };
  if (any && !whole)
    for (int i = ti; i < PART / 16; i += NTH) *(uint4*)(img + 16 * i) = *(const uint4*)(out + at(i));
  __syncthreads();
  if (any) {
    const int g = u / 4, kg = u % 4;
    const int key0 = k0 + 8 * oct;
    const T* src = src0 + b * sb + h * sh + 8 * u;
    // rows outside the new tokens are read as the nearest one inside, and what comes of them is not stored
    typename Octet<T>::type x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = load_octet<T, VEC>(src + (int64_t)(min(max(key0 + e, lo), hi - 1) - start) * st);
    // words as sums of shifted code bits: what KV_MAGIC's bits add up to is taken off beforehand; 8-bit codes run through an offset
    // of 128, so that no byte borrows from the next, and lose it to a flip of every top bit
    constexpr int OFFSET = BITS == 4 ? L::OFF : 128;
    constexpr uint32_t START = 0u - (BITS == 4 ? 0x4B400000u * 0x11111111u : 0x4B400000u * 0x01010101u);
    constexpr uint32_t FLIP = BITS == 4 ? 0u : 0x80808080u;
    uint32_t vw[8][BITS / 4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int w = 0; w < BITS / 4; ++w) vw[j][w] = START;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = key0 + e >= lo && key0 + e < hi;
      uint32_t m = max_magnitude(x[e]);
      m = dpp_max<0xB1>(m);                                    // the 4 lanes of a group are adjacent
      m = dpp_max<0x4E>(m);
      float s, rs;
      const uint16_t scale = group_scale<L::TOP>(m, s, rs);
      const int key = 8 * oct + e;
      if (in && kg == 0) *(uint16_t*)(img + CODE_BYTES + L::scale_at(key, g)) = scale;
      uint32_t kw[BITS / 4];
#pragma unroll
      for (int w = 0; w < BITS / 4; ++w) kw[w] = START;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = (float)x[e][j];
      if (__any(scale == 0x7FC0)) {                            // a broken group in this wave: its NaNs must not reach the sums
        asm volatile("");                                      // (a branch, not selects on every element of every call)
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = scale == 0x7FC0 ? 0.f : f[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t code = code_bits<T, OFFSET>(f[j], s, rs);
        uint32_t& w = KV == 0 ? kw[BITS == 4 ? 0 : j / 4] : vw[j][BITS == 4 ? 0 : e / 4];
        w += code << (BITS == 4 ? 4 * kv_nibble(KV == 0 ? j : e) : 8 * ((KV == 0 ? j : e) % 4));
      }
      if (KV == 0 && in) {
        uint32_t* p = (uint32_t*)(img + key * L::KROW + (kg * L::NG + g) * L::WORD);
#pragma unroll
        for (int w = 0; w < BITS / 4; ++w) p[w] = kw[w] ^ FLIP;
      }
    }
    if constexpr (KV == 1) {
      uint32_t mask[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = key0 + e >= lo && key0 + e < hi;
        if constexpr (BITS == 4) mask[0] |= in ? 15u << (4 * kv_nibble(e)) : 0u;
        else mask[e / 4] |= in ? 255u << (8 * (e % 4)) : 0u;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t* p = (uint32_t*)(img + L::v_word(oct, 8 * u + j) - L::V);
#pragma unroll
        for (int w = 0; w < BITS / 4; ++w) {
          const uint32_t c = vw[j][w] ^ FLIP;
          p[w] = whole ? c : ((p[w] & ~mask[w]) | (c & mask[w]));
        }
      }
    }
  }
  __syncthreads();
  if (any)
    for (int i = ti; i < PART / 16; i += NTH) *(uint4*)(out + at(i)) = *(const uint4*)(img + 16 * i);
}

template <typename T, int BITS, int DH, bool VEC>
__global__ __launch_bounds__(128) void kv_append_tiles_kernel(KvArgs a, const T* k, const T* v, int64_t k_sb, int64_t k_sh, int64_t k_st,
                                                              int64_t v_sb, int64_t v_sh, int64_t v_st, int blocks_per_head) {
  __shared__ __attribute__((aligned(16))) uint8_t image[256 / DH * KvTile<BITS, DH>::BYTES / 2];
  const int half = (int)(gridDim.x / 2);
  if ((int)blockIdx.x < half) append_tiles<T, BITS, DH, VEC, 0>(a, k, k_sb, k_sh, k_st, blockIdx.x, blocks_per_head, image);
  else append_tiles<T, BITS, DH, VEC, 1>(a, v, v_sb, v_sh, v_st, blockIdx.x - half, blocks_per_head, image);
}

// Values back: the same 8 x 8 blocks, codes straight from memory.  Row t of the output is position start + t; rows at or past the
// sequence's count, and positions outside the cache, are zeros.
template <typename T, int BITS, int DH, bool VEC, int KV>
__device__ __forceinline__ void read_tiles(const KvArgs& a, T* out0, int64_t o_sb, int64_t o_sh, int64_t o_st, int blk, int blocks_per_head) {
  using L = KvTile<BITS, DH>;
  constexpr int TPW = 256 / DH, NTH = DH / 2, U = DH / 8;
  const int tid = threadIdx.x, lt = tid / NTH, ti = tid % NTH, u = ti % U, oct = ti / U;
  const int bh = blk / blocks_per_head, b = bh / a.H, h = bh % a.H;
  const int64_t start = a.first(b);
  const int count = a.count(b);
  const int64_t floor_tile = start >= 0 ? start / KV_TILE : -((KV_TILE - 1 - start) / KV_TILE);
  const int64_t tile = floor_tile + (int64_t)(blk % blocks_per_head) * TPW + lt;
  const int64_t pos0 = tile * KV_TILE + 8 * oct;               // this thread's 8 positions
  if (pos0 + 8 <= start || pos0 >= start + a.T) return;
  const int g = u / 4, kg = u % 4;
  const uint8_t* t = a.data + b * a.c_sb + h * a.c_sh + tile * L::BYTES;
  uint32_t w[8][BITS / 4] = {};
  uint16_t sc[8] = {};
  if (tile >= 0 && tile * KV_TILE < a.capacity && pos0 < start + count) {      // the tile exists and holds rows that are asked for
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t* p = KV == 0 ? (const uint32_t*)(t + (8 * oct + i) * L::KROW + (kg * L::NG + g) * L::WORD)
                                  : (const uint32_t*)(t + L::v_word(oct, 8 * u + i));
#pragma unroll
      for (int q = 0; q < BITS / 4; ++q) w[i][q] = p[q];
      sc[i] = *(const uint16_t*)(t + (KV ? L::VS : L::KS) + L::scale_at(8 * oct + i, g));
    }
  }
  T* out = out0 + b * o_sb + h * o_sh + 8 * u;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t pos = pos0 + e;
    const bool held = pos >= start && pos < start + count && pos >= 0 && pos < a.capacity;
    const float s = bf16_bits_to_f32(sc[e]);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int row = KV == 0 ? e : j, el = KV == 0 ? j : e;   // K words run along the channels, V words along the keys
      int code;
      if constexpr (BITS == 4) code = (int)((w[row][0] >> (4 * kv_nibble(el))) & 15u) - L::OFF;
      else code = (int8_t)(w[row][el / 4] >> (8 * (el % 4)));
      x[j] = held ? s * (float)code : 0.f;
    }
    const int64_t row = pos - start;
    if (row >= 0 && row < a.T) store8<T, VEC>(out + row * o_st, x);
  }
}

template <typename T, int BITS, int DH, bool VEC>
__global__ __launch_bounds__(128) void kv_read_kernel(KvArgs a, T* k, T* v, int64_t o_sb, int64_t o_sh, int64_t o_st, int blocks_per_head) {
  const int half = (int)(gridDim.x / 2);
  if ((int)blockIdx.x < half) read_tiles<T, BITS, DH, VEC, 0>(a, k, o_sb, o_sh, o_st, blockIdx.x, blocks_per_head);
  else read_tiles<T, BITS, DH, VEC, 1>(a, v, o_sb, o_sh, o_st, blockIdx.x - half, blocks_per_head);
}

int kv_check(const char* who, const bg_kv_cache* c, const void* data, int dtype, int64_t T) {
  BG_REQUIRE(c && data, "%s: null cache", who);
  BG_REQUIRE(c->bits == 4 || c->bits == 8, "%s: bits=%d (4 or 8)", who, c->bits);
  BG_REQUIRE(c->Dh == 32 || c->Dh == 64 || c->Dh == 128 || c->Dh == 256, "%s: Dh=%d (32, 64, 128 or 256)", who, c->Dh);
  BG_REQUIRE(dtype == BG_F32 || dtype == BG_BF16, "%s: dtype %d", who, dtype);
  BG_REQUIRE(c->B > 0 && c->H > 0 && c->capacity > 0 && c->capacity < (1 << 30) && T > 0 && T < (1 << 30),
             "%s: B=%d H=%d capacity=%d T=%lld", who, c->B, c->H, c->capacity, (long long)T);
  const int64_t tiles = cdiv(c->capacity, KV_TILE), bytes = tiles * (int64_t)bg_kv_cache_tile_bytes(c->bits, c->Dh);
  BG_REQUIRE(((uintptr_t)data & 15) == 0 && c->c_sb % 16 == 0 && c->c_sh % 16 == 0, "%s: the cache must lie on 16-byte boundaries", who);
  // no two (batch, head) share a byte: one of the two strides steps over all that the other reaches
  const int64_t sb = c->B == 1 ? 0 : c->c_sb, sh = c->H == 1 ? 0 : c->c_sh;
  BG_REQUIRE((c->H == 1 || sh >= bytes) && (c->B == 1 || sb >= bytes) && (c->H == 1 || c->B == 1 || sb - bytes >= (c->H - 1) * sh || sh - bytes >= (c->B - 1) * sb),
             "%s: cache strides %lld, %lld overlap (%lld bytes per head)", who, (long long)c->c_sb, (long long)c->c_sh, (long long)bytes);
  return BG_OK;
}

}  // namespace bg

using namespace bg;

extern "C" size_t bg_kv_cache_tile_bytes(int bits, int Dh) {
  if ((bits != 4 && bits != 8) || (Dh != 32 && Dh != 64 && Dh != 128 && Dh != 256)) return 0;
  return (size_t)(2 * KV_TILE * Dh * bits / 8 + 2 * KV_TILE * (Dh / KV_GROUP) * 2);
}

static KvArgs kv_args(const bg_kv_cache* c, void* data, const int32_t* start, const int32_t* counts, int T) {
  KvArgs a;
  a.data = (uint8_t*)data;
  a.B = c->B; a.H = c->H; a.capacity = c->capacity;
  a.c_sb = c->c_sb; a.c_sh = c->c_sh;
  a.start = start; a.counts = counts; a.T = T;
  return a;
}

static bool aligned16(const void* p, int64_t s0, int64_t s1, int64_t s2, int e) {
  return (((uintptr_t)p | (uintptr_t)(s0 * e) | (uintptr_t)(s1 * e) | (uintptr_t)(s2 * e)) & 15) == 0;
}

extern "C" int bg_kv_cache_append(const bg_kv_cache* cache, void* data, const void* k, const void* v, int dtype, int T,
                                  int64_t k_sb, int64_t k_sh, int64_t k_st, int64_t v_sb, int64_t v_sh, int64_t v_st,
                                  const int32_t* start, const int32_t* counts, void* stream) {
  if (int rc = kv_check("bg_kv_cache_append", cache, data, dtype, T)) return rc;
  BG_REQUIRE(k && v, "bg_kv_cache_append: null k / v");
  const KvArgs a = kv_args(cache, data, start, counts, T);
  hipStream_t st = (hipStream_t)stream;
  const int e = dtype == BG_F32 ? 4 : 2;
  const bool vec = aligned16(k, k_sb, k_sh, k_st, e) && aligned16(v, v_sb, v_sh, v_st, e);
  const int64_t heads = (int64_t)cache->B * cache->H;
  if (T == 1) {
    const int64_t blocks = cdiv(2 * heads * cache->Dh, 256);
    BG_REQUIRE(blocks < (1ll << 24), "bg_kv_cache_append: %lld blocks", (long long)blocks);        // a launch has fewer than 2^32 threads
#define BG_GO(BITS, DH)                                                                                                              \
  if (dtype == BG_F32)                                                                                                               \
    hipLaunchKernelGGL((kv_append_token_kernel<float, BITS, DH>), dim3((unsigned)blocks), dim3(256), 0, st, a, (const float*)k,      \
                       (const float*)v, k_sb, k_sh, v_sb, v_sh);                                                                     \
  else                                                                                                                               \
    hipLaunchKernelGGL((kv_append_token_kernel<bf16_t, BITS, DH>), dim3((unsigned)blocks), dim3(256), 0, st, a, (const bf16_t*)k,    \
                       (const bf16_t*)v, k_sb, k_sh, v_sb, v_sh)
    BG_KV_DISPATCH(cache->bits, cache->Dh, BG_GO)
#undef BG_GO
    BG_CHECK_LAUNCH("bg_kv_cache_append");
    return BG_OK;
  }
  const int64_t tiles = cdiv((int64_t)T + KV_TILE - 1, KV_TILE);            // T tokens at any offset touch at most this many
  const int64_t per_head = cdiv(tiles, 256 / cache->Dh), blocks = 2 * per_head * heads;     // keys, values
  BG_REQUIRE(blocks < (1ll << 25), "bg_kv_cache_append: %lld blocks", (long long)blocks);
#define BG_GO2(TT, BITS, DH, VEC)                                                                                                   \
  hipLaunchKernelGGL((kv_append_tiles_kernel<TT, BITS, DH, VEC>), dim3((unsigned)blocks), dim3(128), 0, st, a, (const TT*)k,        \
                     (const TT*)v, k_sb, k_sh, k_st, v_sb, v_sh, v_st, (int)per_head)
#define BG_GO(BITS, DH)                                                                                    \
  if (dtype == BG_F32) { if (vec) BG_GO2(float, BITS, DH, true); else BG_GO2(float, BITS, DH, false); }    \
  else { if (vec) BG_GO2(bf16_t, BITS, DH, true); else BG_GO2(bf16_t, BITS, DH, false); }
  BG_KV_DISPATCH(cache->bits, cache->Dh, BG_GO)
#undef BG_GO
#undef BG_GO2
  BG_CHECK_LAUNCH("bg_kv_cache_append");
  return BG_OK;
}

extern "C" int bg_kv_cache_read(const bg_kv_cache* cache, const void* data, void* k, void* v, int dtype, int T, int64_t o_sb, int64_t o_sh,
                                int64_t o_st, const int32_t* start, const int32_t* counts, void* stream) {
  if (int rc = kv_check("bg_kv_cache_read", cache, data, dtype, T)) return rc;
  BG_REQUIRE(k && v, "bg_kv_cache_read: null k / v");
  const KvArgs a = kv_args(cache, (void*)data, start, counts, T);
  hipStream_t st = (hipStream_t)stream;
  const int e = dtype == BG_F32 ? 4 : 2;
  const bool vec = aligned16(k, o_sb, o_sh, o_st, e) && aligned16(v, 0, 0, 0, e);
  const int64_t tiles = cdiv((int64_t)T + KV_TILE - 1, KV_TILE);
  const int64_t per_head = cdiv(tiles, 256 / cache->Dh), blocks = 2 * per_head * cache->B * cache->H;
  BG_REQUIRE(blocks < (1ll << 25), "bg_kv_cache_read: %lld blocks", (long long)blocks);
#define BG_GO2(TT, BITS, DH, VEC)                                                                                                 \
  hipLaunchKernelGGL((kv_read_kernel<TT, BITS, DH, VEC>), dim3((unsigned)blocks), dim3(128), 0, st, a, (TT*)k, (TT*)v, o_sb,      \
                     o_sh, o_st, (int)per_head)
#define BG_GO(BITS, DH)                                                                                    \
  if (dtype == BG_F32) { if (vec) BG_GO2(float, BITS, DH, true); else BG_GO2(float, BITS, DH, false); }    \
  else { if (vec) BG_GO2(bf16_t, BITS, DH, true); else BG_GO2(bf16_t, BITS, DH, false); }
  BG_KV_DISPATCH(cache->bits, cache->Dh, BG_GO)
#undef BG_GO
#undef BG_GO2
  BG_CHECK_LAUNCH("bg_kv_cache_read");
  return BG_OK;
}
