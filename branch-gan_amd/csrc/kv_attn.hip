// Attention over the quantised key / value cache (bg_kv_cache_attn_fwd).
//
// Mathematics.  With codes c and scales s per 32 channels g,
//   q . k = sum_g s_kg (q_g . c_kg)         o_ch = sum_k (p_k s_vg) c_v,ch
// so the codes themselves are the matrix operands: as bf16 they are exact (see unpack_codes), the scales join in fp32 - on the scores after the product, on the probabilities before it.  Nothing held is rounded again.  bf16
// queries are exact operands; fp32 queries go in as three bf16 pieces (24 bits), probabilities as two (16 bits) for bf16 outputs - at most
// 2^-17 of a probability, 1 / 256 of half a step of the output, where three would cost 7 % (8 sequences of 65537 keys 117 -> 125
// us) - or as three.
//
// Layouts.  One wave takes 4 tiles (128 keys) per turn with v_mfma_f32_16x16x32_bf16 (rows of A x columns of B, 32 deep; lane = (n =
// lane % 16, j = lane / 16) holds 8 elements of A's row n and of B's column n, and results (rows 4 j + r, column n)).
//   Many rows (kv_attn_kernel: prompts, many query heads to a cache head).  Scores: A = K codes, row rr = key 4 t + rr % 4 of tile rr / 4;
//     B = queries, column n = a row; the channel groups are separate products.  Lane (n, j) gets row n's scores against the 32 keys of
//     tile j, which as probabilities are already the A operand of the output, whose B = V codes: P never leaves its lane, no LDS.
//   Few rows (kv_decode_kernel: at most 16 pairs (row, channel group) - the groups' partial products are columns of their own, so
//     that a group costs a lane, not an instruction).  Scores: A = queries, row of pair p zero outside its group; B = K codes, column
//     n = key 8 n + t of the turn: lane (n, j) gets RR = 1, 2 or 4 pairs' scores for 8 keys, a quarter of the vector work of the layout
//     above where RR is 1 (one query head per cache head up to heads of 128).  Sums over a row's pairs by lane swaps.  The
//     probabilities go through LDS once (16 bytes per pair and octet of keys) to become A operands.
//   In both 4-bit codes go from memory to operands of bf16 queries with one shift and one mask-or per pair; signed codes (4 bits with
//   fp32 queries, 8 bits) take a conversion each.
// Softmax.  The running maximum of a row moves only when a score passes it by 2^8 (probabilities stay below 256), so that
//   the usual turn needs no exchange between lanes for it.
// Work.  Four waves per workgroup take turns round robin; the key range is split over workgroups when there are too few of
//   them to fill 256 CUs (kv_attn_plan), the partial states joined by a second kernel.
// Bound.  One token: HBM, 0.5625 or 1.0625 bytes per cached value.  Measured: 8 sequences of 65537 keys, 8 heads of 128, four query heads
//   each, 4 bits, 604 MB in 117 us (5.2 TB/s; the launches of the call included, the part that stays in the last-level cache too);
//   64 uneven sequences of up to 2047 keys, 16 heads of 64, 87 MB in 22 us (4.0 TB/s); 16 of up to 4001, 8 heads of 256, 8 bits,
//   float32 queries, 162 MB in 41 + 5 us (3.5 TB/s: the longest sequences finish alone).  Many rows: vector work - 128 keys x 16 rows
//   of 64 channels are some 930 vector instructions of a wave (exponentials, scales, splitting P, unpacking) against 64 matrix
//   ones; 67 tokens of 4 sequences of 16 heads against about 2000 keys in 20 + 4 us, of which that
//   work is less than half: two turns a wave do not hide the prologue, the joins and every tile's own reading of the keys.
#include "kv_cache.h"

namespace bg {

constexpr int KW = 4;                       // waves per workgroup
constexpr int KV_TURN = 4 * KV_TILE;        // keys a wave takes per turn

struct KvAttnArgs {
  KvArgs kv;
  const void* q;
  int64_t q_sb, q_sh, q_st;
  void* out;
  int64_t o_sb, o_sh, o_st;
  float* lse;
  float* part;                              // [row][split][Dh + 2]: unnormalised output, maximum (log2), sum
  int G, max_keys, splits, rows_per_tile;
  bool negate, q_vec;                       // negative scale; queries on the 16-byte grid
  float scale_log2;                         // |scale| log2(e), times the unit of the codes
};

// Most (returned) and fewest keys that the rows of the tile at row0 see.
__device__ __forceinline__ int tile_keys(const KvAttnArgs& a, int b, int row0, int& fewest) {
  const int count = a.kv.count(b), last = min(row0 + a.rows_per_tile, a.kv.T * a.G) - 1;
  const int t_lo = a.kv.T > 1 ? row0 / a.G : 0, t_hi = a.kv.T > 1 ? last / a.G : 0;
  fewest = t_hi < count ? min(a.kv.visible(b, t_lo), a.max_keys) : 0;
  return t_lo < count ? min(a.kv.visible(b, min(t_hi, count - 1)), a.max_keys) : 0;
}

template <int N> __device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = ((const uint4*)p)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const uint2 v = *(const uint2*)p;
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *(const uint32_t*)p;
  }
}

// 8 neighbouring channels of a query; vec: on the 16-byte grid
template <typename T> __device__ __forceinline__ void load_query(const T* q, bool vec, bool real, bool negate, float (&x)[8]) {
  if (vec && real) {
    if constexpr (sizeof(T) == 2) {
      const bf16x8 v = *(const bf16x8*)q;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
    } else {
      const f32x4 u = *(const f32x4*)q, v = *(const f32x4*)(q + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { x[e] = u[e]; x[4 + e] = v[e]; }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = real ? to_f32(q[e]) : 0.f;
  }
  if (negate) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = -x[e];
  }
}

union Frag {
  uint32_t u[4];
  bf16x8 v;
};

// 8 codes -> 8 bf16 numbers (code + offset) / unit.
// 4 bits, bf16 queries: the nibble as bits 3..6 of a bf16 in [16, 32) is 16 + stored code = code + 24 - a shift and a mask-or per pair.
// (The two constants sit in a vector and a scalar register: as literals they would make the mask-or two instructions.)
// What the offset adds to an output is taken off turn by turn (step by step where there are many rows): sums that kept it grow with
// the number of keys while the output, an average, shrinks - over 65536 random keys 18 % of the bf16 outputs then were not the rounded
// ones, now 0.8 %.  16 subtractions a turn at heads of 64 (64 sequences 21.8 -> 22.2 us, 67 tokens 21.7 -> 21.9); signed codes
// for bf16 queries would cost 26.3 and 23.5.
// To a score, a product of its own for every key, the offset adds rounding of some 24 sum|q| 2^-24 times the key's scale s: a
// hundred-thousandth of what half a code step, s / 2 per channel, may be off in the cache already (2e-7 of a key's largest magnitude at
// heads of 64 and queries of size 1).
// 4 bits, fp32 queries: sums of c + 24 would cost 2 to 3 bits that fp32 results show (error 4e-6 against 4e-7), so the codes come
// signed, by the instruction that reads a signed nibble as sixteenths - twice the instructions.
// 8 bits: signed bytes, converted (a conversion that takes its byte from the word, and half a pack).
template <typename T, int BITS> constexpr float kv_offset() { return BITS == 4 && sizeof(T) == 2 ? 24.f : 0.f; }
template <typename T, int BITS> constexpr float kv_unit() { return BITS == 4 && sizeof(T) == 4 ? 16.f : 1.f; }
struct Nibbles {
  uint32_t mask, base;
  __device__ __forceinline__ Nibbles() : mask(0x00780078u), base(0x41804180u) { asm volatile("" : "+v"(mask), "+s"(base)); }
};
template <typename T, int BITS> __device__ __forceinline__ bf16x8 unpack_codes(const uint32_t* w, const Nibbles& nb) {
  Frag f;
  if constexpr (BITS == 4 && sizeof(T) == 2) {
    f.u[0] = ((w[0] << 3) & nb.mask) | nb.base;
    f.u[1] = ((w[0] >> 1) & nb.mask) | nb.base;
    f.u[2] = ((w[0] >> 5) & nb.mask) | nb.base;
    f.u[3] = ((w[0] >> 9) & nb.mask) | nb.base;
  } else if constexpr (BITS == 4) {
    const uint32_t lo = w[0] ^ 0x88888888u;                // code + 8 to two's complement
    uint32_t hi = lo >> 4;
    asm volatile("" : "+v"(hi));                           // (one shift for four nibbles: the conversion picks its byte)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = i & 1 ? hi : lo;
      f.v[2 * i] = (bf16_t)__builtin_amdgcn_cvt_off_f32_i4((int)((x >> (8 * (i / 2))) & 255u));
      f.v[2 * i + 1] = (bf16_t)__builtin_amdgcn_cvt_off_f32_i4((int)((x >> (8 * (i / 2) + 16)) & 255u));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = (bf16_t)(float)(int8_t)(w[i / 4] >> (8 * (i % 4)));
  }
  return f.v;
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// x -> N bf16 pieces that add up to it (8 bits each)
template <int N> __device__ __forceinline__ void split_bf16(const float (&x)[8], bf16x8 (&piece)[N]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    f32x2 rest = {x[2 * h], x[2 * h + 1]};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bf16x2 p = __builtin_convertvector(rest, bf16x2);
      piece[i][2 * h] = p[0];
      piece[i][2 * h + 1] = p[1];
      if (i + 1 < N) {
        const uint32_t u = __builtin_bit_cast(uint32_t, p);
        rest[0] -= bf16_lo(u);
        rest[1] -= bf16_hi(u);
      }
    }
  }
}

template <int CTRL> __device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
// over the 16 lanes n of a lane group, the result in all of them
__device__ __forceinline__ float sum16(float x) {
  x += dpp<0xB1>(x);                                     // quad_perm 1,0,3,2 and 2,3,0,1, mirrors of 8 and of 16 lanes
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  return x + dpp<0x140>(x);
}
__device__ __forceinline__ float max16(float x) {
  x = fmaxf(x, dpp<0xB1>(x));
  x = fmaxf(x, dpp<0x4E>(x));
  x = fmaxf(x, dpp<0x141>(x));
  return fmaxf(x, dpp<0x140>(x));
}
// over lane groups j, j ^ 1 (and j ^ 2)
__device__ __forceinline__ float sum_j1(float x) {
  const auto v = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(v[0]) + __uint_as_float(v[1]);
}
__device__ __forceinline__ float sum_j2(float x) {
  const auto v = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(v[0]) + __uint_as_float(v[1]);
}
__device__ __forceinline__ float bf16_at(const uint32_t* w, int i) { return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]); }

// Joins the states of the workgroup's waves and writes the rows row0 .. row0 + ROWS - 1, or the split's partial state.
template <typename T, int DH, int ROWS, typename Shared>
__device__ __forceinline__ void write_rows(const KvAttnArgs& a, Shared& sh, int b, int h, int row0, int split) {
  const int R = a.kv.T * a.G;
  for (int i = threadIdx.x; i < ROWS * DH; i += 64 * KW) {
    const int row = i / DH, ch = i % DH, rr = row0 + row;
    if (rr >= R) break;
    float M = sh.m[0][row];
#pragma unroll
    for (int w = 1; w < KW; ++w) M = fmaxf(M, sh.m[w][row]);
    const float Ms = M == -INFINITY ? 0.f : M;
    float S = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const float f = __builtin_amdgcn_exp2f(sh.m[w][row] - Ms);
      S += f * sh.l[w][row];
      o += f * sh.o[w][row][ch];
    }
    if (a.splits == 1) {
      const int t = rr / a.G, hq = h * a.G + rr - t * a.G;
      const bool any = a.kv.visible(b, t) > 0;
      ((T*)a.out)[b * a.o_sb + hq * a.o_sh + t * a.o_st + ch] = from_f32<T>(any ? o / S : 0.f);
      if (a.lse && ch == 0) a.lse[((int64_t)b * a.kv.H * a.G + hq) * a.kv.T + t] = any ? (M + __log2f(S)) * 0.6931471805599453f : -INFINITY;
    } else {
      float* part = a.part + ((((int64_t)b * a.kv.H + h) * R + rr) * a.splits + split) * (DH + 2);
      part[ch] = o;
      if (ch == 0) { part[DH] = M; part[DH + 1] = S; }
    }
  }
}

// The turns of a split: the first `more` of them take one more than the rest.
__device__ __forceinline__ void split_turns(const KvAttnArgs& a, int split, int turns, int& begin, int& end) {
  const int each = (int)((uint32_t)turns / (uint32_t)a.splits), more = turns - each * a.splits;
  begin = split * each + min(split, more);
  end = begin + each + (split < more ? 1 : 0);
}

// ---- few rows --------------------------------------------------------------------------------------------------------------------
template <typename T, int BITS, int DH, int RR> struct DecodeShape {
  static constexpr int NG = DH / KV_GROUP, ROWS = 4 * RR / NG, PAIRS = 4 * RR;
  static constexpr int RL = RR > NG ? RR / NG : 1;                           // rows a lane holds scores of
  // a turn's codes in flight, K and V: whole (16 registers each at most), halves or quarters
  static constexpr int KT = DH * BITS <= 256 ? 8 : DH * BITS <= 1024 ? 4 : 2, VT = KT / 2;
  // waves per SIMD: small heads are bound by vector work and latency as much as by memory.  At RR = 2 that leaves <fp32, 4, 32>, <bf16,
  // 4, 64> and <bf16, 8, 32> 3 to 8 registers short, at RR = 4 the heads of 256 4 to 8: spilled around the loop
  static constexpr int WAVES = DH * BITS > 256 || RR == 4 ? 2 : DH * BITS == 256 && sizeof(T) == 4 ? 3 : 4;
};

template <typename T, int BITS, int DH, int RR>
__global__ __launch_bounds__(64 * KW, (DecodeShape<T, BITS, DH, RR>::WAVES)) void kv_decode_kernel(KvAttnArgs a) {
  using L = KvTile<BITS, DH>;
  using D = DecodeShape<T, BITS, DH, RR>;
  constexpr int NG = L::NG, CB = DH / 16, RL = D::RL, KT = D::KT, VT = D::VT, KP = 8 / KT;
  constexpr int NQ = sizeof(T) == 4 ? 3 : 1, NP = sizeof(T) == 4 ? 3 : 2;   // bf16 pieces of queries / probabilities
  constexpr float OFFT = kv_offset<T, BITS>();
  constexpr bool OWN_Q = NG * NQ > 4;               // keep a lane's one group only, and the zeros of the others as a select per use
  constexpr int KWORDS = NG * L::WORD / 4, VWORDS = CB * L::WORD / 4;
  struct Shared {
    float o[KW][D::ROWS][DH];
    float m[KW][D::ROWS], l[KW][D::ROWS];
    bf16x8 p[KW][NP][D::PAIRS][16];
  };
  __shared__ Shared sh;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, j = lane >> 4;
  const int b = blockIdx.z, h = blockIdx.y, split = blockIdx.x;
  const int R = a.kv.T * a.G;
  const uint8_t* base = a.kv.data + b * a.kv.c_sb + h * a.kv.c_sh;
  const int last_tile = (a.kv.capacity - 1) / KV_TILE;

  // pairs p = row NG + group.  As a query operand lane n's row holds pair n / 4 RR + n % 4 (none for n % 4 >= RR): the scores of that
  // matrix row, 4 j + r, come out in register r of lane group j, which so gets the pairs j RR + r.
  const int q_pair = (n >> 2) * RR + (n & 3), q_row = q_pair / NG, q_g = q_pair % NG;
  const bool q_real = (n & 3) < RR && q_row < R;
  int pair_g[RR], row_vis[RL];
#pragma unroll
  for (int r = 0; r < RR; ++r) pair_g[r] = (j * RR + r) % NG;

  uint32_t kw[KT][KWORDS], ks[RR][4], vw[VT][VWORDS], vs[RR][4];
  int t_begin = 0;
  const auto tile_at = [&](int turn, int i) __attribute__((always_inline)) -> const uint8_t* {
    return base + (int64_t)min(4 * turn + i, last_tile) * L::BYTES;
  };
  const auto load_k = [&](int turn, int piece) __attribute__((always_inline)) {
    const uint8_t* t = tile_at(turn, n >> 2);
#pragma unroll
    for (int i = 0; i < KT; ++i) load_words<KWORDS>(t + (8 * (n & 3) + piece * KT + i) * L::KROW + j * NG * L::WORD, kw[i]);
    if (piece == 0) {
#pragma unroll
      for (int r = 0; r < RR; ++r) load_words<4>(t + L::KS + L::scale_at(8 * (n & 3), pair_g[r]), ks[r]);
    }
  };
  const auto load_v = [&](int turn, int piece) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < VT; ++i) load_words<VWORDS>(tile_at(turn, piece * VT + i) + L::V + (j * 16 + n) * CB * L::WORD, vw[i]);
  };
  const auto load_v_scales = [&](int turn) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < RR; ++r) load_words<4>(tile_at(turn, n >> 2) + L::VS + L::scale_at(8 * (n & 3), pair_g[r]), vs[r]);
  };
  // with the whole key range in this workgroup the first turn's place is known before the sequence's length is
  if (a.splits == 1) load_k(wave, 0);

  bf16x8 qf[OWN_Q ? 1 : NG][NQ];
  float q0[RR];                                                              // what the offset of the codes adds to a score
  {
    const int t_row = a.kv.T > 1 ? (int)((uint32_t)q_row / (uint32_t)a.G) : 0, g_row = q_row - t_row * a.G;
    const T* q = (const T*)a.q + b * a.q_sb + (int64_t)(h * a.G + g_row) * a.q_sh + (int64_t)t_row * a.q_st + 32 * q_g + 8 * j;
    float x[8], sum = 0.f;
    load_query(q, a.q_vec, q_real, a.negate, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += x[e];
    bf16x8 piece[NQ];
    split_bf16<NQ>(x, piece);
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      if constexpr (OWN_Q) {
        qf[0][i] = piece[i];
      } else {
        const Frag own = {.v = piece[i]};
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          Frag f;
#pragma unroll
          for (int w = 0; w < 4; ++w) f.u[w] = g == q_g ? own.u[w] : 0u;
          qf[g][i] = f.v;
        }
      }
    }
    sum = -OFFT * sum_j2(sum_j1(sum));
#pragma unroll
    for (int r = 0; r < RR; ++r) q0[r] = __shfl(sum, 4 * j + r);
  }

  int n_min;
  const int n_max = tile_keys(a, b, 0, n_min);
#pragma unroll
  for (int i = 0; i < RL; ++i) {
    const int row = j * RR / NG + i;
    row_vis[i] = row < R ? min(a.kv.visible(b, a.kv.T > 1 ? row / a.G : 0), a.max_keys) : 0x7FFFFFFF;
  }
  const int turns = (n_max + KV_TURN - 1) / KV_TURN;
  int t_end;
  split_turns(a, split, turns, t_begin, t_end);
  if (a.splits > 1 && t_begin + wave < t_end) load_k(t_begin + wave, 0);

  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 acc[CB], off = zero;                                                 // off: what the codes' offset added in this turn
#pragma unroll
  for (int c = 0; c < CB; ++c) acc[c] = zero;
  float mc[RL], l[RL];                                                       // maximum in log2 units, this lane's share of the sum
#pragma unroll
  for (int i = 0; i < RL; ++i) { mc[i] = -INFINITY; l[i] = 0.f; }
  Frag ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones.v[i] = (bf16_t)OFFT;
  const Nibbles nb;

  // scores of this lane's rows against keys 8 n + t, t of one piece
  float s[8][RL];
  const auto scores = [&](int kp) __attribute__((always_inline)) {
    f32x4 d[KT];
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      d[i] = zero;
#pragma unroll
      for (int r = 0; r < RR; ++r) d[i][r] = q0[r];
    }
    int own_g = q_g;
    if constexpr (OWN_Q) asm volatile("" : "+v"(own_g));      // the selects stay in the loop: ahead of it they would take NG times the registers
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      bf16x8 qg[NQ];
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if constexpr (OWN_Q) {
          const Frag own = {.v = qf[0][i]};
          Frag f;
#pragma unroll
          for (int w = 0; w < 4; ++w) f.u[w] = g == own_g ? own.u[w] : 0u;
          qg[i] = f.v;
        } else {
          qg[i] = qf[g][i];
        }
      }
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const bf16x8 kf = unpack_codes<T, BITS>(&kw[i][g * L::WORD / 4], nb);
#pragma unroll
        for (int q = 0; q < NQ; ++q) d[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qg[q], kf, d[i], 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      const int t = kp * KT + i;
      float v[RR];
#pragma unroll
      for (int r = 0; r < RR; ++r) v[r] = d[i][r] * bf16_at(ks[r], t);
#pragma unroll
      for (int rl = 0; rl < RL; ++rl) {
        float x = v[rl * NG < RR ? rl * NG : 0];
#pragma unroll
        for (int g = 1; g < (NG < RR ? NG : RR); ++g) x += v[rl * NG + g];
        if constexpr (NG >= 2 * RR) x = sum_j1(x);
        if constexpr (NG >= 4 * RR) x = sum_j2(x);
        s[t][rl] = x;
      }
    }
  };
  // the turn's scores to probabilities times scales in LDS: octet n of pair j RR + r
  const auto softmax = [&](int turn, bool first) __attribute__((always_inline)) {
    const int key0 = turn * KV_TURN + 8 * n;
    const bool partial = turn * KV_TURN + KV_TURN > n_min;                   // some row does not see all of this turn
    if (partial) {
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int rl = 0; rl < RL; ++rl) s[t][rl] = key0 + t < row_vis[rl] ? s[t][rl] : -INFINITY;
    }
    float top[RL];
    bool past = first;
#pragma unroll
    for (int rl = 0; rl < RL; ++rl) {
      top[rl] = s[0][rl];
#pragma unroll
      for (int t = 1; t < 8; ++t) top[rl] = fmaxf(top[rl], s[t][rl]);
      top[rl] *= a.scale_log2;
      past = past || top[rl] > mc[rl] + 8.f;
    }
    if (__any(past)) {
      float keep[RL];
#pragma unroll
      for (int rl = 0; rl < RL; ++rl) {
        const float m_new = fmaxf(mc[rl], max16(top[rl]));
        keep[rl] = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mc[rl] - m_new);
        mc[rl] = m_new;
        l[rl] *= keep[rl];
      }
      float f[4];                                                            // of the accumulators' rows, pairs 4 j + r
#pragma unroll
      for (int r = 0; r < 4; ++r) f[r] = __shfl(keep[RL > 1 ? r % RR / NG : 0], 16 * (((4 * j + r) / RR) & 3));
#pragma unroll
      for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[c][r] *= f[r];
    }
    float p[8][RL];
#pragma unroll
    for (int rl = 0; rl < RL; ++rl) {
      const float ms = mc[rl] == -INFINITY ? 0.f : mc[rl];
#pragma unroll
      for (int t = 0; t < 8; ++t) p[t][rl] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][rl], a.scale_log2, -ms));
    }
    if (partial) {                                                           // keys not seen: no weight
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int rl = 0; rl < RL; ++rl) p[t][rl] = key0 + t < row_vis[rl] ? p[t][rl] : 0.f;
    }
#pragma unroll
    for (int rl = 0; rl < RL; ++rl)
#pragma unroll
      for (int t = 0; t < 8; t += 2) l[rl] += p[t][rl] + p[t + 1][rl];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");                   // the previous turn's are read
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      const int rl = RL > 1 ? r / NG : 0;
      float x[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) x[t] = p[t][rl] * bf16_at(vs[r], t);
      if (partial) {                                                         // the scale of a key not seen may be anything
#pragma unroll
        for (int t = 0; t < 8; ++t) x[t] = key0 + t < row_vis[rl] ? x[t] : 0.f;
      }
      bf16x8 piece[NP];
      split_bf16<NP>(x, piece);
#pragma unroll
      for (int i = 0; i < NP; ++i) sh.p[wave][i][j * RR + r][n] = piece[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  // one piece of the output: row n of A is pair n (rows past the pairs repeat them and are not used), octets 4 tile + j.  The offset
  // leaves with its turn: see unpack_codes.
  const auto output = [&](int vp) __attribute__((always_inline)) {
    if (OFFT != 0.f && vp == 0) off = zero;
#pragma unroll
    for (int i = 0; i < VT; ++i) {
      bf16x8 pf[NP];
#pragma unroll
      for (int q = 0; q < NP; ++q) pf[q] = sh.p[wave][q][n & (D::PAIRS - 1)][4 * (vp * VT + i) + j];
      if constexpr (OFFT != 0.f) {
#pragma unroll
        for (int q = 0; q < NP; ++q) off = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[q], ones.v, off, 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        const bf16x8 vf = unpack_codes<T, BITS>(&vw[i][c * L::WORD / 4], nb);
#pragma unroll
        for (int q = 0; q < NP; ++q) acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[q], vf, acc[c], 0, 0, 0);
      }
    }
    if (OFFT != 0.f && vp == KP - 1) {
#pragma unroll
      for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[c][r] -= off[r];
    }
  };

  int turn = t_begin + wave;
  if constexpr (KP == 1) {
    for (; turn < t_end; turn += KW) {
      load_v(turn, 0);
      load_v_scales(turn);
      scores(0);
      if (turn + KW < t_end) load_k(turn + KW, 0);
      softmax(turn, turn == t_begin + wave);
      output(0);
    }
  } else {
    // In pieces: the next turn's scores run between the pieces of this turn's output, so that each piece's loads have the other's
    // arithmetic to hide behind (16 uneven sequences, heads of 256, 8 bits: 61 -> 50 us).
    if (turn < t_end) {
      load_v_scales(turn);
      load_v(turn, 0);
#pragma unroll
      for (int x = 0; x < KP; ++x) {
        scores(x);
        if (x + 1 < KP) load_k(turn, x + 1);
      }
      if (turn + KW < t_end) load_k(turn + KW, 0);
      softmax(turn, true);
    }
    for (; turn < t_end; turn += KW) {
      const int next = turn + KW;
      const bool more = next < t_end;
      if (more) load_v_scales(next);
#pragma unroll
      for (int x = 0; x < KP; ++x) {
        if (more) {
          scores(x);
          if (x + 1 < KP) load_k(next, x + 1);
          else if (next + KW < t_end) load_k(next + KW, 0);
        }
        output(x);
        if (x + 1 < KP) load_v(turn, x + 1);
        else if (more) load_v(next, 0);
      }
      if (more) softmax(next, false);
    }
  }

#pragma unroll
  for (int rl = 0; rl < RL; ++rl) {
    const float sum = sum16(l[rl]);
    if (n == 0 && j * RR % NG == 0) { sh.m[wave][j * RR / NG + rl] = mc[rl]; sh.l[wave][j * RR / NG + rl] = sum; }
  }
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int p = 4 * j + r;
      if (p < D::PAIRS && p % NG == c / 2) sh.o[wave][p / NG][16 * c + n] = acc[c][r] * kv_unit<T, BITS>();
    }
  __syncthreads();
  write_rows<T, DH, D::ROWS>(a, sh, b, h, 0, split);
}

// ---- many rows -------------------------------------------------------------------------------------------------------------------
// steps of a turn, so that the codes in flight fit the registers beside the accumulators; waves per SIMD: one where two would spill far
// more than the 3 registers that <bf16, 4, 256> and <fp32, 8, 256> still do
template <int BITS, int DH> constexpr int kv_steps() { return DH * BITS <= 512 ? 4 : 2; }
template <int BITS, int DH> constexpr int kv_waves() { return DH == 256 || (DH == 128 && BITS == 4) ? 1 : 2; }

template <typename T, int BITS, int DH>
__global__ __launch_bounds__(64 * KW, (kv_waves<BITS, DH>())) void kv_attn_kernel(KvAttnArgs a) {
  using L = KvTile<BITS, DH>;
  constexpr int NG = L::NG, TS = kv_steps<BITS, DH>(), NO = TS / 2, CB = DH / 16, ROWS = 16;
  constexpr int NQ = sizeof(T) == 4 ? 3 : 1, NP = sizeof(T) == 4 ? 3 : 2;   // bf16 pieces of queries / probabilities
  constexpr float OFFT = kv_offset<T, BITS>();
  constexpr bool LDS_Q = NG * NQ > 8;                                        // the pieces of long fp32 rows live in LDS
  constexpr int KWORDS = NG * L::WORD / 4, VWORDS = CB * L::WORD / 4;
  struct Shared {
    float o[KW][ROWS][DH];
    float m[KW][ROWS], l[KW][ROWS];
    bf16x8 q[LDS_Q ? NG : 1][NQ][LDS_Q ? 64 : 1];
  };
  __shared__ Shared sh;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, j = lane >> 4;
  const int b = blockIdx.z, h = blockIdx.y;
  const int rt = (int)(blockIdx.x / (uint32_t)a.splits), split = (int)blockIdx.x - rt * a.splits;
  const int R = a.kv.T * a.G, row0 = rt * ROWS;                             // rows (t, g) of this cache head: rho = t G + g
  const uint8_t* base = a.kv.data + b * a.kv.c_sb + h * a.kv.c_sh;
  const int last_tile = (a.kv.capacity - 1) / KV_TILE;
  constexpr int SUB = 8 / TS;                                                // steps of a turn

  // this lane's column: its row
  const int rho = row0 + n;
  const bool real = rho < R;
  const int t_row = (int)((uint32_t)rho / (uint32_t)a.G), g_row = rho - t_row * a.G;

  uint32_t kw[TS][KWORDS], ks[NG][TS * 2], vw[NO][VWORDS], vs[NG][TS * 2];
  int t_begin = 0;
  auto key_base = [&](int step, int tile_in_turn) __attribute__((always_inline)) -> const uint8_t* {
    const int tile = (t_begin + wave + KW * (step / SUB)) * 4 + tile_in_turn;
    return base + (int64_t)min(tile, last_tile) * L::BYTES;
  };
  auto load_k = [&](int step) __attribute__((always_inline)) {
    const int s = step % SUB;
    const uint8_t* kt = key_base(step, n >> 2);
#pragma unroll
    for (int t = 0; t < TS; ++t) load_words<KWORDS>(kt + (4 * (s * TS + t) + (n & 3)) * L::KROW + j * NG * L::WORD, kw[t]);
    const uint8_t* st = key_base(step, j) + L::KS + s * TS * 8;
#pragma unroll
    for (int g = 0; g < NG; ++g) load_words<TS * 2>(st + g * KV_TILE * 2, ks[g]);
  };
  auto load_v = [&](int step) __attribute__((always_inline)) {
    const int s = step % SUB;
    const uint8_t* vt = key_base(step, j);
#pragma unroll
    for (int o = 0; o < NO; ++o) load_words<VWORDS>(vt + L::V + ((s * NO + o) * 16 + n) * CB * L::WORD, vw[o]);
#pragma unroll
    for (int g = 0; g < NG; ++g) load_words<TS * 2>(vt + L::VS + s * TS * 8 + g * KV_TILE * 2, vs[g]);
  };
  // with the whole key range in this workgroup the first turn's place is known before the sequence's length is
  if (a.splits == 1) load_k(0);

  // queries: B operand of step g = channels 32 g + 8 j + 0..7 of column n's row
  bf16x8 qf[LDS_Q ? 1 : NG][NQ];
  float q0[NG];                                                              // what the offset of the codes adds to a score
  {
    const T* q = (const T*)a.q + b * a.q_sb + (int64_t)(h * a.G + g_row) * a.q_sh + (int64_t)t_row * a.q_st + 8 * j;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float x[8], sum = 0.f;
      load_query(q + 32 * g, a.q_vec, real, a.negate, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += x[e];
      bf16x8 piece[NQ];
      split_bf16<NQ>(x, piece);
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if constexpr (LDS_Q) sh.q[g][i][lane] = piece[i];                    // the four waves write the same values
        else qf[g][i] = piece[i];
      }
      q0[g] = -OFFT * sum_j2(sum_j1(sum));
    }
  }
  if constexpr (LDS_Q) __syncthreads();

  // what the rows of this tile see: all of them at least n_min keys, none more than n_max
  int n_min;
  const int n_max = tile_keys(a, b, row0, n_min);
  const int vis = real ? min(a.kv.visible(b, t_row), a.max_keys) : 0x7FFFFFFF;

  f32x4 acc[CB];
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < CB; ++c) acc[c] = zero;
  float mc = -INFINITY, l = 0.f;                                             // maximum in log2 units, this lane's share of the sum
  Frag ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones.v[i] = (bf16_t)OFFT;
  const Nibbles nb;

  const int turns = (n_max + KV_TURN - 1) / KV_TURN;
  int t_end;
  split_turns(a, split, turns, t_begin, t_end);
  const int my_turns = t_end - t_begin > wave ? (t_end - t_begin - wave + KW - 1) / KW : 0;
  const int steps = my_turns * SUB;
  if (a.splits > 1 && steps > 0) load_k(0);
  for (int step = 0; step < steps; ++step) {
    load_v(step);
    // scores
    f32x4 sc[TS];
#pragma unroll
    for (int t = 0; t < TS; ++t) sc[t] = zero;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      bf16x8 qg[NQ];
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if constexpr (LDS_Q) qg[i] = sh.q[g][i][lane];
        else qg[i] = qf[g][i];
      }
#pragma unroll
      for (int t = 0; t < TS; ++t) {
        const bf16x8 kf = unpack_codes<T, BITS>(&kw[t][g * L::WORD / 4], nb);
        f32x4 d = {q0[g], q0[g], q0[g], q0[g]};
#pragma unroll
        for (int i = 0; i < NQ; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qg[i], d, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[t][r] = __builtin_fmaf(d[r], bf16_at(ks[g], 4 * t + r), sc[t][r]);
      }
    }
    if (step + 1 < steps) load_k(step + 1);
    // keys of this lane: key0 + 4 t + r
    const int turn0 = (t_begin + wave + KW * (step / SUB)) * KV_TURN;
    const bool partial = turn0 + KV_TURN > n_min;                            // some row does not see all of this turn
    const int key0 = turn0 + j * KV_TILE + (step % SUB) * TS * 4;
    if (partial) {
#pragma unroll
      for (int t = 0; t < TS; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[t][r] = key0 + 4 * t + r < vis ? sc[t][r] : -INFINITY;
    }
    float top = sc[0][0];
#pragma unroll
    for (int t = 0; t < TS; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, sc[t][r]);
    top *= a.scale_log2;
    if (step == 0 || __any(top > mc + 8.f)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float m_new = fmaxf(mc, top);
      const float keep = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mc - m_new);
      mc = m_new;
      l *= keep;
      float f[4];                                                            // of the accumulators' rows 4 j + r: lane 4 j + r has it
#pragma unroll
      for (int r = 0; r < 4; ++r) f[r] = __shfl(keep, 4 * j + r);
#pragma unroll
      for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[c][r] *= f[r];
    }
    const float ms = mc == -INFINITY ? 0.f : mc;
    float p[TS][4];
#pragma unroll
    for (int t = 0; t < TS; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) p[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][r], a.scale_log2, -ms));
    if (partial) {                                                           // keys not seen: no weight, and no scale (it may be anything)
#pragma unroll
      for (int t = 0; t < TS; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool seen = key0 + 4 * t + r < vis;
          p[t][r] = seen ? p[t][r] : 0.f;
          if (!seen) {
#pragma unroll
            for (int g = 0; g < NG; ++g) vs[g][2 * t + r / 2] &= r & 1 ? 0x0000FFFFu : 0xFFFF0000u;
          }
        }
    }
#pragma unroll
    for (int t = 0; t < TS; ++t) l += (p[t][0] + p[t][1]) + (p[t][2] + p[t][3]);
    // output
    f32x4 offg[NG];                                                          // what the codes' offset adds in this step
#pragma unroll
    for (int g = 0; g < NG; ++g) offg[g] = zero;
#pragma unroll
    for (int o = 0; o < NO; ++o) {
      bf16x8 pf[NG][NP];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = p[2 * o + e / 4][e % 4] * bf16_at(vs[g], 8 * o + e);
        split_bf16<NP>(x, pf[g]);
        if constexpr (OFFT != 0.f) {
#pragma unroll
          for (int i = 0; i < NP; ++i) offg[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[g][i], ones.v, offg[g], 0, 0, 0);
        }
      }
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        const bf16x8 vf = unpack_codes<T, BITS>(&vw[o][c * L::WORD / 4], nb);
#pragma unroll
        for (int i = 0; i < NP; ++i) acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[c / 2][i], vf, acc[c], 0, 0, 0);
      }
    }
    if constexpr (OFFT != 0.f) {
#pragma unroll
      for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[c][r] -= offg[c / 2][r];
    }
  }

  // this wave's state -> LDS (accumulator row 4 j + r, channel 16 c + n)
  l = sum_j2(sum_j1(l));
  if (j == 0) { sh.m[wave][n] = mc; sh.l[wave][n] = l; }
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r) sh.o[wave][4 * j + r][16 * c + n] = acc[c][r] * kv_unit<T, BITS>();
  __syncthreads();
  write_rows<T, DH, ROWS>(a, sh, b, h, row0, split);
}

// Joins the splits of a row: one wave per row, the states of eight splits under way together.
template <typename T, int DH>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(KvAttnArgs a, uint32_t rows) {
  constexpr int PER = (DH + 63) / 64, U = 8;
  const int lane = threadIdx.x & 63;
  const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const uint32_t R = (uint32_t)(a.kv.T * a.G), bh = row / R;
  const int rr = (int)(row - bh * R), b = (int)(bh / (uint32_t)a.kv.H), h = (int)(bh - b * (uint32_t)a.kv.H);
  const int t = rr / a.G, hq = h * a.G + rr % a.G;
  const int splits = a.splits;
  const float* part = a.part + (int64_t)row * a.splits * (DH + 2);
  float M = -INFINITY, S = 0.f, o[PER] = {};
  for (int s0 = 0; s0 < splits; s0 += U) {
    float m[U], l[U], v[U][PER];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float* ps = part + (int64_t)min(s0 + u, splits - 1) * (DH + 2);
      m[u] = s0 + u < splits ? ps[DH] : -INFINITY;
      l[u] = ps[DH + 1];
#pragma unroll
      for (int i = 0; i < PER; ++i) v[u][i] = ps[min(lane + 64 * i, DH - 1)];
    }
    float top = M;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, m[u]);
    const float ms = top == -INFINITY ? 0.f : top, keep = __builtin_amdgcn_exp2f(M - ms);
    M = top;
    S *= keep;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] *= keep;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float f = s0 + u < splits ? __builtin_amdgcn_exp2f(m[u] - ms) : 0.f;
      const bool in = s0 + u < splits;
      S += in ? f * l[u] : 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] += in ? f * v[u][i] : 0.f;
    }
  }
  const bool any = a.kv.visible(b, t) > 0;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 64 * i < DH) ((T*)a.out)[b * a.o_sb + hq * a.o_sh + t * a.o_st + lane + 64 * i] = from_f32<T>(any ? o[i] / S : 0.f);
  if (a.lse && lane == 0) a.lse[((int64_t)b * a.kv.H * a.G + hq) * a.kv.T + t] = any ? (M + __log2f(S)) * 0.6931471805599453f : -INFINITY;
}

// Which kernel, and how many workgroups share a row tile's key range: at least two per CU (512), none with less than one turn for
// each wave.  512 is what is resident at once for heads of 128 and 256 and few rows, by their registers (smaller heads: three or four per
// CU; many rows at heads of 256, or of 128 in 4 bits: one); the rule rounds up, so it is met exactly only where the heads of the
// batch divide 512 (24 sequences of 12 heads: 576).  More was slower where it was measured: 640, 768 and 1024 took 140, 127 and 121 us against 116 for 8 sequences of 65537 keys
// (8 heads of 128, 4 bits), 58, 60 and 56 against 50 for 16 uneven ones of up to 4001 (8 heads of 256, 8 bits).  Every sequence
// is split evenly: splits of a fixed number of turns, fewer for short sequences, leave CUs idle and were a sixth slower.
struct KvPlan {
  int pairs;                                 // (row, channel group) pairs per cache head; more than 16: kv_attn_kernel
  int row_tiles, splits;
};
static KvPlan kv_attn_plan(const bg_kv_cache* c, int Hq, int T, int max_keys) {
  KvPlan p;
  const int64_t R = (int64_t)T * (Hq / c->H), pairs = R * (c->Dh / KV_GROUP);
  p.pairs = pairs > 16 ? 17 : (int)pairs;
  p.row_tiles = pairs > 16 ? (int)cdiv(R, 16) : 1;
  const int64_t base = (int64_t)c->B * c->H * p.row_tiles;
  const int64_t most = cdiv(max_keys, KV_TURN * KW), want = cdiv(512, base);
  p.splits = (int)(want < most ? want : most);
  return p;
}

}  // namespace bg

using namespace bg;

extern "C" size_t bg_kv_cache_attn_workspace_bytes(const bg_kv_cache* cache, int Hq, int T, int max_keys) {
  if (!cache || cache->H <= 0 || cache->B <= 0 || cache->Dh < 32 || Hq <= 0 || Hq % cache->H || T <= 0 || max_keys <= 0) return 0;
  const KvPlan p = kv_attn_plan(cache, Hq, T, max_keys);
  return p.splits == 1 ? 0 : (size_t)cache->B * Hq * T * p.splits * (cache->Dh + 2) * sizeof(float);
}

template <typename T, int BITS, int DH>
static void kv_attn_launch(const KvAttnArgs& a, const KvPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.row_tiles * p.splits), (unsigned)a.kv.H, (unsigned)a.kv.B), block(64 * KW);
  if (p.pairs > 16) hipLaunchKernelGGL((kv_attn_kernel<T, BITS, DH>), grid, block, 0, st, a);
  else if (p.pairs > 8) hipLaunchKernelGGL((kv_decode_kernel<T, BITS, DH, 4>), grid, block, 0, st, a);
  else if (DH == 256 || p.pairs > 4) hipLaunchKernelGGL((kv_decode_kernel<T, BITS, DH, 2>), grid, block, 0, st, a);
  else if constexpr (DH < 256) hipLaunchKernelGGL((kv_decode_kernel<T, BITS, DH, 1>), grid, block, 0, st, a);
  if (p.splits > 1) {
    const uint32_t rows = (uint32_t)(a.kv.B * a.kv.H) * (uint32_t)(a.kv.T * a.G);
    hipLaunchKernelGGL((kv_attn_join_kernel<T, DH>), dim3((unsigned)cdiv(rows, 4)), dim3(256), 0, st, a, rows);
  }
}

extern "C" int bg_kv_cache_attn_fwd(const bg_kv_cache* cache, const void* data, const void* q, int dtype, int Hq, int T, int64_t q_sb,
                                    int64_t q_sh, int64_t q_st, const int32_t* start, const int32_t* counts, int max_keys, float scale,
                                    void* out, int64_t o_sb, int64_t o_sh, int64_t o_st, float* lse, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  if (int rc = kv_check("bg_kv_cache_attn_fwd", cache, data, dtype, T)) return rc;
  BG_REQUIRE(q && out, "bg_kv_cache_attn_fwd: null q / out");
  BG_REQUIRE(Hq > 0 && Hq % cache->H == 0, "bg_kv_cache_attn_fwd: Hq=%d query heads over %d cache heads", Hq, cache->H);
  BG_REQUIRE(max_keys > 0 && max_keys <= cache->capacity, "bg_kv_cache_attn_fwd: max_keys=%d of capacity %d", max_keys, cache->capacity);
  BG_REQUIRE((int64_t)T * Hq < (1ll << 30), "bg_kv_cache_attn_fwd: T=%d Hq=%d", T, Hq);
  const KvPlan p = kv_attn_plan(cache, Hq, T, max_keys);
  const int64_t rows = (int64_t)cache->B * Hq * T;
  BG_REQUIRE(cache->B <= 65535 && cache->H <= 65535 && (int64_t)p.row_tiles * p.splits < (1ll << 24) && rows < (1ll << 31),
             "bg_kv_cache_attn_fwd: B=%d H=%d, %lld rows", cache->B, cache->H, (long long)rows);
  const size_t need = bg_kv_cache_attn_workspace_bytes(cache, Hq, T, max_keys);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 3))) {
    set_error("bg_kv_cache_attn_fwd: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
    return BG_ERR_WORKSPACE;
  }
  KvAttnArgs a;
  a.kv.data = (uint8_t*)data;
  a.kv.B = cache->B; a.kv.H = cache->H; a.kv.capacity = cache->capacity;
  a.kv.c_sb = cache->c_sb; a.kv.c_sh = cache->c_sh;
  a.kv.start = start; a.kv.counts = counts; a.kv.T = T;
  a.q = q; a.q_sb = q_sb; a.q_sh = q_sh; a.q_st = q_st;
  a.out = out; a.o_sb = o_sb; a.o_sh = o_sh; a.o_st = o_st;
  a.lse = lse; a.part = (float*)workspace;
  a.G = Hq / cache->H; a.max_keys = max_keys; a.splits = p.splits;
  a.rows_per_tile = p.pairs > 16 ? 16 : T * a.G;
  a.negate = scale < 0.f;
  const int64_t es = dtype == BG_F32 ? 4 : 2;
  a.q_vec = (((uintptr_t)q | (uintptr_t)(q_sb * es) | (uintptr_t)(q_sh * es) | (uintptr_t)(q_st * es)) & 15) == 0;
  const double unit = dtype == BG_F32 && cache->bits == 4 ? kv_unit<float, 4>() : 1.0;                 // of the scores
  a.scale_log2 = (float)((scale < 0.f ? -(double)scale : (double)scale) * 1.4426950408889634 * unit);
  hipStream_t st = (hipStream_t)stream;
#define BG_GO(BITS, DH)                                           \
  if (dtype == BG_F32) kv_attn_launch<float, BITS, DH>(a, p, st); \
  else kv_attn_launch<bf16_t, BITS, DH>(a, p, st)
  BG_KV_DISPATCH(cache->bits, cache->Dh, BG_GO)
#undef BG_GO
  BG_CHECK_LAUNCH("bg_kv_cache_attn_fwd");
  return BG_OK;
}
