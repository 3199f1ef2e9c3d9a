// Attention over the quantised key / value cache (bg_kv_cache_attn_fwd).
//
// Mathematics.  With codes c and scales s per 32 channels g,
//   q . k = sum_g s_kg (q_g . c_kg)         o_ch = sum_k (p_k s_vg) c_v,ch
// so the codes themselves are the matrix operands: as bf16 they are exact (4 bits: as c + 24, whose part is taken out of the sums; 8
// bits: signed), the scales join in fp32 - on the scores after the product, on the probabilities before it.  Nothing held is rounded again.  bf16
// queries are exact operands; fp32 queries go in as three bf16 pieces (24 bits), probabilities as two (16 bits, for bf16 outputs) or three.
//
// Layout.  One wave takes 4 tiles (128 keys) per turn with v_mfma_f32_16x16x32_bf16; lane = (n = lane % 16, j = lane / 16).
//   scores   A = K codes: row rr of 16 is key 4 t + rr % 4 of tile rr / 4, B = queries: column n.  The result gives lane (n, j) the
//            scores of column n against keys 4 t + r (r = 0..3) of tile j: over t, the 32 keys of ITS tile.
//   output   A = probabilities: row n, lane group j holds 8 keys of tile j - what the lane already has -, B = V codes: lane (n, j) holds
//            channel n's 8 keys of tile j.  Codes go from memory to operands with one shift and one mask-or per pair; P never
//            leaves its lane; no LDS in the loop.
// Columns.  PACKED (rows <= 16 / NG, decoding): column n = (row n / NG, channel group n % NG), its query zero outside its group: the
//   NG partial scores of a row land in NG adjacent lanes, each with its own scale, and are summed by DPP; the output's A rows
//   are (row, group) pairs, of which a column block uses the ones of its group.  One scale per key and lane instead of NG.
//   Otherwise a column is a row and the groups are separate products.  (Which is faster depends on the rows only: a packed tile holds
//   16 / NG of them at about half the vector work of a general one with 16.)
// Softmax.  The running maximum of a row moves only when a score passes it by 2^8 (probabilities stay below 256), so that
//   the usual turn needs no exchange between lanes.
// Work.  Four waves per workgroup take turns round robin; the key range is split over workgroups when there are too few of
//   them to fill 256 CUs (kv_attn_plan), the partial states joined by a second kernel.
// Bound by HBM: 0.5625 or 1.0625 bytes per cached value.
#include "kv_cache.h"

namespace bg {

constexpr int KW = 4;                       // waves per workgroup
constexpr int KV_TURN = 4 * KV_TILE;        // keys a wave takes per turn

// Turn of a wave in steps of TS rows of four keys per tile, so that the codes in flight fit the registers beside the accumulators
template <typename T, int BITS, int DH, bool PACKED> constexpr int kv_steps() {
  if (!PACKED) return DH * BITS <= 512 ? 4 : 2;
  if (DH * BITS <= 256) return 4;
  if (DH * BITS <= 512) return sizeof(T) == 4 && DH == 128 ? 4 : 8;
  return DH * BITS <= 1024 && !(sizeof(T) == 4 && DH == 256) ? 4 : 2;
}

struct KvAttnArgs {
  KvArgs kv;
  const void* q;
  int64_t q_sb, q_sh, q_st;
  void* out;
  int64_t o_sb, o_sh, o_st;
  float* lse;
  float* part;                              // [row][split][Dh + 2]: unnormalised output, maximum (log2), sum
  int G, max_keys, splits, rows_per_tile, negate;
  float scale_log2;                         // |scale| log2(e)
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

union Frag {
  uint32_t u[4];
  bf16x8 v;
};

// 8 codes -> 8 bf16 numbers code + OFFT.  4 bits: the nibble as bits 3..6 of a bf16 in [16, 32) is 16 + stored code; 8 bits: converted
// (a conversion that takes its byte from the word, and half a pack).
template <int BITS> constexpr float kv_offset() { return BITS == 4 ? 24.f : 0.f; }
// The two constants sit in a vector and a scalar register: as literals they would make the mask-or two instructions.
struct Nibbles {
  uint32_t mask, base;
  __device__ __forceinline__ Nibbles() : mask(0x00780078u), base(0x41804180u) { asm volatile("" : "+v"(mask), "+s"(base)); }
};
template <int BITS> __device__ __forceinline__ bf16x8 unpack_codes(const uint32_t* w, const Nibbles& nb) {
  Frag f;
  if constexpr (BITS == 4) {
    f.u[0] = ((w[0] << 3) & nb.mask) | nb.base;
    f.u[1] = ((w[0] >> 1) & nb.mask) | nb.base;
    f.u[2] = ((w[0] >> 5) & nb.mask) | nb.base;
    f.u[3] = ((w[0] >> 9) & nb.mask) | nb.base;
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

template <int CTRL> __device__ __forceinline__ float dpp_add(float x) {
#pragma clang fp contract(off)          // a fused multiply-add would need the moved value in a register of its own
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
template <int NG> __device__ __forceinline__ float group_sum(float x) {      // over NG adjacent lanes
  if constexpr (NG >= 2) x = dpp_add<0xB1>(x);                              // quad_perm 1,0,3,2
  if constexpr (NG >= 4) x = dpp_add<0x4E>(x);                              // quad_perm 2,3,0,1
  if constexpr (NG >= 8) x = dpp_add<0x141>(x);                             // row_half_mirror
  return x;
}

// Waves per SIMD the kernel is built for: four for small heads, whose turns are short and bound by vector work as much as by
// memory; else two; one (512 registers) where two would spill.
template <typename T, int BITS, int DH, bool PACKED> constexpr int kv_waves() {
  if (PACKED) return DH * BITS <= 256 ? (sizeof(T) == 4 && DH == 64 ? 3 : 4) : 2;
  return DH == 256 || (DH == 128 && BITS == 4) ? 1 : 2;
}

template <typename T, int BITS, int DH, bool PACKED>
__global__ __launch_bounds__(64 * KW, (kv_waves<T, BITS, DH, PACKED>())) void kv_attn_kernel(KvAttnArgs a) {
  using L = KvTile<BITS, DH>;
  constexpr int NG = L::NG, TS = kv_steps<T, BITS, DH, PACKED>(), NO = TS / 2, CB = DH / 16;
  constexpr int ROWS = PACKED ? 16 / NG : 16, GL = PACKED ? 1 : NG;         // rows per tile; groups whose scales a lane needs
  constexpr int NQ = sizeof(T) == 4 ? 3 : 1, NP = sizeof(T) == 4 ? 3 : 2;   // bf16 pieces of queries / probabilities
  constexpr float OFFT = kv_offset<BITS>();
  constexpr bool OWN_Q = PACKED && NG * NQ > 4;     // keep a lane's one group only, and the zeros of the others as a select per use
  constexpr bool LDS_Q = !PACKED && NG * NQ > 8;    // the pieces of long fp32 rows live in LDS
  constexpr int NQF = OWN_Q || LDS_Q ? 1 : NG;
  constexpr int KWORDS = NG * L::WORD / 4, VWORDS = CB * L::WORD / 4;
  __shared__ float sh_o[KW][ROWS][DH];
  __shared__ float sh_m[KW][16], sh_l[KW][16];
  __shared__ bf16x8 sh_q[LDS_Q ? NG : 1][NQ][LDS_Q ? 64 : 1];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, j = lane >> 4;
  const int b = blockIdx.z, h = blockIdx.y;
  const int rt = (int)(blockIdx.x / (uint32_t)a.splits), split = (int)blockIdx.x - rt * a.splits;
  const int R = a.kv.T * a.G, row0 = rt * ROWS;                             // rows (t, g) of this cache head: rho = t G + g
  const uint8_t* base = a.kv.data + b * a.kv.c_sb + h * a.kv.c_sh;
  const int last_tile = (a.kv.capacity - 1) / KV_TILE;
  constexpr int SUB = 8 / TS;                                                // steps of a turn

  // this lane's column: its row
  const int rho = row0 + (PACKED ? n / NG : n), my_g = PACKED ? n % NG : 0;
  const bool real = rho < R;
  int t_row = 0, g_row = rho;                                                // rho = t_row G + g_row
  if (a.kv.T > 1) {
    t_row = (int)((uint32_t)rho / (uint32_t)a.G);
    g_row = rho - t_row * a.G;
  }

  uint32_t kw[TS][KWORDS], ks[GL][TS * 2], vw[NO][VWORDS], vs[GL][TS * 2];
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
    for (int g = 0; g < GL; ++g) load_words<TS * 2>(st + (PACKED ? my_g : g) * KV_TILE * 2, ks[g]);
  };
  auto load_v = [&](int step) __attribute__((always_inline)) {
    const int s = step % SUB;
    const uint8_t* vt = key_base(step, j);
#pragma unroll
    for (int o = 0; o < NO; ++o) load_words<VWORDS>(vt + L::V + ((s * NO + o) * 16 + n) * CB * L::WORD, vw[o]);
#pragma unroll
    for (int g = 0; g < GL; ++g) load_words<TS * 2>(vt + L::VS + s * TS * 8 + (PACKED ? my_g : g) * KV_TILE * 2, vs[g]);
  };
  // with the whole key range in this workgroup the first turn's place is known before the sequence's length is
  if (a.splits == 1) load_k(0);

  // queries: B operand of step g = channels 32 g + 8 j + 0..7 of column n's row
  bf16x8 qf[NQF][NQ];
  float q0[GL];                                                              // what the offset of the codes adds to a score
  {
    const T* q = (const T*)a.q + b * a.q_sb + (int64_t)(h * a.G + g_row) * a.q_sh + (int64_t)t_row * a.q_st + 8 * j;
#pragma unroll
    for (int g = 0; g < (PACKED ? 1 : NG); ++g) {
      float x[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = real ? to_f32(q[32 * (PACKED ? my_g : g) + e]) : 0.f;
        x[e] = a.negate ? -v : v;
        sum += x[e];
      }
      bf16x8 piece[NQ];
      split_bf16<NQ>(x, piece);
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if constexpr (LDS_Q) sh_q[g][i][lane] = piece[i];                    // the four waves write the same values
        else qf[g][i] = piece[i];
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      q0[g] = -OFFT * sum;
    }
    if constexpr (PACKED && !OWN_Q) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const Frag own = {.v = qf[0][i]};
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          Frag f;
#pragma unroll
          for (int w = 0; w < 4; ++w) f.u[w] = g == my_g ? own.u[w] : 0u;
          qf[g][i] = f.v;
        }
      }
    }
  }
  if constexpr (LDS_Q) __syncthreads();
  auto query = [&](int g, int i, int own_g) __attribute__((always_inline)) -> bf16x8 {
    if constexpr (LDS_Q) return sh_q[g][i][lane];
    if constexpr (!OWN_Q) return qf[g][i];
    const Frag own = {.v = qf[0][i]};
    Frag f;
#pragma unroll
    for (int w = 0; w < 4; ++w) f.u[w] = g == own_g ? own.u[w] : 0u;
    return f.v;
  };

  // what the rows of this tile see: all of them at least n_min keys, none more than n_max
  int n_min;
  const int n_max = tile_keys(a, b, row0, n_min);
  const int vis = real ? min(a.kv.visible(b, t_row), a.max_keys) : 0x7FFFFFFF;

  f32x4 acc[CB], off = {0.f, 0.f, 0.f, 0.f};                                 // PACKED: one offset sum; else one per group
  f32x4 offg[PACKED ? 1 : NG];
#pragma unroll
  for (int c = 0; c < CB; ++c) acc[c] = off;
#pragma unroll
  for (int g = 0; g < (PACKED ? 1 : NG); ++g) offg[g] = off;
  float mc = -INFINITY, l = 0.f;                                             // maximum in log2 units, this lane's share of the sum
  Frag ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones.v[i] = (bf16_t)OFFT;

  const Nibbles nb;
  const int turns = (n_max + KV_TURN - 1) / KV_TURN;
  const int each = (int)((uint32_t)turns / (uint32_t)a.splits), more = turns - each * a.splits;        // the first `more` splits take one more
  t_begin = split * each + min(split, more);
  const int t_end = t_begin + each + (split < more ? 1 : 0);
  const int my_turns = t_end - t_begin > wave ? (t_end - t_begin - wave + KW - 1) / KW : 0;
  const int steps = my_turns * SUB;
  if (a.splits > 1 && steps > 0) load_k(0);
  for (int step = 0; step < steps; ++step) {
    load_v(step);
    // scores
    f32x4 sc[TS];
    int own_g = my_g;
    if constexpr (OWN_Q) asm volatile("" : "+v"(own_g));      // the selects stay in the loop: ahead of it they would take NG times the registers
#pragma unroll
    for (int t = 0; t < TS; ++t) sc[t] = PACKED ? f32x4{q0[0], q0[0], q0[0], q0[0]} : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      bf16x8 qg[NQ];
#pragma unroll
      for (int i = 0; i < NQ; ++i) qg[i] = query(g, i, own_g);
#pragma unroll
      for (int t = 0; t < TS; ++t) {
        const bf16x8 kf = unpack_codes<BITS>(&kw[t][g * L::WORD / 4], nb);
        if constexpr (PACKED) {
#pragma unroll
          for (int i = 0; i < NQ; ++i) sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qg[i], sc[t], 0, 0, 0);
        } else {
          f32x4 d = {q0[g], q0[g], q0[g], q0[g]};
#pragma unroll
          for (int i = 0; i < NQ; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qg[i], d, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float k_scale = r & 1 ? bf16_hi(ks[g][2 * t + r / 2]) : bf16_lo(ks[g][2 * t + r / 2]);
            sc[t][r] = __builtin_fmaf(d[r], k_scale, sc[t][r]);
          }
        }
      }
    }
    if constexpr (PACKED) {
#pragma unroll
      for (int t = 0; t < TS; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float k_scale = r & 1 ? bf16_hi(ks[0][2 * t + r / 2]) : bf16_lo(ks[0][2 * t + r / 2]);
          sc[t][r] = group_sum<NG>(sc[t][r] * k_scale);
        }
    }
    // (the sums stay in this block: moved behind the branch below, an add and the lane exchange that feeds it are two instructions)
#pragma unroll
    for (int t = 0; t < TS; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = sc[t][r];
        asm volatile("" : "+v"(v));
        sc[t][r] = v;
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
#pragma unroll
      for (int g = 0; g < (PACKED ? 1 : NG); ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) offg[g][r] *= f[r];
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
            for (int g = 0; g < GL; ++g) vs[g][2 * t + r / 2] &= r & 1 ? 0x0000FFFFu : 0xFFFF0000u;
          }
        }
    }
#pragma unroll
    for (int t = 0; t < TS; ++t) l += (p[t][0] + p[t][1]) + (p[t][2] + p[t][3]);
    // output
#pragma unroll
    for (int o = 0; o < NO; ++o) {
      bf16x8 pf[GL][NP];
#pragma unroll
      for (int g = 0; g < GL; ++g) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t w = vs[g][4 * o + e / 2];
          x[e] = p[2 * o + e / 4][e % 4] * (e & 1 ? bf16_hi(w) : bf16_lo(w));
        }
        split_bf16<NP>(x, pf[g]);
#pragma unroll
        for (int i = 0; i < NP && OFFT != 0.f; ++i) offg[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[g][i], ones.v, offg[g], 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        const bf16x8 vf = unpack_codes<BITS>(&vw[o][c * L::WORD / 4], nb);
#pragma unroll
        for (int i = 0; i < NP; ++i) acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[PACKED ? 0 : c / 2][i], vf, acc[c], 0, 0, 0);
      }
    }
  }

  // this wave's state -> LDS (accumulator row 4 j + r, channel 16 c + n)
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (j == 0 && my_g == 0) { sh_m[wave][rho - row0] = mc; sh_l[wave][rho - row0] = l; }
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int ar = 4 * j + r;
      if (PACKED && ar % NG != c / 2) continue;
      sh_o[wave][PACKED ? ar / NG : ar][16 * c + n] = acc[c][r] - offg[PACKED ? 0 : c / 2][r];
    }
  __syncthreads();
  for (int i = tid; i < ROWS * DH; i += 64 * KW) {
    const int row = i / DH, ch = i % DH, rr = row0 + row;
    if (rr >= R) break;
    float M = sh_m[0][row];
#pragma unroll
    for (int w = 1; w < KW; ++w) M = fmaxf(M, sh_m[w][row]);
    const float Ms = M == -INFINITY ? 0.f : M;
    float S = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const float f = __builtin_amdgcn_exp2f(sh_m[w][row] - Ms);
      S += f * sh_l[w][row];
      o += f * sh_o[w][row][ch];
    }
    const int t = rr / a.G, hq = h * a.G + rr % a.G;
    if (a.splits == 1) {
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

// How many workgroups share a row tile's key range: enough to give every CU two (512), none with less than one turn for each wave.
// (Even splits of every sequence: splits of a fixed number of turns, fewer for short sequences, leave CUs idle - 16 uneven sequences
// of 8 heads, 8 bits, 67 against 79 us.)
struct KvPlan {
  bool packed;
  int row_tiles, splits;
};
static KvPlan kv_attn_plan(const bg_kv_cache* c, int Hq, int T, int max_keys) {
  KvPlan p;
  const int64_t R = (int64_t)T * (Hq / c->H);
  const int ng = c->Dh / KV_GROUP;
  p.packed = R <= 16 / ng;
  p.row_tiles = (int)cdiv(R, p.packed ? 16 / ng : 16);
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
  const dim3 grid((unsigned)(p.row_tiles * p.splits), (unsigned)a.kv.H, (unsigned)a.kv.B);
  if (p.packed) hipLaunchKernelGGL((kv_attn_kernel<T, BITS, DH, true>), grid, dim3(64 * KW), 0, st, a);
  else hipLaunchKernelGGL((kv_attn_kernel<T, BITS, DH, false>), grid, dim3(64 * KW), 0, st, a);
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
  BG_REQUIRE(cache->B <= 65535 && cache->H <= 65535 && (int64_t)p.row_tiles * p.splits < (1ll << 31) && rows < (1ll << 31),
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
  a.rows_per_tile = p.packed ? 16 / (cache->Dh / KV_GROUP) : 16;
  a.negate = scale < 0.f;
  a.scale_log2 = (float)((scale < 0.f ? -(double)scale : (double)scale) * 1.4426950408889634);
  hipStream_t st = (hipStream_t)stream;
#define BG_GO(BITS, DH)                                           \
  if (dtype == BG_F32) kv_attn_launch<float, BITS, DH>(a, p, st); \
  else kv_attn_launch<bf16_t, BITS, DH>(a, p, st)
  BG_KV_DISPATCH(cache->bits, cache->Dh, BG_GO)
#undef BG_GO
  BG_CHECK_LAUNCH("bg_kv_cache_attn_fwd");
  return BG_OK;
}
