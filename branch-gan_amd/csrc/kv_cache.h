// Layout of the quantised key / value cache (include/branchgan.h: bg_kv_cache), shared by the kernels that write, read and attend it.
//
// A (batch, head) holds tiles of 32 consecutive keys.  One tile of head size DH, NG = DH / 32 groups of 32 channels:
//   K codes    [32 keys][4 kg][NG g] words of the channels 32 g + 8 kg + 0..7 (8 codes: 4 bytes at 4 bits, 8 bytes at 8 bits)
//   V codes    [4 octets][16 n][DH / 16 c] words of the keys 8 octet + 0..7 of channel 16 c + n
//   K scales   [NG g][32 keys] bf16
//   V scales   the same
// A word is what one lane feeds to a 32-deep matrix instruction (8 consecutive elements of its row), for K along the channels and
// for V along the keys: the codes go from memory to the matrix operand with no shuffle and no LDS.
// 8-bit codes are signed bytes; 4-bit ones are stored as code + 8, and their words keep element e in nibble (e >> 1) + 4 (e & 1), so that one mask over a
// shifted word leaves elements 2i and 2i + 1 in the two halves of a register, the order of a bf16 pair.
#pragma once
#include "common.h"

namespace bg {

constexpr int KV_TILE = 32;        // keys per tile
constexpr int KV_GROUP = 32;       // channels per scale

template <int BITS, int DH> struct KvTile {
  static constexpr int NG = DH / KV_GROUP;
  static constexpr int TOP = BITS == 4 ? 7 : 127;        // codes are -TOP .. TOP
  static constexpr int OFF = BITS == 4 ? 8 : 0;
  static constexpr int WORD = BITS;                      // bytes of 8 codes
  static constexpr int KROW = DH * BITS / 8;
  static constexpr int V = KV_TILE * KROW;
  static constexpr int KS = V + KV_TILE * DH * BITS / 8;
  static constexpr int VS = KS + KV_TILE * NG * 2;
  static constexpr int BYTES = VS + KV_TILE * NG * 2;
  static constexpr int v_word(int oct, int ch) { return V + ((oct * 16 + ch % 16) * (DH / 16) + ch / 16) * WORD; }
  static constexpr int scale_at(int key, int g) { return (g * KV_TILE + key) * 2; }
};

__device__ __forceinline__ constexpr int kv_nibble(int e) { return (e >> 1) + 4 * (e & 1); }

__device__ __forceinline__ float bf16_bits_to_f32(uint32_t b) { return __uint_as_float(b << 16); }

struct KvArgs {
  uint8_t* data;
  int B, H, capacity;
  int64_t c_sb, c_sh;                      // bytes
  const int32_t* start;                    // NULL: 0
  const int32_t* counts;                   // NULL: T
  int T;
  __device__ __forceinline__ int first(int b) const { return start ? start[b] : 0; }
  __device__ __forceinline__ int count(int b) const {
    const int n = counts ? counts[b] : T;
    return n < 0 ? 0 : (n > T ? T : n);
  }
  // keys of the cache that new token t of sequence b sees: those before it and itself; 0 for a padding row
  __device__ __forceinline__ int visible(int b, int t) const {
    if (t >= count(b)) return 0;
    const int64_t n = (int64_t)first(b) + t + 1;
    return (int)(n < 0 ? 0 : (n > capacity ? capacity : n));
  }
};

// cases of (bits, Dh) the kernels are built for
#define BG_KV_DISPATCH(bits, Dh, F)             \
  switch ((bits) * 1000 + (Dh)) {               \
    case 4032: F(4, 32); break;                 \
    case 4064: F(4, 64); break;                 \
    case 4128: F(4, 128); break;                \
    case 4256: F(4, 256); break;                \
    case 8032: F(8, 32); break;                 \
    case 8064: F(8, 64); break;                 \
    case 8128: F(8, 128); break;                \
    default: F(8, 256); break;                  \
  }

int kv_check(const char* who, const bg_kv_cache* c, const void* data, int dtype, int64_t T);   // kv_cache.hip

}  // namespace bg
