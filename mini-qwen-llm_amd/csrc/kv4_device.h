// The 4-bit paged cache's record: what one key / value head keeps of one page of 16 tokens.
//
// 18 D bytes (D = 64 or 128, groups g of 64 dimensions), in the order in which a wave's
// lanes hold the operands of the 16 x 16 x 32 MFMAs, so that the attention reads whole
// records with wide loads straight into them:
//
//   K codes  8 D bytes  [quarter 4][token 16][g][half 2][8 codes]: dimension 64 g + 16 quarter
//            + 8 half + j; code j = 2 i in nibble i, code j = 2 i + 1 in nibble i + 4 of the
//            word, so that (word >> 4 i) & 0x000F000F is the pair of a packed operand.
//            Lane 16 quarter + token of S^T = K Q^T's left operand reads D / 8 bytes.
//   V codes  8 D bytes  [token / 4][m 16][token % 4][g][4 codes]: dimension 64 g + 4 m + b in
//            nibble b of its 16 bits.  Lane 16 (token / 4) + m of O^T = V^T P^T's left operand
//            reads D / 8 bytes.  A token's codes are whole 16-bit words in both parts:
//            writing one token touches no other's.
//   K, V     D bytes each  [token 16][g][scale, least], 16 bits each, of the model's type
//
// A code n stands for scale * n + least.
#pragma once

#include "mqk_device.h"

namespace mqk {

constexpr int kPage = 16;  // tokens of a page

template <int D>
struct Kv4 {
  static constexpr int kG = D / 64;           // groups of a head
  static constexpr int kRecord = 18 * D;      // bytes
  static constexpr int kV = 8 * D;            // V codes
  static constexpr int kMetaK = 16 * D, kMetaV = 17 * D;
  // word of K codes of (token, 8 dimensions c = d / 8)
  static __device__ __forceinline__ int k_word(int token, int c) {
    const int g = c >> 3, quarter = (c >> 1) & 3, half = c & 1;
    return ((quarter * 16 + token) * kG + g) * 2 + half;
  }
  // 16-bit word of V codes of (token, group, m)
  static __device__ __forceinline__ int v_half(int token, int g, int m) {
    return (((token >> 2) * 16 + m) * 4 + (token & 3)) * kG + g;
  }
};

// Element types the cache's scales and least values come in.
struct KvBf16 : Bf16 {
  static constexpr uint32_t kExp = 0x7F80u, kNaN = 0x7FC0u;
  static __device__ __forceinline__ uint32_t from_f32(float f) { return f32_to_bf16(f); }
};
struct KvFp16 : Fp16 {
  static constexpr uint32_t kExp = 0x7C00u, kNaN = 0x7E00u;
  static __device__ __forceinline__ uint32_t from_f32(float f) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  }
};

// Sequence of packed token t among offsets cu[0..n] (clamped into [0, total]) and the
// values beside it, by one round of loads for 64 candidates: all lanes of the wave must
// call it with the same t.  Returns false for a token behind the last sequence.
struct SeqOf {
  int s;
  int64_t at, n;  // first token and length
  int len;        // lens[s]
};
__device__ __forceinline__ bool find_seq(const int32_t* cu, const int32_t* lens, int n_seqs, int64_t t, SeqOf& r) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < n_seqs; base += 63) {
    // 64 offsets cover 63 sequences
    const int c = base + lane;
    const int32_t off = cu[c <= n_seqs ? c : n_seqs];
    const int32_t len = lens ? lens[c < n_seqs ? c : n_seqs - 1] : 0;
    const int below = __popcll(__ballot(c <= n_seqs && int64_t(off) <= t));
    if (below == 0) return false;
    if (below <= 63) {
      const int i = below - 1;
      if (base + i >= n_seqs) return false;
      r.s = base + i;
      r.at = __builtin_amdgcn_readlane(off, i);
      r.n = int64_t(__builtin_amdgcn_readlane(off, i + 1)) - r.at;
      r.len = __builtin_amdgcn_readlane(len, i);
      return r.at >= 0 && t - r.at < r.n;
    }
  }
  return false;
}

}  // namespace mqk
