// Attention of new tokens over a paged cache of bf16 / fp16 keys and values:
//
//   O[i] = sum_j softmax_j(scale * q[i] . k[j]) v[j],   j < len - n + i + 1
//
// for token i of a sequence's n new ones, position j being in slot j % page of page
// table[j / page]; or, with lists of selected pages, over the keys of those up to the token's
// own.  The reference splits this over paged_attn_prefill and paged_attn_decode
// (mini_qwen/kernels/paged_attn_prefill.py:64-156, paged_attn_decode.py:389-424).
//
// Rows are (token, query head) pairs of one key / value head, so that the heads that share
// keys read them once and a decode step fills a tile as far as it can.  One pass over the keys
// with a running maximum and sum; the scores are computed transposed, S^T = K Q^T, on 32 x 32
// MFMAs, so that a lane has scores of one row only and the probabilities go from S^T into
// O^T = V^T P^T without leaving their registers (a sum over keys has no order; V^T is read
// in that of S^T, transposed on the way out of the LDS).
//
// Two launches share a call's sequences, as their lengths are on the device:
//   few rows (up to 32: decode steps, few proposed tokens)  A workgroup of KS waves, every
//     wave with tiles of 32 keys (heads up to 64: 64) of its own, two buffers and no barrier;
//     what bounds it is reading the cache.  The steps of all sequences and heads stand in one
//     row that is cut into equal parts, one a workgroup, wherever that falls.
//   many rows (chunks)  Four waves with 32 rows each share tiles of 64 keys, two workgroups
//     a CU.  Long key ranges are cut into parts where there are fewer tiles of rows than
//     places for workgroups.
// A third joins the parts of what was cut.  Selected pages run as the first, a list's keys in
// the place of a sequence's, in equal parts that the host can choose.
//
// Scores, maxima, sums and O are fp32; P is rounded once to the tensors' type for the second
// product (as V itself is), the output once.  P, O and the sum have a common factor, 2^7 for fp16,
// that the division by the sum takes out again: fp16 has normal numbers down to 2^-14 only, and
// over thousands of keys the weights below that make a difference together.
#include "attn_device.h"
#include "mqk_attn.h"
#include "mqk_paged.h"

#include <algorithm>

namespace mqk {
namespace {

// A value that every lane has, into scalar registers.
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(v)), hi = __builtin_amdgcn_readfirstlane(uint32_t(v >> 32));
  return int64_t(uint64_t(hi) << 32 | lo);
}
template <class T>
__device__ __forceinline__ const T* uniform_ptr(const T* p) {
  return reinterpret_cast<const T*>(uniform64(reinterpret_cast<int64_t>(p)));
}

// The lane's number, opaque: what is worked out from it stays where it is used.  (The compiler
// would work it out ahead of the loop over a workgroup's parts and keep it in registers.)
__device__ __forceinline__ int here() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

// The rows of one wave over the keys so far: O^T, and the running maximum and sum of each
// lane's row.  KEEP: the lane's places in a tile are worked out once and kept.
template <class E, int DP, int BK, bool KEEP>
struct Rows {
  static constexpr int kRow = DP * 2, kC = DP / 8, kNB = BK / 32, kND = DP / 32;
  static constexpr bool kAhead = !KEEP && DP <= 128;
  f32x16_t o[kND];
  float mx, mraw, sum;  // the maximum as the exponents take it (scaled, less kLift) and as it was
  bool large;           // of the maximum: its fp32 step counts

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int d = 0; d < kND; ++d) o[d] = f32x16_t{};
    mx = mraw = -INFINITY;
    sum = 0.f;
    large = false;
  }

  // A tile of BK keys: bits of the keys that are there, of which the lane's row sees the first
  // `rel`; masked: whether some row does not see them all.
  __device__ __forceinline__ void add(const unsigned char* kt, const unsigned char* vt, const u32x4_t (&qf)[kC / 2],
                                      float scale, bool masked, int rel, const uint32_t (&bits)[kNB]) {
    const int lane = KEEP ? threadIdx.x & 63 : here(), half = lane >> 5, row = lane & 31;
    f32x16_t st[kNB];
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb) st[nb] = f32x16_t{};
    {
      // Fragments are read a group of 4 products ahead; the compiler would read each right
      // before its product and wait for it there.
      constexpr int kAll = kC / 2 * kNB, kGroup = 4;
      static_assert(kAll % kGroup == 0, "whole groups");
      u32x4_t kf[2][kGroup];
      auto fetch = [&](int g) {
#pragma unroll
        for (int e = 0; e < kGroup; ++e) {
          const int t = (g * kGroup + e) / kNB, r = (g * kGroup + e) % kNB * 32 + row;
          kf[g & 1][e] = *reinterpret_cast<const u32x4_t*>(kt + r * kRow + k_slot<kC>(r, 2 * t + half) * 16);
        }
      };
      fetch(0);
#pragma unroll
      for (int g = 0; g < kAll / kGroup; ++g) {
        if (g + 1 < kAll / kGroup) fetch(g + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < kGroup; ++e) {
          const int t = (g * kGroup + e) / kNB, nb = (g * kGroup + e) % kNB;
          st[nb] = E::mfma32(kf[g & 1][e], qf[t], st[nb]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // Left operand V^T: lane = (d = 16 * (lane / 16 % 2) + lane % 16, keys of its half), read
    // as blocks of 4 keys x 16 columns: this lane's address is that of key lane % 16 / 4,
    // columns 4 * (lane % 4), and it receives column lane % 16.
    const int r0 = 4 * half + ((lane & 15) >> 2), c0 = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    auto v_at = [&](int g, int d) {  // 16 keys from 16 g on, columns 32 d ..
      const unsigned char* at = vt + (g * 16 + r0) * kRow + v_slot<kC, 2>(r0, d * 4 + c0) * 16 + (lane & 1) * 8;
      typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * kRow));
      const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo), h2 = __builtin_bit_cast(u32x2_t, hi);
      return u32x4_t{l2[0], l2[1], h2[0], h2[1]};
    };
    // (a wave that has its SIMD to itself reads them under the softmax)
    u32x4_t vf[kAhead ? kNB * 2 : 1][kND];
    if constexpr (kAhead) {
#pragma unroll
      for (int g = 0; g < kNB * 2; ++g)
#pragma unroll
        for (int d = 0; d < kND; ++d) vf[g][d] = v_at(g, d);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (masked) {
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb) {
        const int n = rel - nb * 32;
        const uint32_t w = (n >= 32 ? bits[nb] : n <= 0 ? 0u : bits[nb] & ((1u << n) - 1)) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) st[nb][i] = w & (1u << (8 * (i / 4) + i % 4)) ? st[nb][i] : -INFINITY;
      }
    }
    float top = st[0][0];
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, st[nb][i]);
    // O and the sum are brought to a new maximum only where one grew by more than 2^8: until
    // then the terms stay below 2^(8 + kLift), which no rounding minds.
    if (__any(top * scale > mx + (8.f + E::kLift))) {
      const float traw = max_halves(top);
      const float now = fmaxf(mx, __builtin_fmaf(traw, scale, -E::kLift));
      const float f = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - now);
      mx = now;
      mraw = fmaxf(mraw, traw);
      // scale * s - maximum has the product unrounded and the maximum rounded: off by 2^-24 of
      // the maximum, so a large one is subtracted before the product
      large = __any(fabsf(mx) > 65536.f && mx != -INFINITY);
      sum *= f;
#pragma unroll
      for (int d = 0; d < kND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= f;
    }
    if (large) {
      const float raw = mx == -INFINITY ? 0.f : mraw;
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) st[nb][i] -= raw;
    }
    const float sub = mx == -INFINITY ? 0.f : large ? -E::kLift : mx;
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        st[nb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[nb][i], scale, -sub));
        sum += st[nb][i];
      }
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        u32x4_t pf;
#pragma unroll
        for (int e = 0; e < 4; ++e) pf[e] = E::pack2(st[nb][8 * ks + 2 * e], st[nb][8 * ks + 2 * e + 1]);
#pragma unroll
        for (int d = 0; d < kND; ++d) o[d] = E::mfma32(kAhead ? vf[kAhead ? nb * 2 + ks : 0][d] : v_at(nb * 2 + ks, d), pf, o[d]);
      }
  }
};

// Where a tile of BK keys is in the cache.  A page is a multiple of 8 tokens, so that every 8 keys
// lie in one page; lane i has the place (bytes) of keys 8 (i % (BK / 8)) .. + 7, and how many of
// them are there.
template <int BK>
struct Groups {
  static constexpr int kN = BK / 8;
  uint32_t lo, hi;
  int count;

  // row: of the cache, or -1; n: keys that are there
  __device__ __forceinline__ void set(int row, int n, uint32_t ts) {
    const uint64_t at = uint64_t(uint32_t(max(row, 0))) * ts;
    lo = uint32_t(at);
    hi = uint32_t(at >> 32);
    count = row < 0 ? 0 : min(max(n, 0), 8);
  }
  __device__ __forceinline__ int64_t place(int g) const {
    return int64_t(uint64_t(__builtin_amdgcn_readlane(hi, g)) << 32 | uint32_t(__builtin_amdgcn_readlane(lo, g)));
  }
  __device__ __forceinline__ bool full() const { return __all(count == 8); }
  __device__ __forceinline__ void bits(uint32_t (&to)[BK / 32]) const {
#pragma unroll
    for (int nb = 0; nb < BK / 32; ++nb) to[nb] = 0;
#pragma unroll
    for (int g = 0; g < kN; ++g)
      to[g / 4] |= ((1u << __builtin_amdgcn_readlane(count, g)) - 1) << (8 * (g % 4));
  }
};

// Staging of a tile's rows by QW waves: every load of a wave fills 64 chunks in a row, kPer rows
// (8 at most, of one group).  Rows that are not there hold what their slots, or the cache's
// first ones, hold; columns past a head size that is no whole tile are zeros.
template <int DP, int QW, int BK>
struct Stager {
  static constexpr int kC = DP / 8, kPer = 64 / kC, kTile = BK * DP * 2, kLoads = kTile / (QW * 1024);
  static constexpr int kStep = QW * kPer;  // rows between a wave's loads
  static constexpr int kDist = kStep >= 16 ? 1 : (16 / kStep < kLoads ? 16 / kStep : kLoads);
  static_assert(kPer >= 1 && kPer <= 8 && 8 % kPer == 0, "a load's rows are of one group");
  uint32_t koff[kDist], voff[kDist];  // of the lane, from its load's group on
  uint32_t ts;
  int wave;

  __device__ __forceinline__ Stager(uint32_t token_stride, int w) : ts(token_stride), wave(w) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < kDist; ++i) {
      const int r = (i * QW + wave) * kPer + lane / kC, c = lane % kC;
      koff[i] = uint32_t(r % 8) * ts + uint32_t(k_slot<kC>(r, c)) * 16;
      voff[i] = uint32_t(r % 8) * ts + uint32_t(v_slot<kC, 2>(r, c)) * 16;
    }
  }
  // kbase, vbase: of the caches' head; kto, vto: LDS addresses of the tile
  __device__ __forceinline__ void stage(const unsigned char* kbase, const unsigned char* vbase, const Groups<BK>& g,
                                        int dbytes, uint32_t kto, uint32_t vto) const {
    if (dbytes == DP * 2) {
      auto at = [&](const unsigned char* base, int i) {
        return uniform_ptr(base + g.place((i * QW + wave) * kPer / 8));
      };
      auto all = [&](const unsigned char* base, const uint32_t (&off)[kDist], uint32_t to) {
        to += wave * 1024;
        if constexpr (kLoads % 4 == 0) {
#pragma unroll
          for (int i = 0; i < kLoads; i += 4)
            dma16x4_from<QW * 1024>(at(base, i), at(base, i + 1), at(base, i + 2), at(base, i + 3), off[i % kDist],
                                    off[(i + 1) % kDist], off[(i + 2) % kDist], off[(i + 3) % kDist], to + i * QW * 1024);
        } else {
#pragma unroll
          for (int i = 0; i < kLoads; ++i) dma16_from(at(base, i), off[i % kDist], to + i * QW * 1024);
        }
      };
      all(kbase, koff, kto);
      all(vbase, voff, vto);
      return;
    }
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int i = 0; i < 2 * kLoads; ++i) {
      const bool v = i >= kLoads;
      const int l = (v ? i - kLoads : i) * QW + wave, r = l * kPer + lane / kC, c = lane % kC;
      const int at = (v ? v_slot<kC, 2>(r, c) : k_slot<kC>(r, c)) * 16;
      const unsigned char* from = (v ? vbase : kbase) + g.place(l * kPer / 8) + uint32_t(r % 8) * ts + at;
      if (at >= dbytes) from = reinterpret_cast<const unsigned char*>(&g_zero16);
      dma16(from, (v ? vto : kto) + l * 1024);
    }
  }
};

// Of a staged tile of values, rows that are not there (bits) become 0: they were read from slots
// that may hold anything, and 0 * that need not be 0.  So do values that are not finite
// where FINITE, as some row of queries does not see their key; whether there were some of
// those.  (share, of: this wave's part of the tile)
template <class E, int DP, int BK, bool FINITE>
__device__ __forceinline__ bool take_out(unsigned char* tile, const uint32_t (&bits)[BK / 32], int share, int of) {
  constexpr int kC = DP / 8;
  const int lane = here();
  bool bad = false;
#pragma unroll 2
  for (int i = share * 64 + lane; i < BK * kC; i += of * 64) {
    u32x4_t* w = reinterpret_cast<u32x4_t*>(tile) + i;
    const int r = i / kC;
    const bool there = (BK == 32 ? bits[0] : bits[r / 32]) >> (r % 32) & 1;
    if (!FINITE) {
      if (!there) *w = u32x4_t{0, 0, 0, 0};
      continue;
    }
    const u32x4_t was = *w;
    u32x4_t x = was;
    uint32_t odd = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if ((x[e] & E::kExp) == E::kExp) x[e] &= 0xFFFF0000u;
      if ((x[e] & (E::kExp << 16)) == (E::kExp << 16)) x[e] &= 0xFFFFu;
      odd |= x[e] ^ was[e];
      if (!there) x[e] = 0;
    }
    if (odd != 0 || !there) *w = x;
    bad |= there && odd != 0;
  }
  return __any(bad);
}

// A sequence of the call: its tokens at .. at + n, its length, and the keys its table has.
struct Seq {
  int64_t at;
  int n, len, m;
};
__device__ __forceinline__ Seq seq_of(const PagedAttn& a, int s) {
  Seq q;
  q.at = seq_at(a.cu, a.each, a.T, s);
  const int64_t to = seq_at(a.cu, a.each, a.T, s + 1);
  q.n = int(to > q.at ? to - q.at : 0);
  q.len = max(a.lens[s], 0);
  q.m = int(min(int64_t(q.len), a.cols * a.page));
  return q;
}
// Keys that token i sees: the tokens are the last ones of the length, also where the table ends
// before it.
__device__ __forceinline__ int limit_of(const Seq& q, int i) { return min(q.len - q.n + i + 1, q.m); }

// Sum over the lanes up to this one.
__device__ __forceinline__ int64_t scan_lanes(int64_t x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(x, d);
    if (lane >= d) x += o;
  }
  return x;
}

__device__ __forceinline__ int quotient(Divide d, int x) { return int((uint64_t(uint32_t(x)) * d.mul) >> d.shift); }

// Zeros for the rows behind the last sequence (which only offsets leave: then there is always a
// launch for few rows).
__device__ __forceinline__ void fill_rest(const PagedAttn& a, int threads) {
  if (!a.fill || !a.cu) return;
  const int64_t chunks = int64_t(a.Hq) * a.D / 8;
  const int64_t from = seq_at(a.cu, 0, a.T, a.n_seqs) * chunks, to = a.T * chunks;
  for (int64_t i = from + int64_t(blockIdx.x) * threads + threadIdx.x; i < to; i += int64_t(gridDim.x) * threads)
    *reinterpret_cast<u32x4_t*>(a.out + i * 16) = u32x4_t{0, 0, 0, 0};
}

// A lane's pieces of its row of q.
template <int DP>
__device__ __forceinline__ void load_q(const PagedAttn& a, int64_t token, int head, u32x4_t (&qf)[DP / 16]) {
  const int half = (threadIdx.x & 63) >> 5;
  const unsigned char* src = a.q + token * a.q_ts + int64_t(head) * a.q_hs;
#pragma unroll
  for (int t = 0; t < DP / 16; ++t) {
    const int at = (2 * t + half) * 16;
    qf[t] = DP == a.D || at < a.D * 2 ? *reinterpret_cast<const u32x4_t*>(src + at) : u32x4_t{0, 0, 0, 0};
  }
}

// A wave's rows to the output, divided by their sums.
template <class E, int DP, int BK, bool KEEP>
__device__ __forceinline__ void write_rows(const Rows<E, DP, BK, KEEP>& w, float total, bool live, unsigned char* dst, int dbytes) {
  const int half = here() >> 5;
  const float inv = total == 0.f ? 0.f : 1.f / total;  // (a query that sees no key: 0)
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      // four columns a lane in two runs 8 apart: the halves swap them into runs of 8
      u32x4_t x;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t lo = E::pack2(w.o[d][8 * j + 2 * e] * inv, w.o[d][8 * j + 2 * e + 1] * inv);
        const uint32_t hi = E::pack2(w.o[d][8 * j + 4 + 2 * e] * inv, w.o[d][8 * j + 4 + 2 * e + 1] * inv);
        const u32x2_t r = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
        x[e] = r[0];
        x[2 + e] = r[1];
      }
      const int at = (d * 32 + j * 16 + half * 8) * 2;
      if (live && at < dbytes) *reinterpret_cast<u32x4_t*>(dst + at) = x;
    }
}
// ... or, as they are, to row `at` of the partial results.
template <class E, int DP, int BK, bool KEEP>
__device__ __forceinline__ void write_part(const PagedAttn& a, const Rows<E, DP, BK, KEEP>& w, float total, bool live, int64_t at) {
  const int half = here() >> 5;
  if (!live) return;
  if (half == 0) *reinterpret_cast<f32x2_t*>(a.many.ml + at * 2) = f32x2_t{w.mx, total};
  float* dst = a.many.part + at * a.D;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = d * 32 + j * 8 + half * 4;
      if (col < a.D)
        *reinterpret_cast<f32x4_t*>(dst + col) =
            f32x4_t{w.o[d][4 * j], w.o[d][4 * j + 1], w.o[d][4 * j + 2], w.o[d][4 * j + 3]};
    }
}

// The values that are not finite and were taken out of tiles, of the keys that some row of the
// tile did not see: keys from .. to of a sequence, to the rows that see them.
template <class E, int DP, int BK, bool KEEP>
__device__ __forceinline__ void add_taken_out(const PagedAttn& a, Rows<E, DP, BK, KEEP>& w, int s, int kvh, int from, int to,
                                              int limit) {
  const int half = here() >> 5;
  const int32_t* table = a.table + int64_t(s) * a.cols;
  for (int key = from; key < min(to, limit); ++key) {
    const int j = quotient(a.page8, key >> 3);
    const int id = table[j];
    if (id < 0 || id >= a.num_blocks) continue;
    const unsigned char* src = a.v + ((int64_t(id) * a.page + (key - j * a.page)) * a.Hkv + kvh) * a.D * 2;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = d * 32 + 8 * j + 4 * half;
        if (col >= a.D) continue;
        const u32x2_t x = *reinterpret_cast<const u32x2_t*>(src + col * 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t y = x[e / 2] >> (16 * (e % 2)) & 0xFFFFu;
          if ((y & E::kExp) == E::kExp) w.o[d][4 * j + e] += E::to_f32(y);
        }
      }
      asm volatile("" ::: "memory");  // (a few of these rare loads at a time, for the registers' sake)
    }
  }
}

// --- few rows ----------------------------------------------------------------------------
//
// 64 sequences up to 8192 keys, 8 heads: 242 us for 1.33 GB, 5.5 TB/s (a copy reaches 5.0), and the
// join 5; 168 MB 39 us, of which 8 are launch, lengths, tables, first tiles and drain.  With offsets
// such a step has the launch for many rows beside it, which finds nothing to do: 4 to 10 us.
// Bringing the next head's tiles during a join changed neither, tiles two ahead took 5 % off the
// second and added 3 % to the first.

constexpr int kListPages = 1024;  // entries of a list that a part may have
// Waves of a workgroup, and keys of a wave's tile: what LDS has room for.  (Heads up to 64 with
// tiles of 32 keys: 254 us for the above at their size, with 64 keys 248.)
constexpr int few_waves(int D) { return D > 128 ? 2 : 4; }
constexpr int few_keys(int D) { return D > 64 ? 32 : 64; }

// Steps of one head of a sequence (one at least: one without keys has its zeros written by
// somebody); none of a sequence that is the other launch's.
__device__ __forceinline__ bool few_mine(const PagedAttn& a, const Seq& q) {
  return q.n > 0 && int64_t(q.n) * a.G <= a.few_rows;
}
template <int DP>
__device__ __forceinline__ int few_steps(const PagedAttn& a, const Seq& q) {
  constexpr int kStep = few_keys(DP) * few_waves(DP);
  if (!few_mine(a, q)) return 0;
  return max(1, (q.m + kStep - 1) / kStep);
}
// A workgroup's part of the row of places, and the sequence it starts in.
struct Part {
  int64_t pos, end;   // places (aligned: parts)
  int s, n;           // sequence, its steps a head
  int64_t base;       // its first place (part)
  int64_t per;        // places (aligned: steps) of a part
  bool aligned;       // a workgroup has one part of one head
};
// Equal parts of all the steps there are, wherever their borders fall.  A head has a place more
// than steps, ahead of them: to begin with another head (its lengths, pages and first tile, the
// joining of the last one's waves) takes a workgroup about as long as a step, and without that
// place the ones with the short sequences would be the last to end (32 sequences of 320 to 2240 keys,
// 8 heads: this launch 52 us without it, 44 with it; the call 56 and 48).  Where there is little
// work, parts that begin with a head.
template <int DP>
__device__ __forceinline__ bool find_few(const PagedAttn& a, int64_t bid, int64_t grid, Part& w) {
  const int lane = threadIdx.x & 63;
  if (a.whole) {
    w.s = int(uint32_t(bid) / uint32_t(a.Hkv));
    const Seq q = seq_of(a, w.s);
    w.n = few_steps<DP>(a, q);
    w.pos = int64_t(uint32_t(bid) % uint32_t(a.Hkv));
    w.end = w.pos + 1;
    w.base = 0;
    w.per = w.n;
    w.aligned = true;
    return few_mine(a, q);  // (not w.n: the length need not be there yet)
  }
  int64_t total = 0, heads = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
    const int s = s0 + lane;
    const int64_t n = s < a.n_seqs ? int64_t(few_steps<DP>(a, seq_of(a, s))) * a.Hkv : 0;
    total += uniform64(__shfl(scan_lanes(n), 63));
    heads += int64_t(__popcll(__ballot(n > 0))) * a.Hkv;
  }
  w.per = max(int64_t(1), (total + grid - 1) / grid);
  w.aligned = w.per <= 8 && heads * 2 <= grid;
  if (w.aligned) {
    w.per = max(int64_t(1), (total + grid - heads - 1) / (grid - heads));
  } else {
    total += heads;
    w.per = max(int64_t(2), (total + grid - 1) / grid);
  }
  w.pos = w.aligned ? bid : w.per * bid;
  int64_t base = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
    const int s = s0 + lane;
    const int steps = s < a.n_seqs ? few_steps<DP>(a, seq_of(a, s)) : 0;
    const int64_t places = w.aligned ? (steps + w.per - 1) / w.per : int64_t(steps) + (steps > 0);
    const int64_t n = places * a.Hkv, to = base + scan_lanes(n);
    const uint64_t in = __ballot(w.pos >= to - n && w.pos < to);
    if (in != 0) {
      const int l = __ffsll(static_cast<unsigned long long>(in)) - 1;
      w.s = s0 + l;
      w.n = __builtin_amdgcn_readlane(steps, l);
      w.base = uniform64(__shfl(to - n, l));
      w.end = w.aligned ? w.pos + 1 : min(total, w.pos + w.per);
      return true;
    }
    base = uniform64(__shfl(to, 63));
  }
  return false;
}

template <int DP, bool LISTS>
struct FewLds {
  static constexpr int kTile = few_keys(DP) * DP * 2;
  __align__(16) unsigned char tiles[few_waves(DP) * 4 * kTile];  // of each wave: K buffers, V buffers
  float join_ml[few_waves(DP)][2][64];
  int list_row[LISTS ? kListPages : 1], list_count[LISTS ? kListPages : 1];
};

// Workgroup `bid` of `grid`.
template <class E, int DP, bool LISTS>
__device__ __forceinline__ void few_rows(const PagedAttn& a, FewLds<DP, LISTS>& sh, int64_t bid, int64_t grid) {
  constexpr int KS = few_waves(DP), BK = few_keys(DP);
  using St = Stager<DP, 1, BK>;
  using Rw = Rows<E, DP, BK, false>;
  constexpr int kTile = St::kTile, kND = DP / 32, kC = DP / 8;
  unsigned char* const lds_all = sh.tiles;
  auto& join_ml = sh.join_ml;
  auto& list_row = sh.list_row;
  auto& list_count = sh.list_count;
  const int tid = threadIdx.x, lane = tid & 63, row = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  Part w{};
  int rb = 0;             // (lists) block of 32 rows
  int64_t unit = 0;       // (lists) (token, head, rows)
  int part = 0;
  if constexpr (LISTS) {
    unit = uint32_t(bid) / uint32_t(a.parts);
    part = int(uint32_t(bid) % uint32_t(a.parts));
    const int rbs = (a.G + 31) / 32;
    rb = int(unit % rbs);
    w.pos = 0;
    w.end = 1;
    w.s = 0;
    const int64_t token = unit / rbs / a.Hkv;
    if (a.cu) {
      // the last sequence that does not begin past the token
      int lo = 0, hi = a.n_seqs;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= token) lo = mid;
        else hi = mid;
      }
      w.s = __builtin_amdgcn_readfirstlane(lo);
    } else {
      w.s = int(token / a.each);
    }
  } else {
    if (!a.whole && tid < 2) a.few.joins[2 * bid + tid].parts = 0;
    if (!find_few<DP>(a, bid, grid, w)) return;
  }

  const St stager(uint32_t(a.Hkv) * a.D * 2, 0);
  unsigned char* lds = lds_all + wave * (4 * kTile);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
      uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)lds)));
  const int dbytes = a.D * 2;

  while (w.pos < w.end) {
    const Seq q = seq_of(a, w.s);
    int kvh, first, rows, limit, least, tiles, steps = 0;  // first key, and tiles from there, of this part
    int64_t token;
    bool begins = true;  // whether the head's first step is this workgroup's
    if constexpr (LISTS) {
      const int rbs = (a.G + 31) / 32;
      kvh = int(unit / rbs % a.Hkv);
      token = unit / rbs / a.Hkv;
      if (token < q.at || token >= q.at + q.n) return;  // (behind the last sequence)
      rows = min(32, a.G - rb * 32);
      limit = max(0, limit_of(q, int(token - q.at)));
      const int keys = int(a.n_pages) * a.page;
      first = part * a.part_steps * (BK * KS);
      tiles = (min(keys - first, a.part_steps * (BK * KS)) + BK - 1) / BK;
      least = 0;
      // the part's pages: first row of each in the cache, and how many keys the token sees there
      const int from = first / a.page, to = min(int(a.n_pages), (first + tiles * BK + a.page - 1) / a.page);
      const int32_t* list = a.pages + (token * a.Hkv + kvh) * a.n_pages;
      const int32_t* table = a.table + int64_t(w.s) * a.cols;
      for (int i = from + tid; i < to; i += 64 * KS) {
        const int j = list[i];
        const bool in = j >= 0 && j < a.cols;
        const int id = in ? table[j] : -1;
        list_row[i - from] = id >= 0 && id < a.num_blocks ? id * a.page : -1;
        list_count[i - from] = in ? min(max(int64_t(limit) - int64_t(j) * a.page, int64_t(0)), int64_t(a.page)) : 0;
      }
      __syncthreads();
    } else {
      int step0 = 0;
      if (a.whole) {
        kvh = int(uint32_t(bid) % uint32_t(a.Hkv));
        steps = w.n;
      } else {
        // (the launch sees to it that a sequence's steps fit)
        const uint32_t into = uint32_t(w.pos - w.base), of = w.aligned ? uint32_t((w.n + w.per - 1) / w.per) : uint32_t(w.n) + 1;
        kvh = __builtin_amdgcn_readfirstlane(into / of);
        const uint32_t place = __builtin_amdgcn_readfirstlane(into - uint32_t(kvh) * of);
        if (w.aligned) {
          step0 = int(place) * int(w.per);
          steps = int(min(int64_t(w.n - step0), w.per));
        } else {
          w.pos += place == 0;  // (the head's own place; a part that ends with it has none of the head)
          if (w.pos >= w.end) return;
          step0 = int(place) - (place > 0);
          steps = int(min(int64_t(w.n - step0), w.end - w.pos));
        }
      }
      begins = step0 == 0;
      first = step0 * (BK * KS);
      tiles = (min(q.m - first, steps * (BK * KS)) + BK - 1) / BK;
      rows = q.n * a.G;
      token = q.at + min(row, rows - 1) / a.G;
      limit = limit_of(q, int(token - q.at));
      least = limit_of(q, 0);
    }
    const unsigned char* kbase = a.k + int64_t(kvh) * a.D * 2;
    const unsigned char* vbase = a.v + int64_t(kvh) * a.D * 2;
    const int r = rb * 32 + min(row, rows - 1);
    const int head = kvh * a.G + (LISTS ? r : r % a.G);
    u32x4_t qf[kC / 2];
    load_q<DP>(a, token, head, qf);

    // --- this wave's tiles: numbers wave, wave + KS, .. of the part
    const int used = max(0, (tiles - wave + KS - 1) / KS);
    const int32_t* table = a.table + int64_t(w.s) * a.cols;
    int id = -1, key = 0;  // of this lane's group: page, and (place among the) keys
    auto look = [&](int j) {
      key = first + (j * KS + wave) * BK + 8 * (lane % (BK / 8));
      // (read whatever the length is: it need not be there yet)
      if constexpr (!LISTS) id = table[min(int64_t(quotient(a.page8, key >> 3)), a.cols - 1)];
    };
    auto groups = [&]() {
      Groups<BK> g;
      const int j = quotient(a.page8, key >> 3), off = key - j * a.page;
      if constexpr (LISTS) {
        const int e = j - quotient(a.page8, first >> 3);
        const bool in = key < int(a.n_pages) * a.page;
        const int at = in ? list_row[e] : -1;
        g.set(at < 0 ? -1 : at + off, in ? list_count[e] - off : 0, stager.ts);
      } else {
        g.set(id >= 0 && id < a.num_blocks ? id * a.page + off : -1, q.m - key, stager.ts);
      }
      return g;
    };
    Rw rws;
    rws.clear();
    bool full = true, next_full = true, bad = false;
    uint32_t bits[BK / 32], next_bits[BK / 32];
    auto bring = [&](int buf) {
      const Groups<BK> g = groups();
      next_full = g.full();
#pragma unroll
      for (int i = 0; i < BK / 32; ++i) next_bits[i] = ~0u;
      if (!next_full) g.bits(next_bits);
      stager.stage(kbase, vbase, g, dbytes, lds0 + buf * kTile, lds0 + (2 + buf) * kTile);
    };
    look(0);
    if (used > 0) {
      bring(0);
      look(1);
    }
    // (the compiler does not know of the waits for the direct loads: with loads of its own still
    // open for it, it would wait for everything in every round)
#pragma unroll
    for (int t = 0; t < kC / 2; ++t) asm volatile("" : "+v"(qf[t]));
    for (int j = 0; j < used; ++j) {
      wait_vm<0>();
      asm volatile("" : "+v"(id));
      full = next_full;
#pragma unroll
      for (int i = 0; i < BK / 32; ++i) bits[i] = next_bits[i];
      if (j + 1 < used) {
        bring((j + 1) & 1);
        look(j + 2);
      }
      const int key0 = first + (j * KS + wave) * BK;
      unsigned char* vt = lds + (2 + (j & 1)) * kTile;
      const bool cut = !LISTS && key0 + BK > least;
      if (cut && q.n > 1) bad |= take_out<E, DP, BK, true>(vt, bits, 0, 1);
      else if (!full) take_out<E, DP, BK, false>(vt, bits, 0, 1);
      asm volatile("" ::: "memory");
      rws.add(lds + (j & 1) * kTile, vt, qf, a.scale, cut || !full, LISTS ? BK : limit - key0, bits);
    }
    if (!LISTS && bad)
      for (int j = 0; j < used; ++j) {
        const int key0 = first + (j * KS + wave) * BK;
        if (key0 + BK > least) add_taken_out(a, rws, w.s, kvh, key0, key0 + BK, limit);
      }

    // --- the waves' results joined: all into LDS, then every wave a part of the columns
    constexpr int kQuads = kND * 4, kMine = kQuads / KS;  // runs of 4 columns a lane
    static_assert(KS * kQuads * 1024 <= KS * 4 * kTile && kQuads % KS == 0, "the tiles' place");
    __syncthreads();  // (all waves are past their tiles)
    f32x4_t* join = reinterpret_cast<f32x4_t*>(lds_all) + here();
    join_ml[wave][0][lane] = rws.mx;
    join_ml[wave][1][lane] = rws.sum;
#pragma unroll
    for (int d = 0; d < kND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        join[(wave * kQuads + d * 4 + i) * 64] =
            f32x4_t{rws.o[d][4 * i], rws.o[d][4 * i + 1], rws.o[d][4 * i + 2], rws.o[d][4 * i + 3]};
    __syncthreads();
    {
      float all = -INFINITY, total = 0.f, f[KS];
#pragma unroll
      for (int g = 0; g < KS; ++g) all = fmaxf(all, join_ml[g][0][lane]);
#pragma unroll
      for (int g = 0; g < KS; ++g) {
        // (a wave without a maximum has seen no key, or only scores that are NaN, as its sum is)
        const float mg = join_ml[g][0][lane];
        f[g] = mg == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mg - all);
        total += mg == -INFINITY ? join_ml[g][1][lane] : join_ml[g][1][lane] * f[g];
      }
      total = sum_halves(total);
      const bool live = row < rows, done = LISTS ? a.parts == 1 : steps == w.n;
      // numbers: aligned, the workgroup's; else two for each, as the heads that it has a part of
      // only are one that goes on there and one that begins there
      const int64_t block = bid, id = LISTS || w.aligned ? block : 2 * block + begins;
      const float inv = total == 0.f ? 0.f : 1.f / total;  // (a query that sees no key: 0)
      unsigned char* dst = a.out + (token * a.Hq + head) * dbytes;
      float* part_dst = a.few.part + (id * a.rows + row) * a.D;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int quad = wave * kMine + i, col = (quad >> 2) * 32 + (quad & 3) * 8 + (lane >> 5) * 4;
        f32x4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < KS; ++g) {
          const f32x4_t x = join[(g * kQuads + quad) * 64];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = f[g] == 0.f ? y[e] : __builtin_fmaf(x[e], f[g], y[e]);
        }
        if (!live || col >= a.D) continue;
        if (done)
          *reinterpret_cast<u32x2_t*>(dst + col * 2) = u32x2_t{E::pack2(y[0] * inv, y[1] * inv), E::pack2(y[2] * inv, y[3] * inv)};
        else
          *reinterpret_cast<f32x4_t*>(part_dst + col) = y;
      }
      if (!done && wave == 0) {
        if (live && lane < 32) *reinterpret_cast<f32x2_t*>(a.few.ml + (id * a.rows + row) * 2) = f32x2_t{all, total};
        if (!LISTS && lane == 0) {
          PagedJoin j;
          if (w.aligned) {
            j.parts = int((w.n + w.per - 1) / w.per);
            j.index = int(w.pos - (w.base + int64_t(kvh) * j.parts));
            j.first = block - j.index;
            j.stride = 1;
            j.lead = 0;
          } else {
            const int64_t head0 = w.base + int64_t(kvh) * (w.n + 1) + 1;  // the head's first step
            j.index = int(block - head0 / w.per);
            j.parts = int((head0 + w.n - 1) / w.per - head0 / w.per) + 1;
            j.first = 2 * (block - j.index);
            j.stride = 2;
            j.lead = 1;
          }
          j.at = q.at;
          j.base = 0;
          j.kvh = kvh;
          j.rows = rows;
          a.few.joins[2 * block + begins] = j;
        }
      }
    }
    if constexpr (LISTS) return;
    if (w.aligned) return;
    w.pos += steps;
    if (w.pos >= w.end) return;
    __syncthreads();  // (the join's readers are done)
    if (w.pos >= w.base + (int64_t(w.n) + 1) * a.Hkv) {
      w.base += (int64_t(w.n) + 1) * a.Hkv;
      do {
        w.s += 1;
        if (w.s >= a.n_seqs) return;
        w.n = few_steps<DP>(a, seq_of(a, w.s));
      } while (w.n == 0);
    }
  }
}

template <class E, int DP, bool LISTS>
__global__ void __launch_bounds__(64 * few_waves(DP), 1)
paged_few_kernel(PagedAttn a) {
  __shared__ FewLds<DP, LISTS> sh;
  fill_rest(a, 64 * few_waves(DP));
  few_rows<E, DP, LISTS>(a, sh, blockIdx.x, gridDim.x);
}

// --- many rows ---------------------------------------------------------------------------
//
// 2048 tokens after 30000, 32 / 4 heads: 1070 us, 970 TFLOP/s; the matrix cores are busy 46 % of
// the cycles (2.0 GHz under this load) and take turns with the vector units' softmax, as in
// attn_prefill.hip.  Two workgroups a CU: one's softmax goes under the other's products.

constexpr int kManyRows = 128, kManyKeys = 64;
// Tiles of a part, at least, and of a sequence that is not cut.  (A part of 4 tiles instead of 8: 64
// tokens after 1000, 32 / 8 heads 33 -> 27 us.  To cut 5 to 8 tiles takes longer than it saves, the
// join being a launch: one prompt of 300 19 us whole, 24 cut; of 700, 16 / 8 heads, 32.5 and 30.)
constexpr int kManyLeast = 4, kManyWhole = 8;

__device__ __forceinline__ int many_blocks(const PagedAttn& a, const Seq& q) {
  const int64_t rows = int64_t(q.n) * a.G;
  return rows <= a.few_rows ? 0 : int((rows + kManyRows - 1) / kManyRows);
}
// Tiles of keys that block rb of a sequence's rows sees.
__device__ __forceinline__ int many_steps(const PagedAttn& a, const Seq& q, int rb) {
  const int64_t last = min((int64_t(rb) + 1) * kManyRows, int64_t(q.n) * a.G) - 1;
  return (max(0, limit_of(q, int(last / a.G))) + kManyKeys - 1) / kManyKeys;
}

// Tiles of keys of a part.  As many parts as fill the places for workgroups where there are
// fewer blocks of rows than those (whole numbers of them: 300 blocks of equal length in two
// parts each would take two rounds); else only what is longer than an even share.  Where the
// least part does not let them fill all places, one a CU, if those are no longer than kManyAlone: a
// second workgroup on some of the CUs would be what the others wait for (32 tokens after 20000, 32 /
// 8 heads: 320 parts of 8 tiles 45 us, 256 of 10 40; 300 after 4000, 16 / 8 heads 45 and 39).  How
// much longer was found by timing both: of 29 calls with parts of 8 to 13 tiles so (4 to 7 in
// pairs), 16 to 500 tokens after 1000 to 40000, 25 were as fast or up to 5 us faster with one a CU,
// four 2 to 4 us slower; with 17 and 18 tiles (7 and 8 in pairs) all four were slower.
constexpr int kManyAlone = 13;
struct Cut {
  int64_t blocks, total;
};
__device__ __forceinline__ int64_t many_part(const PagedAttn& a, const Cut& c) {
  if (a.most_split == 0) return 0x3FFFFFFF;
  auto share = [&](int64_t places) {
    const int64_t ways = c.blocks >= places || c.blocks == 0 ? places : c.blocks * (places / c.blocks);
    return (c.total + ways - 1) / ways;
  };
  int64_t per = max(int64_t(kManyLeast), share(a.slots));
  if (per <= kManyWhole && a.D <= 128 && share(a.slots / 2) <= kManyAlone) per = max(per, share(a.slots / 2));
  return min(int64_t(0x3FFFFFFF), per);
}

// A workgroup's part of a sequence's rows and keys, and how many there are in all.
struct Item {
  int s, parts;
  int64_t local, split, per;  // place among the sequence's items, its first partial result, tiles of a part
};
// This workgroup's item; false: there is none.
__device__ __forceinline__ bool find_many(const PagedAttn& a, Item& it) {
  const int lane = threadIdx.x & 63;
  const int64_t bid = blockIdx.x, grid = gridDim.x;
  const bool tell = bid == 0 && threadIdx.x < 64;  // (goes through all, to say how many partial results there are)
  Cut c{0, 0};
  for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
    const int x = s0 + lane;
    int64_t blocks = 0, steps = 0;
    if (x < a.n_seqs) {
      const Seq q = seq_of(a, x);
      blocks = int64_t(many_blocks(a, q)) * a.Hkv;
      steps = blocks * max(1, (q.m + kManyKeys - 1) / kManyKeys);
    }
    c.blocks += uniform64(__shfl(scan_lanes(blocks), 63));
    c.total += uniform64(__shfl(scan_lanes(steps), 63));
  }
  it.s = -1;
  int64_t base = 0, base_split = 0;
  if (c.blocks > 0) {
    it.per = many_part(a, c);
    for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
      const int x = s0 + lane;
      int64_t items = 0;
      int p = 1;
      if (x < a.n_seqs) {
        const Seq q = seq_of(a, x);
        const int steps = (q.m + kManyKeys - 1) / kManyKeys;
        p = steps <= kManyWhole ? 1 : int((steps + it.per - 1) / it.per);
        items = int64_t(many_blocks(a, q)) * a.Hkv * p;
      }
      const int64_t to = base + scan_lanes(items);
      // (offsets out of order can have more than the launch; what has no workgroup is not counted)
      const int64_t ps = p > 1 ? max(int64_t(0), min(items, grid - (to - items))) : 0;
      const int64_t to_split = base_split + scan_lanes(ps);
      const uint64_t in = __ballot(bid >= to - items && bid < to);
      if (in != 0) {
        const int l = __ffsll(static_cast<unsigned long long>(in)) - 1;
        it.s = s0 + l;
        it.parts = __builtin_amdgcn_readlane(p, l);
        it.local = bid - uniform64(__shfl(to - items, l));
        it.split = uniform64(__shfl(to_split - ps, l));
        if (!tell) break;
      }
      base = uniform64(__shfl(to, 63));
      base_split = uniform64(__shfl(to_split, 63));
    }
    if (it.s >= 0 && it.parts == 1) it.per = 0x3FFFFFFF;
  }
  if (tell && lane == 0) *a.n_split = base_split;
  return it.s >= 0;
}

template <int DP>
struct ManyLds {
  __align__(16) unsigned char tiles[4 * kManyKeys * DP * 2];  // K buffers, V buffers
  int taken;
};

template <class E, int DP>
__device__ __forceinline__ void many_rows(const PagedAttn& a, ManyLds<DP>& sh, const Item& it) {
  constexpr int QW = 4, BK = kManyKeys;
  using St = Stager<DP, QW, BK>;
  using Rw = Rows<E, DP, BK, (DP <= 128)>;
  constexpr int kTile = St::kTile, kC = DP / 8;
  unsigned char* const lds = sh.tiles;
  int& taken = sh.taken;
  const int tid = threadIdx.x, lane = tid & 63, row = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int s = __builtin_amdgcn_readfirstlane(it.s), parts = __builtin_amdgcn_readfirstlane(it.parts);
  const int64_t local = uniform64(it.local), split = uniform64(it.split);
  const int per = __builtin_amdgcn_readfirstlane(int(it.per));
  const Seq q = seq_of(a, s);
  const int kvh = int(local % a.Hkv), part = int(local / a.Hkv % parts);
  const int rb = many_blocks(a, q) - 1 - int(local / a.Hkv / parts);  // (the late rows, which see most keys, first)
  const int seen = many_steps(a, q, rb), first = part * per;
  const int tiles = max(0, min(seen - first, per));
  const bool whole = seen <= per;
  const int64_t number = split + local;  // of the partial result
  if (tiles == 0 && part > 0) {
    if (parts > 1 && tid == 0 && number < a.most_split) a.many.joins[number].parts = 0;
    return;
  }

  const int64_t all_rows = int64_t(q.n) * a.G, r0 = int64_t(rb) * kManyRows + wave * 32;
  const int64_t r = min(r0 + row, all_rows - 1);  // (rows past the end repeat the last one)
  const int tok = int(r / a.G), limit = limit_of(q, tok);
  const int least = limit_of(q, int(int64_t(rb) * kManyRows / a.G));  // keys all rows of the workgroup see
  const int least_w = limit_of(q, int(min(r0, all_rows - 1) / a.G));  // of the wave
  const int most_w = limit_of(q, int(min(r0 + 31, all_rows - 1) / a.G));
  const int mine = r0 < all_rows ? max(0, min((max(0, most_w) + BK - 1) / BK - first, tiles)) : 0;
  const int head = kvh * a.G + int(r - int64_t(tok) * a.G);
  u32x4_t qf[kC / 2];
  load_q<DP>(a, q.at + tok, head, qf);

  const St stager(uint32_t(a.Hkv) * a.D * 2, wave);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
      uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)lds)));
  const int dbytes = a.D * 2;
  const unsigned char* kbase = a.k + int64_t(kvh) * a.D * 2;
  const unsigned char* vbase = a.v + int64_t(kvh) * a.D * 2;
  const int32_t* table = a.table + int64_t(s) * a.cols;
  int id = -1, key = 0;
  auto look = [&](int j) {
    key = (first + j) * BK + 8 * (lane & 7);
    id = key < q.m ? table[quotient(a.page8, key >> 3)] : -1;
  };
  bool full = true, next_full = true;
  uint32_t bits[2] = {~0u, ~0u}, next_bits[2] = {~0u, ~0u};
  auto bring = [&](int buf) {
    Groups<BK> g;
    const int j = quotient(a.page8, key >> 3);
    g.set(id >= 0 && id < a.num_blocks ? id * a.page + (key - j * a.page) : -1, q.m - key, stager.ts);
    next_full = g.full();
    if (next_full) next_bits[0] = next_bits[1] = ~0u;
    else g.bits(next_bits);
    stager.stage(kbase, vbase, g, dbytes, lds0 + buf * kTile, lds0 + (2 + buf) * kTile);
  };
  if (tid == 0) taken = 0;
  if (tiles > 0) {
    look(0);
    bring(0);
    look(1);
  }
#pragma unroll
  for (int t = 0; t < kC / 2; ++t) asm volatile("" : "+v"(qf[t]));
  Rw rws;
  rws.clear();
  for (int j = 0; j < tiles; ++j) {
    wait_vm<0>();
    asm volatile("" : "+v"(id));
    __syncthreads();
    full = next_full;
    bits[0] = next_bits[0];
    bits[1] = next_bits[1];
    if (j + 1 < tiles) {
      bring((j + 1) & 1);
      look(j + 2);
    }
    const int key0 = (first + j) * BK;
    unsigned char* vt = lds + (2 + (j & 1)) * kTile;
    const bool cut = q.n > 1 && key0 + BK > least;
    if (cut || !full) {
      if (cut ? take_out<E, DP, BK, true>(vt, bits, wave, QW) : take_out<E, DP, BK, false>(vt, bits, wave, QW)) taken = 1;
      __syncthreads();
    }
    if (j < mine)
      rws.add(lds + (j & 1) * kTile, vt, qf, a.scale, key0 + BK > least_w || !full, limit - key0, bits);
  }
  __syncthreads();
  if (taken) {
    const int from = max(first * BK, max(0, least) / BK * BK);
    add_taken_out(a, rws, s, kvh, from, (first + tiles) * BK, limit);
  }
  const float total = sum_halves(rws.sum);
  const bool live = r0 + row < all_rows;
  if (whole) {
    write_rows(rws, total, live, a.out + ((q.at + tok) * a.Hq + head) * dbytes, dbytes);
  } else if (number < a.most_split) {  // (more: offsets out of order)
    write_part(a, rws, total, live, number * kManyRows + wave * 32 + row);
  }
  if (parts > 1 && tid == 0 && number < a.most_split) {
    PagedJoin j;
    j.index = part;
    j.parts = whole ? 0 : int((seen + per - 1) / per);
    j.first = number - int64_t(part) * a.Hkv;
    j.stride = a.Hkv;
    j.lead = 0;
    j.at = q.at;
    j.base = rb * kManyRows;
    j.kvh = kvh;
    j.rows = int(min(int64_t(kManyRows), all_rows - int64_t(rb) * kManyRows));
    if (j.first + int64_t(j.parts - 1) * a.Hkv >= a.most_split) j.parts = 0;
    a.many.joins[number] = j;
  }
}

template <class E, int DP>
__global__ void __launch_bounds__(256, DP == 256 ? 1 : 2)
paged_many_kernel(PagedAttn a) {
  __shared__ ManyLds<DP> sh;
  Item it;
  if (find_many(a, it)) many_rows<E, DP>(a, sh, it);
}

// --- the parts' results joined -----------------------------------------------------------

enum JoinOf { kFew, kLists, kMany, kBoth };

// Float4s from .. to - 1 of a block's output, `step` at a time with `ways` threads each, ONCE such at
// once.
template <class E, int ONCE>
__device__ __forceinline__ void join_rows(const PagedAttn& a, const PagedOut& o, const PagedJoin& j, int rows, int from, int to,
                                          int step, int ways, float (*part_sum)[6]) {
  constexpr int kOnce = ONCE;
  const int tid = threadIdx.x, way = tid / step, wide = a.D / 4;
  for (int e0 = from; e0 < to; e0 += step * kOnce) {
    f32x4_t y[kOnce];
    float l[kOnce], m[kOnce];
    int64_t at[kOnce];
    int col[kOnce], row[kOnce];
    bool in[kOnce];
#pragma unroll
    for (int u = 0; u < kOnce; ++u) {
      const int e = e0 + u * step + tid % step;
      in[u] = e < to && way < ways;
      row[u] = in[u] ? e / wide : 0;
      col[u] = in[u] ? (e - row[u] * wide) * 4 : 0;
      at[u] = j.first * rows + row[u];
      y[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      l[u] = 0.f;
      m[u] = -INFINITY;
    }
    // a result (maximum mi, sum li, x) into another; one without a maximum has seen no key, or
    // only scores that are NaN, as its sum is
    auto add = [&](int u, float mi, float li, f32x4_t x) {
      const float top = fmaxf(m[u], mi);
      const float f = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi - top);
      const float g = m[u] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[u] - top);
      l[u] = mi == -INFINITY ? l[u] + li : __builtin_fmaf(li, f, l[u] * g);
#pragma unroll
      for (int c = 0; c < 4; ++c) y[u][c] = f == 0.f ? y[u][c] * g : __builtin_fmaf(x[c], f, y[u][c] * g);
      m[u] = top;
    };
#pragma unroll 2
    for (int i = way; i < j.parts; i += ways) {
      f32x2_t ml[kOnce];
      f32x4_t x[kOnce];
#pragma unroll
      for (int u = 0; u < kOnce; ++u) {  // (threads beyond the last one read what is there)
        const int64_t r = at[u] + (int64_t(i) * j.stride + (i == 0 ? j.lead : 0)) * rows;
        ml[u] = *reinterpret_cast<const f32x2_t*>(o.ml + r * 2);
        x[u] = *reinterpret_cast<const f32x4_t*>(o.part + r * a.D + col[u]);
      }
#pragma unroll
      for (int u = 0; u < kOnce; ++u) add(u, ml[u][0], ml[u][1], x[u]);
    }
#pragma unroll
    for (int u = 0; u < kOnce; ++u) {
      if (u > 0 && e0 + u * step >= to) break;
      if (ways > 1) {
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; ++c) part_sum[tid][c] = y[u][c];
        part_sum[tid][4] = l[u];
        part_sum[tid][5] = m[u];
        __syncthreads();
        if (way == 0)
          for (int w = 1; w < ways; ++w) {
            const float* p = part_sum[w * step + tid];
            add(u, p[5], p[4], f32x4_t{p[0], p[1], p[2], p[3]});
          }
      }
      if (!in[u] || way > 0) continue;
      const float inv = l[u] == 0.f ? 0.f : 1.f / l[u];
      const int r = j.base + row[u], tok = r / a.G;
      unsigned char* dst = a.out + (((j.at + tok) * a.Hq + j.kvh * a.G + (r - tok * a.G)) * a.D + col[u]) * 2;
      *reinterpret_cast<u32x2_t*>(dst) =
          u32x2_t{E::pack2(y[u][0] * inv, y[u][1] * inv), E::pack2(y[u][2] * inv, y[u][3] * inv)};
    }
  }
}

// A workgroup for every partial result: an equal share of the block's output, 4 columns of a
// row a thread, the threads that are left over sharing the parts.  4 us where little was cut
// (launch and the descriptors' load), 8 for 14 MB of partial results.
template <class E, int OF>
__global__ void __launch_bounds__(256)
paged_join_kernel(PagedAttn a) {
  __shared__ float part_sum[256][6];
  PagedJoin j;
  // (both: the long sequences' partial results, then the short ones')
  const int64_t bid = OF == kBoth ? int64_t(blockIdx.x) - a.most_split : int64_t(blockIdx.x);
  const bool many = OF == kMany || (OF == kBoth && bid < 0);
  const PagedOut o = many ? a.many : a.few;
  const int rows = many ? kManyRows : a.rows;
  if constexpr (OF == kLists) {
    const int64_t unit = blockIdx.x / a.parts;
    const int rbs = (a.G + 31) / 32, rb = int(unit % rbs);
    j.index = blockIdx.x % a.parts;
    j.parts = a.parts;
    j.first = unit * a.parts;
    j.stride = 1;
    j.lead = 0;
    j.kvh = int(unit / rbs % a.Hkv);
    j.at = unit / rbs / a.Hkv;
    j.base = rb * 32;
    j.rows = min(32, a.G - rb * 32);
    if (a.cu && (j.at >= seq_at(a.cu, 0, a.T, a.n_seqs) || j.at < seq_at(a.cu, 0, a.T, 0))) return;  // (of no sequence)
  } else {
    if (many && int64_t(blockIdx.x) >= *a.n_split) return;
    j = o.joins[many ? int64_t(blockIdx.x) : bid];
    if (j.parts == 0) return;
  }
  const int wide = a.D / 4, all = j.rows * wide;  // float4s
  const int from = int(int64_t(all) * j.index / j.parts), to = int(int64_t(all) * (j.index + 1) / j.parts);
  // this workgroup's float4s `step` at a time, `ways` threads each; or, where there are many, four
  // such at once
  const int step = min(256, max(1, to - from)), ways = min(256 / step, min(16, j.parts));
  if (to - from > 256) join_rows<E, 4>(a, o, j, rows, from, to, step, ways, part_sum);
  else join_rows<E, 1>(a, o, j, rows, from, to, step, ways, part_sum);
}

template <class E, int DP>
hipError_t launch(const PagedAttn& a, const PagedPlan& p, hipStream_t stream) {
  const dim3 few(64 * few_waves(DP)), many(256);
  if (a.pages) {
    hipLaunchKernelGGL((paged_few_kernel<E, DP, true>), dim3(unsigned(p.few)), few, 0, stream, a);
    if (a.parts > 1) hipLaunchKernelGGL((paged_join_kernel<E, kLists>), dim3(unsigned(p.few)), many, 0, stream, a);
    return hipGetLastError();
  }
  if (p.few) hipLaunchKernelGGL((paged_few_kernel<E, DP, false>), dim3(unsigned(p.few)), few, 0, stream, a);
  if (p.many) hipLaunchKernelGGL((paged_many_kernel<E, DP>), dim3(unsigned(p.many)), many, 0, stream, a);
  const bool few_parts = p.few && !a.whole;
  if (few_parts && p.most_split)
    hipLaunchKernelGGL((paged_join_kernel<E, kBoth>), dim3(unsigned(p.most_split + 2 * p.few)), many, 0, stream, a);
  else if (few_parts)
    hipLaunchKernelGGL((paged_join_kernel<E, kFew>), dim3(unsigned(2 * p.few)), many, 0, stream, a);
  else if (p.most_split)
    hipLaunchKernelGGL((paged_join_kernel<E, kMany>), dim3(unsigned(p.most_split)), many, 0, stream, a);
  return hipGetLastError();
}

}  // namespace

PagedPlan plan_paged_attn(int64_t T, int64_t n_seqs, bool cu, int64_t cols, int page, int64_t n_pages, int Hq, int Hkv,
                          int D, int cus) {
  PagedPlan p{};
  const int64_t G = Hq / Hkv;
  const int ks = few_waves(D);
  const int64_t step = int64_t(few_keys(D)) * ks;
  size_t n = 0;
  auto take = [&](size_t bytes) {
    const size_t at = n;
    n += (bytes + 255) / 256 * 256;
    return at;
  };
  auto room = [&](PagedPlan::Room& o, size_t joins, size_t ids, size_t rows) {
    o.joins = take(joins * sizeof(PagedJoin));
    o.ml = take(ids * rows * 2 * 4);
    o.part = take(ids * rows * D * 4);
  };
  p.parts = 1;
  if (n_pages > 0) {
    const int64_t units = T * Hkv * ((G + 31) / 32), steps = (n_pages * page + step - 1) / step;
    // parts: as many as give each CU a workgroup; and a list in LDS
    const int64_t most = std::max<int64_t>(1, (int64_t(kListPages) - 2) * page / step);
    int64_t parts = std::max<int64_t>(1, std::min<int64_t>(steps, cus / units));
    parts = std::max(parts, (steps + most - 1) / most);
    p.part_steps = int((steps + parts - 1) / parts);
    p.parts = int((steps + p.part_steps - 1) / p.part_steps);
    p.rows = int(std::min<int64_t>(32, G));
    p.few = units * p.parts;
    if (p.parts > 1) room(p.few_room, 0, size_t(units) * p.parts, p.rows);
    p.bytes = n;
    return p;
  }
  const int64_t each = cu ? 0 : T / n_seqs;
  const bool few = cu ? true : each * G <= 32, many = cu ? T * G > 32 : each * G > 32;
  p.few_rows = few ? 32 : 0;
  if (many) p.n_split = take(8);
  if (few) {
    const int64_t steps = std::max<int64_t>(1, (cols * page + step - 1) / step);  // of a sequence as long as the table is wide
    const int64_t units = n_seqs * Hkv, full = cus;  // what LDS has room for
    // A head a workgroup, and nothing to join, where parts cannot save what the join's launch costs,
    // whatever the lengths are: 4 us, about 4 steps.  The longest sequence has no more than 4 steps
    // over an equal share (8 in all), and the places that the last round leaves empty are worth 2
    // steps a place at most (40 sequences of 1024 keys, 8 heads: 320 workgroups 48 us, parts 42 and
    // the join 4).  (1 to 96 sequences of similar lengths, 128 to 2048 keys, 4 and 8 heads: of 147 calls
    // that this takes all were 0.8 to 10 us faster so.  So were 71 of the 147 others, by up to 6.7,
    // but for lengths that differ: one of 2048 keys beside short ones would be 16 steps on its own.)
    const int64_t rounds = (units + full - 1) / full;
    p.whole = steps <= 4 + std::min<int64_t>(4, (units * steps + full - 1) / full) &&
              (rounds == 1 || (rounds * full - units) * steps <= 2 * full);
    p.few = p.whole ? units : std::min<int64_t>(full, units * (steps + 1));
    p.rows = int(cu ? 32 : each * G);
    if (!p.whole) room(p.few_room, size_t(p.few) * 2, size_t(p.few) * 2, p.rows);
  }
  if (many) {
    p.slots = (D > 128 ? 1 : 2) * cus;
    // (offsets: a sequence of this launch has 33 rows at least, and so no more blocks than its rows
    // / 33; in a packed step there is room for few, whatever the number of sequences)
    const int64_t blocks = cu ? std::min(T * G / 33, T * G / kManyRows + n_seqs) * Hkv
                              : n_seqs * Hkv * ((each * G + kManyRows - 1) / kManyRows);
    // (equal numbers of tokens: as many blocks as places or more are cut only for unequal lengths)
    const bool cut = (n_seqs > 1 || blocks < p.slots) && cols * page > kManyWhole * kManyKeys;
    p.many = blocks + (cut ? p.slots : 0);
    p.most_split = cut ? 2 * p.slots : 0;
    room(p.many_room, size_t(p.most_split), size_t(p.most_split), kManyRows);
  }
  p.bytes = n;
  return p;
}

hipError_t launch_paged_attn(const PagedAttn& a, const PagedPlan& p, int fp16, hipStream_t stream) {
  if (fp16) return a.D > 128 ? launch<AttnFp16, 256>(a, p, stream) : a.D > 64 ? launch<AttnFp16, 128>(a, p, stream) : launch<AttnFp16, 64>(a, p, stream);
  return a.D > 128 ? launch<AttnBf16, 256>(a, p, stream) : a.D > 64 ? launch<AttnBf16, 128>(a, p, stream) : launch<AttnBf16, 64>(a, p, stream);
}

}  // namespace mqk
