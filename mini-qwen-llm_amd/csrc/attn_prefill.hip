// Causal attention over packed prompts with grouped heads:
//
//   O[i] = sum_j softmax_j(scale * Q[i] . K[j]) V[j],   j < m - n + i + 1
//
// for query i of a sequence's n queries and m keys (m = n for a whole prompt, m > n where
// the prompt continues one whose keys are there already).  The reference runs it as
// paged_attn_prefill (mini_qwen/kernels/paged_attn_prefill.py:64-156).
//
// One pass over the keys with a running maximum and sum.  A wave takes 32 queries of one
// head; QW waves of a workgroup share the tiles of kBK keys that they stage in LDS (two
// buffers, direct loads, one barrier a tile), and KS such groups take every KS-th tile each,
// joined in LDS at the end:
//   QW 4, KS 1  128 queries a workgroup, two workgroups a CU: what long prompts run on
//   QW 4, KS 2  where those would be no more workgroups than CUs: half the tiles for each
//   QW 1, KS 4  where there is even less: 32 queries a workgroup, no barrier until the join
// Few queries over many keys: the keys in parts (QW 4, KS 1), a workgroup each, whose O,
// maxima and sums a second launch joins.
//
// The scores are computed transposed, S^T = K Q^T, on the 32 x 32 MFMAs, so that one lane
// holds scores of one query only: a tile's maximum and sum are lane-local but for one
// exchange between the halves of the wave.  The accumulator's layout is the operand layout
// of the second product up to an order of the keys, and a sum over keys has no order: the
// probabilities go from S^T into O^T = V^T P^T without leaving their registers, if V^T is
// read in the same order of keys.  That read transposes 4 x 16 blocks on the way out of the
// LDS (ds_read_b64_tr_b16).
//
// Scores, maxima, sums and O are fp32; P is rounded once to the tensors' type for the
// second product (2^-8 relative a term for bf16, as V itself carries), the output once.
//
// Measured, bf16, 32 heads of 128: one prompt of 8192 tokens (4 key heads) 520 to 533 us, 1040
// TFLOP/s of the 1430 that a large matrix product reaches; there the matrix cores are busy 48 %
// of the time, the vector units 36 %, and the card lowers its clock under the load (the cycles
// stay the same from launch to launch, the time does not).  1024 queries over 8024 keys 136
// us; 16 prompts of 513 tokens on average 79 us, of which 32 us are its bytes and 36 us its
// products, hardly over one another in workgroups of five tiles.  Heads of 256 (one wave a
// SIMD): 566 TFLOP/s; fp32: 108 of 154.  Small prompts are a launch and a chain of loads: 128
// tokens of 16 heads, fp32, 12.9 us.  Not kept, at 8192 tokens (us, where the form kept took 523
// to 533): 8 waves to a tile of keys (523 to 534; ragged prompts 102 to 110), tiles of 32 keys
// with three waves a SIMD (546; 729 with registers spilled), half a tile's scores ahead of its
// values (560 to 572), loads spread over the products (580 to 600), two barriers a tile with
// some loads left under way (590 to 600), exponents and values interleaved by hand (533 to 541),
// the sum as a product with ones (557), a higher wave priority around the products (541) or by
// the wave's slot (532), scheduling groups (no effect).
#include "mqk_attn.h"
#include "mqk_device.h"

namespace mqk {
namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// 16 bytes of zeros: what the columns past a head size that is no whole tile are read from.
__device__ const u32x4_t g_zero16 = {0, 0, 0, 0};

struct AttnBf16 : Bf16 {
  static constexpr int kBytes = 2;
  static constexpr uint32_t kExp = 0x7F80u;
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) { return mfma_32x32x16(a, b, c); }
};
struct AttnFp16 : Fp16 {
  static constexpr int kBytes = 2;
  static constexpr uint32_t kExp = 0x7C00u;
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0,
                                                  0, 0);
  }
};
struct AttnF32 {
  static constexpr int kBytes = 4;
  static constexpr uint32_t kExp = 0x7F800000u;
  // four k-steps of 2: slot h of step e is element e of half h's four
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
};

// Where chunk c (16 bytes) of row r lies in a staged row of C chunks.  K rows are read a
// chunk column at a time (32 rows, one chunk): 16 neighbouring rows take 16 different bank
// groups.  V rows are read 4 at a time, 4 neighbouring chunks each (16-bit types), or one
// row by each half of the wave, 4 rows apart (fp32).
template <int C>
__device__ __forceinline__ int k_slot(int r, int c) {
  return C >= 16 ? (c ^ (r & 15)) : (c ^ ((r >> 1) & 7));
}
template <int C, int BYTES>
__device__ __forceinline__ int v_slot(int r, int c) {
  if (BYTES == 4) return c ^ (((r >> 2) & 1) << 3);
  return C >= 16 ? (c ^ ((r & 3) << 2)) : (c ^ (((r >> 1) & 1) << 2));
}

__device__ __forceinline__ float max_halves(float x) {  // over lanes l and l + 32, to both
  const u32x2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const u32x2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// First token and length of sequence s: offsets in device memory, clamped into the tensor,
// or equal lengths.
__device__ __forceinline__ int64_t seq_at(const int32_t* cu, int64_t each, int64_t total, int s) {
  const int64_t at = cu ? int64_t(cu[s]) : each * s;
  return at < 0 ? 0 : at > total ? total : at;
}

// L2 -> LDS as dma16, from a wave-uniform base plus a 32-bit offset of the lane.  The load may
// read M0 one wait state after it is written, and its base five after a vector instruction
// wrote that (v_readlane, where the compiler keeps the base in a vector register), of which
// the compiler sees to none inside the asm.
__device__ __forceinline__ void dma16_from(const unsigned char* base, uint32_t off, uint32_t lds_base) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 2\n\t"
      "global_load_lds_dwordx4 %2, %3\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(off), "s"(base)
      : "memory");
}

// kNBuf 2: the next tile is loaded under the present one; 1: what LDS has room for where every
// wave has tiles of its own (fp32 heads past 64).
template <class E, int DP, int QW, int KS>
struct AttnShape {
  static constexpr int kBQ = 32 * QW;
  static constexpr int kBK = QW == 1 || E::kBytes == 4 ? 32 : 64;
  static constexpr int kTile = kBK * DP * E::kBytes;
  static constexpr int kNBuf = KS * 4 * kTile <= 128 * 1024 ? 2 : 1;
  static constexpr int kThreads = 64 * QW * KS;
  static constexpr int kJoin = (KS - 1) * QW * DP * 128;  // bytes of the other groups' O
  static constexpr int kLds = KS * 2 * kNBuf * kTile > kJoin ? KS * 2 * kNBuf * kTile : kJoin;
  static_assert(kLds <= 128 * 1024 + 1024, "LDS");
  static_assert(kNBuf == 2 || QW == 1, "one buffer is staged over without a barrier by the wave that reads it");
  // waves a SIMD that the registers are to allow
  static constexpr int kWaves = DP == 256 ? 1 : QW * KS == 4 && QW == 1 ? 1 : 2;
};

// PARTS: the keys in a.parts parts.  (In one kernel with the rest the code for them cost a long
// prompt 5 % of its time: 546 us, without 518, for 8192 tokens of 32 heads.)
template <class E, int DP, int QW, int KS, bool PARTS>
__global__ void __launch_bounds__(64 * QW * KS, (AttnShape<E, DP, QW, KS>::kWaves))
attn_prefill_kernel(AttnArgs a) {
  using Sh = AttnShape<E, DP, QW, KS>;
  constexpr int kBQ = Sh::kBQ, kBK = Sh::kBK, kTile = Sh::kTile, kNBuf = Sh::kNBuf;
  constexpr int kES = E::kBytes;
  constexpr int kRow = DP * kES;           // bytes of a staged row
  constexpr int kC = kRow / 16;            // its 16-byte chunks
  constexpr int kLoads = kTile / (QW * 1024);
  constexpr int kNB = kBK / 32;            // 32-key blocks of a tile
  constexpr int kND = DP / 32;             // 32-wide blocks of the head
  __shared__ __align__(16) unsigned char lds_all[Sh::kLds];  // of each group: K buffers, V buffers
  __shared__ float join_ml[KS > 1 ? (KS - 1) * QW : 1][2][64];
  __shared__ int redo;

  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, row = lane & 31;
  const int wave_id = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave = wave_id % QW, group = wave_id / QW;

  // --- the tile: head and slot, and of the slot the sequence and its place in it.  Slot
  // numbers leave gaps: sequence s starts at slot cu[s] / kBQ + s, which is monotone and
  // leaves it enough of them, so that no sum over the lengths is needed.
  int head, slot, part;
  {
    const int bid = blockIdx.x, nslots = a.nslots;
    if (a.xcds > 1 && a.Hq % a.xcds == 0) {  // the heads of a group of an XCD share its L2
      const int per = a.Hq / a.xcds, i = bid / a.xcds;
      head = (bid % a.xcds) * per + i % per;
      slot = i / per;
    } else {
      head = bid % a.Hq;
      slot = bid / a.Hq;
    }
    part = PARTS ? slot % a.parts : 0;
    slot = nslots - 1 - (PARTS ? slot / a.parts : slot);  // the late queries, which see most keys, first
  }
  int s;
  int64_t q_at, q_to;  // the sequence's queries (n_seqs: the rows behind the last one)
  if (a.cu_q) {
    // the last sequence whose first slot is not past this one: 64 offsets at a time, which
    // cover 63 sequences
    s = 0;
    q_at = q_to = 0;
    for (int base = 0; base <= a.n_seqs; base += 63) {
      const int c = base + lane;
      const int64_t at = seq_at(a.cu_q, 0, a.T, c <= a.n_seqs ? c : a.n_seqs);
      const int n = __popcll(__ballot(c <= a.n_seqs && at / kBQ + c <= slot));
      if (n == 0) return;  // (offsets out of order)
      if (n <= 63) {
        s = base + n - 1;
        q_at = __builtin_amdgcn_readlane(int(at), n - 1);
        q_to = __builtin_amdgcn_readlane(int(at), n);
        break;
      }
    }
  } else {
    // equal lengths: a whole number of slots each
    s = slot / int((a.each_q + kBQ - 1) / kBQ);
    q_at = a.each_q * s;
    q_to = q_at + a.each_q;
  }
  const int64_t tile = a.cu_q ? slot - (q_at / kBQ + s) : slot % int((a.each_q + kBQ - 1) / kBQ);
  const int64_t orow = int64_t(a.Hq) * a.D * kES;  // bytes of an output token
  if (s >= a.n_seqs) {  // behind the last sequence
    const int64_t t0 = q_at + tile * kBQ;
    if (tile < 0 || !a.fill || part > 0) return;
    const int chunks = a.D * kES / 16;
    for (int i = tid; i < kBQ * chunks; i += Sh::kThreads) {
      const int64_t t = t0 + i / chunks;
      if (t < a.T)
        *reinterpret_cast<u32x4_t*>(a.out + t * orow + (int64_t(head) * chunks + i % chunks) * 16) = u32x4_t{0, 0, 0, 0};
    }
    return;
  }
  const int64_t n64 = q_to - q_at;
  if (tile < 0 || tile * kBQ >= n64) return;
  const int n = int(n64);
  int64_t k_at = q_at, k_to = q_to;
  if (a.cu_k || !a.cu_q) {
    k_at = seq_at(a.cu_k, a.each_k, a.Tk, s);
    k_to = seq_at(a.cu_k, a.each_k, a.Tk, s + 1);
  }
  const int m = k_to < k_at ? 0 : int(k_to - k_at);

  const int q0 = int(tile) * kBQ, w0 = q0 + wave * 32;  // first query of the workgroup and of the wave
  const int qi = min(w0 + row, n - 1);                   // (rows past the end repeat the last one)
  const int shift = m - n;                               // (may be negative: such queries see nothing)
  const int limit = shift + qi + 1;                      // keys this lane's query sees
  auto tiles_to = [&](int queries) { return (max(0, min(m, shift + min(queries, n))) + kBK - 1) / kBK; };
  const int seen = tiles_to(q0 + kBQ);                   // tiles that any query of the workgroup sees
  // of them this part's, first .. first + tiles - 1, and those that one of the wave's sees
  const int per = PARTS ? (seen + a.parts - 1) / a.parts : seen, first = PARTS ? part * per : 0;
  const int tiles = max(0, min(seen - first, per));
  const int mine = w0 < n ? max(0, min(tiles_to(w0 + 32) - first, tiles)) : 0;
  const int least = shift + q0 + 1, least_w = shift + w0 + 1;  // keys all of them see
  const int kvh = head / (a.Hq / a.Hkv);
  const unsigned char* kbase = a.k + k_at * a.k_ts + int64_t(kvh) * a.k_hs;
  const unsigned char* vbase = a.v + k_at * a.v_ts + int64_t(kvh) * a.v_hs;
  const int dbytes = a.D * kES;

  // The queries stay in registers (heads past 128 have the whole of a SIMD's for one wave).
  const unsigned char* qsrc = a.q + (q_at + qi) * a.q_ts + int64_t(head) * a.q_hs;
  auto load_q = [&](int t) {
    const int at = (2 * t + half) * 16;
    return DP == a.D || at < dbytes ? *reinterpret_cast<const u32x4_t*>(qsrc + at) : u32x4_t{0, 0, 0, 0};
  };
  u32x4_t qf[kC / 2];
#pragma unroll
  for (int t = 0; t < kC / 2; ++t) qf[t] = load_q(t);

  unsigned char* lds = lds_all + group * (2 * kNBuf * kTile);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(
      uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)lds)));
  // Staging: every load of a wave fills 64 chunks in a row, kPer rows (or part of one).  Whole
  // tiles are addressed from a uniform base with offsets of the lane that repeat every
  // kDist loads, the period of the chunks' order.
  constexpr int kPer = 64 / kC > 0 ? 64 / kC : 1;
  static_assert(kC <= 64, "a load holds a whole row at least");
  constexpr int kStep = QW * kPer;  // rows between a wave's loads
  constexpr int kDist = kStep >= 16 ? 1 : (16 / kStep < kLoads ? 16 / kStep : kLoads);
  uint32_t koff[kDist], voff[kDist];
#pragma unroll
  for (int i = 0; i < kDist; ++i) {
    const int r = (i * QW + wave) * kPer + lane / kC, c = lane % kC;
    koff[i] = uint32_t(lane / kC) * uint32_t(a.k_ts) + uint32_t(k_slot<kC>(r, c)) * 16;
    voff[i] = uint32_t(lane / kC) * uint32_t(a.v_ts) + uint32_t(v_slot<kC, kES>(r, c)) * 16;
  }
  auto stage = [&](bool is_v, int kt, int buf) {
    const unsigned char* base = is_v ? vbase : kbase;
    const int64_t ts = is_v ? a.v_ts : a.k_ts;
    const uint32_t to = lds0 + uint32_t((is_v ? kNBuf + buf : buf) * kTile + wave * 1024);
    if (DP == a.D && (kt + 1) * kBK <= m && !a.far) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        dma16_from(base + (int64_t(kt) * kBK + (i * QW + wave) * kPer) * ts, is_v ? voff[i % kDist] : koff[i % kDist],
                   to + i * QW * 1024);
      return;
    }
    constexpr int kAtOnce = DP == 256 ? 1 : kLoads;  // (addresses kept for all of them would not fit the registers)
#pragma unroll kAtOnce
    for (int i = 0; i < kLoads; ++i) {
      const int r = (i * QW + wave) * kPer + lane / kC, c = lane % kC;
      const int key = min(kt * kBK + r, m - 1);  // (rows past the last key repeat it; their scores are masked)
      const int at = (is_v ? v_slot<kC, kES>(r, c) : k_slot<kC>(r, c)) * 16;
      const unsigned char* from = base + int64_t(key) * ts + at;
      if (DP != a.D && at >= dbytes) from = reinterpret_cast<const unsigned char*>(&g_zero16);
      dma16(from, to + i * QW * 1024);
    }
  };
  // A group's tiles are those of number first + j * KS + group.  A wave with tiles of its own (QW 1)
  // waits for its loads only, the others for each other too.
  auto arrive = [&]() {
    wait_vm<0>();
    if constexpr (QW > 1) __syncthreads();
  };
  auto of_group = [&](int all) { return (all - group + KS - 1) / KS; };  // (all >= 0)
  const int rounds = (tiles + KS - 1) / KS;    // the same for all groups: barriers
  const int staged = max(0, of_group(tiles));  // tiles this group stages
  const int used = max(0, of_group(mine));     // tiles this wave computes

  if (kNBuf == 2 && staged > 0) {
    stage(false, first + group, 0);
    stage(true, first + group, 0);
  }
  // (the compiler does not know of the waits for the direct loads: with the queries' own
  // loads still open for it, it would wait for everything in every round)
#pragma unroll
  for (int t = 0; t < kC / 2; ++t) asm volatile("" : "+v"(qf[t]));

  f32x16_t o[kND];
  // the running maximum, scaled (as the exponents take it) and as it was, and the sum
  float mx, mraw, sum;
  bool large;  // of the maximum: its fp32 step counts
  bool careful = false;

  auto product = [&](int j, f32x16_t (&st)[kNB]) {  // scores of tile j
    const unsigned char* kt_lds = lds + (kNBuf == 2 ? j & 1 : 0) * kTile;
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb) st[nb] = f32x16_t{};
    // Fragments are read a group of 4 products ahead; the compiler would read each right
    // before its product and wait for it there.
    constexpr int kAll = kC / 2 * kNB, kGroup = DP == 256 && kES == 4 ? 2 : 4;
    static_assert(kAll % kGroup == 0, "whole groups");
    u32x4_t kf[2][kGroup];
    auto fetch = [&](int g) {
#pragma unroll
      for (int e = 0; e < kGroup; ++e) {
        const int t = (g * kGroup + e) / kNB, r = (g * kGroup + e) % kNB * 32 + row;
        kf[g & 1][e] = *reinterpret_cast<const u32x4_t*>(kt_lds + r * kRow + k_slot<kC>(r, 2 * t + half) * 16);
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
  };
  // Masks tile j's scores, takes their maximum into account.
  auto prepare = [&](int j, f32x16_t (&st)[kNB]) {
    const int kt = first + j * KS + group;
    if ((kt + 1) * kBK > least_w) {
      const int rel = limit - kt * kBK - 4 * half;
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          st[nb][i] = nb * 32 + 8 * (i / 4) + i % 4 < rel ? st[nb][i] : -INFINITY;
    }
    float top = st[0][0];
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, st[nb][i]);
    // O and the sum are brought to a new maximum only where one grew by more than 2^8: until
    // then the terms stay below 256, which no rounding minds.
    if (__any(top * a.scale > mx + 8.f)) {
      const float traw = max_halves(top);
      const float now = fmaxf(mx, traw * a.scale);
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
  };
  auto exponents = [&](f32x16_t (&st)[kNB]) {
    const float sub = large || mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        st[nb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[nb][i], a.scale, -sub));
        sum += st[nb][i];
      }
  };
  auto values = [&](int j, f32x16_t (&st)[kNB]) {  // O += V^T P^T of tile j
    const unsigned char* vt_lds = lds + (kNBuf + (kNBuf == 2 ? j & 1 : 0)) * kTile;
    if constexpr (kES == 2) {
      // A operand: V^T, lane = (d = 16 * (lane / 16 % 2) + lane % 16, keys of half), read
      // as blocks of 4 keys x 16 columns: this lane's address is that of key
      // lane % 16 / 4, columns 4 * (lane % 4), and it receives column lane % 16.
      const int r0 = 4 * half + ((lane & 15) >> 2), c0 = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          u32x4_t pf;
#pragma unroll
          for (int e = 0; e < 4; ++e) pf[e] = E::pack2(st[nb][8 * ks + 2 * e], st[nb][8 * ks + 2 * e + 1]);
#pragma unroll
          for (int d = 0; d < kND; ++d) {
            const int kb = nb * 32 + ks * 16;
            const unsigned char* at =
                vt_lds + (kb + r0) * kRow + v_slot<kC, kES>(r0, d * 4 + c0) * 16 + (lane & 1) * 8;
            typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;
            const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
            const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * kRow));
            const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo), h2 = __builtin_bit_cast(u32x2_t, hi);
            o[d] = E::mfma32(u32x4_t{l2[0], l2[1], h2[0], h2[1]}, pf, o[d]);
          }
        }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = 8 * (i / 4) + i % 4 + 4 * half;
#pragma unroll
        for (int d = 0; d < kND; ++d) {
          const int c = (d * 32 + row) / 4;
          const float v = *reinterpret_cast<const float*>(vt_lds + key * kRow + v_slot<kC, kES>(key, c) * 16 + (row & 3) * 4);
          o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, st[0][i], o[d], 0, 0, 0);
        }
      }
    }
  };
  // (careful) values that are not finite leave a tile that some query does not see whole:
  // those that are seen are added at the end
  auto sanitise = [&](int j) {
    if (j < staged && (first + j * KS + group + 1) * kBK > least) {
      uint32_t* w = reinterpret_cast<uint32_t*>(lds + (kNBuf + (kNBuf == 2 ? j & 1 : 0)) * kTile);
      for (int i = wave * 64 + lane; i < kTile / 4; i += QW * 64) {
        uint32_t x = w[i];
        if (kES == 4) {
          if ((x & E::kExp) == E::kExp) x = 0;
        } else {
          if ((x & E::kExp) == E::kExp) x &= 0xFFFF0000u;
          if ((x & (E::kExp << 16)) == (E::kExp << 16)) x &= 0xFFFFu;
        }
        w[i] = x;
      }
    }
    __syncthreads();
  };

  for (;;) {
#pragma unroll
    for (int d = 0; d < kND; ++d) o[d] = f32x16_t{};
    mx = mraw = -INFINITY;
    sum = 0.f;
    large = false;
    {
      f32x16_t st[kNB];
      if (kNBuf == 2 && careful && staged > 0) {
        stage(false, first + group, 0);
        stage(true, first + group, 0);
      }
      for (int j = 0; j < rounds; ++j) {
        const int next = kNBuf == 2 ? j + 1 : j;
        if (kNBuf == 2) arrive();
        if (next < staged) {
          stage(false, first + next * KS + group, kNBuf == 2 ? next & 1 : 0);
          stage(true, first + next * KS + group, kNBuf == 2 ? next & 1 : 0);
        }
        if (kNBuf == 1) arrive();
        if (careful) sanitise(j);
        if (j < used) {
          product(j, st);
          prepare(j, st);
          exponents(st);
          values(j, st);
        }
      }
    }
    if (careful) break;
    // A masked value that is not finite has come in as 0 * V: where the output is not
    // finite, the tile is done again with such values kept apart.
    float bad = 0.f;
#pragma unroll
    for (int d = 0; d < kND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) bad = __builtin_fmaf(o[d][i], 0.f, bad);
    if (tid == 0) redo = 0;
    __syncthreads();
    if (bad != 0.f) redo = 1;
    __syncthreads();
    if (!redo) break;
    careful = true;
  }
  if constexpr (KS > 1) {
    // --- the groups' results, lane by lane (all waves are past their tiles)
    float* part = reinterpret_cast<float*>(lds_all);
    if (careful) __syncthreads();
    if (group > 0) {
      const int at = (group - 1) * QW + wave;
      join_ml[at][0][lane] = mx;
      join_ml[at][1][lane] = sum;
#pragma unroll
      for (int d = 0; d < kND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) part[((at * kND + d) * 16 + i) * 64 + lane] = o[d][i];
    }
    __syncthreads();
    if (group > 0) return;
    float all = mx;
#pragma unroll
    for (int g = 0; g < KS - 1; ++g) all = fmaxf(all, join_ml[g * QW + wave][0][lane]);
    const float f0 = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - all);
    // (a group without a maximum has seen no key, or only scores that are NaN, as its sum is)
    sum = mx == -INFINITY ? sum : sum * f0;
#pragma unroll
    for (int d = 0; d < kND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = mx == -INFINITY ? 0.f : o[d][i] * f0;
#pragma unroll
    for (int g = 0; g < KS - 1; ++g) {
      const int at = g * QW + wave;
      const float mg = join_ml[at][0][lane];
      if (mg == -INFINITY) {
        sum += join_ml[at][1][lane];
        continue;
      }
      const float f = __builtin_amdgcn_exp2f(mg - all);
      sum = __builtin_fmaf(join_ml[at][1][lane], f, sum);
#pragma unroll
      for (int d = 0; d < kND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = __builtin_fmaf(part[((at * kND + d) * 16 + i) * 64 + lane], f, o[d][i]);
    }
  }
  if (careful) {
    // the values that are not finite, of the keys that were masked for some query of the tile
    const int from = max(first * kBK, least / kBK * kBK);
    const int to = min(limit, min(m, (first + tiles) * kBK));
    for (int key = from; key < to; ++key) {
      const unsigned char* src = vbase + int64_t(key) * a.v_ts;
#pragma unroll
      for (int d = 0; d < kND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int col = d * 32 + 8 * (i / 4) + 4 * half + i % 4;
          if (col >= a.D) continue;
          uint32_t x;
          if (kES == 4) x = *reinterpret_cast<const uint32_t*>(src + col * kES);
          else x = *reinterpret_cast<const uint16_t*>(src + col * kES);
          if ((x & E::kExp) == E::kExp) {
            float v;
            if constexpr (kES == 4) v = __uint_as_float(x);
            else v = E::to_f32(x);
            o[d][i] += v;
          }
        }
    }
  }

  const float total = sum_halves(sum);
  if constexpr (PARTS) {  // joined by a second launch
    static_assert(KS == 1, "one group of waves");
    int r = row;
    asm volatile("" : "+v"(r));  // (not worked out ahead and kept through the loop)
    if (w0 + r >= n) return;
    const int64_t at = ((q_at + w0 + r) * a.Hq + head) * a.parts + part;
    if (half == 0) *reinterpret_cast<f32x2_t*>(a.part_ml + at * 2) = f32x2_t{mx, total};
    if (tiles == 0) return;  // (nothing seen, as the maximum says)
    float* dst = a.part + at * a.D;
#pragma unroll
    for (int d = 0; d < kND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = d * 32 + j * 8 + half * 4;
        if (col < a.D)
          *reinterpret_cast<f32x4_t*>(dst + col) = f32x4_t{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
      }
    return;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;  // (a query that sees no key: 0)
  const bool live = w0 + row < n;
  unsigned char* dst = a.out + (q_at + qi) * orow + int64_t(head) * dbytes;
#pragma unroll
  for (int d = 0; d < kND; ++d) {
    if constexpr (kES == 2) {
      // four columns a lane in two runs 8 apart: the halves swap them into runs of 8
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        u32x4_t w;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t x = E::pack2(o[d][8 * j + 2 * e] * inv, o[d][8 * j + 2 * e + 1] * inv);
          const uint32_t y = E::pack2(o[d][8 * j + 4 + 2 * e] * inv, o[d][8 * j + 4 + 2 * e + 1] * inv);
          const u32x2_t r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
          w[e] = r[0];
          w[2 + e] = r[1];
        }
        const int at = (d * 32 + j * 16 + half * 8) * kES;
        if (live && at < dbytes) *reinterpret_cast<u32x4_t*>(dst + at) = w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4_t w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = o[d][4 * j + e] * inv;
        const int at = (d * 32 + j * 8 + half * 4) * kES;
        if (live && at < dbytes) *reinterpret_cast<f32x4_t*>(dst + at) = w;
      }
    }
  }
}

// Joins the parts of a row (a token's head): DP / 4 lanes a row, 4 columns each.
template <class E, int DP>
__global__ void __launch_bounds__(256)
attn_join_kernel(AttnArgs a) {
  constexpr int kLanes = DP / 4;
  const int64_t r = int64_t(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  const int col = threadIdx.x % kLanes * 4;
  if (r >= a.T * a.Hq || col >= a.D) return;
  if (a.cu_q && r / a.Hq >= seq_at(a.cu_q, 0, a.T, a.n_seqs)) return;  // (behind the last sequence)
  const f32x2_t* ml = reinterpret_cast<const f32x2_t*>(a.part_ml) + r * a.parts;
  const float* src = a.part + r * a.parts * a.D + col;
  float all = -INFINITY;
  for (int p = 0; p < a.parts; ++p) all = fmaxf(all, ml[p][0]);
  float sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < a.parts; ++p) {
    const float mx = ml[p][0];
    // (a part without a maximum has seen no key, or only scores that are NaN, as its sum is)
    const float f = mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - all);
    sum = __builtin_fmaf(ml[p][1], f, sum);
    if (mx == -INFINITY) continue;
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(src + int64_t(p) * a.D);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[e], f, o[e]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  unsigned char* dst = a.out + (r * a.D + col) * E::kBytes;
  if constexpr (E::kBytes == 2)
    *reinterpret_cast<u32x2_t*>(dst) = u32x2_t{E::pack2(o[0] * inv, o[1] * inv), E::pack2(o[2] * inv, o[3] * inv)};
  else
    *reinterpret_cast<f32x4_t*>(dst) = f32x4_t{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
}

template <class E, int DP, int QW, int KS>
hipError_t launch_shape(AttnArgs a, hipStream_t stream) {
  using Sh = AttnShape<E, DP, QW, KS>;
  // slots: whole tiles of the tokens, one more a sequence, one for the rows behind them
  const int64_t slots = a.cu_q ? a.T / Sh::kBQ + a.n_seqs + 1 : int64_t(a.n_seqs) * ((a.each_q + Sh::kBQ - 1) / Sh::kBQ);
  const int64_t blocks = (a.T * a.Hq * (DP / 4) + 255) / 256;  // of the join
  if (slots * a.Hq * a.parts > kMostThreads / Sh::kThreads || (a.parts > 1 && blocks > kMostThreads / 256))
    return hipErrorInvalidConfiguration;
  a.nslots = int(slots);
  // (lane offsets of a staged tile: at most kBK rows, in 32 bits without a sign)
  auto is_far = [](int64_t ts) { return ts < 0 || ts > 0x7FFFFFFFll / Sh::kBK; };
  a.far = is_far(a.k_ts) || is_far(a.v_ts);
  const dim3 grid(unsigned(slots * a.Hq * a.parts)), t(Sh::kThreads);
  if constexpr (KS == 1) {
    if (a.parts > 1) {
      hipLaunchKernelGGL((attn_prefill_kernel<E, DP, QW, KS, true>), grid, t, 0, stream, a);
      hipLaunchKernelGGL((attn_join_kernel<E, DP>), dim3(unsigned(blocks)), dim3(256), 0, stream, a);
      return hipGetLastError();
    }
  }
  hipLaunchKernelGGL((attn_prefill_kernel<E, DP, QW, KS, false>), grid, t, 0, stream, a);
  return hipGetLastError();
}

template <class E>
hipError_t launch(const AttnArgs& a, int split, hipStream_t stream) {
  if (a.D > 128) return launch_shape<E, 256, 4, 1>(a, stream);
  if (a.D > 64) {
    if (split == 4) return launch_shape<E, 128, 1, 4>(a, stream);
    return split == 2 ? launch_shape<E, 128, 4, 2>(a, stream) : launch_shape<E, 128, 4, 1>(a, stream);
  }
  if (split == 4) return launch_shape<E, 64, 1, 4>(a, stream);
  return split == 2 ? launch_shape<E, 64, 4, 2>(a, stream) : launch_shape<E, 64, 4, 1>(a, stream);
}

}  // namespace

// How a call is cut: a model of its time (us) for each way, which came within 1.5 % of the best
// measured one on average over 70 calls (1 to 64 sequences of 16 to 3000 queries over up to
// 8500 keys, heads of 64 to 256, all types), 24 % at worst.  Some of them, bf16, 32
// heads of 128 (us): KS 1, 2, 4, then KS 1 with the keys in 4 and 8 parts
//   one sequence of 512                15.9   15.3   21.8   27.1   36.2
//   four of 512                        24.0   30.1   79.5   69.3  107.6
//   one of 1024                        26.8   23.9   52.2   46.9   65.7
//   64 queries over 4064 keys          80.1   59.7   49.7   31.6   27.2
// and fp32, 16 heads of 64
//   one sequence of 512                43.2   41.1   17.7   23.9   26.6
//   64 queries over 1064 keys          83.0   76.5   29.9   30.5   24.1
AttnPlan plan_attn_prefill(int dtype, int64_t T, int64_t Tk, int64_t n_seqs, bool cu, int Hq, int D, int cus, int split,
                           int parts) {
  AttnPlan p{};
  p.split = split ? split : 1;
  p.parts = split || parts == 0 ? 1 : parts;
  const bool wide = D > 64, widest = D > 128, f32 = dtype == 2;
  if (split == 0 && parts < 2) {
    const double rows = double(T) / n_seqs, keys = double(Tk) / n_seqs, mean = keys - 0.5 * rows;
    double best = 0.;
    auto weigh = [&](int ks, int n) {
      // us a workgroup takes for a key
      const double a_key = f32 ? (widest ? .280 : !wide ? (ks == 1 ? .078 : ks == 2 ? .072 : .027)
                                               : ks == 1 ? .133 : ks == 2 ? .128 : .045)
                               : (widest ? .045 : !wide ? (ks == 1 ? .0145 : ks == 2 ? .0112 : .0078)
                                                : ks == 1 ? .0190 : ks == 2 ? .0145 : .0115);
      const int height = ks == 4 ? 32 : 128;
      const double tiles = n_seqs * (n_seqs == 1 || !cu ? ceil(rows / height) : fmax(1., rows / height + .5));
      const double wgs = tiles * Hq * n;
      const int a_cu = ks == 1 ? (widest ? 1 : 2) : ks == 4 && !wide ? 2 : 1;
      // (two on a CU, with the workgroups that find no queries among those that take their places)
      const double grid = n_seqs == 1 || !cu ? wgs : (double(T) / height + n_seqs + 1) * Hq * n;
      const double key = a_key * (a_cu == 2 && grid > cus ? (f32 ? 1.9 : 1.3) : 1.);
      const double start = ks == 1 ? 4. : 7.;
      double us = fmax((ks == 1 ? 5. : 6.5) + keys / n * key, wgs / (a_cu * cus) * (start + mean / n * key) + 1.);
      if (n > 1) us += 4. + .35 * n + double(T) * Hq * n * (8. * D + 16.) / 4.5e6;
      if (best == 0. || us < best) {
        best = us;
        p.split = ks;
        p.parts = n;
      }
    };
    for (int n = 1; n <= (parts == 1 ? 1 : 16); n *= 2) weigh(1, n);
    if (!widest) {
      weigh(2, 1);
      weigh(4, 1);
    }
  }
  if (widest) p.split = 1;
  if (p.parts > 1) {
    const size_t rows = size_t(T) * Hq * p.parts;
    p.ml = 0;
    p.part = (rows * 8 + 255) / 256 * 256;
    p.bytes = p.part + rows * D * 4;
  }
  return p;
}

hipError_t launch_attn_prefill(const AttnArgs& a, int dtype, int split, hipStream_t stream) {
  switch (dtype) {
    case 0: return launch<AttnBf16>(a, split, stream);
    case 1: return launch<AttnFp16>(a, split, stream);
    default: return launch<AttnF32>(a, split, stream);
  }
}

}  // namespace mqk
