// Causal attention over packed prompts with grouped heads:
//
//   O[i] = sum_j softmax_j(scale * Q[i] . K[j]) V[j],   j < m - n + i + 1
//
// for query i of a sequence's n queries and m keys (m = n for a whole prompt, m > n where
// the prompt continues one whose keys are there already).  The reference runs it as
// paged_attn_prefill (mini_qwen/kernels/paged_attn_prefill.py:64-156).
//
// One pass over the keys with a running maximum and sum: a workgroup of four waves takes
// 128 queries of one head, each wave 32 of them, and walks the keys in tiles of kBK that
// the waves stage together in LDS (two buffers, direct loads, one barrier a tile).
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
// second product (2^-9 relative a term for bf16, as V itself carries), the output once.
#include "mqk_attn.h"
#include "mqk_device.h"

namespace mqk {
namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));

constexpr int kBQ = 128;     // queries of a workgroup
constexpr int kThreads = 256;

// 16 bytes of zeros: what the columns past a head size that is no whole tile are read from.
__device__ const u32x4_t g_zero16 = {0, 0, 0, 0};

struct AttnBf16 : Bf16 {
  static constexpr int kBytes = 2;
  static constexpr int kBK = 64;
  static constexpr uint32_t kExp = 0x7F80u;
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) { return mfma_32x32x16(a, b, c); }
};
struct AttnFp16 : Fp16 {
  static constexpr int kBytes = 2;
  static constexpr int kBK = 64;
  static constexpr uint32_t kExp = 0x7C00u;
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0,
                                                  0, 0);
  }
};
struct AttnF32 {
  static constexpr int kBytes = 4;
  static constexpr int kBK = 32;
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

template <class E, int DP>
__global__ void __launch_bounds__(kThreads, DP == 256 ? 1 : 2)
attn_prefill_kernel(AttnArgs a) {
  constexpr int kBK = E::kBK;
  constexpr int kES = E::kBytes;
  constexpr int kRow = DP * kES;           // bytes of a staged row
  constexpr int kC = kRow / 16;            // its 16-byte chunks
  constexpr int kTile = kBK * kRow;        // bytes of a staged tile
  constexpr int kLoads = kTile / (kThreads * 16);
  constexpr int kNB = kBK / 32;            // 32-key blocks of a tile
  constexpr int kND = DP / 32;             // 32-wide blocks of the head
  __shared__ __align__(16) unsigned char lds[4 * kTile];  // K, K, V, V
  __shared__ int redo;

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, row = lane & 31;

  // --- the tile: head and slot, and of the slot the sequence and its place in it.  Slot
  // numbers leave gaps: sequence s starts at slot cu[s] / 128 + s, which is monotone and
  // leaves it enough of them, so that no sum over the lengths is needed.
  int head, slot;
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
    slot = nslots - 1 - slot;  // the late queries, which see most keys, first
  }
  int s = 0;
  if (a.cu_q) {
    // the last sequence whose first slot is not past this one, 64 candidates at a time
    for (int base = 0; base <= a.n_seqs; base += 64) {
      const int c = base + lane;
      const bool in = c <= a.n_seqs && int(seq_at(a.cu_q, 0, a.T, c <= a.n_seqs ? c : 0) / kBQ) + c <= slot;
      const int n = __popcll(__ballot(in));
      s = base + n - 1;
      if (n < 64) break;
    }
    if (s < 0) s = 0;
    if (s > a.n_seqs) s = a.n_seqs;
  } else {
    // equal lengths: a whole number of slots each
    const int per = int((a.each_q + kBQ - 1) / kBQ);
    s = slot / per;
  }
  s = __builtin_amdgcn_readfirstlane(s);
  const int64_t q_at = seq_at(a.cu_q, a.each_q, a.T, s);
  const int64_t tile = a.cu_q ? slot - (q_at / kBQ + s) : slot % int((a.each_q + kBQ - 1) / kBQ);
  const int64_t orow = int64_t(a.Hq) * a.D * kES;  // bytes of an output token
  if (s >= a.n_seqs) {  // behind the last sequence
    const int64_t t0 = q_at + tile * kBQ;
    if (tile < 0 || !a.fill) return;
    const int chunks = a.D * kES / 16;
    for (int i = tid; i < kBQ * chunks; i += kThreads) {
      const int64_t t = t0 + i / chunks;
      if (t < a.T)
        *reinterpret_cast<u32x4_t*>(a.out + t * orow + (int64_t(head) * chunks + i % chunks) * 16) = u32x4_t{0, 0, 0, 0};
    }
    return;
  }
  const int64_t n = seq_at(a.cu_q, a.each_q, a.T, s + 1) - q_at;
  if (tile < 0 || tile * kBQ >= n) return;
  const int32_t* cu_k = a.cu_k ? a.cu_k : a.cu_q;
  const int64_t k_at = seq_at(cu_k, a.each_k, a.Tk, s);
  int64_t m64 = seq_at(cu_k, a.each_k, a.Tk, s + 1) - k_at;
  const int m = m64 < 0 ? 0 : int(m64);

  const int q0 = int(tile) * kBQ;
  const int qi = min(q0 + wave * 32 + row, int(n) - 1);  // (rows past the end repeat the last one)
  const int shift = m - int(n);                          // (may be negative: such queries see nothing)
  const int limit = shift + qi + 1;                      // keys this lane's query sees
  const int most = max(0, min(m, shift + min(q0 + kBQ, int(n))));  // keys any query of the tile sees
  const int least = shift + q0 + 1;                      // keys all of them see
  const int tiles = (most + kBK - 1) / kBK;
  const int kvh = head / (a.Hq / a.Hkv);
  const unsigned char* kbase = a.k + k_at * a.k_ts + int64_t(kvh) * a.k_hs;
  const unsigned char* vbase = a.v + k_at * a.v_ts + int64_t(kvh) * a.v_hs;
  const int dbytes = a.D * kES;

  // The queries stay in registers, but for heads past 128, which would not leave enough of
  // them: those are read again (from the caches) for every tile.
  constexpr bool kHeld = DP <= 128;
  const unsigned char* qsrc = a.q + (q_at + qi) * a.q_ts + int64_t(head) * a.q_hs;
  auto load_q = [&](int t) {
    const int at = (2 * t + half) * 16;
    return DP == a.D || at < dbytes ? *reinterpret_cast<const u32x4_t*>(qsrc + at) : u32x4_t{0, 0, 0, 0};
  };
  u32x4_t qf[kHeld ? kC / 2 : 1];
  if constexpr (kHeld) {
#pragma unroll
    for (int t = 0; t < kC / 2; ++t) qf[t] = load_q(t);
  }

  const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)lds));
  // Stages tile kt into buffer b: every load of the wave fills 64 chunks in a row.
  auto stage = [&](int kt, int b) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int p = (i * 4 + wave) * 64 + lane;
      const int r = p / kC, c = p % kC;
      const int key = min(kt * kBK + r, m - 1);  // (rows past the last key repeat it; their scores are masked)
      const int ck = k_slot<kC>(r, c) * 16, cv = v_slot<kC, kES>(r, c) * 16;
      const unsigned char* pk = kbase + int64_t(key) * a.k_ts + ck;
      const unsigned char* pv = vbase + int64_t(key) * a.v_ts + cv;
      const unsigned char* z = reinterpret_cast<const unsigned char*>(&g_zero16);
      if (DP != a.D) {
        pk = ck < dbytes ? pk : z;
        pv = cv < dbytes ? pv : z;
      }
      const uint32_t at = uint32_t((i * 4 + wave) * 1024);
      dma16(pk, lds0 + b * kTile + at);
      dma16(pv, lds0 + (2 + b) * kTile + at);
    }
  };

  f32x16_t o[kND];
  float mx, mraw, sum;  // the running maximum, scaled (as the exponents take it) and as it was
  bool careful = false;
  for (;;) {
#pragma unroll
    for (int d = 0; d < kND; ++d) o[d] = f32x16_t{};
    mx = mraw = -INFINITY;
    sum = 0.f;
    if (tiles > 0) stage(0, 0);
    for (int kt = 0; kt < tiles; ++kt) {
      const int b = kt & 1;
      wait_vm<0>();
      __syncthreads();
      if (kt + 1 < tiles) stage(kt + 1, b ^ 1);
      const unsigned char* kt_lds = lds + b * kTile;
      unsigned char* vt_lds = lds + (2 + b) * kTile;
      const bool diag = (kt + 1) * kBK > least;
      if (careful && diag) {
        // values that are not finite leave the tile: those that are seen are added below
        for (int i = tid; i < kTile / 4; i += kThreads) {
          uint32_t* w = reinterpret_cast<uint32_t*>(vt_lds) + i;
          uint32_t x = *w;
          if (kES == 4) {
            if ((x & E::kExp) == E::kExp) x = 0;
          } else {
            if ((x & E::kExp) == E::kExp) x &= 0xFFFF0000u;
            if ((x & (E::kExp << 16)) == (E::kExp << 16)) x &= 0xFFFFu;
          }
          *w = x;
        }
        __syncthreads();
      }

      f32x16_t st[kNB];
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb) st[nb] = f32x16_t{};
#pragma unroll
      for (int t = 0; t < kC / 2; ++t) {
        const u32x4_t qt = kHeld ? qf[kHeld ? t : 0] : load_q(t);
#pragma unroll
        for (int nb = 0; nb < kNB; ++nb) {
          const int r = nb * 32 + row;
          const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(kt_lds + r * kRow + k_slot<kC>(r, 2 * t + half) * 16);
          st[nb] = E::mfma32(kf, qt, st[nb]);
        }
      }
      if (diag) {
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
      const float traw = max_halves(top);
      top = traw * a.scale;
      // O and the sum are brought to a new maximum only where it grew by more than 2^8:
      // until then the terms stay below 256, which no rounding minds.
      if (__any(top > mx + 8.f)) {
        const float now = fmaxf(mx, top);
        const float f = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - now);
        mx = now;
        mraw = fmaxf(mraw, traw);
        sum *= f;
#pragma unroll
        for (int d = 0; d < kND; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[d][i] *= f;
      }
      // scale * s - maximum, the product unrounded and the maximum rounded: off by 2^-24 of
      // the maximum, so a large one is subtracted before the product
      const float sub = mx == -INFINITY ? 0.f : mx;
      const bool large = __any(fabsf(sub) > 65536.f);
      if (!large) {
#pragma unroll
        for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
          for (int i = 0; i < 16; ++i) st[nb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[nb][i], a.scale, -sub));
      } else {
        const float raw = mx == -INFINITY ? 0.f : mraw;
#pragma unroll
        for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
          for (int i = 0; i < 16; ++i) st[nb][i] = __builtin_amdgcn_exp2f((st[nb][i] - raw) * a.scale);
      }
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += st[nb][i];

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
  if (careful) {
    // the values that are not finite, of the keys that were masked for some query of the tile
    const int from = max(0, least / kBK * kBK);
    const int to = min(limit, m);
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
  const float inv = total == 0.f ? 0.f : 1.f / total;  // (a query that sees no key: 0)
  const bool live = q0 + wave * 32 + row < int(n);
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

template <class E>
hipError_t launch(const AttnArgs& a, unsigned grid, hipStream_t stream) {
  const dim3 g(grid), t(kThreads);
  if (a.D <= 64) hipLaunchKernelGGL((attn_prefill_kernel<E, 64>), g, t, 0, stream, a);
  else if (a.D <= 128) hipLaunchKernelGGL((attn_prefill_kernel<E, 128>), g, t, 0, stream, a);
  else hipLaunchKernelGGL((attn_prefill_kernel<E, 256>), g, t, 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attn_prefill(AttnArgs a, int dtype, hipStream_t stream) {
  // slots: whole tiles of the tokens, one more a sequence, one for the rows behind them
  const int64_t slots = a.cu_q ? a.T / kBQ + a.n_seqs + 1 : int64_t(a.n_seqs) * ((a.each_q + kBQ - 1) / kBQ);
  if (slots * a.Hq > 0x7FFFFFFFll) return hipErrorInvalidConfiguration;
  a.nslots = int(slots);
  const unsigned grid = unsigned(slots * a.Hq);
  switch (dtype) {
    case 0: return launch<AttnBf16>(a, grid, stream);
    case 1: return launch<AttnFp16>(a, grid, stream);
    default: return launch<AttnF32>(a, grid, stream);
  }
}

}  // namespace mqk
