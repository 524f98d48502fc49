// Decode attention over the 4-bit paged cache, S new tokens a sequence (the last ones of it):
//
//   O[s] = sum_j p_j v_j,  p = softmax_j(scale * q[s] . k_j),  j < len - S + s + 1
//   k_j[d] = s_g n + m_g  (code n, scale and least value of token j's group g of 64 dims)
//
// The reference decodes over a bf16 cache (paged_attn_decode,
// mini_qwen/kernels/paged_attn_decode.py:389-424).  What bounds it is reading the cache
// (1.125 D bytes a key and head), so the codes go into the matrix cores as they are:
//
//   q . k = sum_g (s_g sum_d q_d n_d + m_g sum_d q_d)
//   O     = sum_g sum_j (p_j s_g,j) n_j,d + p_j m_g,j
//
// i.e. the products run on whole numbers 0 .. 15 (exact in bf16) and scales and least values
// are applied to their sums.  A code is put into the fraction bits of 1.0: the operand is
// 1 + n / 16 (a shift and an and-or for two codes), and what the 1 adds is taken off again
// with a sum: for the scores by starting the sum at -sum_d q_d, for O by a product with a
// matrix of ones.
//
// A workgroup of four waves takes a split of a sequence's keys for one key / value head and
// up to 16 rows (S tokens x Hq / Hkv heads); its waves take pages of 16 tokens two by two and
// keep a running softmax each, joined in LDS at the end.  Splits are cut on the device from
// the lengths, so that all sequences together fill the chip whatever their lengths are;
// their partial results are joined by a second launch, which also adds up the weights of
// each key where the caller keeps them (it needs every row's total).
//
// fp16 tensors: q and the probabilities are split into two bf16 terms each (11 bits of q
// exactly, 16 of the probabilities), with twice the products; the matrix cores have room.
#include "kv4_device.h"
#include "mqk_attn.h"

namespace mqk {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kChunk = 32;              // keys a wave takes at a time: two pages
constexpr int kStep = kChunk * kWaves;  // of the workgroup

// How the sequences are cut: `chunk` keys a split, from the sum of the lengths.  Every
// workgroup computes the same from the lengths in device memory.
__device__ __forceinline__ int seq_len(const Kv4Attn& a, int b) {
  const int64_t n = a.lens[b], cap = a.cols * kPage;
  return int(n < 0 ? 0 : n > cap ? cap : n);
}
// Sum of `v` over the workgroup's threads and over those before this one.
__device__ __forceinline__ uint32_t scan_wg(uint32_t v, uint32_t* lds, uint32_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(x, d);
    if (lane >= d) x += o;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  uint32_t before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += lds[w];
    all += lds[w];
  }
  return before + x - v;
}
__device__ __forceinline__ int split_keys(const Kv4Attn& a, uint32_t* lds) {
  int64_t total = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    uint32_t all;
    scan_wg(b < a.B ? uint32_t((seq_len(a, b) + kStep - 1) / kStep) : 0u, lds, all);
    total += all;
  }
  // steps of 128 keys over the target number of workgroups
  const int64_t each = (total * a.Hkv * a.RB + a.target - 1) / a.target;
  return int(max(int64_t(a.least_chunk), each * kStep));
}

struct Work {
  int b, split, splits, hr;  // hr: head * RB + row block
  int chunk;
  uint32_t first;            // first item of the sequence
};
// The work of item `id` of the launch, or false past the last one.
__device__ __forceinline__ bool find_work(const Kv4Attn& a, uint32_t id, uint32_t* lds, Work& w) {
  __shared__ int found[4];
  w.chunk = split_keys(a, lds);
  const uint32_t hr = uint32_t(a.Hkv * a.RB);
  if (threadIdx.x == 0) found[0] = -1;
  uint32_t base = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    const uint32_t splits = b < a.B ? uint32_t(max(1, (seq_len(a, b) + w.chunk - 1) / w.chunk)) : 0u;
    uint32_t all;
    const uint32_t at = base + scan_wg(splits * hr, lds, all);
    if (blockIdx.x == 0 && a.sched && b < a.B) {
      a.sched[2 * b] = int32_t(at);
      a.sched[2 * b + 1] = int32_t(splits);
    }
    if (b < a.B && id >= at && id < at + splits * hr) {
      found[0] = b;
      found[1] = int((id - at) / hr);
      found[2] = int(splits);
      found[3] = int(at);
    }
    base += all;
  }
  __syncthreads();
  w.b = __builtin_amdgcn_readfirstlane(found[0]);
  if (w.b < 0) return false;
  w.split = __builtin_amdgcn_readfirstlane(found[1]);
  w.splits = __builtin_amdgcn_readfirstlane(found[2]);
  w.first = uint32_t(__builtin_amdgcn_readfirstlane(found[3]));
  w.hr = int((id - w.first) % hr);
  return true;
}

// What one lane holds of a page: K codes, V codes, and the scales and least values of the
// tokens 4 (lane / 16) .. +3, group by group.
template <int D>
struct PageRegs {
  static constexpr int kW = D / 32;
  uint32_t k[kW], v[kW], mk[kW * 2], mv[kW * 2];
};
template <int W>
__device__ __forceinline__ void load_words(const unsigned char* p, uint32_t (&to)[W]) {
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    if constexpr (W >= 4) {
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(p + i * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[i + e] = x[e];
    } else {
      const u32x2_t x = *reinterpret_cast<const u32x2_t*>(p);
      to[0] = x[0];
      to[1] = x[1];
    }
  }
}
template <int D, bool WITH_V>
__device__ __forceinline__ void load_page(const unsigned char* rec, int lane, PageRegs<D>& r) {
  using R = Kv4<D>;
  load_words(rec + lane * (D / 8), r.k);
  load_words(rec + R::kMetaK + (lane >> 4) * (D / 4), r.mk);
  if constexpr (WITH_V) {
    load_words(rec + R::kV + lane * (D / 8), r.v);
    load_words(rec + R::kMetaV + (lane >> 4) * (D / 4), r.mv);
  }
}

// Two codes of `word` (nibbles i and i + 4) as bf16 1 + n / 16 each.
template <int I>
__device__ __forceinline__ uint32_t pair_of(uint32_t word) {
  const uint32_t x = I == 0 ? word << 3 : word >> (4 * I - 3);
  return (x & 0x00780078u) | 0x3F803F80u;
}
__device__ __forceinline__ u32x4_t codes_of(uint32_t word) {
  return u32x4_t{pair_of<0>(word), pair_of<1>(word), pair_of<2>(word), pair_of<3>(word)};
}

// bf16 terms of values: one (bf16 tensors) or a second one for the rest (fp16 tensors).
template <int NS>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&to)[NS]) {
  to[0] = pack_bf16x2(x, y);
  if constexpr (NS == 2) to[1] = pack_bf16x2(x - bf16_to_f32(to[0] & 0xFFFFu), y - bf16_to_f32(to[0] >> 16));
}

// The left-over operand of the scores: 16 q of this lane's row, and -16 sum q, per group.
template <class E, int D, int NS>
struct QRegs {
  static constexpr int kG = D / 64;
  u32x4_t q[kG * 2][NS];
  float sum[kG];  // sum_d q_d over the group
};
template <class E, int D, int NS>
__device__ __forceinline__ void load_q(const Kv4Attn& a, int b, int kvh, int r, int lane, QRegs<E, D, NS>& to) {
  using Q = QRegs<E, D, NS>;
  const int quad = lane >> 4;
  const bool live = r < a.S * a.G;
  const int s = live ? r / a.G : 0, h = kvh * a.G + (live ? r % a.G : 0);
  const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + ((int64_t(b) * a.S + s) * a.Hq + h) * D;
#pragma unroll
  for (int g = 0; g < Q::kG; ++g) {
    float sum = 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const u32x4_t x =
          live ? *reinterpret_cast<const u32x4_t*>(src + g * 64 + quad * 16 + half * 8) : u32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = E::to_f32(x[e] & 0xFFFFu), hi = E::to_f32(x[e] >> 16);
        sum += lo;
        sum += hi;
        uint32_t t[NS];
        split_pair<NS>(16.f * lo, 16.f * hi, t);
#pragma unroll
        for (int n = 0; n < NS; ++n) to.q[g * 2 + half][n][e] = t[n];
      }
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    to.sum[g] = sum;
  }
}

// Scores (unscaled) of a page's 16 tokens for the lane's row: x[r] of token 4 (lane / 16) + r.
template <class E, int D, int NS>
__device__ __forceinline__ void scores_of(const PageRegs<D>& p, const QRegs<E, D, NS>& q, float (&x)[4]) {
  constexpr int kG = D / 64;
#pragma unroll
  for (int g = 0; g < kG; ++g) {
    const float start = -16.f * q.sum[g];
    f32x4_t acc = {start, start, start, start};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const u32x4_t k = codes_of(p.k[g * 2 + half]);
#pragma unroll
      for (int n = 0; n < NS; ++n) acc = mfma_16x16x32(k, q.q[g * 2 + half][n], acc);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t meta = p.mk[r * kG + g];
      const float s = E::to_f32(meta & 0xFFFFu), m = E::to_f32(meta >> 16);
      x[r] = g == 0 ? s * acc[r] : __builtin_fmaf(s, acc[r], x[r]);
      x[r] = __builtin_fmaf(m, q.sum[g], x[r]);
    }
  }
}

// The pages of a wave's chunks: 32 chunks' table entries at a time, one a lane.
struct PageIds {
  int ids;
  int from;
};

template <class E, int D, int NS>
__global__ void __launch_bounds__(kThreads, 2)
kv4_attn_kernel(Kv4Attn a) {
  using R = Kv4<D>;
  constexpr int kG = D / 64;
  constexpr int kPitch = D + 4;
  __shared__ uint32_t scan[kWaves];
  __shared__ float ml[2][kWaves][16];
  __shared__ __align__(16) float part[kWaves][16][kPitch];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, quad = lane >> 4, row = lane & 15;
  Work w;
  if (!find_work(a, blockIdx.x, scan, w)) return;
  const int kvh = w.hr / a.RB, rb = w.hr % a.RB;
  const int len = seq_len(a, w.b);
  const int r = rb * 16 + row;
  const int rows = min(16, a.S * a.G - rb * 16);
  const int limit = row < rows ? len - a.S + r / a.G + 1 : len;  // keys this lane's row sees
  const int least = len - a.S + rb * 16 / a.G + 1;               // keys every row sees
  const int from = w.split * w.chunk, to = min(len, from + w.chunk);

  QRegs<E, D, NS> q;
  load_q(a, w.b, kvh, r, lane, q);

  const int32_t* table = a.table + int64_t(w.b) * a.cols;
  const int64_t step = int64_t(a.Hkv) * R::kRecord;
  const unsigned char* cache = a.cache + int64_t(kvh) * R::kRecord;
  // chunk i of this wave: keys from + (4 i + wave) * 32 ..
  const int chunks = max(0, (to - from - wave * kChunk + kStep - 1) / kStep);
  auto ids_from = [&](int i) -> int {  // lane l: page l % 2 of chunk i + l / 2
    const int key = from + ((i + (lane >> 1)) * kWaves + wave) * kChunk + (lane & 1) * kPage;
    return key < to ? table[key / kPage] : -1;
  };
  int ids = ids_from(0);
  int ids_at = 0;

  f32x4_t o[kG][4], ones[kG];
  float tm[kG];
  float mx = -INFINITY, sum = 0.f;
#pragma unroll
  for (int g = 0; g < kG; ++g) {
#pragma unroll
    for (int n = 0; n < 4; ++n) o[g][n] = f32x4_t{0, 0, 0, 0};
    ones[g] = f32x4_t{0, 0, 0, 0};
    tm[g] = 0.f;
  }
  constexpr uint32_t kOne = 0x3F803F80u;
  const u32x4_t one = {kOne, kOne, kOne, kOne};

  struct Chunk {
    PageRegs<D> p[2];
    bool in[2];
  };
  auto load = [&](int i, Chunk& c) {
    if (i - ids_at >= 32) {
      ids = ids_from(i);
      ids_at = i;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int id = __builtin_amdgcn_readlane(ids, (i - ids_at) * 2 + j);
      // (a page that is not there: the first one's bytes, which nothing sees)
      c.in[j] = id >= 0 && id < a.num_blocks;
      load_page<D, true>(cache + (c.in[j] ? int64_t(id) : 0) * step, lane, c.p[j]);
    }
  };
  auto compute = [&](int i, Chunk& c) {
    const int key0 = from + (i * kWaves + wave) * kChunk;
    float x[2][4];
    scores_of<E, D, NS>(c.p[0], q, x[0]);
    scores_of<E, D, NS>(c.p[1], q, x[1]);
    if (key0 + kChunk > min(least, to) || !c.in[0] || !c.in[1]) {
      // what a row does not see: no score, and of V no scale and no least value either
      // (a page's unused slots may hold anything)
      const int most = min(limit, to);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const bool seen = c.in[j] && key0 + j * kPage + quad * 4 + t < most;
          x[j][t] = seen ? x[j][t] : -INFINITY;
#pragma unroll
          for (int g = 0; g < kG; ++g) c.p[j].mv[t * kG + g] = seen ? c.p[j].mv[t * kG + g] : 0u;
        }
    }
    float top = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3]));
    top = fmaxf(top, fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
    // a new maximum only where one grew by more than 2^8 (terms stay below 256 until then)
    if (__any((top - mx) * a.scale > 8.f)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float now = fmaxf(mx, top);
      const float f = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mx - now) * a.scale);
      mx = now;
      sum *= f;
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        tm[g] *= f;
        ones[g] *= f;
#pragma unroll
        for (int n = 0; n < 4; ++n) o[g][n] *= f;
      }
    }
    const float raw = mx == -INFINITY ? 0.f : mx;
    float p[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        p[j][t] = __builtin_amdgcn_exp2f((x[j][t] - raw) * a.scale);
        sum += p[j][t];
      }
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      u32x4_t ps[NS];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t m0 = c.p[j].mv[2 * e * kG + g], m1 = c.p[j].mv[(2 * e + 1) * kG + g];
          uint32_t t[NS];
          split_pair<NS>(p[j][2 * e] * E::to_f32(m0 & 0xFFFFu), p[j][2 * e + 1] * E::to_f32(m1 & 0xFFFFu), t);
#pragma unroll
          for (int n = 0; n < NS; ++n) ps[n][2 * j + e] = t[n];
          tm[g] = __builtin_fmaf(p[j][2 * e], E::to_f32(m0 >> 16), tm[g]);
          tm[g] = __builtin_fmaf(p[j][2 * e + 1], E::to_f32(m1 >> 16), tm[g]);
        }
      // left operand: V^T, codes of dimension 64 g + 4 m + b for tokens 4 quad + 0 .. 3 of both pages
      uint32_t vw[4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if constexpr (kG == 2) {
            const uint32_t v0 = c.p[j].v[2 * e], v1 = c.p[j].v[2 * e + 1];
            vw[2 * j + e] = g == 0 ? __builtin_amdgcn_perm(v1, v0, 0x05040100u) : __builtin_amdgcn_perm(v1, v0, 0x07060302u);
          } else {
            vw[2 * j + e] = c.p[j].v[e];
          }
        }
      const u32x4_t a0 = {pair_of<0>(vw[0]), pair_of<0>(vw[1]), pair_of<0>(vw[2]), pair_of<0>(vw[3])};
      const u32x4_t a1 = {pair_of<1>(vw[0]), pair_of<1>(vw[1]), pair_of<1>(vw[2]), pair_of<1>(vw[3])};
      const u32x4_t a2 = {pair_of<2>(vw[0]), pair_of<2>(vw[1]), pair_of<2>(vw[2]), pair_of<2>(vw[3])};
      const u32x4_t a3 = {pair_of<3>(vw[0]), pair_of<3>(vw[1]), pair_of<3>(vw[2]), pair_of<3>(vw[3])};
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        ones[g] = mfma_16x16x32(one, ps[n], ones[g]);
        o[g][0] = mfma_16x16x32(a0, ps[n], o[g][0]);
        o[g][1] = mfma_16x16x32(a1, ps[n], o[g][1]);
        o[g][2] = mfma_16x16x32(a2, ps[n], o[g][2]);
        o[g][3] = mfma_16x16x32(a3, ps[n], o[g][3]);
      }
    }
  };

  Chunk c0, c1;
  if (chunks > 0) load(0, c0);
  for (int i = 0; i < chunks; i += 2) {
    if (i + 1 < chunks) load(i + 1, c1);
    compute(i, c0);
    if (i + 1 < chunks) {
      if (i + 2 < chunks) load(i + 2, c0);
      compute(i + 1, c1);
    }
  }

  // --- the waves' results joined: maxima first, then the scaled sums
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
#pragma unroll
  for (int g = 0; g < kG; ++g) {
    tm[g] += __shfl_xor(tm[g], 16);
    tm[g] += __shfl_xor(tm[g], 32);
  }
  if (quad == 0) {
    ml[0][wave][row] = mx;
    ml[1][wave][row] = sum;
  }
  __syncthreads();
  float all = -INFINITY;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) all = fmaxf(all, ml[0][k][row]);
  const float f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mx - all) * a.scale);
#pragma unroll
  for (int g = 0; g < kG; ++g)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4_t y;
#pragma unroll
      for (int n = 0; n < 4; ++n)  // dimension 64 g + 4 (4 quad + t) + n
        y[n] = mx == -INFINITY ? 0.f : f * __builtin_fmaf(16.f, o[g][n][t] - ones[g][t], tm[g]);
      *reinterpret_cast<f32x4_t*>(&part[wave][row][64 * g + 16 * quad + 4 * t]) = y;
    }
  __syncthreads();
  // 8 dimensions a thread
  constexpr int kLanes = D / 8;
  for (int i = tid; i < 16 * kLanes; i += kThreads) {
    const int rr = i / kLanes, d = i % kLanes * 8;
    if (rr >= rows) continue;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = 0.f;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) m = fmaxf(m, ml[0][k][rr]);
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const float mk = ml[0][k][rr];
      l += mk == -INFINITY ? 0.f : ml[1][k][rr] * __builtin_amdgcn_exp2f((mk - m) * a.scale);
      const f32x4_t y0 = *reinterpret_cast<const f32x4_t*>(&part[k][rr][d]);
      const f32x4_t y1 = *reinterpret_cast<const f32x4_t*>(&part[k][rr][d + 4]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] += y0[e];
        y[4 + e] += y1[e];
      }
    }
    if (w.splits == 1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      u32x4_t out;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = E::pack2(y[2 * e] * inv, y[2 * e + 1] * inv);
      const int rg = rb * 16 + rr;
      const int64_t at = ((int64_t(w.b) * a.S + rg / a.G) * a.Hq + kvh * a.G + rg % a.G) * D + d;
      *reinterpret_cast<u32x4_t*>(reinterpret_cast<uint16_t*>(a.out) + at) = out;
    } else {
      float* dst = a.part + (int64_t(blockIdx.x) * 16 + rr) * D + d;
      *reinterpret_cast<f32x4_t*>(dst) = f32x4_t{y[0], y[1], y[2], y[3]};
      *reinterpret_cast<f32x4_t*>(dst + 4) = f32x4_t{y[4], y[5], y[6], y[7]};
    }
    if (a.part_ml && d == 0) {
      float* ml_out = a.part_ml + (int64_t(blockIdx.x) * 16 + rr) * 2;
      ml_out[0] = m;
      ml_out[1] = l;
    }
  }
}

// Joins the splits of one row: one wave per (sequence, token, query head).
template <class E, int D>
__global__ void __launch_bounds__(256)
kv4_join_kernel(Kv4Attn a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (item >= int64_t(a.B) * a.S * a.Hq) return;
  const int b = int(item / (a.S * a.Hq)), rest = int(item % (a.S * a.Hq));
  const int s = rest / a.Hq, h = rest % a.Hq, kvh = h / a.G, r = s * a.G + h % a.G;
  const int first = a.sched[2 * b], splits = a.sched[2 * b + 1];
  if (splits <= 1) return;
  const int hr = a.Hkv * a.RB;
  const int64_t at0 = (int64_t(first) + kvh * a.RB + r / 16) * 16 + r % 16, step = int64_t(hr) * 16;
  float m = -INFINITY;
  for (int i = lane; i < splits; i += 64) m = fmaxf(m, a.part_ml[(at0 + i * step) * 2]);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  constexpr int kE = D / 64;
  float y[kE], l = 0.f;
#pragma unroll
  for (int e = 0; e < kE; ++e) y[e] = 0.f;
  for (int i = 0; i < splits; ++i) {
    const int64_t at = at0 + i * step;
    const float mi = a.part_ml[at * 2], li = a.part_ml[at * 2 + 1];
    const float f = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mi - m) * a.scale);
    l = __builtin_fmaf(li, f, l);
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const float p = a.part[at * D + lane * kE + e];
      y[e] = mi == -INFINITY ? y[e] : __builtin_fmaf(p, f, y[e]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + item * D + lane * kE;
  if constexpr (kE == 2) *reinterpret_cast<uint32_t*>(out) = E::pack2(y[0] * inv, y[1] * inv);
  else *out = uint16_t(E::pack2(y[0] * inv, 0.f));
}

// Adds every key's weight, summed over the call's tokens and the query heads of its head, to
// its score: a workgroup per split of 512 keys of a sequence's head, the scores of the rows
// computed again from K's codes and each row's maximum and sum.
template <class E, int D, int NS>
__global__ void __launch_bounds__(kThreads)
kv4_weights_kernel(Kv4Attn a, int per) {
  using R = Kv4<D>;
  __shared__ float ref[2][64];  // of up to 64 rows: maximum, and 1 / sum
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, quad = lane >> 4, row = lane & 15;
  const int b = blockIdx.x / (per * a.Hkv), rest = blockIdx.x % (per * a.Hkv);
  const int kvh = rest / per, part = rest % per;
  const int len = seq_len(a, b);
  constexpr int kKeys = 512;
  const int from = part * kKeys, to = min(len, from + kKeys);
  if (from >= to) return;
  const int first = a.sched[2 * b], splits = a.sched[2 * b + 1];
  const int hr = a.Hkv * a.RB, all_rows = a.S * a.G;
  const int32_t* table = a.table + int64_t(b) * a.cols;
  constexpr int kMine = kKeys / kPage / kWaves;  // pages a wave takes: part's pages wave, wave + 4, ...
  float add[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) add[i] = 0.f;
  for (int r0 = 0; r0 < all_rows; r0 += 64) {
    __syncthreads();
    for (int i = tid; i < 64; i += kThreads) {
      const int r = r0 + i;
      float m = -INFINITY, l = 0.f;
      if (r < all_rows) {
        const int64_t at0 = (int64_t(first) + kvh * a.RB + r / 16) * 16 + r % 16, step = int64_t(hr) * 16;
        for (int k = 0; k < splits; ++k) m = fmaxf(m, a.part_ml[(at0 + k * step) * 2]);
        for (int k = 0; k < splits; ++k) {
          const float mk = a.part_ml[(at0 + k * step) * 2];
          if (mk != -INFINITY) l += a.part_ml[(at0 + k * step) * 2 + 1] * __builtin_amdgcn_exp2f((mk - m) * a.scale);
        }
      }
      ref[0][i] = m;
      ref[1][i] = l == 0.f ? 0.f : 1.f / l;
    }
    __syncthreads();
    for (int rb = r0 / 16; rb * 16 < min(all_rows, r0 + 64); ++rb) {
      const int r = rb * 16 + row;
      QRegs<E, D, NS> q;
      load_q(a, b, kvh, r, lane, q);
      const float m = ref[0][r - r0], inv = ref[1][r - r0];
      const float raw = m == -INFINITY ? 0.f : m;
      const int limit = r < all_rows ? min(to, len - a.S + r / a.G + 1) : 0;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int key0 = from + (i * kWaves + wave) * kPage;
        if (key0 >= to) break;
        const int id = table[key0 / kPage];
        if (id < 0 || id >= a.num_blocks) continue;
        PageRegs<D> p;
        load_page<D, false>(a.cache + (int64_t(id) * a.Hkv + kvh) * R::kRecord, lane, p);
        float x[4];
        scores_of<E, D, NS>(p, q, x);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          float y = key0 + quad * 4 + t < limit ? __builtin_amdgcn_exp2f((x[t] - raw) * a.scale) * inv : 0.f;
          // over the 16 rows
          y += dpp_move<0xB1>(y);
          y += dpp_move<0x4E>(y);
          y += dpp_move<0x141>(y);
          y += dpp_move<0x140>(y);
          if (row == t) add[i] += y;
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int key0 = from + (i * kWaves + wave) * kPage;
    const int key = key0 + quad * 4 + row;
    if (row < 4 && key < to) {
      const int id = table[key0 / kPage];
      if (id >= 0 && id < a.num_blocks) a.scores[(int64_t(id) * a.Hkv + kvh) * kPage + quad * 4 + row] += add[i];
    }
  }
}

template <class E, int D, int NS>
hipError_t launch(const Kv4Attn& a, unsigned grid, bool split, hipStream_t stream) {
  hipLaunchKernelGGL((kv4_attn_kernel<E, D, NS>), dim3(grid), dim3(kThreads), 0, stream, a);
  if (split) {
    const unsigned rows = unsigned((int64_t(a.B) * a.S * a.Hq + 3) / 4);
    hipLaunchKernelGGL((kv4_join_kernel<E, D>), dim3(rows), dim3(256), 0, stream, a);
  }
  if (a.scores) {
    const int per = int((a.cols * kPage + 511) / 512);
    hipLaunchKernelGGL((kv4_weights_kernel<E, D, NS>), dim3(unsigned(int64_t(a.B) * a.Hkv * per)), dim3(kThreads), 0,
                       stream, a, per);
  }
  return hipGetLastError();
}

}  // namespace

Kv4Plan plan_kv4_attn(int B, int S, int Hq, int Hkv, int D, int64_t cols, bool scores, int cus) {
  Kv4Plan p{};
  const int64_t G = Hq / Hkv, RB = (S * G + 15) / 16;
  p.target = 4 * cus;
  p.least_chunk = 512;
  const int64_t cap = cols * kPage;
  p.split = cap > p.least_chunk;
  // items: what `target` workgroups leave over, one more a sequence and head; never more than
  // the table's width allows
  const int64_t hr = B * int64_t(Hkv) * RB, widest = (cap + p.least_chunk - 1) / p.least_chunk;
  p.items = p.split ? (hr * widest < p.target + hr ? hr * widest : p.target + hr) : hr;
  if (p.items < hr) p.items = hr;
  size_t n = 0;
  if (p.split || scores) {
    p.sched = n;
    n += (size_t(B) * 8 + 255) / 256 * 256;
    p.ml = n;
    n += (size_t(p.items) * 16 * 2 * 4 + 255) / 256 * 256;
  }
  if (p.split) {
    p.part = n;
    n += size_t(p.items) * 16 * D * 4;
  }
  p.bytes = n;
  return p;
}

hipError_t launch_kv4_attn(const Kv4Attn& a, int64_t items, bool split, int fp16, int D, hipStream_t stream) {
  const unsigned grid = unsigned(items);
  if (fp16) return D == 128 ? launch<KvFp16, 128, 2>(a, grid, split, stream) : launch<KvFp16, 64, 2>(a, grid, split, stream);
  return D == 128 ? launch<KvBf16, 128, 1>(a, grid, split, stream) : launch<KvBf16, 64, 1>(a, grid, split, stream);
}

}  // namespace mqk
