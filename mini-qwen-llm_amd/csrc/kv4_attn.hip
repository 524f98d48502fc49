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
// The V codes are taken relative to 8, with least + 8 scale in the place of the least value:
// the rounding of p_j s_g,j to bf16 then weighs |n - 8| and not n.
//
// A workgroup of four waves walks 128 keys a step, each wave pages of 16 tokens two by two,
// with up to 16 rows (S tokens x Hq / Hkv heads) of one key / value head, and a running
// softmax a wave, joined in LDS at the end.  The steps of all sequences and heads stand in
// one row, cut into equal parts, one a workgroup, wherever that falls: so every workgroup
// has the same work whatever the lengths are.  The cut is made on the device, from the
// lengths there.  A sequence's head that lies in one part is finished there; the partial
// results of the others are joined by a second launch.  A third one adds up the weights of
// each key where the caller keeps them (it needs every row's total).
//
// fp16 tensors: K's codes meet q in fp16 (1 + n / 16 is exact there too); the probabilities
// times V's scales do not have fp16's range and are split into two bf16 terms (16 bits), with
// twice the products.  At D 128 that leaves room for two waves a SIMD, not three: 64
// sequences of 4096 keys, 32 / 8 heads, 96 us where bf16 takes 74.
//
// Measured, bf16, heads of 128: 64 sequences of 2048 to 8192 keys, 32 / 8 heads, 92 us in all
// for 401 MB (4.4 TB/s, a copy runs at 5.2); 4 of 8192 to 32768 keys, 32 / 4 heads, with the
// weights 38 us (main launch 21, join 5, weights 12).  There the waves' turn-around between a
// chunk's scores and its values is what is left, three waves a SIMD over one another.  A
// single sequence is bound by latency: of 300 keys 7.6 us, of 4096 11.4, 4 of them the
// second launch's.
#include "kv4_device.h"
#include "mqk_attn.h"

namespace mqk {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kChunk = 32;              // keys a wave takes at a time: two pages
constexpr int kStep = kChunk * kWaves;  // of the workgroup

__device__ __forceinline__ int seq_len(const Kv4Attn& a, int b) {
  const int64_t n = a.lens[b], cap = a.cols * kPage;
  return int(n < 0 ? 0 : n > cap ? cap : n);
}
// Keys that a sequence's first query sees (none: 0 or less): the queries are the last tokens of
// its length, also where the table ends before it.
__device__ __forceinline__ int first_limit(const Kv4Attn& a, int b) { return max(a.lens[b], 0) - a.S + 1; }
// Steps of one head and row block of a sequence (one at least: a sequence without keys has
// its zeros written by somebody).
__device__ __forceinline__ int seq_steps(int len) { return max(1, (len + kStep - 1) / kStep); }

// Equal parts of all the steps there are, of 4 at least (3 would cut the usual lengths' heads
// across: 32 sequences of 1024 keys 19.7 us, with 4 15.4); of 2 where those are no more than
// the CUs take at once (one sequence of 4096 keys: 7.6 us, with 4 9.6).
__device__ __forceinline__ int64_t steps_a_part(const Kv4Attn& a, int64_t total) {
  return total <= a.few ? 2 : max(int64_t(4), (total + gridDim.x - 1) / int64_t(gridDim.x));
}

// Sum of `v` over the workgroup's threads before this one, and over all.
__device__ __forceinline__ int64_t scan_wg(int64_t v, int64_t* lds, int64_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(x, d);
    if (lane >= d) x += o;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int64_t before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += lds[w];
    all += lds[w];
  }
  return before + x - v;
}

// A value that every lane has, into scalar registers.
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(v)), hi = __builtin_amdgcn_readfirstlane(uint32_t(v >> 32));
  return int64_t(uint64_t(hi) << 32 | lo);
}

// A workgroup's part of the row of steps, and the sequence it starts in.
struct Part {
  int64_t pos, end;   // steps
  int b, n;           // sequence, its steps a head
  int64_t base;       // its first step
};
__device__ __forceinline__ bool find_part(const Kv4Attn& a, Part& w) {
  __shared__ int64_t scan[kWaves];
  __shared__ int64_t found[2];
  const int hr = a.Hkv * a.RB;
  if (a.whole) {  // a part a head
    w.b = blockIdx.x / hr;
    w.n = seq_steps(seq_len(a, w.b));
    w.base = 0;
    w.pos = int64_t(blockIdx.x % hr) * w.n;
    w.end = w.pos + w.n;
    return true;
  }
  int64_t total = 0, all, mine = 0, before = 0;
  if (a.B <= 64) {  // every wave for itself
    const int lane = threadIdx.x & 63;
    const int n = lane < a.B ? seq_steps(seq_len(a, lane)) : 0;
    mine = int64_t(n) * hr;
    int64_t at = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t o = __shfl_up(at, d);
      if (lane >= d) at += o;
    }
    total = uniform64(__shfl(at, 63));
    at -= mine;
    const int64_t per = steps_a_part(a, total);
    w.pos = per * blockIdx.x;
    w.end = min(total, w.pos + per);
    if (blockIdx.x == 0) {
      if (threadIdx.x < a.B) a.sched[1 + threadIdx.x] = at;
      if (threadIdx.x == 0) a.sched[0] = per;
    }
    const uint64_t in = __ballot(w.pos >= at && w.pos < at + mine);
    if (in == 0) return false;
    w.b = __ffsll(static_cast<unsigned long long>(in)) - 1;
    w.base = uniform64(__shfl(at, w.b));
    w.n = __builtin_amdgcn_readlane(n, w.b);
    return true;
  }
  const bool one = a.B <= kThreads;  // the sequences' sums stay in registers
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    mine = b < a.B ? int64_t(seq_steps(seq_len(a, b))) * hr : 0;
    before = scan_wg(mine, scan, all);
    total += all;
  }
  total = uniform64(total);
  const int64_t per = steps_a_part(a, total);
  w.pos = per * blockIdx.x;
  w.end = min(total, w.pos + per);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.sched[0] = per;
  int64_t base = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    if (!one) {
      mine = b < a.B ? int64_t(seq_steps(seq_len(a, b))) * hr : 0;
      before = scan_wg(mine, scan, all);
    }
    const int64_t at = base + before;
    if (b < a.B) {
      if (blockIdx.x == 0) a.sched[1 + b] = at;
      if (w.pos >= at && w.pos < at + mine) {
        found[0] = b;
        found[1] = at;
      }
    }
    base += one ? total : all;
  }
  __syncthreads();
  if (w.pos >= total) return false;
  w.b = __builtin_amdgcn_readfirstlane(int(found[0]));
  w.base = uniform64(found[1]);
  w.n = seq_steps(seq_len(a, w.b));
  return true;
}

// What one lane holds of a page: D / 8 bytes of K codes and of V codes, and one scale and
// least value.  The 16 lanes of a quarter hold those of its tokens 4 (lane / 16) .. +3, K's
// in lanes 0 .. 7 (token % 4 and group), V's in lanes 8 .. 15; an operand that all of them
// need is spread over the quarter by the instruction that uses it.  kg: K's scale and least
// value of token lane % 16 and group lane / 16, the left operand of an fp32 product.
template <int D>
struct PageRegs {
  static constexpr int kW = D / 32;
  uint32_t k[kW], v[kW], meta, kg;
};
template <int W>
__device__ __forceinline__ void load_words(const unsigned char* p, uint32_t (&to)[W]) {
  if constexpr (W == 4) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = x[e];
  } else {
    const u32x2_t x = *reinterpret_cast<const u32x2_t*>(p);
    to[0] = x[0];
    to[1] = x[1];
  }
}
template <int D>
__device__ __forceinline__ int meta_at(int lane) {  // byte of the lane's word in the record
  using R = Kv4<D>;
  const int n = lane & 7;
  return ((lane & 8) ? R::kMetaV : R::kMetaK) + (lane >> 4) * (D / 4) + (n < 4 * R::kG ? n : 0) * 4;
}
template <int D>
__device__ __forceinline__ void load_keys(const unsigned char* rec, int lane, PageRegs<D>& r) {
  using R = Kv4<D>;
  load_words(rec + lane * (D / 8), r.k);
  r.meta = *reinterpret_cast<const uint32_t*>(rec + meta_at<D>(lane));
  const int g = lane >> 4;  // (groups past the head's: another's, times 0)
  r.kg = *reinterpret_cast<const uint32_t*>(rec + R::kMetaK + ((lane & 15) * R::kG + (g < R::kG ? g : 0)) * 4);
}
template <int D>
__device__ __forceinline__ void load_values(const unsigned char* rec, int lane, PageRegs<D>& r) {
  load_words(rec + Kv4<D>::kV + lane * (D / 8), r.v);
}
// A number that a generic lambda takes as a constant.
template <int N>
struct Const {
  static constexpr int value = N;
};

// Lane N of each 16, to all of them.
template <int N>
__device__ __forceinline__ float spread(float v) {
  return __uint_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x150 + N, 0xF, 0xF, true));
}

// Lane (i + N) % 16 of each 16, to its lane i.
template <int N>
__device__ __forceinline__ float rotate(float v) {
  return __uint_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x120 + (16 - N), 0xF, 0xF, true));
}

// Two codes of `word` (nibbles i and i + 4) as 1 + n / 16 each, in bf16 or (HALF) fp16.  One
// instruction ands and ors if one constant is in a scalar and the other in a vector register
// (it takes no literals and one scalar), where the compiler would use two.
template <bool HALF>
struct CodeMask {
  uint32_t keep = HALF ? 0x03C003C0u : 0x00780078u, one = HALF ? 0x3C003C00u : 0x3F803F80u;
  __device__ __forceinline__ CodeMask() { asm("" : "+s"(keep), "+v"(one)); }
};
template <int I, bool HALF>
__device__ __forceinline__ uint32_t pair_of(uint32_t word, const CodeMask<HALF>& c) {
  constexpr int kUp = (HALF ? 6 : 3) - 4 * I;  // to the highest fraction bits
  const uint32_t x = kUp >= 0 ? word << (kUp & 31) : word >> (-kUp & 31);
  return (x & c.keep) | c.one;
}
template <bool HALF>
__device__ __forceinline__ u32x4_t codes_of(uint32_t word, const CodeMask<HALF>& c) {
  return u32x4_t{pair_of<0>(word, c), pair_of<1>(word, c), pair_of<2>(word, c), pair_of<3>(word, c)};
}
// K's codes meet q in the tensors' type, V's the probabilities in bf16.
template <class E>
constexpr bool kHalf = E::kExp == 0x7C00u;
template <bool HALF>
struct Masks {
  CodeMask<HALF> k;
  CodeMask<false> other;
  __device__ __forceinline__ const CodeMask<false>& v() const { return other; }
};
template <>
struct Masks<false> {
  CodeMask<false> k;
  __device__ __forceinline__ const CodeMask<false>& v() const { return k; }
};
template <class E>
__device__ __forceinline__ f32x4_t mfma_keys(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (kHalf<E>) {
    typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0, 0, 0);
  } else {
    return mfma_16x16x32(a, b, c);
  }
}

// bf16 terms of values: one (bf16 tensors) or a second one for the rest (fp16 tensors).
template <int NS>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&to)[NS]) {
  to[0] = pack_bf16x2(x, y);
  if constexpr (NS == 2) to[1] = pack_bf16x2(x - bf16_to_f32(to[0] & 0xFFFFu), y - bf16_to_f32(to[0] >> 16));
}

// The right operand of the scores: q of this lane's row, and -sum q, per group.
template <int D>
struct QRegs {
  static constexpr int kG = D / 64;
  u32x4_t q[kG * 2];
  float start[kG];  // -sum_d q_d over the group
  float sum;        // sum_d q_d over group lane / 16, 0 past the last
};
// Row r's 16-byte pieces of this lane: dimensions 64 (i / 2) + 16 (lane / 16) + 8 (i % 2) ..
template <int D>
__device__ __forceinline__ void fetch_q(const Kv4Attn& a, int b, int kvh, int r, int lane, u32x4_t (&to)[D / 32]) {
  const bool live = r < a.S * a.G;
  const int s = live ? r / a.G : 0, h = kvh * a.G + (live ? r % a.G : 0);
  const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + ((int64_t(b) * a.S + s) * a.Hq + h) * D + (lane >> 4) * 16;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
    to[i] = live ? *reinterpret_cast<const u32x4_t*>(src + i / 2 * 64 + i % 2 * 8) : u32x4_t{0, 0, 0, 0};
}
template <class E, int D>
__device__ __forceinline__ void take_q(const u32x4_t (&raw)[D / 32], int lane, QRegs<D>& to) {
  const int quad = lane >> 4;
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
    float sum = 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      to.q[g * 2 + half] = raw[g * 2 + half];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sum += E::to_f32(raw[g * 2 + half][e] & 0xFFFFu);
        sum += E::to_f32(raw[g * 2 + half][e] >> 16);
      }
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    to.start[g] = -sum;
    to.sum = quad == g ? sum : g == 0 ? 0.f : to.sum;
  }
}

// Scores of a page's 16 tokens for the lane's row: x[r] of token 4 (lane / 16) + r.  s: the
// lane's scale; m: K's least value of token lane % 16, group lane / 16 (their part of the
// scores is a product over the groups).  Both times the softmax scale, log2(e) in it.
template <class E, int D>
__device__ __forceinline__ void scores_of(const uint32_t (&k)[D / 32], float s, float m, const QRegs<D>& q,
                                          const CodeMask<kHalf<E>>& cm, float (&x)[4]) {
  constexpr int kG = D / 64;
  f32x4_t acc[kG];
#pragma unroll
  for (int g = 0; g < kG; ++g) {
    acc[g] = f32x4_t{q.start[g], q.start[g], q.start[g], q.start[g]};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      acc[g] = mfma_keys<E>(codes_of(k[g * 2 + half], cm), q.q[g * 2 + half], acc[g]);
    }
  }
  const f32x4_t low = __builtin_amdgcn_mfma_f32_16x16x4f32(m, q.sum, f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
  auto token = [&](auto r) {
    constexpr int R = decltype(r)::value;
    x[R] = __builtin_fmaf(spread<R * kG>(s), acc[0][R], low[R]);
    if constexpr (kG == 2) x[R] = __builtin_fmaf(spread<R * kG + 1>(s), acc[kG - 1][R], x[R]);
  };
  token(Const<0>{});
  token(Const<1>{});
  token(Const<2>{});
  token(Const<3>{});
}

template <class E, int D, int NS>
__global__ void __launch_bounds__(kThreads, NS == 2 && D == 128 ? 2 : 3)
kv4_attn_kernel(Kv4Attn a) {
  using R = Kv4<D>;
  constexpr int kG = D / 64;
  constexpr int kPitch = D + 4;
  __shared__ float ml[2][kWaves][16];
  __shared__ __align__(16) float part[kWaves][16][kPitch];
  const int tid = threadIdx.x, lane = tid & 63, quad = lane >> 4, row = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Part w;
  if (!find_part(a, w)) return;
  const int hr_all = a.Hkv * a.RB;

  while (w.pos < w.end) {
    const uint32_t into = uint32_t(w.pos - w.base);  // (the launch checks that a sequence's steps fit)
    const int hr = int(into / uint32_t(w.n)), step0 = int(into % uint32_t(w.n));
    const int steps = int(min(int64_t(w.n - step0), w.end - w.pos));
    const int kvh = hr / a.RB, rb = hr % a.RB;
    const int len = seq_len(a, w.b);
    const int r = rb * 16 + row;
    const int rows = min(16, a.S * a.G - rb * 16);
    const int limit = row < rows ? first_limit(a, w.b) + r / a.G : len;  // keys this lane's row sees
    const int least = first_limit(a, w.b) + rb * 16 / a.G;               // keys every row sees
    const int from = step0 * kStep, to = min(len, from + steps * kStep);

    const int32_t* table = a.table + int64_t(w.b) * a.cols;
    const int64_t stride = int64_t(a.Hkv) * R::kRecord;
    const unsigned char* cache = a.cache + int64_t(kvh) * R::kRecord;
    // chunk i of this wave: keys from + (4 i + wave) * 32 ..
    const int chunks = max(0, (to - from - wave * kChunk + kStep - 1) / kStep);
    auto ids_from = [&](int i) -> int {  // lane l: page l % 2 of chunk i + l / 2
      const int key = from + ((i + (lane >> 1)) * kWaves + wave) * kChunk + (lane & 1) * kPage;
      return key < to ? table[key / kPage] : -1;
    };
    int ids = ids_from(0);
    int ids_at = 0;

    u32x4_t raw[D / 32];
    fetch_q<D>(a, w.b, kvh, r, lane, raw);
    QRegs<D> q;

    const Masks<kHalf<E>> cm;
    const float scale16 = 16.f * a.scale;
    f32x4_t o[kG][4], ones[kG];
    f32x4_t mid = {0.f, 0.f, 0.f, 0.f};  // sum_j p_j (least + 8 scale): of group g in quarter 0's element g
    float mx = -INFINITY, sum = 0.f;  // running maximum of the scores, and sum
#pragma unroll
    for (int g = 0; g < kG; ++g) {
#pragma unroll
      for (int n = 0; n < 4; ++n) o[g][n] = f32x4_t{0, 0, 0, 0};
      ones[g] = f32x4_t{0, 0, 0, 0};
    }
    constexpr uint32_t kOne = 0x3F803F80u;
    const u32x4_t one = {kOne, kOne, kOne, kOne};

    // The chunk at hand; its registers are filled again as soon as they have been read: with
    // the next chunk's keys once its scores are there, with the next values after them.  (A
    // second set of them would leave room for two waves a SIMD, not three.)
    PageRegs<D> page[2];
    const unsigned char* rec[2];  // of the keys in `page`
    bool in[2];
    auto next_keys = [&](int i) {
      if (i - ids_at >= 32) {
        ids = ids_from(i);
        ids_at = i;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int id = __builtin_amdgcn_readlane(ids, (i - ids_at) * 2 + j);
        // (a page that is not there: the first one's bytes, which nothing sees)
        in[j] = id >= 0 && id < a.num_blocks;
        rec[j] = cache + (in[j] ? int64_t(id) : 0) * stride;
        load_keys<D>(rec[j], lane, page[j]);
      }
    };
    auto next_values = [&]() {
#pragma unroll
      for (int j = 0; j < 2; ++j) load_values<D>(rec[j], lane, page[j]);
    };
    auto compute = [&](int i) {
      const int key0 = from + (i * kWaves + wave) * kChunk;
      const bool masked = key0 + kChunk > min(least, to) || !in[0] || !in[1];
      float x[2][4], ms[2], mm[2];  // mm: V's middle values, least + 8 scale
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (masked) {
          // slots that hold no key of the sequence may hold anything: no scale, no least value
          const int token = quad * 4 + (lane & 7) / kG;
          if (!in[j] || key0 + j * kPage + token >= to) page[j].meta = 0u;
        }
        ms[j] = E::to_f32(page[j].meta & 0xFFFFu);
        mm[j] = __builtin_fmaf(8.f, ms[j], E::to_f32(page[j].meta >> 16));
        scores_of<E, D>(page[j].k, ms[j] * scale16, E::to_f32(page[j].kg >> 16) * a.scale, q, cm.k, x[j]);
      }
      if (masked) {
        const int most = min(limit, to);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int t = 0; t < 4; ++t)
            x[j][t] = in[j] && key0 + j * kPage + quad * 4 + t < most ? x[j][t] : -INFINITY;
      }
      if (masked && __any(mm[0] != mm[0] || mm[1] != mm[1])) {
        // V groups that are not finite, which some row may see and another not: they leave the
        // sums, and go to the rows that see them
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float nan[kG];
#pragma unroll
          for (int g = 0; g < kG; ++g) nan[g] = 0.f;
          auto token = [&](auto t) {
            constexpr int T = decltype(t)::value;
            const float z0 = spread<8 + T * kG>(mm[j]);
            if (z0 != z0 && x[j][T] != -INFINITY) nan[0] = z0;
            if constexpr (kG == 2) {
              const float z1 = spread<8 + T * kG + 1>(mm[j]);
              if (z1 != z1 && x[j][T] != -INFINITY) nan[kG - 1] = z1;
            }
          };
          token(Const<0>{});
          token(Const<1>{});
          token(Const<2>{});
          token(Const<3>{});
          if (mm[j] != mm[j]) mm[j] = 0.f;
#pragma unroll
          for (int g = 0; g < kG; ++g) {
            nan[g] += __shfl_xor(nan[g], 16);
            nan[g] += __shfl_xor(nan[g], 32);
#pragma unroll
            for (int n = 0; n < 4; ++n) o[g][n] += nan[g];
          }
        }
      }
      if (i + 1 < chunks) next_keys(i + 1);
      float top = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3]));
      top = fmaxf(top, fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
      // a new maximum only where one grew by more than 2^8 (terms stay below 256 until then)
      if (__any(top > mx + 8.f)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float now = fmaxf(mx, top);
        const float f = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - now);
        mx = now;
        sum *= f;
        mid *= f;
#pragma unroll
        for (int g = 0; g < kG; ++g) {
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
          p[j][t] = __builtin_amdgcn_exp2f(x[j][t] - raw);
          sum += p[j][t];
        }
      // probabilities times V's scales, as right operands
      u32x4_t ps[kG][NS];
      auto weigh = [&](auto page, auto token, auto group) {
        constexpr int J = decltype(page)::value, T = decltype(token)::value, G = decltype(group)::value;
        float y0 = p[J][T] * spread<8 + T * kG + G>(ms[J]);
        float y1 = p[J][T + 1] * spread<8 + (T + 1) * kG + G>(ms[J]);
        uint32_t t[NS];
        split_pair<NS>(y0, y1, t);
#pragma unroll
        for (int n = 0; n < NS; ++n) ps[G][n][2 * J + T / 2] = t[n];
      };
      auto weigh_group = [&](auto g) {
        weigh(Const<0>{}, Const<0>{}, g);
        weigh(Const<0>{}, Const<2>{}, g);
        weigh(Const<1>{}, Const<0>{}, g);
        weigh(Const<1>{}, Const<2>{}, g);
      };
      weigh_group(Const<0>{});
      if constexpr (kG == 2) weigh_group(Const<kG - 1>{});
      // and their sums with V's middle values, 4 tokens a product in fp32: its left operand
      // has group g's in lane g of each quarter (what the other lanes hold goes to rows that
      // nothing reads)
      auto middle = [&](auto token) {
        constexpr int T = decltype(token)::value;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          mid = __builtin_amdgcn_mfma_f32_16x16x4f32(rotate<8 + T * kG>(mm[j]), p[j][T], mid, 0, 0, 0);
      };
      middle(Const<0>{});
      middle(Const<1>{});
      middle(Const<2>{});
      middle(Const<3>{});
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        __builtin_amdgcn_sched_barrier(0);  // (one group's operands at a time: the registers are all in use)
        // left operand: V^T, codes of dimension 64 g + 4 m + b for tokens 4 quad + 0 .. 3 of both pages
        uint32_t vw[4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if constexpr (kG == 2) {
              const uint32_t v0 = page[j].v[2 * e], v1 = page[j].v[2 * e + 1];
              vw[2 * j + e] = g == 0 ? __builtin_amdgcn_perm(v1, v0, 0x05040100u) : __builtin_amdgcn_perm(v1, v0, 0x07060302u);
            } else {
              vw[2 * j + e] = page[j].v[e];
            }
          }
        const u32x4_t a0 = {pair_of<0>(vw[0], cm.v()), pair_of<0>(vw[1], cm.v()), pair_of<0>(vw[2], cm.v()), pair_of<0>(vw[3], cm.v())};
        const u32x4_t a1 = {pair_of<1>(vw[0], cm.v()), pair_of<1>(vw[1], cm.v()), pair_of<1>(vw[2], cm.v()), pair_of<1>(vw[3], cm.v())};
        const u32x4_t a2 = {pair_of<2>(vw[0], cm.v()), pair_of<2>(vw[1], cm.v()), pair_of<2>(vw[2], cm.v()), pair_of<2>(vw[3], cm.v())};
        const u32x4_t a3 = {pair_of<3>(vw[0], cm.v()), pair_of<3>(vw[1], cm.v()), pair_of<3>(vw[2], cm.v()), pair_of<3>(vw[3], cm.v())};
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          ones[g] = mfma_16x16x32(one, ps[g][n], ones[g]);
          o[g][0] = mfma_16x16x32(a0, ps[g][n], o[g][0]);
          o[g][1] = mfma_16x16x32(a1, ps[g][n], o[g][1]);
          o[g][2] = mfma_16x16x32(a2, ps[g][n], o[g][2]);
          o[g][3] = mfma_16x16x32(a3, ps[g][n], o[g][3]);
        }
      }
    };

    if (chunks > 0) {
      next_keys(0);
      next_values();
    }
    take_q<E, D>(raw, lane, q);  // (under the first loads)
    for (int i = 0; i < chunks; ++i) {
      compute(i);
      if (i + 1 < chunks) next_values();
    }

    // --- the waves' results joined: maxima first, then the scaled sums
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    float tm[kG];
#pragma unroll
    for (int g = 0; g < kG; ++g) tm[g] = __shfl(mid[g], row);
    __syncthreads();  // (the last part's readers are done)
    if (quad == 0) {
      ml[0][wave][row] = mx;
      ml[1][wave][row] = sum;
    }
    __syncthreads();
    float all = -INFINITY;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) all = fmaxf(all, ml[0][k][row]);
    const float f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - all);
#pragma unroll
    for (int g = 0; g < kG; ++g)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4_t y;
#pragma unroll
        for (int n = 0; n < 4; ++n)  // dimension 64 g + 4 (4 quad + t) + n: 16 (w - 1.5) = code - 8
          y[n] = mx == -INFINITY ? 0.f
                                 : f * __builtin_fmaf(16.f, __builtin_fmaf(-1.5f, ones[g][t], o[g][n][t]), tm[g]);
        *reinterpret_cast<f32x4_t*>(&part[wave][row][64 * g + 16 * quad + 4 * t]) = y;
      }
    __syncthreads();
    // 8 dimensions a thread
    constexpr int kLanes = D / 8;
    const int64_t id = int64_t(blockIdx.x) + int64_t(w.b) * hr_all + hr;  // of this partial result
    const bool done = steps == w.n;
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
        // (a wave without a maximum has seen no key, or only scores that are NaN, as its sum is)
        l += mk == -INFINITY ? ml[1][k][rr] : ml[1][k][rr] * __builtin_amdgcn_exp2f(mk - m);
        const f32x4_t y0 = *reinterpret_cast<const f32x4_t*>(&part[k][rr][d]);
        const f32x4_t y1 = *reinterpret_cast<const f32x4_t*>(&part[k][rr][d + 4]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[e] += y0[e];
          y[4 + e] += y1[e];
        }
      }
      const int rg = rb * 16 + rr;
      const int64_t at = (int64_t(w.b) * a.S + rg / a.G) * a.Hq + kvh * a.G + rg % a.G;
      if (done) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        u32x4_t out;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = E::pack2(y[2 * e] * inv, y[2 * e + 1] * inv);
        *reinterpret_cast<u32x4_t*>(reinterpret_cast<uint16_t*>(a.out) + at * D + d) = out;
        if (a.fin && d == 0) {
          a.fin[2 * at] = m;
          a.fin[2 * at + 1] = inv;
        }
      } else {
        float* dst = a.part + (id * 16 + rr) * D + d;
        *reinterpret_cast<f32x4_t*>(dst) = f32x4_t{y[0], y[1], y[2], y[3]};
        *reinterpret_cast<f32x4_t*>(dst + 4) = f32x4_t{y[4], y[5], y[6], y[7]};
        if (d == 0) {
          a.part_ml[(id * 16 + rr) * 2] = m;
          a.part_ml[(id * 16 + rr) * 2 + 1] = l;
        }
      }
    }
    w.pos += steps;
    if (w.pos >= w.base + int64_t(w.n) * hr_all && w.pos < w.end) {
      w.base += int64_t(w.n) * hr_all;
      w.b += 1;
      w.n = seq_steps(seq_len(a, w.b));
    }
  }
}

// Joins the partial results of one row (sequence, token, query head): a workgroup a row, its
// waves take every fourth of them.
template <class E, int D>
__global__ void __launch_bounds__(kThreads)
kv4_join_kernel(Kv4Attn a) {
  constexpr int kE = D / 64;
  __shared__ float wl[kWaves], wy[kWaves][D];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t item = blockIdx.x;
  const int b = int(item / (a.S * a.Hq)), rest = int(item % (a.S * a.Hq));
  const int s = rest / a.Hq, h = rest % a.Hq, kvh = h / a.G, r = s * a.G + h % a.G;
  const int64_t per = a.sched[0], base = a.sched[1 + b];
  const int n = seq_steps(seq_len(a, b));
  const int hr = kvh * a.RB + r / 16;
  const int64_t first = base + int64_t(hr) * n;
  const int64_t w0 = first / per;
  const int parts = int((first + n - 1) / per - w0) + 1;
  if (parts <= 1) return;
  const int64_t id0 = (w0 + int64_t(b) * a.Hkv * a.RB + hr) * 16 + r % 16;  // then 16 rows a part
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 64) m = fmaxf(m, a.part_ml[(id0 + int64_t(i) * 16) * 2]);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  float y[kE], l = 0.f;
#pragma unroll
  for (int e = 0; e < kE; ++e) y[e] = 0.f;
#pragma unroll 4
  for (int i = wave; i < parts; i += kWaves) {
    const int64_t at = id0 + int64_t(i) * 16;
    const float mi = a.part_ml[at * 2], li = a.part_ml[at * 2 + 1];
    const float f = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi - m);
    l = __builtin_fmaf(li, f, l);
#pragma unroll
    for (int e = 0; e < kE; ++e) y[e] = __builtin_fmaf(a.part[at * D + lane * kE + e], f, y[e]);
  }
  if (lane == 0) wl[wave] = l;
#pragma unroll
  for (int e = 0; e < kE; ++e) wy[wave][lane * kE + e] = y[e];
  __syncthreads();
  if (wave > 0) return;
  l = 0.f;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) l += wl[k];
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    y[e] = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) y[e] += wy[k][lane * kE + e];
    y[e] *= inv;
  }
  uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + item * D + lane * kE;
  if constexpr (kE == 2) *reinterpret_cast<uint32_t*>(out) = E::pack2(y[0], y[kE - 1]);
  else *out = uint16_t(E::pack2(y[0], 0.f));
  if (a.fin && lane == 0) {
    a.fin[2 * item] = m;
    a.fin[2 * item + 1] = inv;
  }
}

// Adds every key's weight, summed over the call's tokens and the query heads of its head, to
// its score: a wave per a.run pages of a sequence's head, two at a time with the next two
// under way, the scores of the rows computed again from K's codes and each row's maximum
// and sum (half the cache once more; keeping them would take 4 bytes a key and row).
typedef float f32x2_t __attribute__((ext_vector_type(2)));

template <class E, int D>
__global__ void __launch_bounds__(kThreads, 4)
kv4_weights_kernel(Kv4Attn a, int per) {
  using R = Kv4<D>;
  const int tid = threadIdx.x, lane = tid & 63, quad = lane >> 4, row = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / (per * a.Hkv), rest = blockIdx.x % (per * a.Hkv);
  const int kvh = rest / per;
  const int len = seq_len(a, b);
  const int page0 = (rest % per * kWaves + wave) * a.run;
  const int pages = min(a.run, (len - page0 * kPage + kPage - 1) / kPage);
  if (pages <= 0) return;
  const int32_t* table = a.table + int64_t(b) * a.cols;
  const int rows = a.S * a.G;
  const CodeMask<kHalf<E>> cm;
  const float scale16 = 16.f * a.scale;
  u32x4_t raw[D / 32];
  f32x2_t fin;
  auto fetch = [&](int r) {  // the row's q, maximum and 1 / sum
    fetch_q<D>(a, b, kvh, r, lane, raw);
    const int rg = r < rows ? r : 0;
    fin = *reinterpret_cast<const f32x2_t*>(a.fin + 2 * ((int64_t(b) * a.S + rg / a.G) * a.Hq + kvh * a.G + rg % a.G));
  };
  struct Pair {
    PageRegs<D> p[2];
    int id[2];
    float score[2];  // of the lane's key: token 4 quad + row, row < 4
  };
  auto load = [&](int i, Pair& c) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int page = page0 + i + j;
      const int id = i + j < pages ? __builtin_amdgcn_readfirstlane(table[page]) : -1;
      c.id[j] = id < a.num_blocks ? id : -1;
      const int64_t rec = int64_t(max(c.id[j], 0)) * a.Hkv + kvh;
      load_keys<D>(a.cache + rec * R::kRecord, lane, c.p[j]);
      c.score[j] = a.scores[rec * kPage + quad * 4 + (row & 3)];
    }
  };
  for (int rb = 0; rb * 16 < rows; ++rb) {
    const int r = rb * 16 + row;
    fetch(r);
    Pair c0, c1;
    load(0, c0);
    QRegs<D> q;
    take_q<E, D>(raw, lane, q);
    const float m = fin[0], inv = fin[1];
    const float base = m == -INFINITY ? 0.f : m;
    const int limit = r < rows ? min(len, first_limit(a, b) + r / a.G) : 0;
    auto weigh = [&](int i, Pair& c) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (c.id[j] < 0) continue;
        const int key0 = (page0 + i + j) * kPage + quad * 4;
        float x[4], add = 0.f;
        scores_of<E, D>(c.p[j].k, E::to_f32(c.p[j].meta & 0xFFFFu) * scale16, E::to_f32(c.p[j].kg >> 16) * a.scale, q, cm, x);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          float y = key0 + t < limit ? __builtin_amdgcn_exp2f(x[t] - base) * inv : 0.f;
          // over the 16 rows
          y += dpp_move<0xB1>(y);
          y += dpp_move<0x4E>(y);
          y += dpp_move<0x141>(y);
          y += dpp_move<0x140>(y);
          add = row == t ? y : add;
        }
        if (row < 4 && key0 + row < len) a.scores[(int64_t(c.id[j]) * a.Hkv + kvh) * kPage + quad * 4 + row] = c.score[j] + add;
      }
    };
    for (int i = 0; i < pages; i += 4) {
      if (i + 2 < pages) load(i + 2, c1);
      weigh(i, c0);
      if (i + 4 < pages) load(i + 4, c0);
      if (i + 2 < pages) weigh(i + 2, c1);
    }
  }
}

template <class E, int D, int NS>
hipError_t launch(const Kv4Attn& a, const Kv4Plan& p, hipStream_t stream) {
  const dim3 t(kThreads);
  hipLaunchKernelGGL((kv4_attn_kernel<E, D, NS>), dim3(unsigned(p.grid)), t, 0, stream, a);
  if (p.join) hipLaunchKernelGGL((kv4_join_kernel<E, D>), dim3(unsigned(p.join)), t, 0, stream, a);
  if (p.weigh)
    hipLaunchKernelGGL((kv4_weights_kernel<E, D>), dim3(unsigned(p.weigh)), t, 0, stream, a,
                       int(p.weigh / (int64_t(a.B) * a.Hkv)));
  return hipGetLastError();
}

}  // namespace

Kv4Plan plan_kv4_attn(int B, int S, int Hq, int Hkv, int D, int64_t cols, bool scores, int cus) {
  Kv4Plan p{};
  const int64_t G = Hq / Hkv, RB = (S * G + 15) / 16, items = int64_t(B) * Hkv * RB;
  const int64_t steps = (cols * kPage + kStep - 1) / kStep;  // of a sequence as long as the table is wide
  const int64_t full = int64_t(3) * cus;
  // A part a head where no sequence can be long enough for the second launch to pay (D 128, 8
  // heads: one sequence of 512 keys 8.6 us, in parts 11.1; one of 1024 12.6 and 11.1; with
  // more heads than parts of two steps need, 32 sequences of 1024 keys, 16.3 and 19.6).
  p.whole = steps <= 6 || (steps <= 8 && items * steps > full);
  // Parts: three workgroups a CU, what its registers hold, fewer where the tables are not wide
  // enough for them.  (Two, three, four a CU with ragged lengths, D 128: 64 sequences of up to
  // 8192 keys and 8 heads 105.5, 96.0, 100.7 us; 128 of up to 2500 69.7, 62.4, 65.9.)
  const int64_t most = (items * steps + 1) / 2;
  p.few = int(full);
  p.grid = p.whole ? items : most < full ? most : full;
  size_t n = 0;
  auto take = [&](size_t bytes) {
    const size_t at = n;
    n += (bytes + 255) / 256 * 256;
    return at;
  };
  if (scores) p.fin = take(size_t(B) * S * Hq * 2 * 4);
  if (!p.whole) {
    const size_t ids = size_t(p.grid + items);  // a partial result ends where its part or its head does
    p.sched = take((size_t(B) + 1) * 8);
    p.ml = take(ids * 16 * 2 * 4);
    p.part = take(ids * 16 * D * 4);
  }
  // Pages a wave weighs: few while that leaves CUs idle, more to keep its loads under way.
  // The weights kernel with 4, 8 and 16, D 128: one sequence of 2048 keys and 8 heads 4.4,
  // 6.1, 9.9 us; 32 of 1024 keys 9.1, 9.2, 11.6; 4 of 32768 keys and 4 heads 14.9, 14.0,
  // 14.9; 128 of 2048 keys and 8 heads 49.0, 44.1, 42.1.
  const int64_t all = int64_t(B) * Hkv * cols;
  p.run = all <= 4 * 16 * int64_t(cus) ? 4 : all <= 16 * 16 * int64_t(cus) ? 8 : 16;
  p.join = p.whole ? 0 : int64_t(B) * S * Hq;
  p.weigh = scores ? int64_t(B) * Hkv * ((cols + p.run * kWaves - 1) / (p.run * kWaves)) : 0;
  p.bytes = n;
  return p;
}

hipError_t launch_kv4_attn(const Kv4Attn& a, const Kv4Plan& p, int fp16, int D, hipStream_t stream) {
  if (fp16) return D == 128 ? launch<KvFp16, 128, 2>(a, p, stream) : launch<KvFp16, 64, 2>(a, p, stream);
  return D == 128 ? launch<KvBf16, 128, 1>(a, p, stream) : launch<KvBf16, 64, 1>(a, p, stream);
}

}  // namespace mqk
