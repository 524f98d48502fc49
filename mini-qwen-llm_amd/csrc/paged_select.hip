// Selection of a cache's pages by a cheap score, for attention over contexts that are too long
// to be read whole.
//
// Of every page and key / value head the least and the largest key are kept, dimension by
// dimension (lo, hi).  The largest sum of scores that the G query heads of that head could have
// with a key inside the box is
//
//   score = sum_h sum_d max(q_hd lo_d, q_hd hi_d) = sum_d hi_d Qp_d + lo_d Qn_d,
//   Qp_d = sum_h max(q_hd, 0),  Qn_d = sum_h min(q_hd, 0)
//
// so that the heads cost nothing: one product with the box, 4 D operations a page, bound by
// reading it (1/16 of the cache's bytes at 16 tokens a page).  Which page is chosen must not
// hang on the order of a sum, so it is decided in 64 bits, where products of 16-bit values are
// exact and their sums as good as exact.  But 64-bit numbers made of 16-bit ones keep the vector
// units busy for twice the time that the bytes take, so that only the border is:
//
//   scores  On the matrix cores, boxes as they are (16 pages, 32 dimensions an instruction)
//           against Q as three 16-bit numbers that add up to it, in three columns; a fourth one,
//           with |box|, bounds the score's error.  Four tokens of a sequence share the boxes.
//           (16 sequences up to 40000 keys, 8 heads: 41 us for 111 MB from memory, 2.7 TB/s; 33
//           where the boxes are in the Infinity Cache, in 64 bits 42 there.  All sequences have
//           the runs of a table's width: a third of the workgroups' turns are empty here, more
//           where tables are wider: 53 us at 8192 pages.  With offsets four tokens of four
//           sequences follow each other in a workgroup: 58.)
//   choice  The take-th largest score by a radix selection, a workgroup a (token, head).  What is
//           above it by more than the errors is chosen, what is below is not; the few pages
//           between get their exact scores and places.  (14 us there, 15 for 6250 pages: steps
//           that wait for each other, not throughput.  Three tokens a sequence there: scores 55
//           us, choice 23.)
#include "mqk_device.h"
#include "mqk_paged.h"

#include <algorithm>

namespace mqk {
namespace {

// The type, how much a 16-bit number for |Q| may be below it (to the power of 2), and what is added
// to it for parts of Q below the type's smallest number.
struct SelBf16 : Bf16 {
  static constexpr float kUp = 1.f + 0x1p-7f, kLeast = 0x1p-100f;
};
struct SelFp16 : Fp16 {
  static constexpr float kUp = 1.f + 0x1p-10f, kLeast = 0x1p-6f;
};

// First token of sequence s, clamped into the call.
__device__ __forceinline__ int64_t token_of(const int32_t* cu, int64_t each, int64_t T, int s) {
  const int64_t at = cu ? int64_t(cu[s]) : each * s;
  return at < 0 ? 0 : at > T ? T : at;
}
// The last of the first n + 1 sequences whose f does not go past x (f rises; all lanes the same x).
template <class F>
__device__ __forceinline__ int last_sequence(int n, int64_t x, F f) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base <= n; base += 64) {
    const int c = base + lane;
    const int in = __popcll(__ballot(c <= n && f(min(c, n)) <= x));
    if (in == 0) return base - 1;
    if (in < 64) return base + in - 1;
  }
  return n;
}

// --- bounds ------------------------------------------------------------------------------

// A slot is a page that new tokens touch: sequence s has those from cu[s] / page + 2 s on, which
// rises and leaves it enough of them (n tokens touch (n - 1) / page + 2 pages at most), so that
// no sum over the lengths is needed.  Threads of a slot take 8 dimensions each of all heads
// (16 bytes of every token, whole rows of the page together).  8214 tokens of 8 heads 6.7 us
// (19 MB), a step of 64 sequences 5: launch, the search, and a page's loads at once.
template <class E>
__global__ void __launch_bounds__(256)
paged_bounds_kernel(PagedBounds a, int per) {
  const int64_t slot = int64_t(blockIdx.x) * (256 / per) + __builtin_amdgcn_readfirstlane(threadIdx.x / per);
  int s;
  int64_t j, from;
  int len;
  if (a.T < 0) {  // whole sequences
    if (slot >= a.n_seqs * a.cols) return;
    s = int(slot / a.cols);
    j = slot - s * a.cols;
    len = max(a.lens[s], 0);
  } else {
    auto first = [&](int c) { return token_of(a.cu, a.each, a.T, c) / a.page + 2 * int64_t(c); };
    s = last_sequence(a.n_seqs, slot, first);
    if (s < 0 || s >= a.n_seqs) return;
    const int64_t n = max(int64_t(0), token_of(a.cu, a.each, a.T, s + 1) - token_of(a.cu, a.each, a.T, s));
    len = max(a.lens[s], 0);
    if (n == 0) return;
    j = max(int64_t(0), len - n) / a.page + (slot - first(s));
  }
  from = j * a.page;
  if (j < 0 || j >= a.cols || from >= len) return;  // (below 0: offsets out of order)
  const int64_t id = a.table[s * a.cols + j];
  if (id < 0 || id >= a.num_blocks) return;
  const int n = int(min(int64_t(a.page), len - from));
  const int64_t row = int64_t(a.Hkv) * a.D * 2;
  const int chunks = a.Hkv * a.D / 8, of_head = a.D / 8;
  for (int c = threadIdx.x % per; c < chunks; c += per) {
    const unsigned char* src = a.k + id * a.page * row + c * 16;
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = INFINITY;
      hi[e] = -INFINITY;
    }
#pragma unroll 8
    for (int t = 0; t < n; ++t) {
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(src + t * row);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = E::to_f32(x[e / 2] >> (16 * (e % 2)) & 0xFFFFu);
        lo[e] = __builtin_elementwise_minimum(lo[e], f);  // (a NaN stays one)
        hi[e] = __builtin_elementwise_maximum(hi[e], f);
      }
    }
    unsigned char* dst = a.bounds + ((id * a.Hkv + c / of_head) * 2 * a.D + c % of_head * 8) * 2;
    u32x4_t l, h;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      l[e] = E::pack2(lo[2 * e], lo[2 * e + 1]);
      h[e] = E::pack2(hi[2 * e], hi[2 * e + 1]);
    }
    *reinterpret_cast<u32x4_t*>(dst) = l;
    *reinterpret_cast<u32x4_t*>(dst + a.D * 2) = h;
  }
}

// --- scores ------------------------------------------------------------------------------

// A number's place in ascending order, above 0; -0 as 0, every NaN as one value above infinity.
__device__ __forceinline__ uint64_t order_key(double f) {
  uint64_t b = __builtin_bit_cast(uint64_t, f + 0.0);
  if ((b & 0x7FFFFFFFFFFFFFFFull) > 0x7FF0000000000000ull) return ~0ull;
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f + 0.f);
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return ~0u;
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }

// A token's own page (past the table, if its length is), and its sequence and that one's end;
// false: behind the last one, or before the first key.
struct Own {
  int s;
  int64_t page, to;
};
__device__ __forceinline__ bool own_page(const PagedSelect& a, int64_t token, Own& o) {
  if (a.cu) {
    o.s = last_sequence(a.n_seqs, token, [&](int c) { return token_of(a.cu, 0, a.T, c); });
    if (o.s < 0 || o.s >= a.n_seqs) return false;
  } else {
    o.s = int(uint32_t(token) / uint32_t(a.each));
  }
  o.to = token_of(a.cu, a.each, a.T, o.s + 1);
  const int64_t pos = int64_t(max(a.lens[o.s], 0)) - (o.to - token);
  if (pos < 0) return false;
  o.page = uint32_t(pos) / uint32_t(a.page);
  return true;
}

// Sums over the G heads of q's negative and of its positive numbers, in dimension d: heads way,
// way + WAYS, ..
template <class E, int WAYS, class F>
__device__ __forceinline__ void sum_heads(const PagedSelect& a, int64_t token, int kvh, int d, int way, F& neg, F& pos) {
  constexpr int kOnce = 8 / WAYS > 4 ? 8 / WAYS : 4;  // loads under way
  const unsigned char* src = a.q + token * a.q_ts + int64_t(kvh) * a.G * a.q_hs + d * 2;
  neg = pos = F(0);
  for (int g0 = way; g0 < a.G; g0 += kOnce * WAYS) {
    uint16_t x[kOnce];
#pragma unroll
    for (int i = 0; i < kOnce; ++i) x[i] = *reinterpret_cast<const uint16_t*>(src + min(g0 + i * WAYS, a.G - 1) * a.q_hs);
#pragma unroll
    for (int i = 0; i < kOnce; ++i) {
      const float f = g0 + i * WAYS < a.G ? E::to_f32(x[i]) : 0.f;
      neg += F(__builtin_elementwise_minimum(f, 0.f));
      pos += F(__builtin_elementwise_maximum(f, 0.f));
    }
  }
}

// A page's score, and how far it may be from the exact one; below 0: the page is not there.
struct Score {
  float at, off;
};

// A workgroup has a run of pages for one head and `group` tokens (1 or 4), its waves 16 pages
// at a time.  Right operand: column 4 i + part of token i: Q as three numbers of the type that
// add up to it, and |Q|.
template <class E, int DP>
__global__ void __launch_bounds__(256, DP == 256 ? 1 : 3)
paged_score_kernel(PagedSelect a, int run, int group) {
  constexpr int kC = DP / 32;  // 32-dimension pieces of lo, and of hi
  __shared__ __align__(16) float q_sum[4][2 * DP];
  const int lane = threadIdx.x & 63, quarter = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t y = blockIdx.y + blockIdx.z * gridDim.y;
  const int64_t first = a.from + int64_t(y / uint32_t(a.Hkv)) * group;
  const int kvh = int(y % uint32_t(a.Hkv));
  if (first >= a.to) return;
  const int64_t last = min(first + group, a.to);
  // (the length, which everything else waits for, is under way with q)
  int32_t ahead = a.cu ? 0 : a.lens[uint32_t(first) / uint32_t(a.each)];
  for (int i = threadIdx.x; i < int(last - first) * DP; i += 256) {
    float neg = 0.f, pos = 0.f;
    if (i % DP < a.D) sum_heads<E, 1>(a, first + i / DP, kvh, i % DP, 0, neg, pos);
    q_sum[i / DP][i % DP] = neg;
    q_sum[i / DP][DP + i % DP] = pos;
  }
  asm volatile("" : "+v"(ahead));
  __syncthreads();
  for (int64_t token = first; token < last;) {  // (tokens of one sequence at a time)
    Own o;
    if (!own_page(a, token, o)) {
      ++token;
      continue;
    }
    const int n = int(min(last, o.to) - token);
    if (n <= 0) return;  // (offsets out of order)
    const int begin = a.first + int(blockIdx.x) * run;
    // the last token sees most; position and page of token i are this one's + i
    const int64_t pos = int64_t(a.lens[o.s]) - (o.to - token);
    auto end_of = [&](int i) {
      return int(min(min(int64_t(uint32_t(pos + i) / uint32_t(a.page)) + 1 - a.recent, a.cols), int64_t(begin) + run));
    };
    const int most = end_of(n - 1);
    int p0 = begin + wave * 16;
    const int32_t* table = a.table + o.s * a.cols;
    int next = p0 + col < most ? table[p0 + col] : -1;
    // --- Q
    const int mine = col >> 2, part = col & 3, from = int(token - first) + min(mine, n - 1);
    u32x4_t qn[kC], qp[kC];
    float qsum = 0.f;
    {
      auto piece = [&](const float* v) {
        u32x4_t r;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float x[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float q = v[2 * w + h];
            auto round = [](float f) { return E::to_f32(E::pack2(f, 0.f) & 0xFFFFu); };
            const float hi = round(q), mid = round(q - hi);
            x[h] = part == 0 ? hi : part == 1 ? mid : part == 2 ? q - hi - mid : fabsf(q) * E::kUp + E::kLeast;
            if (part == 3) qsum += x[h];
          }
          r[w] = E::pack2(x[0], x[1]);
        }
        return r;
      };
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        qn[c] = piece(&q_sum[from][c * 32 + quarter * 8]);
        qp[c] = piece(&q_sum[from][DP + c * 32 + quarter * 8]);
      }
    }
    // The error: every one of 2 DP products and sums may be off by 2^-23 of the terms' size, Q
    // itself by G of that; a bf16 box's number below the smallest normal one may count as 0.  (An
    // fp16 one, or a part of Q, must not: the matrix instructions read subnormal fp16 numbers as
    // they are.)  Of the 6 DP products with Q's parts, their sums and the bound itself, what is below
    // fp32's smallest normal number may count as 0: 2^-126 each, less than 2^-115 in all.
    qsum += __shfl_xor(qsum, 16);
    qsum += __shfl_xor(qsum, 32);
    const float rel = float(2 * DP + 32 + a.G) * 0x1p-23f * 1.01f;
    Score* const out = reinterpret_cast<Score*>(a.keys) + ((token - a.from + min(mine, n - 1)) * a.Hkv + kvh) * a.cols;
    const int my_end = end_of(min(mine, n - 1));
    // the next pages' boxes, and the ids of those after them, are under way
    int id = next < a.num_blocks ? next : -1;  // page p0 + col
    u32x4_t lo[kC], hi[kC], lo_next[kC], hi_next[kC];
    auto fetch = [&](int block, u32x4_t (&l)[kC], u32x4_t (&h)[kC]) {
      const unsigned char* box = a.bounds + (int64_t(max(block, 0)) * a.Hkv + kvh) * a.D * 4 + quarter * 16;
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        const bool in = DP == a.D || c * 32 + quarter * 8 < a.D;
        l[c] = in ? *reinterpret_cast<const u32x4_t*>(box + c * 64) : u32x4_t{0, 0, 0, 0};
        h[c] = in ? *reinterpret_cast<const u32x4_t*>(box + c * 64 + a.D * 2) : u32x4_t{0, 0, 0, 0};
      }
    };
    auto id_at = [&](int p) {
      const int i = p + col < most ? table[p + col] : -1;
      return i < a.num_blocks ? i : -1;
    };
    if (p0 < most) fetch(id, lo, hi);
    int id_next = id_at(p0 + 64);
    for (; p0 < most; p0 += 64) {
      if (p0 + 64 < most) fetch(id_next, lo_next, hi_next);
      const int id_after = id_at(p0 + 128);
      f32x4_t x = {0.f, 0.f, 0.f, 0.f}, size = x;
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        x = E::mfma(lo[c], qn[c], x);
        x = E::mfma(hi[c], qp[c], x);
        size = E::mfma(lo[c] & 0x7FFF7FFFu, qn[c], size);
        size = E::mfma(hi[c] & 0x7FFF7FFFu, qp[c], size);
      }
      // lane: pages p0 + 4 quarter + j, column col
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s = x[j], m = __shfl_xor(s, 1), l = __shfl_xor(s, 2);  // (parts 0, 1, 2 meet in part 0)
        const float bound = __shfl_xor(size[j], 3), all = __shfl_xor(qsum, 3);
        const int page = p0 + 4 * quarter + j;
        const bool there = __shfl(id, 4 * quarter + j) >= 0;
        if (part == 0 && mine < n && page < my_end)
          out[page] = there ? Score{s + (m + l), __builtin_fmaf(bound, rel, all * 0x1p-125f) + 0x1p-115f} : Score{0.f, -1.f};
      }
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        lo[c] = lo_next[c];
        hi[c] = hi_next[c];
      }
      id = id_next;
      id_next = id_after;
    }
    token += n;
  }
}

// --- selection ---------------------------------------------------------------------------

constexpr int kSelThreads = 512, kSelWaves = 8, kSelHeld = 16, kSelPart = kSelThreads * kSelHeld;
constexpr int kSelBins = 2048;
constexpr int kSelNear = kSelThreads;  // pages at the border that are looked at one by one
constexpr int kSelBin = 64;            // ... as many need no finer border

struct SelShared {
  uint32_t hist[kSelBins], sums[kSelWaves], pick[3];
  uint64_t ands[kSelWaves], ors[kSelWaves];
  double q[512];
  float top[kSelWaves];
  uint64_t near_key[kSelNear];
  uint32_t near_score[kSelNear];
  int near_page[kSelNear];
  uint32_t n_near, n_in, n_open;
  uint32_t chosen[kSelPart / 32];  // a bit a page of a part
};

// Sum over the wave's lanes up to this one: within rows of 16, then over the rows.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t add_dpp(uint32_t x) {
  return x + uint32_t(__builtin_amdgcn_update_dpp(0, int(x), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t scan_wave(uint32_t x) {
  x = add_dpp<0x111, 0xF>(x);
  x = add_dpp<0x112, 0xF>(x);
  x = add_dpp<0x114, 0xF>(x);
  x = add_dpp<0x118, 0xF>(x);
  x = add_dpp<0x142, 0xA>(x);     // row 0's sum to row 1, row 2's to row 3
  return add_dpp<0x143, 0xC>(x);  // rows 0 and 1's to rows 2 and 3
}
// Sum over the threads before this one, and over all of the workgroup.
__device__ __forceinline__ uint32_t scan_sel(uint32_t v, uint32_t* lds, uint32_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t x = scan_wave(v);
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  uint32_t before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    if (w < wave) before += lds[w];
    all += lds[w];
  }
  return before + x - v;
}

// The border of the `take` largest keys: those with key >> shift above `prefix`, and of those equal
// to it the first `left`.  A radix selection over the keys' bits, from the first on which they
// differ, 11 at a time, until what is left of a bin is taken whole, or the bin has no more than
// `enough` keys.  for_all(f) calls f with every key above 0 of the thread; there are more than
// `take`, which is above 0.
template <class K>
struct Border {
  K prefix;
  int shift;
  uint32_t left;
};
template <class K, class F>
__device__ __forceinline__ Border<K> find_border(SelShared& sh, uint32_t take, uint32_t enough, K ands, K ors, F for_all) {
  constexpr int kBits = 8 * sizeof(K);
  const int tid = threadIdx.x;
  Border<K> b{ands, 0, take};
  if (ands == ors) return b;
  int bits = kBits - (kBits == 64 ? __clzll(ands ^ ors) : __clz(uint32_t(ands ^ ors)));
  b.prefix = bits == kBits ? 0 : ands >> bits;
  while (bits > 0) {
    b.shift = max(0, bits - 11);
    for (int i = tid; i < kSelBins; i += kSelThreads) sh.hist[i] = 0;
    __syncthreads();
    for_all([&](K k) {
      if (bits == kBits || k >> bits == b.prefix) atomicAdd(&sh.hist[(k >> b.shift) & ((1u << (bits - b.shift)) - 1)], 1u);
    });
    __syncthreads();
    // bins from the largest on, 4 a thread
    constexpr int kMine = kSelBins / kSelThreads;
    uint32_t c[kMine], mine = 0, sum;
#pragma unroll
    for (int i = 0; i < kMine; ++i) mine += c[i] = sh.hist[kSelBins - 1 - kMine * tid - i];
    uint32_t before = scan_sel(mine, sh.sums, sum);
    if (before < b.left && before + mine >= b.left)
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        if (before < b.left && before + c[i] >= b.left) {
          sh.pick[0] = kSelBins - 1 - kMine * tid - i;
          sh.pick[1] = b.left - before;
          sh.pick[2] = c[i];
        }
        before += c[i];
      }
    __syncthreads();
    b.prefix = bits == kBits ? K(sh.pick[0]) : b.prefix << (bits - b.shift) | sh.pick[0];
    b.left = sh.pick[1];
    bits = b.shift;
    const bool done = sh.pick[2] == b.left || sh.pick[2] <= enough;
    __syncthreads();
    if (done) break;
  }
  return b;
}

// Exact scores, LANES lanes a page, 8 dimensions of lo or hi each.  A bound that is infinite has
// no part where no head's q has its sign, one that is NaN where no head has any q.
template <class E, int LANES>
struct Exact {
  double qs[8];
  uint32_t other;  // dimensions in which some head's q has the other sign
  const unsigned char* bounds;
  int64_t stride;
  bool in;

  // q: sums of the negative numbers, then [LANES * 4 on] of the positive ones
  __device__ __forceinline__ Exact(const PagedSelect& a, const double* q, int kvh) {
    const int lane = threadIdx.x % LANES, part = lane / (LANES / 2), d0 = lane % (LANES / 2) * 8;
    in = d0 < a.D;
    other = 0;
    stride = int64_t(a.Hkv) * a.D * 4;
    bounds = a.bounds + (int64_t(kvh) * 2 * a.D + part * a.D + d0) * 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      qs[e] = q[part * LANES * 4 + d0 + e];
      other |= uint32_t(q[(1 - part) * LANES * 4 + d0 + e] != 0.) << e;
    }
  }
  // (all LANES lanes with the same block)
  __device__ __forceinline__ uint64_t key(int64_t block) const {
    double y = 0.;
    if (in) {
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(bounds + block * stride);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = E::to_f32(x[e / 2] >> (16 * (e % 2)) & 0xFFFFu);
        if (qs[e] != 0. || (f != f && other >> e & 1)) y = __builtin_fma(qs[e], double(f), y);
      }
    }
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) y += __shfl_xor(y, m);
    return order_key(y);
  }
};

template <class E, int LANES>
__global__ void __launch_bounds__(kSelThreads)
paged_select_kernel(PagedSelect a) {
  __shared__ SelShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t unit = blockIdx.x, token = a.from + unit / a.Hkv;
  const int kvh = int(unit % a.Hkv);
  int32_t* out = a.pages + (token * a.Hkv + kvh) * a.take;
  Own o;
  if (!own_page(a, token, o)) {
    for (int i = tid; i < a.take; i += kSelThreads) out[i] = -1;
    return;
  }
  o.s = __builtin_amdgcn_readfirstlane(o.s);
  o.page = __builtin_amdgcn_readfirstlane(int(o.page));  // (so that what follows is the scalar unit's)
  const int32_t* table = a.table + o.s * a.cols;
  // candidates: lo .. hi - 1 (pages past the table are not there, recent ones among them)
  const int64_t end = min(o.page + 1, a.cols);
  const int64_t lo = min(int64_t(a.first), end), hi = max(lo, min(o.page + 1 - a.recent, end));
  auto there = [&](int64_t j) {
    const int id = table[j];
    return id >= 0 && id < a.num_blocks;
  };
  const int64_t parts = hi > lo ? (hi + kSelPart - 1) / kSelPart : 0;
  const Score* const scores = reinterpret_cast<const Score*>(a.keys) + unit * a.cols;
  // A part's scores as keys (0: not there), number e * kSelThreads + tid the thread's e-th: 64
  // pages in a row are a wave's, a bit each.  Vector instructions are what bounds this kernel, one
  // CU's for a head: so keys once, in registers, and no more of them than there are pages (2500
  // of them 16.8 us with 16 a thread read out of LDS as scores in every pass, 14.0 so).
  uint32_t key[kSelHeld];
  Score x[kSelHeld];
  float worst = 0.f;  // the largest error; infinite: some score is no number
  int64_t held = -1;
  int each = 0;       // keys of a thread
  auto fetch = [&](int64_t part) {
    const int64_t from = part * kSelPart;
    const int count = int(min(hi - from, int64_t(kSelPart)));
    each = (count + kSelThreads - 1) / kSelThreads;
#pragma unroll
    for (int e = 0; e < kSelHeld; ++e)
      if (e < each) x[e] = scores[from + min(e * kSelThreads + tid, count - 1)];
  };
  auto keep = [&](int64_t part) {
    held = part;
    const int64_t from = part * kSelPart;
    const int count = int(min(hi - from, int64_t(kSelPart))), least = int(max(lo - from, int64_t(0)));
#pragma unroll
    for (int e = 0; e < kSelHeld; ++e)
      if (e < each) {
        const int i = e * kSelThreads + tid;
        const bool is = !(x[e].off < 0.f) && i >= least && i < count;
        const bool fine = fabsf(x[e].at) < INFINITY && x[e].off < INFINITY;
        key[e] = is ? order_key(fine ? x[e].at : 0.f) : 0;
        worst = fmaxf(worst, !is ? 0.f : fine ? x[e].off : INFINITY);
      }
  };
  // f(key, number in the part) of all the thread's, keys 0 among them
  auto of_part = [&](int64_t part, auto f) {
    if (part != held) {
      fetch(part);
      keep(part);
    }
#pragma unroll
    for (int e = 0; e < kSelHeld; ++e)
      if (e < each) f(key[e], e * kSelThreads + tid);
  };
  if (parts > 0) fetch(0);
  for (int i = tid; i < LANES * 16; i += kSelThreads) {  // (for exact scores: four threads a dimension)
    const int d = i / 4;
    double neg = 0., pos = 0.;
    if (d < a.D) sum_heads<E, 4>(a, token, kvh, d, i % 4, neg, pos);
#pragma unroll
    for (int m = 1; m < 4; m <<= 1) {
      neg += __shfl_xor(neg, m);
      pos += __shfl_xor(pos, m);
    }
    if (i % 4 == 0) {
      sh.q[d] = neg;
      sh.q[LANES * 4 + d] = pos;
    }
  }
  // --- what is kept in any case, and how many of the candidates are there
  uint32_t n = 0, all, sum;
  for (int64_t j = tid; j < lo; j += kSelThreads) n += there(j);
  for (int64_t j = hi + tid; j < end; j += kSelThreads) n += there(j);
  uint32_t ands = ~0u, ors = 0;
  uint32_t found = 0;
  if (parts > 0) keep(0);
  for (int64_t p = 0; p < parts; ++p)
    of_part(p, [&](uint32_t k, int) {
      found += k != 0;
      ands &= k != 0 ? k : ~0u;
      ors |= k;
    });
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    ands &= __shfl_xor(ands, d);
    ors |= __shfl_xor(ors, d);
    worst = fmaxf(worst, __shfl_xor(worst, d));
  }
  if (lane == 0) {
    sh.ands[wave] = ands;
    sh.ors[wave] = ors;
    sh.top[wave] = worst;
  }
  scan_sel(found << 12 | n, sh.sums, all);  // (at most 16 of the first a thread a part, few of the second)
  const bool packed = parts <= 8 && lo + (end - hi) < 4096;
  uint32_t forced = all & 0xFFFu;
  all >>= 12;
  if (!packed) {
    scan_sel(n, sh.sums, forced);
    scan_sel(found, sh.sums, all);
  }
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    ands &= uint32_t(sh.ands[w]);
    ors |= uint32_t(sh.ors[w]);
    worst = fmaxf(worst, sh.top[w]);
  }
  const uint32_t take = uint32_t(a.take) - min(uint32_t(a.take), forced);

  // --- which are chosen: those with keys above one, and some of the pages near the border
  const bool every = all <= take;
  bool exact = false;
  uint32_t above = every ? 0 : ~0u;
  uint32_t near = 0;
  bool near_in = true;                // of the pages near the border, whether number tid is
  Border<uint64_t> border{0, 0, 0};
  if (!every && take > 0) {
    exact = !(worst < INFINITY);
    if (!exact) {
      const Border<uint32_t> b = find_border<uint32_t>(sh, take, kSelBin, ands, ors, [&](auto f) {
        for (int64_t p = 0; p < parts; ++p)
          of_part(p, [&](uint32_t k, int) {
            if (k != 0) f(k);
          });
      });
      // The take-th largest score is one of the bin's, the exact one within `worst` of them; and so
      // is every other page's: above and below that the scores decide.  (Rounded outwards, by the
      // next number each.)
      above = order_key(of_key((b.prefix << b.shift) | ((1u << b.shift) - 1)) + 2.f * worst) + 1;
      const uint32_t below = order_key(of_key(b.prefix << b.shift) - 2.f * worst) - 1;
      uint32_t sure = 0;
      if (tid == 0) sh.n_near = sh.n_in = sh.n_open = 0;
      __syncthreads();
      for (int64_t p = 0; p < parts; ++p)
        of_part(p, [&](uint32_t k, int number) {
          sure += k > above;
          if (k <= above && k >= below) {  // (above 0)
            const uint32_t i = atomicAdd(&sh.n_near, 1u);
            if (i < kSelNear) {
              sh.near_score[i] = k;
              sh.near_page[i] = int(p * kSelPart + number);
            }
          }
        });
      scan_sel(sure, sh.sums, sum);
      near = sh.n_near;
      exact = near > kSelNear;
      const uint32_t want = take - sum;  // of the near ones
      if (!exact && want < near) {
        // The same among them with the want-th largest score itself, and exact scores for those
        // that are still open.
        const uint32_t mine = uint32_t(tid) < near ? sh.near_score[tid] : 0;
        if (uint32_t(tid) < near) {
          uint32_t more = 0, same = 0;
          for (uint32_t i = 0; i < near; ++i) {
            more += sh.near_score[i] > mine;
            same += sh.near_score[i] == mine;
          }
          if (more < want && more + same >= want) sh.pick[0] = mine;
        }
        __syncthreads();
        const float at = of_key(sh.pick[0]);
        const uint32_t in = order_key(at + 2.f * worst) + 1, out_of = order_key(at - 2.f * worst) - 1;
        const bool open = uint32_t(tid) < near && mine <= in && mine >= out_of;
        near_in = mine > in;
        if (open) atomicAdd(&sh.n_open, 1u);
        else if (near_in) atomicAdd(&sh.n_in, 1u);
        __syncthreads();
        const uint32_t left = want - sh.n_in;  // of the open ones
        if (left >= sh.n_open) {
          near_in |= open;
        } else {
          const Exact<E, LANES> ex(a, sh.q, kvh);
          for (uint32_t i = tid / LANES; i < near; i += kSelThreads / LANES) {
            if (sh.near_score[i] > in || sh.near_score[i] < out_of) continue;
            const int id = table[sh.near_page[i]];  // (not there: offsets out of order, and no scores)
            const uint64_t k = ex.key(id >= 0 && id < a.num_blocks ? id : 0);
            if (tid % LANES == 0) sh.near_key[i] = k;
          }
          __syncthreads();
          if (open) {
            const uint64_t k = sh.near_key[tid];
            const int j = sh.near_page[tid];
            uint32_t rank = 0;
            for (uint32_t i = 0; i < near; ++i) {
              const uint32_t s = sh.near_score[i];
              if (s <= in && s >= out_of) rank += sh.near_key[i] > k || (sh.near_key[i] == k && sh.near_page[i] < j);
            }
            near_in = rank < left;
          }
        }
      }
    }
  }
  uint64_t* const keys = a.keys + unit * a.cols;
  if (exact) {
    // All exact scores, in the place of the others: where some are no numbers, or too many are as
    // good as equal.
    __syncthreads();
    const Exact<E, LANES> ex(a, sh.q, kvh);
    uint64_t and64 = ~0ull, or64 = 0;
    for (int64_t j = lo + tid / LANES; j < hi; j += kSelThreads / LANES) {
      const int id = table[j];
      const bool is = id >= 0 && id < a.num_blocks;
      const uint64_t k = ex.key(is ? id : 0);
      if (tid % LANES == 0) keys[j] = is ? k : 0;
      if (is) {
        and64 &= k;
        or64 |= k;
      }
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      and64 &= __shfl_xor(and64, d);
      or64 |= __shfl_xor(or64, d);
    }
    __syncthreads();
    if (lane == 0) {
      sh.ands[wave] = and64;
      sh.ors[wave] = or64;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) {
      and64 &= sh.ands[w];
      or64 |= sh.ors[w];
    }
    border = find_border<uint64_t>(sh, take, 0, and64, or64, [&](auto f) {
      for (int64_t j = lo + tid; j < hi; j += kSelThreads)
        if (keys[j] != 0) f(keys[j]);
    });
  }

  // --- the chosen pages in their order
  uint32_t at = 0, equal = 0;
  auto emit = [&](int64_t from, int64_t to) {  // (every wave counts, the first one writes)
    for (int64_t j0 = from; j0 < to; j0 += 64) {
      const bool chosen = j0 + lane < to && there(j0 + lane);
      const uint64_t in = __ballot(chosen);
      const uint32_t i = at + __popcll(in & ((1ull << lane) - 1));
      if (chosen && wave == 0 && i < uint32_t(a.take)) out[i] = int32_t(j0 + lane);
      at += __popcll(in);
    }
  };
  emit(0, lo);
  if (take > 0)
    for (int64_t p = 0; p < parts; ++p) {
      const int64_t from = p * kSelPart;
      uint32_t up = 0;    // a bit for each of the thread's pages
      int64_t first = 0;  // ... from this one on
      if (exact) {
        uint32_t eq = 0;  // at the border
        first = from + kSelHeld * tid;
#pragma unroll 1
        for (int e = 0; e < kSelHeld; ++e) {
          const int64_t j = first + e;
          const uint64_t k = j >= lo && j < hi ? keys[j] : 0, top = k >> border.shift;
          up |= uint32_t(k != 0 && top > border.prefix) << e;
          eq |= uint32_t(k != 0 && top == border.prefix) << e;
        }
        const uint32_t before = equal + scan_sel(__popc(eq), sh.sums, sum);
        equal += sum;
        // (the first ones at the border)
        uint32_t some = before < border.left ? border.left - before : 0;
        for (uint32_t rest = eq; rest != 0 && some > 0; --some) {
          up |= rest & -rest;
          rest &= rest - 1;
        }
      } else {
        if (p != held) {
          fetch(p);
          keep(p);
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kSelHeld; ++e) {
          if (e < each) {
            const uint64_t in = __ballot(key[e] > above);  // (every: above 0)
            if (lane < 2) sh.chosen[(e * kSelWaves + wave) * 2 + lane] = uint32_t(in >> (32 * lane));
          }
        }
        __syncthreads();
        if (near > 0) {
          if (uint32_t(tid) < near && near_in) {
            const int64_t i = sh.near_page[tid] - from;
            if (i >= 0 && i < kSelPart) atomicOr(&sh.chosen[i / 32], 1u << (i % 32));
          }
          __syncthreads();
        }
        static_assert(kSelPart / 32 <= kSelThreads, "a word a thread at most");
        first = from + 32 * tid;
        up = tid < each * (kSelThreads / 32) ? sh.chosen[tid] : 0;
      }
      uint32_t i = at + scan_sel(__popc(up), sh.sums, sum);
      at += sum;
      for (; up != 0; up &= up - 1, ++i)
        if (i < uint32_t(a.take)) out[i] = int32_t(first + __ffs(up) - 1);
    }
  emit(hi, end);
  for (uint32_t i = at + tid; i < uint32_t(a.take); i += kSelThreads) out[i] = -1;
}

// Scores: workgroups of runs of pages, all equal, as many as run at once (three a CU; more of them
// only make Q more often: 16 sequences up to 40000 keys 55 us with three, 58 with five; two runs of
// 6 and 2 where one of 8 would do: 64 sequences up to 8000 keys 70 us, 53 with one).
template <class E, int DP>
void launch(const PagedSelect& a, int cus, hipStream_t stream) {
  const int group = !a.cu && a.each == 1 ? 1 : 4;
  const int64_t units = (a.to - a.from + group - 1) / group * a.Hkv, times = (std::max<int64_t>(0, a.cols - a.first) + 63) / 64;
  if (times > 0) {
    const int64_t runs = std::max<int64_t>(1, 3 * cus / units), each = (times + runs - 1) / runs;
    const unsigned y = unsigned(std::min<int64_t>(units, 32768));
    hipLaunchKernelGGL((paged_score_kernel<E, DP>), dim3(unsigned((times + each - 1) / each), y, unsigned((units + y - 1) / y)),
                       dim3(256), 0, stream, a, int(each * 64), group);
  }
  hipLaunchKernelGGL((paged_select_kernel<E, DP / 4>), dim3(unsigned((a.to - a.from) * a.Hkv)), dim3(kSelThreads), 0, stream, a);
}

}  // namespace

hipError_t launch_paged_bounds(const PagedBounds& a, int fp16, hipStream_t stream) {
  const int chunks = a.Hkv * a.D / 8;
  const int per = chunks <= 64 ? 64 : chunks <= 128 ? 128 : 256;
  const int64_t slots = a.T < 0 ? a.n_seqs * a.cols : a.T / a.page + 2 * int64_t(a.n_seqs);
  const int64_t grid = (slots * per + 255) / 256;
  if (grid > 0x7FFFFFFF / 256) return hipErrorInvalidConfiguration;
  if (fp16) hipLaunchKernelGGL(paged_bounds_kernel<SelFp16>, dim3(unsigned(grid)), dim3(256), 0, stream, a, per);
  else hipLaunchKernelGGL(paged_bounds_kernel<SelBf16>, dim3(unsigned(grid)), dim3(256), 0, stream, a, per);
  return hipGetLastError();
}

hipError_t launch_paged_select(PagedSelect a, int fp16, int cus, hipStream_t stream) {
  const int64_t round = select_round(a.T, a.Hkv, a.cols);
  hipError_t err = hipSuccess;
  for (a.from = 0; a.from < a.T && err == hipSuccess; a.from = a.to) {
    a.to = std::min(a.T, a.from + round);
    if (fp16) {
      if (a.D > 128) launch<SelFp16, 256>(a, cus, stream);
      else if (a.D > 64) launch<SelFp16, 128>(a, cus, stream);
      else launch<SelFp16, 64>(a, cus, stream);
    } else {
      if (a.D > 128) launch<SelBf16, 256>(a, cus, stream);
      else if (a.D > 64) launch<SelBf16, 128>(a, cus, stream);
      else launch<SelBf16, 64>(a, cus, stream);
    }
    err = hipGetLastError();
  }
  return err;
}

}  // namespace mqk
