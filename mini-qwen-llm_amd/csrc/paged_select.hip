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
// reading it (1/16 of the cache's bytes at 16 tokens a page).  It is computed in 64 bits: the
// products of 16-bit values are exact there and their sums as good as exact, so which page
// is chosen does not hang on the order of a sum (in 32 bits, scores next to each other at the
// border of the choice would change places).  The vector units do that as fast as the
// bytes come.
#include "mqk_device.h"
#include "mqk_paged.h"

#include <algorithm>
#include <type_traits>

namespace mqk {
namespace {

struct SelBf16 {
  static __device__ __forceinline__ float to_f32(uint32_t x) { return bf16_to_f32(x); }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) { return Bf16::pack2(a, b); }
};
struct SelFp16 {
  static __device__ __forceinline__ float to_f32(uint32_t x) { return f16_to_f32(x); }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) { return Fp16::pack2(a, b); }
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
// (16 bytes of every token, whole rows of the page together).
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
  if (j >= a.cols || from >= len) return;
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

// A double's place in ascending order, above 0; -0 as 0, every NaN as one value above infinity.
__device__ __forceinline__ uint64_t order_key(double f) {
  uint64_t b = __builtin_bit_cast(uint64_t, f + 0.0);
  if ((b & 0x7FFFFFFFFFFFFFFFull) > 0x7FF0000000000000ull) return ~0ull;
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// A token's own page (past the table, if its length is), and its sequence; false: behind the last one, or before the first key.
struct Own {
  int s;
  int64_t page;
};
__device__ __forceinline__ bool own_page(const PagedSelect& a, int64_t token, Own& o) {
  if (a.cu) {
    o.s = last_sequence(a.n_seqs, token, [&](int c) { return token_of(a.cu, 0, a.T, c); });
    if (o.s < 0 || o.s >= a.n_seqs) return false;
  } else {
    o.s = int(token / a.each);
  }
  const int64_t to = token_of(a.cu, a.each, a.T, o.s + 1);
  const int64_t pos = int64_t(max(a.lens[o.s], 0)) - (to - token);
  if (pos < 0) return false;
  o.page = pos / a.page;
  return true;
}

constexpr int kScorePages = 16;  // a lane's at a time

// LANES of a wave share a page's box: 8 dimensions of lo or hi each.
template <class E, int LANES>
__global__ void __launch_bounds__(256)
paged_score_kernel(PagedSelect a, int chunks) {
  constexpr int kTogether = 64 / LANES, kPages = kScorePages * kTogether;  // of a wave
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t unit = blockIdx.x / chunks;
  const int64_t token = unit / a.Hkv;
  const int kvh = int(unit % a.Hkv);
  Own o;
  if (!own_page(a, token, o)) return;
  const int64_t from = a.first, to = min(o.page + 1 - a.recent, a.cols);  // candidates
  const int64_t p0 = from + (int64_t(blockIdx.x % chunks) * 4 + wave) * kPages;
  if (p0 >= to) return;
  // --- pages: lane i has that of the wave's i-th
  static_assert(kPages <= 64, "a lane for every page");
  const int32_t* table = a.table + o.s * a.cols;
  int id = lane < kPages && p0 + lane < to ? table[p0 + lane] : -1;
  if (id >= a.num_blocks) id = -1;
  // --- this lane's 8 dimensions of Qn (with lo) or Qp (with hi), and where no head has any q
  const int part = lane % LANES / (LANES / 2), d0 = lane % (LANES / 2) * 8;
  const bool in = d0 < a.D;
  double qs[8];
  uint32_t other = 0;  // dimensions in which some head's q has the other sign
#pragma unroll
  for (int e = 0; e < 8; ++e) qs[e] = 0.;
  if (in) {
    const unsigned char* src = a.q + token * a.q_ts + int64_t(kvh) * a.G * a.q_hs + d0 * 2;
    for (int g = 0; g < a.G; ++g) {
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(src + g * a.q_hs);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = E::to_f32(x[e / 2] >> (16 * (e % 2)) & 0xFFFFu);
        const float mine = part ? __builtin_elementwise_maximum(f, 0.f) : __builtin_elementwise_minimum(f, 0.f);
        qs[e] += double(mine);
        other |= uint32_t(mine != f) << e;
      }
    }
  }
  u32x4_t box[kScorePages];
#pragma unroll
  for (int i = 0; i < kScorePages; ++i) {
    const int64_t page = __shfl(id, i * kTogether + lane / LANES);
    box[i] = u32x4_t{0, 0, 0, 0};
    if (page >= 0 && in)
      box[i] = *reinterpret_cast<const u32x4_t*>(a.bounds + ((page * a.Hkv + kvh) * 2 * a.D + part * a.D + d0) * 2);
  }
  // CAREFUL: a bound that is infinite has no part where no head's q has its sign, one that is
  // NaN where no head has any q (0 * infinity would be NaN; all finite bounds do without)
  int mine = 0;
  auto score = [&](auto careful) {
    double sum[kScorePages];
#pragma unroll
    for (int i = 0; i < kScorePages; ++i) {
      sum[i] = 0.;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float f = E::to_f32(box[i][e / 2] >> (16 * (e % 2)) & 0xFFFFu);
        if (careful) f = qs[e] != 0. || (f != f && other >> e & 1) ? f : 0.f;
        sum[i] = __builtin_fma(qs[e], double(f), sum[i]);
      }
    }
    // sums over the lanes: of 16 pages every exchange halves those that a lane goes on with
    mine = 0;
#pragma unroll
    for (int m = 1, left = kScorePages / 2; m < 16; m <<= 1, left >>= 1) {
      const bool up = lane & m;
      if (up) mine += left;
#pragma unroll
      for (int i = 0; i < kScorePages / 2; ++i) {
        if (i >= left) continue;
        const double keep = up ? sum[i + left] : sum[i], send = up ? sum[i] : sum[i + left];
        sum[i] = keep + __shfl_xor(send, m);
      }
    }
#pragma unroll
    for (int m = 16; m < LANES; m <<= 1) sum[0] += __shfl_xor(sum[0], m);
    return sum[0];
  };
  double sum = score(std::false_type{});
  if (__any(!(fabs(sum) < INFINITY))) {
#pragma unroll
    for (int i = 0; i < kScorePages; ++i) asm volatile("" : "+v"(box[i]));  // (nothing kept for this)
    sum = score(std::true_type{});
  }
  const int64_t page = p0 + mine * kTogether + lane / LANES;
  const bool there = __shfl(id, mine * kTogether + lane / LANES) >= 0;
  if (lane % LANES < 16 && page < to) a.keys[unit * a.cols + page] = there ? order_key(sum) : 0;
}

// --- selection ---------------------------------------------------------------------------

constexpr int kSelThreads = 1024, kSelWaves = 16, kSelHeld = 16, kSelPart = kSelThreads * kSelHeld;
constexpr int kSelBins = 2048;

// Sum over the threads before this one, and over all of the workgroup.
__device__ __forceinline__ uint32_t scan_sel(uint32_t v, uint32_t* lds, uint32_t& all) {
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
  for (int w = 0; w < kSelWaves; ++w) {
    if (w < wave) before += lds[w];
    all += lds[w];
  }
  return before + x - v;
}

// A workgroup a (token, head): the take-th largest key by a radix selection over the keys' bits,
// from the first on which they differ, 11 at a time, until what is left of a bin is taken
// whole; then the chosen pages in their order.  Keys stay in registers, 16 a thread (longer
// sequences: a part of them at a time).
__global__ void __launch_bounds__(kSelThreads)
paged_select_kernel(PagedSelect a) {
  __shared__ uint32_t hist[kSelBins], sums[kSelWaves], pick[3];
  __shared__ uint64_t ands[kSelWaves], ors[kSelWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t unit = blockIdx.x, token = unit / a.Hkv;
  int32_t* out = a.pages + unit * a.take;
  Own o;
  if (!own_page(a, token, o)) {
    for (int i = tid; i < a.take; i += kSelThreads) out[i] = -1;
    return;
  }
  const int32_t* table = a.table + o.s * a.cols;
  // candidates: lo .. hi - 1 (pages past the table are not there, recent ones among them)
  const int64_t end = min(o.page + 1, a.cols);
  const int64_t lo = min(int64_t(a.first), end), hi = max(lo, min(o.page + 1 - a.recent, end));
  auto there = [&](int64_t j) {
    const int id = table[j];
    return id >= 0 && id < a.num_blocks;
  };
  const uint64_t* keys = a.keys + unit * a.cols;
  uint64_t key[kSelHeld];
  int64_t held = -1;
  auto hold = [&](int64_t part) {
    if (part == held) return;
    held = part;
#pragma unroll
    for (int e = 0; e < kSelHeld; ++e) {
      const int64_t j = lo + part * kSelPart + e * kSelThreads + tid;
      key[e] = j < hi ? keys[j] : 0;
    }
  };
  const int64_t parts = (hi - lo + kSelPart - 1) / kSelPart;
  // --- what is kept in any case, and how many of the candidates are there
  uint32_t n = 0, all;
  for (int64_t j = tid; j < lo; j += kSelThreads) n += there(j);
  for (int64_t j = hi + tid; j < end; j += kSelThreads) n += there(j);
  scan_sel(n, sums, all);
  const uint32_t forced = all;
  uint64_t aw = ~0ull, ow = 0;
  n = 0;
  for (int64_t p = 0; p < parts; ++p) {
    hold(p);
#pragma unroll
    for (int e = 0; e < kSelHeld; ++e)
      if (key[e] != 0) {
        ++n;
        aw &= key[e];
        ow |= key[e];
      }
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    aw &= __shfl_xor(aw, d);
    ow |= __shfl_xor(ow, d);
  }
  if (lane == 0) {
    ands[wave] = aw;
    ors[wave] = ow;
  }
  scan_sel(n, sums, all);
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    aw &= ands[w];
    ow |= ors[w];
  }
  const uint32_t take = uint32_t(a.take) - min(uint32_t(a.take), forced);
  // --- the border: pages with key >> shift above `prefix` are chosen, and of those equal to it
  // the first `left`
  int shift = 0;
  uint64_t prefix = 0;
  uint32_t left = 0;
  if (all > take && take > 0) {
    left = take;
    int bits = ow == aw ? 0 : 64 - __clzll(ow ^ aw);
    prefix = bits == 64 ? 0 : aw >> bits;
    while (bits > 0) {
      shift = max(0, bits - 11);
      for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int64_t p = 0; p < parts; ++p) {
        hold(p);
#pragma unroll
        for (int e = 0; e < kSelHeld; ++e)
          if (key[e] != 0 && (bits == 64 || key[e] >> bits == prefix))
            atomicAdd(&hist[(key[e] >> shift) & ((1u << (bits - shift)) - 1)], 1u);
      }
      __syncthreads();
      // bins from the largest on: thread i has two of them
      const int b1 = kSelBins - 1 - 2 * tid, b0 = b1 - 1;
      const uint32_t c1 = hist[b1], c0 = hist[b0];
      uint32_t sum;
      const uint32_t before = scan_sel(c1 + c0, sums, sum);
      if (before < left && before + c1 + c0 >= left) {
        const bool hi_bin = before + c1 >= left;
        pick[0] = hi_bin ? b1 : b0;
        pick[1] = left - before - (hi_bin ? 0 : c1);
        pick[2] = hi_bin ? c1 : c0;
      }
      __syncthreads();
      prefix = bits == 64 ? pick[0] : prefix << (bits - shift) | pick[0];
      left = pick[1];
      bits = shift;
      if (pick[2] == left) break;  // (a bin that is taken whole)
      __syncthreads();
    }
    if (ow == aw) {
      shift = 0;
      prefix = aw;
    }
  }
  const bool every = all <= take;
  // --- the chosen pages in their order
  uint32_t at = 0, equal = 0;
  auto emit = [&](bool chosen, int64_t j) {
    uint32_t sum;
    const uint32_t i = scan_sel(chosen, sums, sum);
    if (chosen && at + i < uint32_t(a.take)) out[at + i] = int32_t(j);
    at += sum;
  };
  for (int64_t j0 = 0; j0 < lo; j0 += kSelThreads) emit(j0 + tid < lo && there(j0 + tid), j0 + tid);
  if (take > 0)
    for (int64_t p = 0; p < parts; ++p) {
      hold(p);
#pragma unroll 1
      for (int e = 0; e < kSelHeld; ++e) {
        const int64_t j0 = lo + p * kSelPart + e * kSelThreads;
        if (j0 >= hi) break;
        uint64_t k = 0;
#pragma unroll
        for (int x = 0; x < kSelHeld; ++x) k = x == e ? key[x] : k;
        bool chosen = k != 0;
        if (!every) {
          const uint64_t top = k >> shift;
          const bool eq = chosen && top == prefix;
          uint32_t sum;
          const uint32_t rank = equal + scan_sel(eq, sums, sum);
          equal += sum;
          chosen = chosen && (top > prefix || (eq && rank < left));
        }
        emit(chosen, j0 + tid);
      }
    }
  for (int64_t j0 = hi; j0 < end; j0 += kSelThreads) emit(j0 + tid < end && there(j0 + tid), j0 + tid);
  for (uint32_t i = at + tid; i < uint32_t(a.take); i += kSelThreads) out[i] = -1;
}

template <class E, int LANES>
void score(const PagedSelect& a, hipStream_t stream) {
  constexpr int kPages = 4 * kScorePages * (64 / LANES);  // of a workgroup
  const int64_t chunks = (std::max<int64_t>(0, a.cols - a.first) + kPages - 1) / kPages;
  if (chunks == 0) return;
  hipLaunchKernelGGL((paged_score_kernel<E, LANES>), dim3(unsigned(a.T * a.Hkv * chunks)), dim3(256), 0, stream, a,
                     int(chunks));
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

hipError_t launch_paged_select(const PagedSelect& a, int fp16, int cus, hipStream_t stream) {
  (void)cus;
  if (fp16) {
    if (a.D > 128) score<SelFp16, 64>(a, stream);
    else if (a.D > 64) score<SelFp16, 32>(a, stream);
    else score<SelFp16, 16>(a, stream);
  } else {
    if (a.D > 128) score<SelBf16, 64>(a, stream);
    else if (a.D > 64) score<SelBf16, 32>(a, stream);
    else score<SelBf16, 16>(a, stream);
  }
  hipLaunchKernelGGL(paged_select_kernel, dim3(unsigned(a.T * a.Hkv)), dim3(kSelThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mqk
