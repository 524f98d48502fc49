// Writing into, reading from and evicting from the 4-bit paged cache (kv4_device.h has the
// record's layout).
#include "kv4_device.h"
#include "mqk_attn.h"

namespace mqk {
namespace {

// Where token t of the call lives: its sequence's page and slot, or false.
// (A wave's lanes ask for the same token.)
struct Place {
  int64_t page;
  int slot;
};
__device__ __forceinline__ bool locate(const Kv4Tokens& a, int64_t t, Place& p) {
  SeqOf q;
  if (a.cu) {
    if (!find_seq(a.cu, a.lens, a.n_seqs, t, q)) return false;
  } else {
    q.s = int(uint32_t(t) / uint32_t(a.each));
    q.at = int64_t(q.s) * a.each;
    q.n = a.each;
    q.len = a.lens[q.s];
  }
  const int64_t pos = int64_t(q.len) - q.n + (t - q.at);
  if (pos < 0 || pos >= a.cols * kPage) return false;
  p.page = a.table[int64_t(q.s) * a.cols + pos / kPage];
  p.slot = int(pos % kPage);
  return p.page >= 0 && p.page < a.num_blocks;
}

__device__ __forceinline__ float min8(float v) {
  v = fminf(v, dpp_move<0xB1>(v));
  v = fminf(v, dpp_move<0x4E>(v));
  return fminf(v, dpp_move<0x141>(v));
}

// x - y = d + err exactly, err as returned (not finite where d is not).
__device__ __forceinline__ float difference_error(float x, float y, float d) {
  const float v = x - d, u = d + v;
  return (x - u) + (v - y);
}

// round(d / s) to the even one of two nearest, exactly, in a type that holds d, s and n * s:
// the whole number that an approximate quotient rounds to is corrected by the remainder.
template <class T>
__device__ __forceinline__ T nearest_code(T d, T s, T n) {
  const T rem2 = T(2) * __builtin_elementwise_fma(-n, s, d);
  const bool odd = (int(n) & 1) != 0;
  if (rem2 > s || (rem2 == s && odd)) n += T(1);
  else if (rem2 < -s || (rem2 == -s && odd)) n -= T(1);
  return n < T(0) ? T(0) : n > T(15) ? T(15) : n;
}

// Scale and least value of a group, from its smallest and largest value, and its codes.
// The definition is exact (quotients of exact differences); it is computed in fp32 where
// the differences are exact there, as they are but for values of very different sizes, and
// in 64 bits otherwise.
template <class E>
struct Group {
  uint32_t bits;  // scale, least
  float s, lo, inv;
  bool far;       // the scale is too small or large to divide by in fp32
  __device__ __forceinline__ Group(float least, float most, bool bad) : lo(least) {
    const float d = most - least;
    float q = d / 15.f;
    if (difference_error(most, least, d) != 0.f) q = static_cast<float>((double(most) - double(least)) / 15.0);
    uint32_t sb = E::from_f32(q), mb = E::from_f32(least);
    if (bad) {  // a group that holds what is not finite reads back as NaN
      sb = 0;
      mb = E::kNaN;
    }
    bits = sb | mb << 16;
    s = E::to_f32(sb);
    far = !(s > 1e-30f && s < 1e30f);
    inv = far ? 0.f : __builtin_amdgcn_rcpf(s);
  }
  // The quotient in fp32 is off by less than 2^-17: only what lands nearer than 2^-15 to the
  // border between two codes, ties among it, is decided by the remainder.  Sets `again`
  // where the difference is not exact: exact_code then.
  __device__ __forceinline__ uint32_t quick_code(float x, bool& again) const {
    const float diff = x - lo, d = diff * inv;
    float n = rintf(d);
    const bool near = fabsf(d - n) > 0.5f - 0x1p-15f;
    if (__any(near) && near) {
      again = again || difference_error(x, lo, diff) != 0.f;
      n = nearest_code(diff, s, n);
    }
    return uint32_t(fminf(n, 15.f));
  }
  __device__ __forceinline__ uint32_t exact_code(float x) const {
    const double d = double(x) - double(lo), t = s;
    return s > 0.f ? uint32_t(nearest_code(d, t, rint(d * (1.0 / t)))) : 0u;
  }
};

// A token a workgroup; D / 8 lanes per head of K or V, 8 elements each.  A group of 64 is 8
// lanes: its least and largest value by three lane moves.  What a decode step takes: its
// time is that of a launch and three loads that wait for each other (64 tokens of 8 heads of
// 128: 4.1 us).
template <class E, int D>
__global__ void __launch_bounds__(256)
kv4_write_kernel(Kv4Tokens a, const unsigned char* __restrict__ k, const unsigned char* __restrict__ v, int64_t k_ts,
                 int64_t k_hs, int64_t v_ts, int64_t v_hs, float* __restrict__ scores) {
  using R = Kv4<D>;
  constexpr int kLanes = D / 8;
  const int64_t t = blockIdx.x;
  const int units = 2 * a.Hkv;
  const int c = threadIdx.x % kLanes;  // dimensions 8 c ..
  Place p;
  if (!locate(a, t, p)) return;
  // (a wave's lanes stay together: the lane moves below need all of a group)
  for (int u0 = threadIdx.x / kLanes; u0 < (units + 7) / 8 * 8; u0 += 256 / kLanes) {
    const int u = min(u0, units - 1);
    const bool is_v = u >= a.Hkv;
    const int h = is_v ? u - a.Hkv : u;
    const unsigned char* src = is_v ? v + t * v_ts + h * v_hs : k + t * k_ts + h * k_hs;
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(src + c * 16);
    float f[8];
    float lo = INFINITY, hi = -INFINITY, bad = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t b = (x[e / 2] >> (16 * (e & 1))) & 0xFFFFu;
      f[e] = E::to_f32(b);
      lo = fminf(lo, f[e]);
      hi = fmaxf(hi, f[e]);
      if ((b & E::kExp) == E::kExp) bad = -1.f;
    }
    lo = min8(lo);
    hi = -min8(-hi);
    bad = min8(bad);
    const Group<E> q(lo, hi, bad != 0.f);
    uint32_t n[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      bool again = q.far;
      n[e] = q.quick_code(f[e], again);
      if (again) n[e] = q.exact_code(f[e]);
    }
    if (u0 >= units) continue;
    unsigned char* rec = a.cache + (p.page * a.Hkv + h) * R::kRecord;
    const int g = c >> 3;
    if (!is_v) {
      const uint32_t w = n[0] | n[2] << 4 | n[4] << 8 | n[6] << 12 | n[1] << 16 | n[3] << 20 | n[5] << 24 | n[7] << 28;
      reinterpret_cast<uint32_t*>(rec)[R::k_word(p.slot, c)] = w;
    } else {
      uint16_t* w = reinterpret_cast<uint16_t*>(rec + R::kV);
      const int m = (c & 7) * 2;
      w[R::v_half(p.slot, g, m)] = uint16_t(n[0] | n[1] << 4 | n[2] << 8 | n[3] << 12);
      w[R::v_half(p.slot, g, m + 1)] = uint16_t(n[4] | n[5] << 4 | n[6] << 8 | n[7] << 12);
    }
    if ((c & 7) == 0)
      reinterpret_cast<uint32_t*>(rec + (is_v ? R::kMetaV : R::kMetaK))[p.slot * R::kG + g] = q.bits;
    if (scores && !is_v && c == 0) scores[(p.page * a.Hkv + h) * kPage + p.slot] = 0.f;
  }
}

// The values of the call's tokens, dense [T, Hkv, D]: a token a workgroup, D / 8 lanes per
// head of K or V.  Tokens that are nowhere in the cache give 0.
template <class E, int D>
__global__ void __launch_bounds__(256)
kv4_read_kernel(Kv4Tokens a, unsigned char* __restrict__ k, unsigned char* __restrict__ v) {
  using R = Kv4<D>;
  constexpr int kLanes = D / 8;
  const int64_t t = blockIdx.x;
  Place p{0, 0};
  const bool there = locate(a, t, p);
  for (int u = threadIdx.x / kLanes; u < 2 * a.Hkv; u += 256 / kLanes) {
    const bool is_v = u >= a.Hkv;
    const int h = is_v ? u - a.Hkv : u;
    const int c = threadIdx.x % kLanes, g = c >> 3;
    u32x4_t out = {0, 0, 0, 0};
    if (there) {
      const unsigned char* rec = a.cache + (p.page * a.Hkv + h) * R::kRecord;
      const uint32_t meta = reinterpret_cast<const uint32_t*>(rec + (is_v ? R::kMetaV : R::kMetaK))[p.slot * R::kG + g];
      const float s = E::to_f32(meta & 0xFFFFu), m = E::to_f32(meta >> 16);
      float f[8];
      if (!is_v) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(rec)[R::k_word(p.slot, c)];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __builtin_fmaf(float((w >> (4 * (e / 2) + 16 * (e & 1))) & 15u), s, m);
      } else {
        const uint16_t* w = reinterpret_cast<const uint16_t*>(rec + R::kV);
        const uint32_t x = w[R::v_half(p.slot, g, (c & 7) * 2)], y = w[R::v_half(p.slot, g, (c & 7) * 2 + 1)];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[e] = __builtin_fmaf(float((x >> (4 * e)) & 15u), s, m);
          f[4 + e] = __builtin_fmaf(float((y >> (4 * e)) & 15u), s, m);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = E::pack2(f[2 * e], f[2 * e + 1]);
    }
    *reinterpret_cast<u32x4_t*>((is_v ? v : k) + ((t * a.Hkv + h) * D + c * 8) * 2) = out;
  }
}

// ---------------------------------------------------------------------------------------
// Whole pages: runs of tokens, a wave per page and head.  Its lanes hold the record's words
// as they lie (kv4_device.h), so that a page is written and read in whole cache lines; token
// by token the V codes go out as 2-byte stores 16 bytes apart.  Bound by memory and, writing,
// by the vector instructions of the codes (20 for a value): 8192 tokens of 8 heads of 128 are
// written in 15.0 us (2.9 TB/s of what is read and written), read in 10.6 us (4.1 TB/s).
// ---------------------------------------------------------------------------------------

template <int W>
__device__ __forceinline__ void load_words(const uint32_t* from, uint32_t (&w)[W]) {
  if constexpr (W == 4) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(from);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = x[e];
  } else {
    const u32x2_t x = *reinterpret_cast<const u32x2_t*>(from);
    w[0] = x[0];
    w[1] = x[1];
  }
}
template <int W>
__device__ __forceinline__ void store_words(uint32_t* to, const uint32_t (&w)[W]) {
  if constexpr (W == 4) *reinterpret_cast<u32x4_t*>(to) = u32x4_t{w[0], w[1], w[2], w[3]};
  else *reinterpret_cast<u32x2_t*>(to) = u32x2_t{w[0], w[1]};
}
template <int G>
__device__ __forceinline__ void store_meta(unsigned char* to, int token, const uint32_t (&bits)[G]) {
  if constexpr (G == 2) reinterpret_cast<u32x2_t*>(to)[token] = u32x2_t{bits[0], bits[1]};
  else reinterpret_cast<uint32_t*>(to)[token] = bits[0];
}

// A page of a call's tokens.  Sequence s of n tokens at cu[s] touches at most n / 16 + 2
// pages; its slots start at cu[s] / 16 + 2 s, which leaves it that many without a sum over
// the lengths.  The slots past the last sequence's hold the tokens behind it.
struct PageOf {
  int64_t page;   // in the cache, or -1: its tokens are nowhere there
  int64_t token;  // of the page's slot 0 (may lie before the sequence's first new one)
  int from, to;   // slots that hold tokens of the call
};
__device__ __forceinline__ PageOf page_of(const Kv4Tokens& a, int64_t slot) {
  const int lane = threadIdx.x & 63;
  PageOf p{-1, 0, 0, 0};
  int s = -1;
  int64_t at = 0, n = 0, len = 0;
  if (a.cu) {
    for (int base = 0; base <= a.n_seqs; base += 63) {  // 64 offsets cover 63 sequences
      const int c = base + lane;
      int64_t off = a.cu[c <= a.n_seqs ? c : a.n_seqs];
      const int32_t l = a.lens[c < a.n_seqs ? c : a.n_seqs - 1];
      off = off < 0 ? 0 : off > a.T ? a.T : off;
      const int below = __popcll(__ballot(c <= a.n_seqs && off / kPage + 2 * int64_t(c) <= slot));
      if (below == 0) return p;
      if (below <= 63) {
        const int i = below - 1;
        s = base + i;
        at = __builtin_amdgcn_readlane(int(off), i);
        if (s >= a.n_seqs) {
          p.token = at + (slot - (at / kPage + 2 * int64_t(a.n_seqs))) * kPage;
          p.to = int(max(int64_t(0), min(int64_t(kPage), a.T - p.token)));
          return p;
        }
        n = __builtin_amdgcn_readlane(int(off), i + 1) - at;
        len = __builtin_amdgcn_readlane(l, i);
        break;
      }
    }
    if (s < 0) return p;
  } else {
    // (equal lengths: the last sequence whose first slot is not past this one)
    int64_t lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
      const int64_t m = (lo + hi) / 2;
      if (m * a.each / kPage + 2 * m <= slot) lo = m;
      else hi = m;
    }
    s = int(lo);
    at = lo * a.each;
    n = a.each;
    len = a.lens[s];
  }
  if (n <= 0) return p;
  const int64_t pos0 = len - n;                                      // of the first new token
  const int64_t first = pos0 >= 0 ? pos0 / kPage : -((15 - pos0) / kPage);  // its page (rounded down)
  const int64_t index = first + (slot - (at / kPage + 2 * int64_t(s)));
  const int64_t start = index * kPage - pos0;  // of slot 0 among the new tokens
  p.token = at + start;
  p.from = int(start < 0 ? min(-start, int64_t(kPage)) : 0);
  p.to = int(max(int64_t(0), min(int64_t(kPage), n - start)));
  if (p.from >= p.to || index < 0 || index >= a.cols) return p;
  const int64_t id = a.table[int64_t(s) * a.cols + index];
  if (id >= 0 && id < a.num_blocks) p.page = id;
  return p;
}

// A wave takes a page of a head of K or V (both in one wave: 18.5 us for 8214 tokens of 8
// heads, where this takes 16.3): lane = (quarter, token), 16 dimensions of each group, the
// order of K's words; V's go through LDS into theirs.
template <class E, int D>
__global__ void __launch_bounds__(256)
kv4_write_pages_kernel(Kv4Tokens a, const unsigned char* __restrict__ k, const unsigned char* __restrict__ v,
                       int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs, float* __restrict__ scores, int64_t slots) {
  using R = Kv4<D>;
  constexpr int kG = R::kG;
  constexpr int kW = 2 * kG;  // words of a lane's codes
  __shared__ __align__(16) uint32_t turn[4][64 * kW];
  const int lane = threadIdx.x & 63, quad = lane >> 4, row = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = int64_t(blockIdx.x) * 4 + wave;
  const int units = 2 * a.Hkv;  // K's heads, then V's
  if (item >= slots * units) return;
  const int unit = int(item % units);
  const bool is_v = unit >= a.Hkv;
  const int h = is_v ? unit - a.Hkv : unit;
  const PageOf p = page_of(a, item / units);
  if (p.page < 0) return;
  unsigned char* rec = a.cache + (p.page * a.Hkv + h) * R::kRecord;
  const bool mine = row >= p.from && row < p.to;
  const int64_t t = mine ? p.token + row : p.token + p.from;
  const unsigned char* src = (is_v ? v + t * v_ts + h * v_hs : k + t * k_ts + h * k_hs) + quad * 32;
  u32x4_t x[kG][2];
#pragma unroll
  for (int g = 0; g < kG; ++g)
#pragma unroll
    for (int half = 0; half < 2; ++half) x[g][half] = *reinterpret_cast<const u32x4_t*>(src + g * 128 + half * 16);
  {
    uint32_t words[kW], bits[kG];
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      float f[16], lo = INFINITY, hi = -INFINITY, bad = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        f[e] = E::to_f32((x[g][e / 8][e / 2 % 4] >> (16 * (e & 1))) & 0xFFFFu);
        lo = fminf(lo, f[e]);
        hi = fmaxf(hi, f[e]);
        bad = __builtin_fmaf(f[e], 0.f, bad);  // (NaN where one is not finite)
      }
      lo = fminf(lo, __shfl_xor(lo, 16));
      hi = fmaxf(hi, __shfl_xor(hi, 16));
      lo = fminf(lo, __shfl_xor(lo, 32));
      hi = fmaxf(hi, __shfl_xor(hi, 32));
      if (__any(bad != 0.f)) {  // (rare: no moves for it otherwise)
        bad += __shfl_xor(bad, 16);
        bad += __shfl_xor(bad, 32);
      }
      const Group<E> q(lo, hi, bad != 0.f);
      bits[g] = q.bits;
      uint32_t n[16];
      bool again = q.far;
#pragma unroll
      for (int e = 0; e < 16; ++e) n[e] = q.quick_code(f[e], again);
      if (__any(again)) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (again) n[e] = q.exact_code(f[e]);
      }
      if (!is_v) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t w = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) w |= n[half * 8 + j] << (4 * (j / 2) + 16 * (j & 1));
          words[g * 2 + half] = w;
        }
      } else {
        // 4 dimensions, m = 4 quad + i, of this token: 16 bits in V's place for it
#pragma unroll
        for (int i = 0; i < 4; ++i)
          reinterpret_cast<uint16_t*>(turn[wave])[R::v_half(row, g, quad * 4 + i)] =
              uint16_t(n[4 * i] | n[4 * i + 1] << 4 | n[4 * i + 2] << 8 | n[4 * i + 3] << 12);
      }
    }
    if (!is_v) {
      if (mine) {
        store_words(reinterpret_cast<uint32_t*>(rec) + lane * kW, words);
        if (quad == 0) store_meta<kG>(rec + R::kMetaK, row, bits);
        if (scores && quad == 1) scores[(p.page * a.Hkv + h) * kPage + row] = 0.f;
      }
      return;
    }
    if (mine && quad == 0) store_meta<kG>(rec + R::kMetaV, row, bits);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (the wave's own LDS words, in order)
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int i = 0; i < kW; ++i) words[i] = turn[wave][lane * kW + i];
    // lane = (token / 4, m): whole where its 4 tokens are all of the call's
    uint32_t* dst = reinterpret_cast<uint32_t*>(rec + R::kV) + lane * kW;
    if (quad * 4 >= p.from && quad * 4 + 4 <= p.to) {
      store_words(dst, words);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (quad * 4 + r >= p.from && quad * 4 + r < p.to) {
          if constexpr (kG == 2) dst[r] = words[r % kW];
          else reinterpret_cast<uint16_t*>(dst)[r] = uint16_t(words[r / 2] >> (16 * (r & 1)));
        }
    }
  }
}

// A wave a page and head, K and V: their words as they lie, a lane's output 32 bytes of K's
// rows and 8 of V's.
template <class E, int D>
__global__ void __launch_bounds__(256)
kv4_read_pages_kernel(Kv4Tokens a, unsigned char* __restrict__ k, unsigned char* __restrict__ v, int64_t slots) {
  using R = Kv4<D>;
  constexpr int kG = R::kG;
  const int lane = threadIdx.x & 63, quad = lane >> 4, row = lane & 15;
  const int64_t item = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= slots * a.Hkv) return;
  const int h = int(item % a.Hkv);
  const PageOf p = page_of(a, item / a.Hkv);
  if (p.from >= p.to) return;
  // (a page that is not there: zeros)
  const bool there = p.page >= 0;
  const unsigned char* rec = a.cache + ((there ? p.page : 0) * a.Hkv + h) * R::kRecord;
  uint32_t kw[2 * kG], vw[2 * kG], km[kG], vm[4][kG];
#pragma unroll
  for (int i = 0; i < 2 * kG; ++i) {
    kw[i] = reinterpret_cast<const uint32_t*>(rec)[lane * 2 * kG + i];
    vw[i] = reinterpret_cast<const uint32_t*>(rec + R::kV)[lane * 2 * kG + i];
  }
#pragma unroll
  for (int g = 0; g < kG; ++g) {
    km[g] = reinterpret_cast<const uint32_t*>(rec + R::kMetaK)[row * kG + g];
#pragma unroll
    for (int r = 0; r < 4; ++r) vm[r][g] = reinterpret_cast<const uint32_t*>(rec + R::kMetaV)[(quad * 4 + r) * kG + g];
  }
  if (row >= p.from && row < p.to) {
    unsigned char* dst = k + ((p.token + row) * a.Hkv + h) * D * 2;
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      const float s = E::to_f32(km[g] & 0xFFFFu), m = E::to_f32(km[g] >> 16);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t w = kw[g * 2 + half];
        u32x4_t out;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          out[e] = there ? E::pack2(__builtin_fmaf(float(w >> (4 * e) & 15u), s, m),
                                    __builtin_fmaf(float(w >> (16 + 4 * e) & 15u), s, m))
                         : 0u;
        *reinterpret_cast<u32x4_t*>(dst + (g * 64 + quad * 16 + half * 8) * 2) = out;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int slot = quad * 4 + r;
    if (slot < p.from || slot >= p.to) continue;
    unsigned char* dst = v + ((p.token + slot) * a.Hkv + h) * D * 2;
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      const float s = E::to_f32(vm[r][g] & 0xFFFFu), m = E::to_f32(vm[r][g] >> 16);
      const uint32_t w = kG == 2 ? vw[r % (2 * kG)] >> (16 * g) : vw[r / 2 % (2 * kG)] >> (16 * (r & 1));
      u32x2_t out;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        out[e] = there ? E::pack2(__builtin_fmaf(float(w >> (8 * e) & 15u), s, m),
                                  __builtin_fmaf(float(w >> (8 * e + 4) & 15u), s, m))
                       : 0u;
      *reinterpret_cast<u32x2_t*>(dst + (g * 64 + row * 4) * 2) = out;
    }
  }
}

// ---------------------------------------------------------------------------------------
// Eviction: a workgroup per (sequence, head).  The budget-th largest score is found by a radix
// selection over the scores' bits, 11 at a time (counts in LDS, two bins a thread; a score's
// first 11 bits are its sign, exponent and two more), then the kept tokens are numbered in
// their order by a sum over the workgroup, and moved to the front a batch of pages at a time.
// A token only ever moves forward: once the tokens of a batch and of those before it have
// been read, writing the batch touches nothing that a later one reads.  Scores stay in
// registers, 16 a thread (longer sequences: a part of them at a time).
// A token that is not there (past the table, or in a page outside the cache) is never kept:
// its place at the front would go on holding the token that stood there before.  A sequence
// has the same tokens in every head, so its new length is the same in all of them.
// Moving in place ties a piece of the record to one workgroup, but not the whole record:
// where heads are few, a second launch moves it with four workgroups a head (half of K's
// quarters or of V's columns each), as one CU's loads would bound it otherwise.
// Down to 2048 from 4096 tokens of 8 heads of 128, in one launch and in two: one sequence
// 26.0 and 19.0 us (12.6 of them the selection and the list), 8 sequences 28.3 and 21.7, 16
// 30.6 and 30.5, 32 37.6 and 44.3; the sum that leaves out recent tokens that are not there
// has added 0.3 to 0.7 us to each.  32 sequences of up to 6000 tokens: 54 us, 141 MB read and 75
// written (4.0 TB/s, the selection's time in it).  75 MB of what is read are kept tokens and
// scores: a line comes whole for every kept part of it.
// ---------------------------------------------------------------------------------------

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;
constexpr int kEvictHeld = 16;
constexpr int kEvictPart = kEvictThreads * kEvictHeld;
constexpr int kEvictBins = 2048;
constexpr int kEvictList = 8192;  // kept positions that stay in LDS

// A float's place in ascending order; -0 as 0, every NaN as one value above infinity.
__device__ __forceinline__ uint32_t order_key(float f) {
  uint32_t b = __float_as_uint(f);
  if (b == 0x80000000u) b = 0;
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

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
  x = add_dpp<0x142, 0xA>(x);  // row 0's sum to row 1, row 2's to row 3
  return add_dpp<0x143, 0xC>(x);  // rows 0 and 1's to rows 2 and 3
}
// Sum over the threads before this one, and over all of the workgroup.
__device__ __forceinline__ uint32_t scan_evict(uint32_t v, uint32_t* lds, uint32_t& all) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t x = scan_wave(v);
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  const uint32_t w = scan_wave(lane < kEvictWaves ? lds[lane] : 0u);
  all = __builtin_amdgcn_readlane(w, kEvictWaves - 1);
  return (wave > 0 ? __builtin_amdgcn_readlane(w, wave - 1) : 0u) + x - v;
}

// D > 0: the move in the same launch; 0: not.
template <int D>
__global__ void __launch_bounds__(kEvictThreads)
kv4_evict_kernel(Kv4Evict a) {
  __shared__ uint32_t hist[kEvictBins];
  __shared__ uint32_t sums[kEvictWaves];
  __shared__ uint32_t counts[2][kEvictHeld * kEvictWaves];
  __shared__ uint32_t pick[3];  // digit, what is left to take in its bin, and what is there
  __shared__ int32_t list[D > 0 ? kEvictList : 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / a.Hkv, h = blockIdx.x % a.Hkv;
  const int64_t cap = a.cols * kPage;
  const int len = max(a.lens[b], 0);
  const int budget = a.budget;
  int32_t* kept = a.kept + (int64_t(b) * a.Hkv + h) * budget;
  if (len <= budget) {
    if (h == 0 && tid == 0) a.new_lens[b] = len;
    for (int i = tid; i < budget; i += kEvictThreads) kept[i] = i < len ? i : -1;
    return;
  }
  const int32_t* table = a.table + int64_t(b) * a.cols;
  const int recent = min(a.recent, budget);
  const int last = len - recent;          // the first of the recent tokens
  const int old = int(min(int64_t(last), cap));  // candidates: the tokens before it in the table
  const int take = budget - recent;       // of them to keep
  auto recent_there = [&](int i) {        // is the i-th recent token there?
    if (i >= recent || last + i >= cap) return false;
    const int page = table[(last + i) / kPage];
    return page >= 0 && page < a.num_blocks;
  };
  const bool there0 = recent_there(tid);  // (the first ones' loads under the selection)

  uint32_t keys[kEvictHeld];
  int held = -1;
  auto hold = [&](int part) {  // token part * kEvictPart + e * 1024 + tid in keys[e]; 0 past the last
    if (part == held) return;
    held = part;
    int ids[kEvictHeld];
#pragma unroll
    for (int e = 0; e < kEvictHeld; ++e) {
      const int i = part * kEvictPart + e * kEvictThreads + tid;
      ids[e] = i < old ? table[i / kPage] : -1;
    }
#pragma unroll
    for (int e = 0; e < kEvictHeld; ++e) {
      // (a page that is not there: below every score)
      const int64_t page = ids[e];
      keys[e] = 0;
      if (page >= 0 && page < a.num_blocks) keys[e] = order_key(a.scores[(page * a.Hkv + h) * kPage + tid % kPage]);
    }
  };
  const int parts = (old + kEvictPart - 1) / kEvictPart;
  auto left_of = [&](int part) { return old - part * kEvictPart; };  // tokens from this part's first on

  // threshold: the take-th largest key, and how many equal to it are kept (fewer candidates:
  // all that are there, whose keys are above 0)
  uint32_t prefix = 0, left = 0;
  if (take > 0 && take <= old) {
    left = uint32_t(take);
    int bits = 32;  // still to be decided
    while (bits > 0) {
      const int shift = bits - min(bits, 11);
      hist[tid] = hist[tid + kEvictThreads] = 0;
      __syncthreads();
      for (int part = 0; part < parts; ++part) {
        hold(part);
        const int n = left_of(part);
#pragma unroll
        for (int e = 0; e < kEvictHeld; ++e)
          if (e * kEvictThreads < n) {
            if (e * kEvictThreads + tid < n && (bits == 32 || keys[e] >> bits == prefix >> bits))
              atomicAdd(&hist[(keys[e] >> shift) & (kEvictBins - 1)], 1u);
          }
      }
      __syncthreads();
      // bins from the highest down, two a thread
      const uint32_t n0 = hist[kEvictBins - 1 - 2 * tid], n1 = hist[kEvictBins - 2 - 2 * tid];
      uint32_t all;
      const uint32_t above = scan_evict(n0 + n1, sums, all);
      if (above < left && above + n0 + n1 >= left) {
        const bool second = above + n0 < left;
        pick[0] = uint32_t(kEvictBins - 1 - 2 * tid - second);
        pick[1] = left - above - (second ? n0 : 0u);
        pick[2] = second ? n1 : n0;
      }
      __syncthreads();
      prefix |= pick[0] << shift;
      left = pick[1];
      bits = shift;
      if (pick[2] == left && prefix > 0) {
        // all of the bin are kept: those above the number before it, none equal to that
        prefix -= 1;
        left = 0;
        break;
      }
    }
    if (prefix == 0) left = 0;  // (key 0: tokens that are not there)
  }

  // the kept tokens in order: those above the threshold, and the first `left` equal to it
  uint32_t more_base = 0, tie_base = 0;
  for (int part = 0; part < parts && take > 0; ++part) {
    hold(part);
    const uint64_t below = (1ull << lane) - 1;
    const int n = left_of(part), runs = min(kEvictHeld, (n + kEvictThreads - 1) / kEvictThreads) * kEvictWaves;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEvictHeld; ++e) {
      if (e * kEvictThreads >= n) break;
      const bool in = e * kEvictThreads + tid < n;
      const uint64_t bm = __ballot(in && keys[e] > prefix), bt = __ballot(in && keys[e] == prefix);
      if (lane == 0) {
        counts[0][e * kEvictWaves + wave] = __popcll(bm);
        counts[1][e * kEvictWaves + wave] = __popcll(bt);
      }
    }
    __syncthreads();
    // sums over the runs of 64 before, in the tokens' order
    uint32_t more_all, tie_all;
    const uint32_t m0 = scan_evict(tid < runs ? counts[0][tid] : 0u, sums, more_all);
    const uint32_t t0 = scan_evict(tid < runs ? counts[1][tid] : 0u, sums, tie_all);
    if (tid < runs) {
      counts[0][tid] = m0;
      counts[1][tid] = t0;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEvictHeld; ++e) {
      if (e * kEvictThreads >= n) break;
      const bool in = e * kEvictThreads + tid < n;
      const bool more = in && keys[e] > prefix, tie = in && keys[e] == prefix;
      const uint64_t bm = __ballot(more), bt = __ballot(tie);
      const uint32_t m = more_base + counts[0][e * kEvictWaves + wave] + __popcll(bm & below);
      const uint32_t t = tie_base + counts[1][e * kEvictWaves + wave] + __popcll(bt & below);
      const uint32_t at = m + min(t, left);
      if ((more || (tie && t < left)) && at < uint32_t(take)) {
        const int i = part * kEvictPart + e * kEvictThreads + tid;
        kept[at] = i;
        if (D > 0 && at < kEvictList) list[at] = i;
      }
    }
    more_base += more_all;
    tie_base += tie_all;
  }
  int now = min(int(more_base + min(tie_base, left)), take);
  for (int i0 = 0; i0 < recent; i0 += kEvictThreads) {
    const bool there = i0 == 0 ? there0 : recent_there(i0 + tid);
    uint32_t all;
    const int at = now + int(scan_evict(there, sums, all));
    if (there) {
      kept[at] = last + i0 + tid;
      if (D > 0 && at < kEvictList) list[at] = last + i0 + tid;
    }
    now += int(all);
  }
  if (h == 0 && tid == 0) a.new_lens[b] = now;
  for (int i = now + tid; i < budget; i += kEvictThreads) kept[i] = -1;
  if constexpr (D == 0) return;
  using R = Kv4<D == 0 ? 128 : D>;
  __threadfence_block();
  __syncthreads();

  // move: kPages pages a wave and batch
  constexpr int kPages = 4;
  constexpr int kW = R::kG * 2;  // words of a lane's codes of one page
  const int pages = (now + kPage - 1) / kPage;
  const int row = lane & 15, quad = lane >> 4;
  for (int p0 = 0; p0 < pages; p0 += kEvictWaves * kPages) {
    uint32_t kc[kPages][kW], vc[kPages][kW], meta[kPages];
    float sc[kPages];
    int from[kPages], id[kPages], to[kPages];
#pragma unroll
    for (int j = 0; j < kPages; ++j) {
      const int p = p0 + j * kEvictWaves + wave;
      const int at = p * kPage + row;
      from[j] = -1;
      if (at < now) from[j] = at < kEvictList ? list[at] : kept[at];
      to[j] = p < pages ? table[p] : -1;
    }
#pragma unroll
    for (int j = 0; j < kPages; ++j) {
      id[j] = from[j] >= 0 ? table[from[j] / kPage] : -1;
      if (id[j] >= a.num_blocks) id[j] = -1;
      from[j] &= kPage - 1;
    }
#pragma unroll
    for (int j = 0; j < kPages; ++j) {
#pragma unroll
      for (int e = 0; e < kW; ++e) kc[j][e] = vc[j][e] = 0;
      meta[j] = 0;
      sc[j] = 0.f;
      if (id[j] >= 0) {
        // K: this lane's quarter of token `row`; scale and least value of group quad % 2 of K
        // (quarters 0, 1) and V; the score
        const unsigned char* rec = a.cache + (int64_t(id[j]) * a.Hkv + h) * R::kRecord;
        const uint32_t* w = reinterpret_cast<const uint32_t*>(rec) + (quad * 16 + from[j]) * kW;
#pragma unroll
        for (int e = 0; e < kW; ++e) kc[j][e] = w[e];
        const int g = quad & 1;
        if (g < R::kG)
          meta[j] = reinterpret_cast<const uint32_t*>(rec + (quad < 2 ? R::kMetaK : R::kMetaV))[from[j] * R::kG + g];
        if (quad == 0) sc[j] = a.scores[(int64_t(id[j]) * a.Hkv + h) * kPage + from[j]];
      }
      // V: tokens 4 quad .. 4 quad + 3, column block m = row
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int vid = __shfl(id[j], 4 * quad + r), f = __shfl(from[j], 4 * quad + r);
        if (vid < 0) continue;
        const unsigned char* w = a.cache + (int64_t(vid) * a.Hkv + h) * R::kRecord + R::kV + R::v_half(f, 0, row) * 2;
        if constexpr (R::kG == 2) vc[j][r % kW] = *reinterpret_cast<const uint32_t*>(w);
        else vc[j][r / 2] |= uint32_t(*reinterpret_cast<const uint16_t*>(w)) << (16 * (r & 1));
      }
    }
    wait_vm<0>();  // every wave's loads are there before any wave writes
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPages; ++j) {
      if (to[j] < 0 || to[j] >= a.num_blocks) continue;
      unsigned char* rec = a.cache + (int64_t(to[j]) * a.Hkv + h) * R::kRecord;
      if (id[j] >= 0) {
        uint32_t* w = reinterpret_cast<uint32_t*>(rec) + (quad * 16 + row) * kW;
        store_words(w, kc[j]);
        const int g = quad & 1;
        if (g < R::kG)
          reinterpret_cast<uint32_t*>(rec + (quad < 2 ? R::kMetaK : R::kMetaV))[row * R::kG + g] = meta[j];
        if (quad == 0) a.scores[(int64_t(to[j]) * a.Hkv + h) * kPage + row] = sc[j];
      }
      uint32_t* w = reinterpret_cast<uint32_t*>(rec + R::kV) + (quad * 16 + row) * kW;
      const uint64_t there = __ballot(id[j] >= 0);  // of a page's tokens in lanes 0 .. 15
      const uint32_t mine = uint32_t(there >> (4 * quad)) & 15u;
      if (mine == 15u) {
        store_words(w, vc[j]);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (mine >> r & 1) {
            if constexpr (R::kG == 2) w[r] = vc[j][r % kW];
            else reinterpret_cast<uint16_t*>(w)[r] = uint16_t(vc[j][r / 2] >> (16 * (r & 1)));
          }
      }
    }
  }
}

constexpr int kMoveThreads = 512;
constexpr int kMoveWaves = kMoveThreads / 64;
constexpr int kMovePages = 8;  // a wave and batch, two a step
constexpr int kMoveParts = 4;   // of the record

template <int D>
__global__ void __launch_bounds__(kMoveThreads)
kv4_move_kernel(Kv4Evict a) {
  using R = Kv4<D>;
  constexpr int kW = D / 32;  // words of a lane's codes of one page
  constexpr int kSteps = kMovePages / 2;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = blockIdx.x % kMoveParts, bh = blockIdx.x / kMoveParts;
  const int b = bh / a.Hkv, h = bh % a.Hkv;
  if (a.lens[b] <= a.budget) return;
  const int32_t* table = a.table + int64_t(b) * a.cols;
  const int32_t* kept = a.kept + int64_t(bh) * a.budget;  // (-1 behind the last kept one)
  const int pages = int(min(int64_t((a.budget + kPage - 1) / kPage), a.cols));
  auto record = [&](int id) { return a.cache + (int64_t(id) * a.Hkv + h) * R::kRecord; };
  // every wave's loads are there before any wave writes
  auto turn = [&]() {
    wait_vm<0>();
    __syncthreads();
  };
  for (int p0 = 0; p0 < pages; p0 += kMoveWaves * kMovePages) {
    // (loads without branches between them, so that they are all under way: from the first
    // record where there is nothing to load)
    int from[kSteps], id[kSteps], to[kSteps];  // of the lane's token (lane % 16) of its page
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const int p = p0 + (j * kMoveWaves + wave) * 2 + half, at = p * kPage + (lane & 15);
      from[j] = at < a.budget ? kept[at] : -1;
      to[j] = table[min(p, pages - 1)];
      if (p >= pages || to[j] >= a.num_blocks) to[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      id[j] = table[max(from[j], 0) / kPage];
      if (from[j] < 0 || id[j] >= a.num_blocks) id[j] = -1;
      from[j] &= kPage - 1;
    }
    uint32_t words[kSteps][kW];
    if (part < 2) {
      // K: lane = (page, quarter, token), and beside the codes, of quarter % 2: K's scale and
      // least value of that group (part 0), or V's and, in quarter 2's lanes, the score
      const int token = lane & 15, g = (lane >> 4) & 1, quarter = part * 2 + g;
      const int meta_at = part == 0 ? R::kMetaK : R::kMetaV, mg = g < R::kG ? g : 0;
      uint32_t meta[kSteps];
      float score[kSteps];
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        const unsigned char* rec = record(max(id[j], 0));
        load_words(reinterpret_cast<const uint32_t*>(rec) + (quarter * 16 + from[j]) * kW, words[j]);
        meta[j] = reinterpret_cast<const uint32_t*>(rec + meta_at)[from[j] * R::kG + mg];
        if (part == 1) score[j] = a.scores[(int64_t(max(id[j], 0)) * a.Hkv + h) * kPage + from[j]];
      }
      turn();
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        if (id[j] < 0 || to[j] < 0) continue;
        unsigned char* rec = record(to[j]);
        store_words(reinterpret_cast<uint32_t*>(rec) + (quarter * 16 + token) * kW, words[j]);
        if (g < R::kG) reinterpret_cast<uint32_t*>(rec + meta_at)[token * R::kG + g] = meta[j];
        if (quarter == 2) a.scores[(int64_t(to[j]) * a.Hkv + h) * kPage + token] = score[j];
      }
    } else {
      // V: lane = (page, four tokens, column block m)
      const int quad = (lane >> 3) & 3, m = (part - 2) * 8 + (lane & 7);
      uint32_t there = 0;  // four bits a step
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
#pragma unroll
        for (int e = 0; e < kW; ++e) words[j][e] = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int vid = __shfl(id[j], half * 32 + quad * 4 + r), f = __shfl(from[j], half * 32 + quad * 4 + r);
          there |= uint32_t(vid >= 0) << (4 * j + r);
          const unsigned char* w = record(max(vid, 0)) + R::kV + R::v_half(f, 0, m) * 2;
          if constexpr (R::kG == 2) words[j][r % kW] = *reinterpret_cast<const uint32_t*>(w);
          else words[j][r / 2] |= uint32_t(*reinterpret_cast<const uint16_t*>(w)) << (16 * (r & 1));
        }
      }
      turn();
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        if (to[j] < 0) continue;
        uint32_t* w = reinterpret_cast<uint32_t*>(record(to[j]) + R::kV) + (quad * 16 + m) * kW;
        const uint32_t mine = there >> (4 * j) & 15u;
        if (mine == 15u) {
          store_words(w, words[j]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (mine >> r & 1) {
              if constexpr (R::kG == 2) w[r] = words[j][r % kW];
              else reinterpret_cast<uint16_t*>(w)[r] = uint16_t(words[j][r / 2] >> (16 * (r & 1)));
            }
        }
      }
    }
  }
}

}  // namespace

// Long runs of tokens go page by page, others token by token, and so do few tokens, where a
// wave a page and head is too few waves.  By pages and by tokens at 8 heads of 128 (us):
//   one sequence of 8192     write 15.0, 21.7   read 10.6, 16.7
//   512 sequences of 16      write 33.7, 29.7   read 16.5, 24.1
//   64 sequences of 32       write  9.3,  8.4   read  6.8,  5.4
//   one sequence of 1024     write  6.6,  5.8   read  4.7,  4.4
bool write_by_pages(const Kv4Tokens& a) { return a.T >= 64 * int64_t(a.n_seqs) && a.T * a.Hkv >= 16384; }
bool read_by_pages(const Kv4Tokens& a) { return a.T >= kPage * int64_t(a.n_seqs) && a.T * a.Hkv >= 32768; }

hipError_t launch_kv4_write(const Kv4Tokens& a, const unsigned char* k, const unsigned char* v, int64_t k_ts,
                            int64_t k_hs, int64_t v_ts, int64_t v_hs, float* scores, int D, int fp16,
                            hipStream_t stream) {
  const dim3 t(256);
  const int64_t slots = a.T / kPage + 2 * int64_t(a.n_seqs) + 2;
  const dim3 pages(unsigned((slots * a.Hkv * 2 + 3) / 4));
#define MQK_WRITE(E, DD)                                                                                              \
  if (write_by_pages(a))                                                                                              \
    hipLaunchKernelGGL((kv4_write_pages_kernel<E, DD>), pages, t, 0, stream, a, k, v, k_ts, k_hs, v_ts, v_hs, scores,  \
                       slots);                                                                                        \
  else                                                                                                                \
    hipLaunchKernelGGL((kv4_write_kernel<E, DD>), dim3(unsigned(a.T)), t, 0, stream, a, k, v, k_ts, k_hs, v_ts, v_hs,  \
                       scores)
  if (fp16) {
    if (D == 128) { MQK_WRITE(KvFp16, 128); }
    else { MQK_WRITE(KvFp16, 64); }
  } else {
    if (D == 128) { MQK_WRITE(KvBf16, 128); }
    else { MQK_WRITE(KvBf16, 64); }
  }
#undef MQK_WRITE
  return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4Tokens& a, unsigned char* k, unsigned char* v, int D, int fp16, hipStream_t stream) {
  const dim3 t(256);
  const int64_t slots = a.T / kPage + 2 * int64_t(a.n_seqs) + 2;
  const dim3 pages(unsigned((slots * a.Hkv + 3) / 4));
#define MQK_READ(E, DD)                                                                                       \
  if (read_by_pages(a))                                                                                       \
    hipLaunchKernelGGL((kv4_read_pages_kernel<E, DD>), pages, t, 0, stream, a, k, v, slots);                   \
  else                                                                                                        \
    hipLaunchKernelGGL((kv4_read_kernel<E, DD>), dim3(unsigned(a.T)), t, 0, stream, a, k, v)
  if (fp16) {
    if (D == 128) { MQK_READ(KvFp16, 128); }
    else { MQK_READ(KvFp16, 64); }
  } else {
    if (D == 128) { MQK_READ(KvBf16, 128); }
    else { MQK_READ(KvBf16, 64); }
  }
#undef MQK_READ
  return hipGetLastError();
}

hipError_t launch_kv4_evict(const Kv4Evict& a, int64_t n_seqs, int D, int cus, hipStream_t stream) {
  const int64_t heads = n_seqs * a.Hkv;
  const dim3 e{unsigned(heads)}, et(kEvictThreads);
  // (both sides measured above; to 16 of 4096 tokens one sequence takes 12.8 us in one launch,
  // 14.4 in two, to 500 of 1000 13.6 and 13.0)
  if (2 * heads >= cus || a.budget < 256) {
    if (D == 128) hipLaunchKernelGGL(kv4_evict_kernel<128>, e, et, 0, stream, a);
    else hipLaunchKernelGGL(kv4_evict_kernel<64>, e, et, 0, stream, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(kv4_evict_kernel<0>, e, et, 0, stream, a);
  const dim3 m{unsigned(heads * kMoveParts)}, mt(kMoveThreads);
  if (D == 128) hipLaunchKernelGGL(kv4_move_kernel<128>, m, mt, 0, stream, a);
  else hipLaunchKernelGGL(kv4_move_kernel<64>, m, mt, 0, stream, a);
  return hipGetLastError();
}

}  // namespace mqk
