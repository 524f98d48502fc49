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
    q.s = int(t / a.each);
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

// round(d / s) to the even one of two nearest, exactly: d * (1 / s) is off by 2^-52, so the
// whole number it rounds to is corrected by the (exact) remainder.
__device__ __forceinline__ int nearest_code(double d, double s, double inv) {
  double n = rint(d * inv);
  const double rem2 = 2.0 * __builtin_fma(-n, s, d);
  const bool odd = (int(n) & 1) != 0;
  if (rem2 > s || (rem2 == s && odd)) n += 1.0;
  else if (rem2 < -s || (rem2 == -s && odd)) n -= 1.0;
  return n < 0.0 ? 0 : n > 15.0 ? 15 : int(n);
}

// One workgroup per token; D / 8 lanes per head of K or V, 8 elements each.  A group of 64
// is 8 lanes: its least and largest value by three lane moves.
template <class E, int D>
__global__ void __launch_bounds__(256)
kv4_write_kernel(Kv4Tokens a, const unsigned char* __restrict__ k, const unsigned char* __restrict__ v, int64_t k_ts,
                 int64_t k_hs, int64_t v_ts, int64_t v_hs, float* __restrict__ scores) {
  using R = Kv4<D>;
  constexpr int kLanes = D / 8;
  const int64_t t = blockIdx.x;
  Place p;
  if (!locate(a, t, p)) return;
  const int lane = threadIdx.x & 63;
  const int units = 2 * a.Hkv;
  for (int u = threadIdx.x / kLanes; u < (units + 7) / 8 * 8; u += blockDim.x / kLanes) {
    // (lanes of a wave stay together: the lane moves below need all of a group)
    const bool live = u < units;
    const int uu = live ? u : 0;
    const bool is_v = uu >= a.Hkv;
    const int h = is_v ? uu - a.Hkv : uu;
    const int c = threadIdx.x % kLanes;  // dimensions 8 c ..
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
    // scale: in 64 bits, rounded to float and then to the type.  A group that holds what is
    // not finite reads back as NaN.
    uint32_t sb = E::from_f32(static_cast<float>((double(hi) - double(lo)) / 15.0));
    uint32_t mb = E::from_f32(lo);
    if (bad != 0.f) {
      sb = 0;
      mb = E::kNaN;
    }
    const double s = E::to_f32(sb), least = lo;
    const double inv = s > 0.0 ? 1.0 / s : 0.0;
    uint32_t n[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] = s > 0.0 ? uint32_t(nearest_code(double(f[e]) - least, s, inv)) : 0u;
    unsigned char* rec = a.cache + (p.page * a.Hkv + h) * R::kRecord;
    const int g = c >> 3;
    if (!is_v) {
      const uint32_t w = n[0] | n[2] << 4 | n[4] << 8 | n[6] << 12 | n[1] << 16 | n[3] << 20 | n[5] << 24 | n[7] << 28;
      if (live) reinterpret_cast<uint32_t*>(rec)[R::k_word(p.slot, c)] = w;
    } else if (live) {
      uint16_t* w = reinterpret_cast<uint16_t*>(rec + R::kV);
      const int m = (c & 7) * 2;
      w[R::v_half(p.slot, g, m)] = uint16_t(n[0] | n[1] << 4 | n[2] << 8 | n[3] << 12);
      w[R::v_half(p.slot, g, m + 1)] = uint16_t(n[4] | n[5] << 4 | n[6] << 8 | n[7] << 12);
    }
    if (live && (c & 7) == 0)
      reinterpret_cast<uint32_t*>(rec + (is_v ? R::kMetaV : R::kMetaK))[p.slot * R::kG + g] = sb | mb << 16;
    if (scores && live && !is_v && c == 0) scores[(p.page * a.Hkv + h) * kPage + p.slot] = 0.f;
  }
  (void)lane;
}

// The values of the call's tokens, dense [T, Hkv, D]: one workgroup per token, D / 8 lanes
// per head of K or V.  Tokens that are nowhere in the cache give 0.
template <class E, int D>
__global__ void __launch_bounds__(256)
kv4_read_kernel(Kv4Tokens a, unsigned char* __restrict__ k, unsigned char* __restrict__ v) {
  using R = Kv4<D>;
  constexpr int kLanes = D / 8;
  const int64_t t = blockIdx.x;
  Place p{0, 0};
  const bool there = locate(a, t, p);
  for (int u = threadIdx.x / kLanes; u < 2 * a.Hkv; u += blockDim.x / kLanes) {
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
// Eviction: one workgroup per (sequence, head).  The budget-th largest score is found by a
// radix selection over the scores' bits (8 at a time, counts in LDS), then the kept tokens
// are numbered in their order by a sum over the workgroup, and moved to the front a batch of
// pages at a time: a token only ever moves forward, so once a batch's tokens have all been
// read, writing them touches nothing that a later batch reads.
// ---------------------------------------------------------------------------------------

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;

// A float's place in ascending order; -0 as 0, every NaN as one value above infinity.
__device__ __forceinline__ uint32_t order_key(float f) {
  uint32_t b = __float_as_uint(f);
  if (b == 0x80000000u) b = 0;
  if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <int D>
__global__ void __launch_bounds__(kEvictThreads)
kv4_evict_kernel(Kv4Evict a) {
  using R = Kv4<D>;
  __shared__ uint32_t hist[256];
  __shared__ uint32_t wave_sum[2][kEvictWaves];
  __shared__ uint32_t pick[3];  // digit, what is left to take in it
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / a.Hkv, h = blockIdx.x % a.Hkv;
  const int64_t cap = a.cols * kPage;
  const int len = int(min(int64_t(max(a.lens[b], 0)), cap));
  const int budget = a.budget;
  int32_t* kept = a.kept + (int64_t(b) * a.Hkv + h) * budget;
  const int now = min(len, budget);
  if (h == 0 && tid == 0) a.new_lens[b] = now;
  for (int i = now + tid; i < budget; i += kEvictThreads) kept[i] = -1;
  if (len <= budget) {
    for (int i = tid; i < len; i += kEvictThreads) kept[i] = i;
    return;
  }
  const int32_t* table = a.table + int64_t(b) * a.cols;
  auto key_of = [&](int i) -> uint32_t {
    const int64_t page = table[i / kPage];
    return page < 0 || page >= a.num_blocks ? 0u : order_key(a.scores[(page * a.Hkv + h) * kPage + i % kPage]);
  };
  const int recent = min(a.recent, budget);
  const int old = len - recent;           // candidates
  const int take = budget - recent;       // of them to keep
  // threshold: the take-th largest key, and how many equal to it are kept
  uint32_t prefix = 0, left = uint32_t(take);
  if (take > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < old; i += kEvictThreads) {
        const uint32_t key = key_of(i);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (wave == 0) {
        // lane l has the counts of digits 255 - 4 l .. 252 - 4 l; digits from the top down
        uint32_t n[4], mine = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          n[e] = hist[255 - 4 * lane - e];
          mine += n[e];
        }
        uint32_t above = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const uint32_t o = __shfl_up(above, d);
          if (lane >= d) above += o;
        }
        above -= mine;  // counts of the digits above this lane's
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (above < left && above + n[e] >= left) {
            pick[0] = uint32_t(255 - 4 * lane - e);
            pick[1] = left - above;
          }
          above += n[e];
        }
      }
      __syncthreads();
      prefix |= pick[0] << shift;
      left = pick[1];
      __syncthreads();
    }
  }
  // the kept tokens in order: of those equal to the threshold the first `left`
  int base = 0;
  uint32_t ties = 0;
  for (int i0 = 0; i0 < old && take > 0; i0 += kEvictThreads) {
    const int i = i0 + tid;
    const uint32_t key = i < old ? key_of(i) : 0u;
    const bool more = i < old && key > prefix, tie = i < old && key == prefix;
    const uint64_t bm = __ballot(more), bt = __ballot(tie);
    const uint64_t below = (1ull << lane) - 1;
    if (lane == 0) {
      wave_sum[0][wave] = __popcll(bm);
      wave_sum[1][wave] = __popcll(bt);
    }
    __syncthreads();
    uint32_t m0 = 0, t0 = 0, mall = 0, tall = 0;
#pragma unroll
    for (int w = 0; w < kEvictWaves; ++w) {
      if (w < wave) {
        m0 += wave_sum[0][w];
        t0 += wave_sum[1][w];
      }
      mall += wave_sum[0][w];
      tall += wave_sum[1][w];
    }
    const uint32_t tbefore = ties + t0 + __popcll(bt & below);    // ties before this one
    const uint32_t mbefore = m0 + __popcll(bm & below);
    const bool keep = more || (tie && tbefore < left);
    // tokens kept before this one: the larger ones, and the ties taken before it
    const uint32_t at = uint32_t(base) + mbefore + (min(tbefore, left) - min(ties, left));
    if (keep && at < uint32_t(budget)) kept[at] = i;
    base += int(mall + min(ties + tall, left) - min(ties, left));
    ties += tall;
    __syncthreads();
  }
  for (int i = tid; i < recent; i += kEvictThreads) kept[take + i] = old + i;
  __threadfence_block();
  __syncthreads();

  // move: kPages pages a wave and batch, whole batch read before any of it is written
  constexpr int kPages = 2;
  constexpr int kW = D / 32;  // words of a lane's codes of one page
  const int pages = (budget + kPage - 1) / kPage;
  const int row = lane & 15, quad = lane >> 4;
  for (int p0 = 0; p0 < pages; p0 += kEvictWaves * kPages) {
    uint32_t kc[kPages][kW], vc[kPages][kW], meta[kPages];
    float sc[kPages];
    bool ok_k[kPages];
    uint32_t ok_v[kPages];
#pragma unroll
    for (int j = 0; j < kPages; ++j) {
      const int p = p0 + j * kEvictWaves + wave;
      auto source = [&](int slot, int64_t& page) -> int {  // token kept at this place of the page, or -1
        const int at = p * kPage + slot;
        const int i = at < budget ? kept[at] : -1;
        page = i < 0 ? -1 : table[i / kPage];
        return page >= 0 && page < a.num_blocks ? i % kPage : -1;
      };
      int64_t page;
      // K: this lane's quarter of token `row`
      int from = source(row, page);
      ok_k[j] = from >= 0;
      meta[j] = 0;
      sc[j] = 0.f;
#pragma unroll
      for (int e = 0; e < kW; ++e) kc[j][e] = 0;
      if (from >= 0) {
        const unsigned char* rec = a.cache + (page * a.Hkv + h) * R::kRecord;
        const uint32_t* w = reinterpret_cast<const uint32_t*>(rec) + (quad * 16 + from) * kW;
#pragma unroll
        for (int e = 0; e < kW; ++e) kc[j][e] = w[e];
        // scale and least: quarter g of K, quarter 2 + g of V; the score: quarter 3 or 1
        const int g = quad & 1;
        if (g < R::kG)
          meta[j] = reinterpret_cast<const uint32_t*>(rec + (quad < 2 ? R::kMetaK : R::kMetaV))[from * R::kG + g];
        if (quad == 0) sc[j] = a.scores[(page * a.Hkv + h) * kPage + from];
      }
      // V: tokens 4 quad .. 4 quad + 3, column block m = row
      ok_v[j] = 0;
      uint16_t hv[4][R::kG];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int f = source(4 * quad + r, page);
#pragma unroll
        for (int g = 0; g < R::kG; ++g) hv[r][g] = 0;
        if (f >= 0) {
          const uint16_t* w = reinterpret_cast<const uint16_t*>(a.cache + (page * a.Hkv + h) * R::kRecord + R::kV);
#pragma unroll
          for (int g = 0; g < R::kG; ++g) hv[r][g] = w[R::v_half(f, g, row)];
          ok_v[j] |= 1u << r;
        }
      }
#pragma unroll
      for (int e = 0; e < kW; ++e) {
        if (R::kG == 2) vc[j][e] = hv[e][0] | uint32_t(hv[e][R::kG - 1]) << 16;
        else vc[j][e] = hv[2 * e][0] | uint32_t(hv[2 * e + 1][0]) << 16;
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPages; ++j) {
      const int p = p0 + j * kEvictWaves + wave;
      if (p >= pages) continue;
      const int64_t page = table[p];
      if (page < 0 || page >= a.num_blocks) continue;
      unsigned char* rec = a.cache + (page * a.Hkv + h) * R::kRecord;
      if (ok_k[j]) {
        uint32_t* w = reinterpret_cast<uint32_t*>(rec) + (quad * 16 + row) * kW;
#pragma unroll
        for (int e = 0; e < kW; ++e) w[e] = kc[j][e];
        const int g = quad & 1;
        if (g < R::kG)
          reinterpret_cast<uint32_t*>(rec + (quad < 2 ? R::kMetaK : R::kMetaV))[row * R::kG + g] = meta[j];
        if (quad == 0) a.scores[(page * a.Hkv + h) * kPage + row] = sc[j];
      }
      uint16_t* w = reinterpret_cast<uint16_t*>(rec + R::kV);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (ok_v[j] >> r & 1) {
#pragma unroll
          for (int g = 0; g < R::kG; ++g) {
            const uint32_t x = R::kG == 2 ? vc[j][r % kW] >> (16 * g) : vc[j][(r / 2) % kW] >> (16 * (r & 1));
            w[R::v_half(4 * quad + r, g, row)] = uint16_t(x);
          }
        }
    }
    __syncthreads();
  }
}

}  // namespace

hipError_t launch_kv4_write(const Kv4Tokens& a, const unsigned char* k, const unsigned char* v, int64_t k_ts,
                            int64_t k_hs, int64_t v_ts, int64_t v_hs, float* scores, int D, int fp16,
                            hipStream_t stream) {
  const dim3 g{unsigned(a.T)}, t(256);
#define MQK_WRITE(E, DD) hipLaunchKernelGGL((kv4_write_kernel<E, DD>), g, t, 0, stream, a, k, v, k_ts, k_hs, v_ts, v_hs, scores)
  if (fp16) {
    if (D == 128) MQK_WRITE(KvFp16, 128);
    else MQK_WRITE(KvFp16, 64);
  } else {
    if (D == 128) MQK_WRITE(KvBf16, 128);
    else MQK_WRITE(KvBf16, 64);
  }
#undef MQK_WRITE
  return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4Tokens& a, unsigned char* k, unsigned char* v, int D, int fp16, hipStream_t stream) {
  const dim3 g{unsigned(a.T)}, t(256);
  if (fp16) {
    if (D == 128) hipLaunchKernelGGL((kv4_read_kernel<KvFp16, 128>), g, t, 0, stream, a, k, v);
    else hipLaunchKernelGGL((kv4_read_kernel<KvFp16, 64>), g, t, 0, stream, a, k, v);
  } else {
    if (D == 128) hipLaunchKernelGGL((kv4_read_kernel<KvBf16, 128>), g, t, 0, stream, a, k, v);
    else hipLaunchKernelGGL((kv4_read_kernel<KvBf16, 64>), g, t, 0, stream, a, k, v);
  }
  return hipGetLastError();
}

hipError_t launch_kv4_evict(const Kv4Evict& a, int64_t n_seqs, int D, hipStream_t stream) {
  const dim3 g(unsigned(n_seqs * a.Hkv)), t(kEvictThreads);
  if (D == 128) hipLaunchKernelGGL(kv4_evict_kernel<128>, g, t, 0, stream, a);
  else hipLaunchKernelGGL(kv4_evict_kernel<64>, g, t, 0, stream, a);
  return hipGetLastError();
}

}  // namespace mqk
