// A step's block tables and slots from its requests' lengths.
//
// Sequence s has old[s] tokens and gets new[s] (what of them fits the call's n_tokens): with
// pages of P tokens it has ceil(old / P) pages and takes ceil((old + new) / P) less those from
// the list of free ones, in the order of the sequences.  So the place of a sequence's first
// new page in the list, and of its first token among the call's, are sums over the sequences
// before it, and everything else follows for each page and token by itself.
//
// Nothing here costs but latency (a few hundred KB at most): one launch, in which every
// workgroup makes the sums over all sequences for itself in LDS (a launch of its own for
// them would take longer than reading the lengths again), then writes its share of pages and
// tokens, each found by bisection among the sums.  A step of 48 sequences 4.8 us, 300 sequences
// with 8214 new tokens 7.3: loads, scans and bisections that wait for each other.
#include "mqk_device.h"
#include "mqk_paged.h"

#include <algorithm>

namespace mqk {
namespace {

// Sum over the threads before this one, and over all of the workgroup (WAVES waves).
template <int WAVES>
__device__ __forceinline__ int64_t scan_before(int64_t v, int64_t* lds, int64_t& all) {
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
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += lds[w];
    all += lds[w];
  }
  return before + x - v;
}

// The last of sums[0 .. n - 1] that is not above x (sums[0] is 0 or less than it).
__device__ __forceinline__ int last_not_above(const int32_t* sums, int n, int32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int THREADS, int EACH>
__global__ void __launch_bounds__(THREADS)
paged_tables_kernel(PagedTables a) {
  constexpr int kMost = THREADS * EACH;
  __shared__ int32_t token_at[kMost], page_at[kMost];
  __shared__ int64_t sums[THREADS / 64];
  const int tid = threadIdx.x;
  const bool first = blockIdx.x == 0;
  auto pages_of = [&](int32_t n) { return (uint32_t(n) + uint32_t(a.page) - 1) / uint32_t(a.page); };
  // --- sums over the sequences: thread i has EACH of them in a row
  auto counts = [&](int s, int32_t& old, int32_t& fresh) {  // tokens before, and new ones
    old = s < a.n_seqs ? max(a.old_lens[s], 0) : 0;
    fresh = s < a.n_seqs ? min(max(a.new_lens[s], 0), 0x7FFFFFFF - old) : 0;  // (a length stays within its type)
  };
  int32_t old, fresh;
  int64_t mine = 0, tokens, pages;
#pragma unroll 4
  for (int e = 0; e < EACH; ++e) {
    counts(tid * EACH + e, old, fresh);
    mine += fresh;
  }
  int64_t at = scan_before<THREADS / 64>(mine, sums, tokens);
  tokens = min(tokens, a.n_tokens);
  mine = 0;
#pragma unroll 4
  for (int e = 0; e < EACH; ++e) {
    const int s = tid * EACH + e;
    counts(s, old, fresh);
    const int64_t from = min(at, a.n_tokens);
    at += fresh;
    fresh = int32_t(min(at, a.n_tokens) - from);
    const int32_t want = max(0, int(min(int64_t(pages_of(old + fresh)), a.cols)) - int(pages_of(old)));
    mine += want;
    token_at[s] = s < a.n_seqs ? int32_t(from) : 0x7FFFFFFF;
    page_at[s] = want;
    if (first && s < a.n_seqs) {
      a.lens[s] = old + fresh;
      a.cu[s] = int32_t(from);
    }
  }
  int64_t page = scan_before<THREADS / 64>(mine, sums, pages);
#pragma unroll 4
  for (int e = 0; e < EACH; ++e) {
    const int s = tid * EACH + e;
    const int32_t want = page_at[s];
    page_at[s] = s < a.n_seqs ? int32_t(min(page, int64_t(0x7FFFFFFF))) : 0x7FFFFFFF;
    page += want;
  }
  const int64_t cursor = a.cursor ? max(a.cursor[0], 0) : 0;
  if (first && tid == 0) {
    a.cu[a.n_seqs] = int32_t(tokens);
    a.taken[0] = int32_t(min(cursor + pages, int64_t(0x7FFFFFFF)));
  }
  __syncthreads();
  auto free_page = [&](int64_t i) { return cursor + i < a.n_free ? a.free_pages[cursor + i] : -1; };
  const int64_t step = int64_t(gridDim.x) * THREADS, self = int64_t(blockIdx.x) * THREADS + tid;
  // --- the new pages' entries
  const int64_t fit = min(pages, int64_t(0x7FFFFFFF));
  for (int64_t i = self; i < fit; i += step) {
    const int s = last_not_above(page_at, a.n_seqs, int32_t(i));
    a.table[s * a.cols + pages_of(max(a.old_lens[s], 0)) + (i - page_at[s])] = free_page(i);
  }
  // --- the tokens
  for (int64_t t = self; t < a.n_tokens; t += step) {
    int seq = -1, pos = -1;
    int64_t slot = -1;
    if (t < tokens) {
      seq = last_not_above(token_at, a.n_seqs, int32_t(t));
      const int32_t have = max(a.old_lens[seq], 0);
      pos = have + int32_t(t - token_at[seq]);
      const uint32_t j = uint32_t(pos) / uint32_t(a.page), has = pages_of(have);
      if (j < a.cols) {
        const int32_t id = j < has ? a.table[seq * a.cols + j] : free_page(page_at[seq] + (j - has));
        if (id >= 0) slot = int64_t(id) * a.page + (uint32_t(pos) - j * uint32_t(a.page));
      }
    }
    a.kv_seq[t] = seq;
    a.kv_pos[t] = pos;
    a.slots[t] = slot;
  }
}

}  // namespace

// A workgroup for every 512 tokens and pages there may be, up to one a CU.
hipError_t launch_paged_tables(const PagedTables& a, int cus, hipStream_t stream) {
  const int64_t items = a.n_tokens + a.n_tokens / a.page + a.n_seqs;
  const unsigned grid = unsigned(std::min<int64_t>(std::max<int64_t>((items + 511) / 512, 1), cus));
  if (a.n_seqs <= 1024) hipLaunchKernelGGL((paged_tables_kernel<256, 4>), dim3(grid), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((paged_tables_kernel<1024, 16>), dim3(grid), dim3(1024), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mqk
