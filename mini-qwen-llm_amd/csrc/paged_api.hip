// C ABI of the operators around the bf16 / fp16 paged cache: argument validation and launch.
// Declarations and the contract of every entry point: include/mqk.h.
#include "../../include/mqk.h"
#include "mqk_attn.h"
#include "mqk_kernels.h"
#include "mqk_paged.h"
#include "mqk_status.h"

#include <algorithm>

using namespace mqk;

namespace {

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kMostScale = 3e38f / kLog2e;   // whose product with log2(e) is finite
constexpr int64_t kMostTokens = 0x7FFF0000ll;  // tile arithmetic stays inside 32 bits

// Whether n bytes at a and m bytes at b have one in common.
bool meet(const void* a, int64_t n, const void* b, int64_t m) {
  if (!a || !b || n <= 0 || m <= 0) return false;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + uintptr_t(m) && y < x + uintptr_t(n);
}

// The sizes of a cache and of the tables into it (its pointers are the entry points' matter).
int check_cache(const mqk_paged_cache* c) {
  if (!c) return fail(MQK_ERR_NULL_POINTER, "cache descriptor is NULL");
  if (c->dtype != MQK_BF16 && c->dtype != MQK_F16) return fail(MQK_ERR_UNSUPPORTED, "cache dtype %d: bf16 or fp16", c->dtype);
  if (c->D <= 0 || c->D % 8 != 0 || c->D > 256) return fail(MQK_ERR_UNSUPPORTED, "head_dim %d: a multiple of 8 up to 256", c->D);
  if (c->Hkv <= 0 || c->Hkv > 4096) return fail(MQK_ERR_BAD_SHAPE, "Hkv = %d out of range", c->Hkv);
  if (c->page <= 0 || c->page % 8 != 0 || c->page > (1 << 20))
    return fail(MQK_ERR_UNSUPPORTED, "page of %d tokens: a multiple of 8", c->page);
  if (c->num_blocks <= 0 || c->bt_cols <= 0 || c->num_blocks > kMostTokens / c->page || c->bt_cols > kMostTokens / c->page)
    return fail(MQK_ERR_BAD_SHAPE, "num_blocks = %lld, bt_cols = %lld out of range", (long long)c->num_blocks,
                (long long)c->bt_cols);
  if (c->n_seqs < 0 || c->n_seqs > (1 << 20)) return fail(MQK_ERR_BAD_SHAPE, "n_seqs = %lld out of range", (long long)c->n_seqs);
  return MQK_OK;
}
int check_tokens(const mqk_paged_cache* c, const int32_t* cu, int64_t T) {
  if (T < 0 || T > kMostTokens) return fail(MQK_ERR_BAD_SHAPE, "T = %lld out of range", (long long)T);
  if (T > 0 && c->n_seqs == 0) return fail(MQK_ERR_BAD_SHAPE, "tokens of no sequence");
  if (!cu && T > 0 && T % c->n_seqs != 0)
    return fail(MQK_ERR_BAD_SHAPE, "without cu_seqlens, T must be a multiple of n_seqs = %lld", (long long)c->n_seqs);
  return MQK_OK;
}
int check_heads(const mqk_paged_cache* c, int Hq) {
  if (Hq <= 0 || Hq % c->Hkv != 0 || Hq > 65536)
    return fail(MQK_ERR_BAD_SHAPE, "Hq = %d must be a positive multiple of Hkv = %d", Hq, c->Hkv);
  return MQK_OK;
}
// q's data and strides (elements): whole 16-byte chunks.
int check_q(const mqk_attn_tensor* q, int64_t T, int Hq) {
  if (!q->data) return fail(MQK_ERR_NULL_POINTER, "q is NULL");
  if (!aligned16(q->data) || (T > 1 && q->token_stride % 8 != 0) || (Hq > 1 && q->head_stride % 8 != 0))
    return fail(MQK_ERR_MISALIGNED, "q must be 16-byte aligned, its strides multiples of 16 bytes");
  return MQK_OK;
}

int attn_shape(const mqk_paged_cache* c, int64_t T, int Hq, const int32_t* cu, int64_t n_pages) {
  if (int st = check_cache(c); st != MQK_OK) return st;
  if (int st = check_heads(c, Hq); st != MQK_OK) return st;
  if (int st = check_tokens(c, cu, T); st != MQK_OK) return st;
  if (n_pages < 0 || n_pages > kMostTokens / c->page)
    return fail(MQK_ERR_BAD_SHAPE, "n_pages = %lld out of range", (long long)n_pages);
  if ((c->bt_cols * c->page / 64 + 2) * c->Hkv > 0x7FFFFFFFll)  // (the steps of a sequence, in 32 bits)
    return fail(MQK_ERR_BAD_SHAPE, "block tables of %lld tokens for %d heads: too many", (long long)(c->bt_cols * c->page), c->Hkv);
  if (T * Hq > 0x3FFFFFFFll) return fail(MQK_ERR_BAD_SHAPE, "T = %lld tokens of %d heads: too many", (long long)T, Hq);
  return MQK_OK;
}
PagedPlan plan_of(const mqk_paged_cache* c, int64_t T, int Hq, bool cu, int64_t n_pages) {
  return plan_paged_attn(T, c->n_seqs, cu, c->bt_cols, c->page, n_pages, Hq, c->Hkv, c->D, device_topology().cus);
}

}  // namespace

extern "C" {

int mqk_paged_tables(const int32_t* seq_lens, const int32_t* new_lens, int64_t n_seqs, int32_t* block_table,
                     int64_t bt_cols, const int32_t* free_pages, int64_t n_free, const int32_t* cursor, int page,
                     int64_t n_tokens, int32_t* lens, int32_t* cu_seqlens, int32_t* kv_seq, int32_t* kv_pos,
                     int64_t* slots, int32_t* taken, void* stream) {
  if (n_seqs <= 0 || n_seqs > kTablesMostSeqs)
    return fail(MQK_ERR_BAD_SHAPE, "n_seqs = %lld: 1 to %d", (long long)n_seqs, kTablesMostSeqs);
  if (page <= 0 || page > (1 << 20)) return fail(MQK_ERR_BAD_SHAPE, "page of %d tokens out of range", page);
  if (bt_cols <= 0 || bt_cols > kMostTokens || n_free < 0 || n_free > 0x7FFFFFFFll)
    return fail(MQK_ERR_BAD_SHAPE, "bt_cols = %lld, n_free = %lld out of range", (long long)bt_cols, (long long)n_free);
  if (n_tokens < 0 || n_tokens > kMostTokens) return fail(MQK_ERR_BAD_SHAPE, "n_tokens = %lld out of range", (long long)n_tokens);
  if (!seq_lens || !new_lens || !block_table || (n_free > 0 && !free_pages) || !lens || !cu_seqlens || !taken ||
      (n_tokens > 0 && (!kv_seq || !kv_pos || !slots)))
    return fail(MQK_ERR_NULL_POINTER, "a required pointer is NULL");
  // (workgroups read all lengths while others write: what is written overlaps nothing else)
  const struct {
    const void* at;
    int64_t bytes;
  } out[7] = {{block_table, n_seqs * bt_cols * 4}, {lens, n_seqs * 4},      {cu_seqlens, (n_seqs + 1) * 4}, {taken, 4},
              {kv_seq, n_tokens * 4},              {kv_pos, n_tokens * 4}, {slots, n_tokens * 8}},
    in[4] = {{seq_lens, n_seqs * 4}, {new_lens, n_seqs * 4}, {free_pages, n_free * 4}, {cursor, 4}};
  for (int i = 0; i < 7; ++i) {
    for (const auto& r : in)
      if (meet(out[i].at, out[i].bytes, r.at, r.bytes)) return fail(MQK_ERR_BAD_SHAPE, "what is written must not overlap what is read");
    for (int j = 0; j < i; ++j)
      if (meet(out[i].at, out[i].bytes, out[j].at, out[j].bytes)) return fail(MQK_ERR_BAD_SHAPE, "outputs must not overlap each other");
  }
  PagedTables a{};
  a.old_lens = seq_lens;
  a.new_lens = new_lens;
  a.table = block_table;
  a.free_pages = free_pages;
  a.cursor = cursor;
  a.lens = lens;
  a.cu = cu_seqlens;
  a.kv_seq = kv_seq;
  a.kv_pos = kv_pos;
  a.slots = slots;
  a.taken = taken;
  a.cols = bt_cols;
  a.n_free = n_free;
  a.n_tokens = n_tokens;
  a.n_seqs = int(n_seqs);
  a.page = page;
  return hip_status(launch_paged_tables(a, device_topology().cus, static_cast<hipStream_t>(stream)),
                    "paged_tables kernel launch");
}

size_t mqk_paged_attn_workspace_size(const mqk_paged_cache* cache, int64_t T, int Hq, int with_cu, int64_t n_pages) {
  static const int32_t some = 0;
  if (attn_shape(cache, T, Hq, with_cu ? &some : nullptr, n_pages) != MQK_OK || T == 0) return 0;
  const size_t n = plan_of(cache, T, Hq, with_cu != 0, n_pages).bytes;
  return n ? kDecodeCounterBytes + n : 0;
}

int mqk_paged_attn(const mqk_attn_tensor* q, const mqk_paged_cache* cache, const int32_t* seq_lens,
                   const int32_t* cu_seqlens, int64_t T, int Hq, float scale, const int32_t* pages, int64_t n_pages,
                   int fill, void* out, void* workspace, size_t ws_bytes, void* stream) {
  if (!q) return fail(MQK_ERR_NULL_POINTER, "q descriptor is NULL");
  if (int st = attn_shape(cache, T, Hq, cu_seqlens, n_pages); st != MQK_OK) return st;
  if (!(scale > 0.f) || scale > kMostScale) return fail(MQK_ERR_BAD_SHAPE, "scale must be positive, and finite times log2(e)");
  if ((pages != nullptr) != (n_pages > 0)) return fail(MQK_ERR_BAD_SHAPE, "pages and n_pages belong together");
  if (T == 0) return ok();
  if (!cache->k || !cache->v || !cache->block_table || !seq_lens || !out)
    return fail(MQK_ERR_NULL_POINTER, "k, v, block_table, seq_lens or out is NULL");
  if (int st = check_q(q, T, Hq); st != MQK_OK) return st;
  if (!aligned16(cache->k) || !aligned16(cache->v) || !aligned16(out))
    return fail(MQK_ERR_MISALIGNED, "k, v and out must be 16-byte aligned");
  PagedAttn a{};
  a.q = static_cast<const unsigned char*>(q->data);
  a.k = static_cast<const unsigned char*>(cache->k);
  a.v = static_cast<const unsigned char*>(cache->v);
  a.out = static_cast<unsigned char*>(out);
  a.q_ts = q->token_stride * 2;
  a.q_hs = q->head_stride * 2;
  a.table = cache->block_table;
  a.lens = seq_lens;
  a.cu = cu_seqlens;
  a.pages = pages;
  a.T = T;
  a.each = cu_seqlens ? 0 : T / cache->n_seqs;
  a.cols = cache->bt_cols;
  a.num_blocks = cache->num_blocks;
  a.n_pages = n_pages;
  a.n_seqs = int(cache->n_seqs);
  a.Hq = Hq;
  a.Hkv = cache->Hkv;
  a.G = Hq / cache->Hkv;
  a.D = cache->D;
  a.page = cache->page;
  a.page8 = divide_by(uint32_t(cache->page / 8));
  a.scale = scale * kLog2e;
  a.fill = fill;
  const PagedPlan p = plan_of(cache, T, Hq, cu_seqlens != nullptr, n_pages);
  if (std::max(p.few, p.many) > kMostThreads / 512) return fail(MQK_ERR_BAD_SHAPE, "too much work for one call");
  a.few_rows = p.few_rows;
  a.rows = p.rows;
  a.parts = p.parts;
  a.part_steps = p.part_steps;
  a.slots = p.slots;
  a.most_split = p.most_split;
  a.whole = p.whole;
  std::unique_lock<std::recursive_mutex> lock;
  if (p.bytes) {
    if (!workspace || ws_bytes < kDecodeCounterBytes + p.bytes)
      return fail(MQK_ERR_WORKSPACE, "needs a workspace of %zu bytes", kDecodeCounterBytes + p.bytes);
    if (!aligned16(workspace)) return fail(MQK_ERR_MISALIGNED, "workspace must be 16-byte aligned");
    // (behind the counters that the projection's kernels keep at zero)
    unsigned char* ws = static_cast<unsigned char*>(workspace) + kDecodeCounterBytes;
    a.n_split = reinterpret_cast<int64_t*>(ws + p.n_split);
    auto out = [&](const PagedPlan::Room& r) {
      return PagedOut{reinterpret_cast<PagedJoin*>(ws + r.joins), reinterpret_cast<float*>(ws + r.ml),
                      reinterpret_cast<float*>(ws + r.part)};
    };
    a.few = out(p.few_room);
    a.many = out(p.many_room);
    lock = handover_lock(workspace);
  }
  return hip_status(launch_paged_attn(a, p, cache->dtype == MQK_F16, static_cast<hipStream_t>(stream)),
                    "paged_attn kernel launch");
}

int mqk_paged_bounds(const mqk_paged_cache* cache, const int32_t* seq_lens, const int32_t* cu_seqlens, int64_t T,
                     void* bounds, void* stream) {
  if (int st = check_cache(cache); st != MQK_OK) return st;
  const bool whole = T == -1;
  if (whole && cu_seqlens) return fail(MQK_ERR_BAD_SHAPE, "whole sequences (T = -1) have no cu_seqlens");
  if (!whole)
    if (int st = check_tokens(cache, cu_seqlens, T); st != MQK_OK) return st;
  if (T == 0 || cache->n_seqs == 0) return ok();
  if (!cache->k || !cache->block_table || !seq_lens || !bounds)
    return fail(MQK_ERR_NULL_POINTER, "k, block_table, seq_lens or bounds is NULL");
  if (!aligned16(cache->k) || !aligned16(bounds)) return fail(MQK_ERR_MISALIGNED, "k and bounds must be 16-byte aligned");
  PagedBounds a{};
  a.k = static_cast<const unsigned char*>(cache->k);
  a.bounds = static_cast<unsigned char*>(bounds);
  a.table = cache->block_table;
  a.lens = seq_lens;
  a.cu = cu_seqlens;
  a.T = T;
  a.each = whole || cu_seqlens ? 0 : T / cache->n_seqs;
  a.cols = cache->bt_cols;
  a.num_blocks = cache->num_blocks;
  a.n_seqs = int(cache->n_seqs);
  a.Hkv = cache->Hkv;
  a.D = cache->D;
  a.page = cache->page;
  const hipError_t err = launch_paged_bounds(a, cache->dtype == MQK_F16, static_cast<hipStream_t>(stream));
  if (err == hipErrorInvalidConfiguration) return fail(MQK_ERR_BAD_SHAPE, "too much work for one call");
  return hip_status(err, "paged_bounds kernel launch");
}

size_t mqk_paged_select_workspace_size(const mqk_paged_cache* cache, int64_t T) {
  if (check_cache(cache) != MQK_OK || T <= 0 || T > kMostTokens / cache->Hkv) return 0;
  return kDecodeCounterBytes + size_t(select_round(T, cache->Hkv, cache->bt_cols)) * cache->Hkv * cache->bt_cols * 8;
}

int mqk_paged_select(const mqk_attn_tensor* q, const void* bounds, const mqk_paged_cache* cache, const int32_t* seq_lens,
                     const int32_t* cu_seqlens, int64_t T, int Hq, int64_t n_pages, int first, int recent, int32_t* pages,
                     void* workspace, size_t ws_bytes, void* stream) {
  if (!q) return fail(MQK_ERR_NULL_POINTER, "q descriptor is NULL");
  if (int st = check_cache(cache); st != MQK_OK) return st;
  if (int st = check_heads(cache, Hq); st != MQK_OK) return st;
  if (int st = check_tokens(cache, cu_seqlens, T); st != MQK_OK) return st;
  if (n_pages <= 0 || n_pages > (1 << 24) || first < 0 || recent < 1 || int64_t(first) + recent > n_pages)
    return fail(MQK_ERR_BAD_SHAPE, "first = %d and recent = %d (1 at least) must fit n_pages = %lld", first, recent,
                (long long)n_pages);
  if (T == 0) return ok();
  if (!bounds || !cache->block_table || !seq_lens || !pages)
    return fail(MQK_ERR_NULL_POINTER, "bounds, block_table, seq_lens or pages is NULL");
  if (int st = check_q(q, T, Hq); st != MQK_OK) return st;
  if (!aligned16(bounds)) return fail(MQK_ERR_MISALIGNED, "bounds must be 16-byte aligned");
  if (T * cache->Hkv > kMostThreads / 1024) return fail(MQK_ERR_BAD_SHAPE, "too much work for one call");
  const size_t need = mqk_paged_select_workspace_size(cache, T);
  if (!workspace || ws_bytes < need) return fail(MQK_ERR_WORKSPACE, "needs a workspace of %zu bytes", need);
  if (!aligned16(workspace)) return fail(MQK_ERR_MISALIGNED, "workspace must be 16-byte aligned");
  PagedSelect a{};
  a.q = static_cast<const unsigned char*>(q->data);
  a.bounds = static_cast<const unsigned char*>(bounds);
  a.q_ts = q->token_stride * 2;
  a.q_hs = q->head_stride * 2;
  a.table = cache->block_table;
  a.lens = seq_lens;
  a.cu = cu_seqlens;
  a.pages = pages;
  a.keys = reinterpret_cast<uint64_t*>(static_cast<unsigned char*>(workspace) + kDecodeCounterBytes);
  a.T = T;
  a.each = cu_seqlens ? 0 : T / cache->n_seqs;
  a.cols = cache->bt_cols;
  a.num_blocks = cache->num_blocks;
  a.n_seqs = int(cache->n_seqs);
  a.Hq = Hq;
  a.Hkv = cache->Hkv;
  a.G = Hq / cache->Hkv;
  a.D = cache->D;
  a.page = cache->page;
  a.take = int(n_pages);
  a.first = first;
  a.recent = recent;
  const auto lock = handover_lock(workspace);
  return hip_status(launch_paged_select(a, cache->dtype == MQK_F16, device_topology().cus, static_cast<hipStream_t>(stream)),
                    "paged_select kernel launch");
}

}  // extern "C"
