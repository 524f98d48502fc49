// C ABI of the attention operators behind the projection front: argument validation and
// launch.  Declarations and the contract of every entry point: include/mqk.h.
#include "../../include/mqk.h"
#include "mqk_attn.h"
#include "mqk_kernels.h"
#include "mqk_status.h"

#include <algorithm>

using namespace mqk;

std::atomic<int64_t> mqk::g_attn_split{0}, mqk::g_attn_parts{0};

namespace {

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

constexpr float kLog2e = 1.44269504088896340736f;
// The largest scale whose product with log2(e) is finite; the decode kernel's with 16 more.
constexpr float kMostScale = 3e38f / kLog2e;
constexpr int64_t kMostTokens = 0x7FFF0000ll;  // tile arithmetic stays inside 32 bits

// A head's stride and a token's (elements): whole 16-byte chunks, or the tensor is not
// read at all with that stride.
bool chunked(int64_t stride, int64_t count, int bytes) { return count <= 1 || stride * bytes % 16 == 0; }

// Whether n bytes at a and m bytes at b have one in common.
bool meet(const void* a, int64_t n, const void* b, int64_t m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + uintptr_t(m) && y < x + uintptr_t(n);
}

// The descriptor every entry point of the 4-bit cache takes.
int check_cache(const mqk_kv4_cache* c) {
  if (!c || !c->cache || !c->block_table) return fail(MQK_ERR_NULL_POINTER, "cache or block_table is NULL");
  if (c->dtype != MQK_BF16 && c->dtype != MQK_F16) return fail(MQK_ERR_UNSUPPORTED, "cache dtype %d: bf16 or fp16", c->dtype);
  if (c->D != 64 && c->D != 128) return fail(MQK_ERR_UNSUPPORTED, "head_dim %d: 64 or 128", c->D);
  if (c->Hkv <= 0 || c->Hkv > 4096) return fail(MQK_ERR_BAD_SHAPE, "Hkv = %d out of range", c->Hkv);
  if (c->num_blocks <= 0 || c->num_blocks > 0x7FFFFFFFll || c->bt_cols <= 0 || c->bt_cols > 0x7FFFFFFFll / 32)
    return fail(MQK_ERR_BAD_SHAPE, "num_blocks = %lld, bt_cols = %lld out of range", (long long)c->num_blocks,
                (long long)c->bt_cols);
  if (c->n_seqs < 0 || c->n_seqs > (1 << 20)) return fail(MQK_ERR_BAD_SHAPE, "n_seqs = %lld out of range", (long long)c->n_seqs);
  if (!aligned16(c->cache)) return fail(MQK_ERR_MISALIGNED, "cache must be 16-byte aligned");
  return MQK_OK;
}

int tokens_of(const mqk_kv4_cache* c, const int32_t* seq_lens, const int32_t* cu, int64_t T, Kv4Tokens& a) {
  if (int st = check_cache(c); st != MQK_OK) return st;
  if (T < 0 || T > kMostTokens) return fail(MQK_ERR_BAD_SHAPE, "T = %lld out of range", (long long)T);
  // (more would be past any memory, and past 32 bits of workgroups)
  if (T * c->Hkv > 0x7FFFFFFFll) return fail(MQK_ERR_BAD_SHAPE, "T = %lld tokens of %d heads: too many", (long long)T, c->Hkv);
  if (T > 0 && c->n_seqs == 0) return fail(MQK_ERR_BAD_SHAPE, "tokens of no sequence");
  if (!cu && T > 0 && T % c->n_seqs != 0)
    return fail(MQK_ERR_BAD_SHAPE, "without cu_seqlens, T must be a multiple of n_seqs = %lld", (long long)c->n_seqs);
  if (T > 0 && !seq_lens) return fail(MQK_ERR_NULL_POINTER, "seq_lens is NULL");
  a.cache = static_cast<unsigned char*>(c->cache);
  a.table = c->block_table;
  a.lens = seq_lens;
  a.cu = cu;
  a.T = T;
  a.each = cu || T == 0 ? 0 : T / c->n_seqs;
  a.cols = c->bt_cols;
  a.num_blocks = c->num_blocks;
  a.n_seqs = int(c->n_seqs);
  a.Hkv = c->Hkv;
  return MQK_OK;
}

int attn_shape(const mqk_kv4_cache* c, int64_t S, int Hq) {
  if (int st = check_cache(c); st != MQK_OK) return st;
  if (S <= 0 || Hq <= 0 || Hq % c->Hkv != 0 || Hq > 65536)
    return fail(MQK_ERR_BAD_SHAPE, "Hq = %d must be a positive multiple of Hkv = %d, S = %lld positive", Hq, c->Hkv,
                (long long)S);
  if (S * Hq > (1 << 20) || c->n_seqs * S * Hq > 0x3FFFFFFFll)
    return fail(MQK_ERR_BAD_SHAPE, "S = %lld tokens of %lld sequences: too many rows for a decode call", (long long)S,
                (long long)c->n_seqs);
  return MQK_OK;
}

int prefill_shape(int dtype, int64_t T, int64_t Tk, int64_t n_seqs, int Hq, int Hkv, int D) {
  if (dtype != MQK_BF16 && dtype != MQK_F16 && dtype != MQK_F32)
    return fail(MQK_ERR_UNSUPPORTED, "dtype %d unknown", dtype);
  if (T < 0 || Tk < 0 || T > kMostTokens || Tk > kMostTokens)
    return fail(MQK_ERR_BAD_SHAPE, "T = %lld, Tk = %lld out of range", (long long)T, (long long)Tk);
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0)
    return fail(MQK_ERR_BAD_SHAPE, "Hq = %d must be a positive multiple of Hkv = %d", Hq, Hkv);
  if (D <= 0 || D % 8 != 0 || D > 256) return fail(MQK_ERR_UNSUPPORTED, "head_dim %d: a multiple of 8 up to 256", D);
  if (n_seqs <= 0 || n_seqs > (1 << 20)) return fail(MQK_ERR_BAD_SHAPE, "n_seqs = %lld out of range", (long long)n_seqs);
  return MQK_OK;
}

AttnPlan plan_of(int dtype, int64_t T, int64_t Tk, int64_t n_seqs, bool cu, int Hq, int D) {
  return plan_attn_prefill(dtype, T, Tk, n_seqs, cu, Hq, D, device_topology().cus, int(g_attn_split.load()),
                           int(g_attn_parts.load()));
}

}  // namespace

extern "C" {

int mqk_kv4_write(const mqk_attn_tensor* k, const mqk_attn_tensor* v, const mqk_kv4_cache* cache,
                  const int32_t* seq_lens, const int32_t* cu_seqlens, int64_t T, float* scores, void* stream) {
  if (!k || !v) return fail(MQK_ERR_NULL_POINTER, "k or v descriptor is NULL");
  Kv4Tokens a{};
  if (int st = tokens_of(cache, seq_lens, cu_seqlens, T, a); st != MQK_OK) return st;
  if (T == 0) return ok();
  if (!k->data || !v->data) return fail(MQK_ERR_NULL_POINTER, "k or v is NULL");
  if (!aligned16(k->data) || !aligned16(v->data) || !chunked(k->token_stride, T, 2) ||
      !chunked(k->head_stride, a.Hkv, 2) || !chunked(v->token_stride, T, 2) || !chunked(v->head_stride, a.Hkv, 2))
    return fail(MQK_ERR_MISALIGNED, "k and v must be 16-byte aligned, their strides multiples of 16 bytes");
  return hip_status(launch_kv4_write(a, static_cast<const unsigned char*>(k->data),
                                     static_cast<const unsigned char*>(v->data), k->token_stride * 2,
                                     k->head_stride * 2, v->token_stride * 2, v->head_stride * 2, scores, cache->D,
                                     cache->dtype == MQK_F16, static_cast<hipStream_t>(stream)),
                    "kv4_write kernel launch");
}

int mqk_kv4_read(const mqk_kv4_cache* cache, const int32_t* seq_lens, const int32_t* cu_seqlens, int64_t T, void* k,
                 void* v, void* stream) {
  Kv4Tokens a{};
  if (int st = tokens_of(cache, seq_lens, cu_seqlens, T, a); st != MQK_OK) return st;
  if (T == 0) return ok();
  if (!k || !v) return fail(MQK_ERR_NULL_POINTER, "k or v is NULL");
  if (!aligned16(k) || !aligned16(v)) return fail(MQK_ERR_MISALIGNED, "k and v must be 16-byte aligned");
  return hip_status(launch_kv4_read(a, static_cast<unsigned char*>(k), static_cast<unsigned char*>(v), cache->D,
                                    cache->dtype == MQK_F16, static_cast<hipStream_t>(stream)),
                    "kv4_read kernel launch");
}

size_t mqk_kv4_attn_workspace_size(const mqk_kv4_cache* cache, int64_t S, int Hq, int with_scores) {
  if (attn_shape(cache, S, Hq) != MQK_OK || cache->n_seqs == 0) return 0;
  const size_t n = plan_kv4_attn(int(cache->n_seqs), int(S), Hq, cache->Hkv, cache->D, cache->bt_cols, with_scores != 0,
                                 device_topology().cus)
                       .bytes;
  return n ? kDecodeCounterBytes + n : 0;
}

int mqk_kv4_attn(const void* q, const mqk_kv4_cache* cache, const int32_t* seq_lens, int64_t S, int Hq, float scale,
                 float* scores, void* out, void* workspace, size_t ws_bytes, void* stream) {
  if (int st = attn_shape(cache, S, Hq); st != MQK_OK) return st;
  if (!(scale > 0.f) || scale > kMostScale / 16.f) return fail(MQK_ERR_BAD_SHAPE, "scale must be positive, and finite times log2(e)");
  if (cache->n_seqs == 0) return ok();
  if (!q || !out || !seq_lens) return fail(MQK_ERR_NULL_POINTER, "q, seq_lens or out is NULL");
  if (!aligned16(q) || !aligned16(out)) return fail(MQK_ERR_MISALIGNED, "q and out must be 16-byte aligned");
  Kv4Attn a{};
  a.q = static_cast<const unsigned char*>(q);
  a.cache = static_cast<const unsigned char*>(cache->cache);
  a.table = cache->block_table;
  a.lens = seq_lens;
  a.out = static_cast<unsigned char*>(out);
  a.scores = scores;
  a.cols = cache->bt_cols;
  a.num_blocks = cache->num_blocks;
  a.B = int(cache->n_seqs);
  a.S = int(S);
  a.Hq = Hq;
  a.Hkv = cache->Hkv;
  a.G = Hq / cache->Hkv;
  a.RB = (a.S * a.G + 15) / 16;
  a.scale = scale * kLog2e;
  const Kv4Plan p = plan_kv4_attn(a.B, a.S, Hq, a.Hkv, cache->D, a.cols, scores != nullptr, device_topology().cus);
  if (std::max({p.grid, p.join, p.weigh}) > kMostThreads / 256 || (a.cols * 16 / 128 + 1) * a.Hkv * a.RB > 0x7FFFFFFFll)
    return fail(MQK_ERR_BAD_SHAPE, "too much work for one call");
  a.whole = p.whole;
  a.few = p.few;
  a.run = p.run;
  std::unique_lock<std::recursive_mutex> lock;
  if (p.bytes) {
    if (!workspace || ws_bytes < kDecodeCounterBytes + p.bytes)
      return fail(MQK_ERR_WORKSPACE, "needs a workspace of %zu bytes", kDecodeCounterBytes + p.bytes);
    if (!aligned16(workspace)) return fail(MQK_ERR_MISALIGNED, "workspace must be 16-byte aligned");
    // (behind the counters that the projection's kernels keep at zero)
    unsigned char* ws = static_cast<unsigned char*>(workspace) + kDecodeCounterBytes;
    if (scores) a.fin = reinterpret_cast<float*>(ws + p.fin);
    if (!p.whole) {
      a.sched = reinterpret_cast<int64_t*>(ws + p.sched);
      a.part_ml = reinterpret_cast<float*>(ws + p.ml);
      a.part = reinterpret_cast<float*>(ws + p.part);
    }
    lock = handover_lock(workspace);
  }
  return hip_status(launch_kv4_attn(a, p, cache->dtype == MQK_F16, cache->D,
                                    static_cast<hipStream_t>(stream)),
                    "kv4_attn kernel launch");
}

int mqk_kv4_evict(const mqk_kv4_cache* cache, float* scores, const int32_t* seq_lens, int budget, int recent,
                  int32_t* new_lens, int32_t* kept, void* stream) {
  if (int st = check_cache(cache); st != MQK_OK) return st;
  if (budget <= 0 || budget > (1 << 24) || recent < 0 || recent > budget)
    return fail(MQK_ERR_BAD_SHAPE, "budget = %d must be positive, recent = %d within it", budget, recent);
  if (cache->n_seqs == 0) return ok();
  if (!scores || !seq_lens || !new_lens || !kept) return fail(MQK_ERR_NULL_POINTER, "scores, seq_lens, new_lens or kept is NULL");
  if (cache->n_seqs * cache->Hkv > kMostThreads / 1024) return fail(MQK_ERR_BAD_SHAPE, "too many sequences");
  // (a workgroup a head: what one writes, others would read)
  const int64_t heads = cache->n_seqs * cache->Hkv, records = cache->num_blocks * cache->Hkv;
  const struct {
    const void* at;
    int64_t bytes;
  } out[2] = {{new_lens, cache->n_seqs * 4}, {kept, heads * budget * 4}},
    in[4] = {{seq_lens, cache->n_seqs * 4}, {cache->block_table, cache->n_seqs * cache->bt_cols * 4},
             {scores, records * 16 * 4}, {cache->cache, records * 18 * cache->D}};
  bool over = meet(new_lens, out[0].bytes, kept, out[1].bytes);
  for (const auto& o : out)
    for (const auto& i : in) over = over || meet(o.at, o.bytes, i.at, i.bytes);
  if (over) return fail(MQK_ERR_BAD_SHAPE, "new_lens and kept must not overlap what the call reads, nor each other");
  Kv4Evict a{};
  a.cache = static_cast<unsigned char*>(cache->cache);
  a.scores = scores;
  a.table = cache->block_table;
  a.lens = seq_lens;
  a.new_lens = new_lens;
  a.kept = kept;
  a.cols = cache->bt_cols;
  a.num_blocks = cache->num_blocks;
  a.Hkv = cache->Hkv;
  a.budget = budget;
  a.recent = recent;
  return hip_status(launch_kv4_evict(a, cache->n_seqs, cache->D, device_topology().cus, static_cast<hipStream_t>(stream)),
                    "kv4_evict kernel launch");
}

size_t mqk_attn_prefill_workspace_size(int dtype, int64_t T, int64_t Tk, int64_t n_seqs, int with_cu, int Hq, int Hkv,
                                       int D) {
  if (prefill_shape(dtype, T, Tk, n_seqs, Hq, Hkv, D) != MQK_OK || T == 0) return 0;
  const size_t n = plan_of(dtype, T, Tk, n_seqs, with_cu != 0, Hq, D).bytes;
  return n ? kDecodeCounterBytes + n : 0;
}

int mqk_attn_prefill(const mqk_attn_tensor* q, const mqk_attn_tensor* k, const mqk_attn_tensor* v, int dtype,
                     const int32_t* cu_q, const int32_t* cu_k, int64_t T, int64_t Tk, int64_t n_seqs, int Hq, int Hkv,
                     int D, float scale, int fill, void* out, void* workspace, size_t ws_bytes, void* stream) {
  if (!q || !k || !v) return fail(MQK_ERR_NULL_POINTER, "q, k or v descriptor is NULL");
  if (int st = prefill_shape(dtype, T, Tk, n_seqs, Hq, Hkv, D); st != MQK_OK) return st;
  if (!(scale > 0.f) || scale > kMostScale) return fail(MQK_ERR_BAD_SHAPE, "scale must be positive, and finite times log2(e)");
  if (!cu_q && (T % n_seqs != 0 || (!cu_k && Tk % n_seqs != 0)))
    return fail(MQK_ERR_BAD_SHAPE, "without cu_seqlens, T and Tk must be multiples of n_seqs = %lld", (long long)n_seqs);
  if (cu_q && !cu_k && T != Tk) return fail(MQK_ERR_BAD_SHAPE, "without cu_k, k must have q's tokens");
  if (T == 0) return ok();
  const int es = dtype == MQK_F32 ? 4 : 2;
  if (!q->data || !out || (Tk > 0 && (!k->data || !v->data))) return fail(MQK_ERR_NULL_POINTER, "q, k, v or out is NULL");
  if (!aligned16(q->data) || !aligned16(k->data) || !aligned16(v->data) || !aligned16(out))
    return fail(MQK_ERR_MISALIGNED, "q, k, v and out must be 16-byte aligned");
  if (!chunked(q->token_stride, T, es) || !chunked(q->head_stride, Hq, es) || !chunked(k->token_stride, Tk, es) ||
      !chunked(k->head_stride, Hkv, es) || !chunked(v->token_stride, Tk, es) || !chunked(v->head_stride, Hkv, es))
    return fail(MQK_ERR_MISALIGNED, "token and head strides must be multiples of 16 bytes");
  AttnArgs a{};
  a.q = static_cast<const unsigned char*>(q->data);
  a.k = static_cast<const unsigned char*>(k->data);
  a.v = static_cast<const unsigned char*>(v->data);
  a.out = static_cast<unsigned char*>(out);
  a.q_ts = q->token_stride * es;
  a.q_hs = q->head_stride * es;
  a.k_ts = k->token_stride * es;
  a.k_hs = k->head_stride * es;
  a.v_ts = v->token_stride * es;
  a.v_hs = v->head_stride * es;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.T = T;
  a.Tk = Tk;
  a.n_seqs = int(n_seqs);
  a.each_q = cu_q ? 0 : T / n_seqs;
  a.each_k = cu_q || cu_k ? 0 : Tk / n_seqs;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.D = D;
  a.scale = scale * kLog2e;
  a.fill = fill;
  a.xcds = device_topology().xcds;
  const AttnPlan p = plan_of(dtype, T, Tk, n_seqs, cu_q != nullptr, Hq, D);
  a.parts = p.parts;
  std::unique_lock<std::recursive_mutex> lock;
  if (p.bytes) {
    if (!workspace || ws_bytes < kDecodeCounterBytes + p.bytes)
      return fail(MQK_ERR_WORKSPACE, "needs a workspace of %zu bytes", kDecodeCounterBytes + p.bytes);
    if (!aligned16(workspace)) return fail(MQK_ERR_MISALIGNED, "workspace must be 16-byte aligned");
    unsigned char* ws = static_cast<unsigned char*>(workspace) + kDecodeCounterBytes;
    a.part_ml = reinterpret_cast<float*>(ws + p.ml);
    a.part = reinterpret_cast<float*>(ws + p.part);
    lock = handover_lock(workspace);
  }
  const hipError_t err = launch_attn_prefill(a, dtype, p.split, static_cast<hipStream_t>(stream));
  if (err == hipErrorInvalidConfiguration) return fail(MQK_ERR_BAD_SHAPE, "too much work for one call");
  return hip_status(err, "attn_prefill kernel launch");
}

}  // extern "C"
