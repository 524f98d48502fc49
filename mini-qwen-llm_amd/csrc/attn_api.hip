// C ABI of the attention operators behind the projection front: argument validation and
// launch.  Declarations and the contract of every entry point: include/mqk.h.
#include "../../include/mqk.h"
#include "mqk_attn.h"
#include "mqk_status.h"

using namespace mqk;

namespace {

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int64_t kMostTokens = 0x7FFF0000ll;  // tile arithmetic stays inside 32 bits

// A head's stride and a token's (elements): whole 16-byte chunks, or the tensor is not
// read at all with that stride.
bool chunked(int64_t stride, int64_t count, int bytes) { return count <= 1 || stride * bytes % 16 == 0; }

}  // namespace

extern "C" {

int mqk_attn_prefill(const mqk_attn_tensor* q, const mqk_attn_tensor* k, const mqk_attn_tensor* v, int dtype,
                     const int32_t* cu_q, const int32_t* cu_k, int64_t T, int64_t Tk, int64_t n_seqs, int Hq, int Hkv,
                     int D, float scale, int fill, void* out, void* stream) {
  if (!q || !k || !v) return fail(MQK_ERR_NULL_POINTER, "q, k or v descriptor is NULL");
  if (dtype != MQK_BF16 && dtype != MQK_F16 && dtype != MQK_F32)
    return fail(MQK_ERR_UNSUPPORTED, "dtype %d unknown", dtype);
  if (T < 0 || Tk < 0 || T > kMostTokens || Tk > kMostTokens)
    return fail(MQK_ERR_BAD_SHAPE, "T = %lld, Tk = %lld out of range", (long long)T, (long long)Tk);
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0)
    return fail(MQK_ERR_BAD_SHAPE, "Hq = %d must be a positive multiple of Hkv = %d", Hq, Hkv);
  if (D <= 0 || D % 8 != 0 || D > 256) return fail(MQK_ERR_UNSUPPORTED, "head_dim %d: a multiple of 8 up to 256", D);
  if (!(scale > 0.f) || scale > 3e38f) return fail(MQK_ERR_BAD_SHAPE, "scale must be positive and finite");
  if (n_seqs <= 0 || n_seqs > (1 << 20)) return fail(MQK_ERR_BAD_SHAPE, "n_seqs = %lld out of range", (long long)n_seqs);
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
  return hip_status(launch_attn_prefill(a, dtype, static_cast<hipStream_t>(stream)), "attn_prefill kernel launch");
}

}  // extern "C"
