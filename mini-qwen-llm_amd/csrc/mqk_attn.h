// Host-side launch interface of the attention operators (prompt attention, the 4-bit
// paged cache and what reads it) between the C ABI (attn_api.hip) and the kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mqk {

struct AttnArgs {
  const unsigned char* q;    // tokens and heads at byte strides, dense in the head
  const unsigned char* k;
  const unsigned char* v;
  unsigned char* out;        // [T, Hq, D]
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  const int32_t* cu_q;       // [n_seqs + 1] or null: n_seqs sequences of each_q tokens
  const int32_t* cu_k;       // [n_seqs + 1] or null: cu_q's, or each_k keys
  int64_t T, Tk, each_q, each_k;
  int n_seqs, Hq, Hkv, D;
  float scale;               // softmax scale times log2(e)
  int fill;                  // 1: rows behind the last sequence become 0; 0: stay as they are
  int xcds;
  int nslots;                // (set by the launch)
};

// dtype: 0 bf16, 1 fp16, 2 fp32.
hipError_t launch_attn_prefill(AttnArgs a, int dtype, hipStream_t stream);

}  // namespace mqk
