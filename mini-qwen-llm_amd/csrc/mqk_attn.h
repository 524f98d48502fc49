// Host-side launch interface of the attention operators (prompt attention, the 4-bit
// paged cache and what reads it) between the C ABI (attn_api.hip) and the kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mqk {

constexpr int64_t kMostThreads = 0xFFFFFFFFll;  // of a launch

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
  int parts;                 // of the keys, by a workgroup each; more than one:
  float* part_ml;            // workspace: [T, Hq, parts][2] maximum and sum of each
  float* part;               // [T, Hq, parts][D]
  int nslots, far;           // (set by the launch)
};
// How a call is cut, and the workspace's layout (byte offsets, all of it scratch).
struct AttnPlan {
  int split;                 // groups of waves of a workgroup that share a head's keys (1, 2, 4)
  int parts;
  size_t ml, part, bytes;
};
// dtype: 0 bf16, 1 fp16, 2 fp32.  split, parts: as forced, or 0.
AttnPlan plan_attn_prefill(int dtype, int64_t T, int64_t Tk, int64_t n_seqs, bool cu, int Hq, int D, int cus, int split,
                           int parts);
// hipErrorInvalidConfiguration: a launch would have too many threads, and none is made.
hipError_t launch_attn_prefill(const AttnArgs& a, int dtype, int split, hipStream_t stream);

// Tokens of a call and their places in the 4-bit paged cache: the last ones of each
// sequence, of which lens[s] are there in all.
struct Kv4Tokens {
  unsigned char* cache;      // [num_blocks, Hkv] records of 18 D bytes
  const int32_t* table;      // [n_seqs, cols]
  const int32_t* lens;       // [n_seqs]
  const int32_t* cu;         // [n_seqs + 1] or null: `each` tokens a sequence
  int64_t T, each, cols, num_blocks;
  int n_seqs, Hkv;
};
hipError_t launch_kv4_write(const Kv4Tokens& a, const unsigned char* k, const unsigned char* v, int64_t k_ts,
                            int64_t k_hs, int64_t v_ts, int64_t v_hs, float* scores, int D, int fp16,
                            hipStream_t stream);
hipError_t launch_kv4_read(const Kv4Tokens& a, unsigned char* k, unsigned char* v, int D, int fp16, hipStream_t stream);

struct Kv4Evict {
  unsigned char* cache;
  float* scores;             // [num_blocks, Hkv, 16]
  const int32_t* table;      // [n_seqs, cols]
  const int32_t* lens;       // [n_seqs]
  int32_t* new_lens;         // [n_seqs]
  int32_t* kept;             // [n_seqs, Hkv, budget]
  int64_t cols, num_blocks;
  int Hkv, budget, recent;
};
hipError_t launch_kv4_evict(const Kv4Evict& a, int64_t n_seqs, int D, int cus, hipStream_t stream);

struct Kv4Attn {
  const unsigned char* q;      // [B, S, Hq, D]
  const unsigned char* cache;
  const int32_t* table;        // [B, cols]
  const int32_t* lens;         // [B]
  unsigned char* out;          // [B, S, Hq, D]
  float* scores;               // [num_blocks, Hkv, 16] or null
  int64_t* sched;              // workspace: steps of a part, then the first step of each sequence
  float* part_ml;              // [partial results][16][2] maximum and sum
  float* part;                 // [partial results][16][D]
  float* fin;                  // [B, S, Hq][2] maximum and 1 / sum of each row (with scores)
  int64_t cols, num_blocks;
  int B, S, Hq, Hkv, G, RB;    // G = Hq / Hkv; RB blocks of 16 rows (S * G of them)
  int whole, few;              // a part a head; or steps that are few for the card
  int run;                     // pages a wave adds the weights of
  float scale;                 // softmax scale times log2(e)
};
// Launches of a call, in workgroups of 256 (0: no such launch), and the workspace's layout (byte
// offsets, all of it scratch).
struct Kv4Plan {
  int64_t grid, join, weigh;
  int whole, few, run;
  size_t sched, ml, part, fin, bytes;
};
Kv4Plan plan_kv4_attn(int B, int S, int Hq, int Hkv, int D, int64_t cols, bool scores, int cus);
hipError_t launch_kv4_attn(const Kv4Attn& a, const Kv4Plan& p, int fp16, int D, hipStream_t stream);

}  // namespace mqk
