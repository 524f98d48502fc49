// Host-side launch interface of the operators around the bf16 / fp16 paged cache, between the
// C ABI (paged_api.hip) and the kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mqk {

// x / d for x < 2^28 as (x * mul) >> shift: with d <= 2^s and mul = ceil(2^(28 + s) / d), the
// product is over x / d * 2^(28 + s) by less than x * d <= 2^28 * 2^s, so the quotient by
// less than 1 / d.
struct Divide {
  uint32_t mul, shift;
};
inline Divide divide_by(uint32_t d) {
  uint32_t s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  return {uint32_t(((uint64_t(1) << (28 + s)) + d - 1) / d), 28 + s};
}

struct PagedTables {
  const int32_t* old_lens;   // [n_seqs] tokens before the step
  const int32_t* new_lens;   // [n_seqs] tokens of the step
  int32_t* table;            // [n_seqs, cols]
  const int32_t* free_pages; // [n_free]
  const int32_t* cursor;     // [1] where in it to begin, or null: at 0
  int32_t* lens;             // [n_seqs]
  int32_t* cu;               // [n_seqs + 1]
  int32_t* kv_seq;           // [n_tokens]
  int32_t* kv_pos;           // [n_tokens]
  int64_t* slots;            // [n_tokens]
  int32_t* taken;            // [1]
  int64_t cols, n_free, n_tokens;
  int n_seqs, page;
};
constexpr int kTablesMostSeqs = 16384;
hipError_t launch_paged_tables(const PagedTables& a, int cus, hipStream_t stream);

// How the partial results of a block of rows are joined: `parts` of them from number `first` on,
// `stride` apart, the first one `lead` further; row r of them is row base + r of the (token, head)
// rows from token `at` on.  Whoever wrote one has a share of the joining: number `index`.
struct PagedJoin {
  int64_t first, at;
  int32_t base, kvh, rows, parts, index, stride, lead;
};

// Partial results: [..][rows][2] maximum and sum, [..][rows][D], and how they are joined.
struct PagedOut {
  PagedJoin* joins;
  float* ml;
  float* part;
};

struct PagedAttn {
  const unsigned char* q;    // tokens and heads at byte strides
  const unsigned char* k;    // [num_blocks, page, Hkv, D]
  const unsigned char* v;
  unsigned char* out;        // [T, Hq, D]
  int64_t q_ts, q_hs;
  const int32_t* table;      // [n_seqs, cols]
  const int32_t* lens;       // [n_seqs]
  const int32_t* cu;         // [n_seqs + 1] or null: `each` tokens a sequence
  const int32_t* pages;      // [T, Hkv, n_pages] or null: all keys
  int64_t T, each, cols, num_blocks, n_pages;
  int n_seqs, Hq, Hkv, G, D, page;
  Divide page8;              // by page / 8
  float scale;               // softmax scale times log2(e)
  int fill;                  // 1: rows behind the last sequence become 0; 0: stay as they are
  int few_rows;              // sequences with up to this many rows are the short launch's
  int rows;                  // rows of a partial result
  int parts, part_steps;     // (selected pages) of a unit, and steps of a part
  int slots;                 // (long launch) workgroups the card takes at once
  int64_t most_split;        // (long launch) partial results there is room for
  int whole;                 // (short launch) a workgroup a head: nothing to join
  int64_t* n_split;          // workspace: how many partial results the long launch has
  PagedOut few, many;        // workspace: [workgroups][2] and [most_split]
};
// Launches of a call (workgroups; 0: no such launch) and the workspace's layout (byte offsets).
struct PagedPlan {
  int64_t few, many;         // short sequences (or selected pages), long ones
  int few_rows, rows, parts, part_steps, slots, whole;
  int64_t most_split;
  struct Room {
    size_t joins, ml, part;
  } few_room, many_room;
  size_t n_split, bytes;
};
PagedPlan plan_paged_attn(int64_t T, int64_t n_seqs, bool cu, int64_t cols, int page, int64_t n_pages, int Hq, int Hkv,
                          int D, int cus);
hipError_t launch_paged_attn(const PagedAttn& a, const PagedPlan& p, int fp16, hipStream_t stream);

struct PagedBounds {
  const unsigned char* k;    // [num_blocks, page, Hkv, D]
  unsigned char* bounds;     // [num_blocks, Hkv, 2, D]
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;         // or null: `each` tokens a sequence
  int64_t T, each, cols, num_blocks;
  int n_seqs, Hkv, D, page;
};
hipError_t launch_paged_bounds(const PagedBounds& a, int fp16, hipStream_t stream);

// Tokens whose scores (8 bytes a page and head) are in the workspace at a time, in whole groups of
// 4: equal rounds of what 256 MiB hold, or one group.  (2048 tokens over 2628 pages, 8 heads: 1285 us
// in one round of 329 MiB, 1295 in two; 1350 where the second had what the first left.)
inline int64_t select_round(int64_t T, int64_t Hkv, int64_t cols) {
  const int64_t groups = (T + 3) / 4, fit = (int64_t(1) << 28) / (Hkv * cols * 32);
  const int64_t rounds = fit > 0 ? (groups + fit - 1) / fit : groups;
  const int64_t each = (groups + rounds - 1) / rounds * 4;
  return each < T ? each : T;
}
struct PagedSelect {
  const unsigned char* q;    // tokens and heads at byte strides
  const unsigned char* bounds;
  int64_t q_ts, q_hs;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;         // or null: `each` tokens a sequence
  int32_t* pages;            // [T, Hkv, take]
  uint64_t* keys;            // workspace: [to - from, Hkv, cols]
  int64_t T, each, cols, num_blocks;
  int64_t from, to;          // a round's tokens
  int n_seqs, Hq, Hkv, G, D, page, take, first, recent;
};
hipError_t launch_paged_select(PagedSelect a, int fp16, int cus, hipStream_t stream);

}  // namespace mqk
