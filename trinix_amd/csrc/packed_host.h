// Host-only argument checks of attention over packed sequences and behind a
// shared prefix (plain C++; see host_plan.h).
#pragma once
#include "host_plan.h"
#include "trinix_attn.h"

namespace trinix {

// head_dim that a call's kernels are built for (at least the tensors'), and whether
// they take it: multiples of 8, fp32 of 4, up to 256.
inline int packed_kernel_dim(int64_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
// Columns that the packed-sequence kernels compute: 96 of 128 where that is enough
// (us, forward and forward with backward, all 128 | 96: 8 heads of 80, 1090 rows in five
// documents, fp32 44 and 176 | 36 and 143; bf16 32/8 heads of 96, 8192 rows 500 and 2815 |
// 426 and 2384; 12 heads of 96, 1024 rows 19.5 and 69.8 | 17.8 and 62.6).
inline int packed_columns(int64_t head_dim) { return head_dim > 64 && head_dim <= 96 ? 96 : packed_kernel_dim(head_dim); }
inline bool packed_head_dim_ok(int64_t head_dim, int32_t dtype) {
  return head_dim > 0 && head_dim <= 256 && head_dim % (dtype == TRINIX_F32 ? 4 : 8) == 0;
}

// TRINIX_OK or the status to return; no launch.  `backward`: the gradient
// pointers and strides too.
int validate_packed(const trinix_packed_args* a, bool backward);
// Workgroups that share the query heads of a KV head in dK and dV (1: none), each
// leaving fp32 partial sums of all keys.
int packed_head_splits(const trinix_packed_args* a);
// Bytes of those partial sums.
int64_t packed_partial_bytes(const trinix_packed_args* a);
// Workgroups that share the keys of a block of rows in the forward, at most (1:
// none), and the bytes of their fp32 partial results.
int packed_key_chunks(const trinix_packed_args* a);
int64_t packed_chunk_bytes(const trinix_packed_args* a);

// Attention behind a shared prefix: the same checks, and the launch plan.
int validate_shared(const trinix_shared_prefix_args* a);
// A row is a (request, query, head of the KV group): row r = (b * Sq + i) * G + g
// of a KV head.  Partial results (fp32, per row and chunk of keys) of n_p prefix
// chunks and n_s chunks of the own keys are merged by a second kernel; the whole
// kinds have none.
enum class SharedKind {
  kRows16,    // 16 rows by a chunk of keys (fp32)
  kSplit,     // 64 rows by a chunk of keys (head_dim 256: 128)
  kWhole64,   // 64 rows of a request by all its keys
  kWhole128,  // 128 rows
};
struct SharedPlan {
  SharedKind kind;
  int rows;            // rows per KV head
  int n_p, chunk_p;    // chunks of the prefix, keys per chunk
  int n_s, chunk_s;    // the same for the own keys (at the cache's capacity)
  int64_t wg_p, wg_s;  // workgroups of the prefix and of the own keys (whole: all in wg_s)
  int64_t ws_bytes;
};
// TRINIX_OK, or TRINIX_ERR_BAD_SHAPE where the grid or the workspace leaves 32
// bits of workgroups.  For validated arguments.
int plan_shared(const trinix_shared_prefix_args* a, SharedPlan* pl);

}  // namespace trinix
