// Host-only argument checks (declared in packed_host.h).
#include "packed_host.h"

#ifndef __host__  // plain C++: the attributes are empty
#define __host__
#define __device__
#endif
#include "packed_map.h"

namespace trinix {
namespace {

// (rows, heads, head_dim) tensor of at least one row: head_dim stride 1; 16-bit
// rows on 16 bytes, a row stride that the kernels' 32-bit in-tile offsets reach.
int check_rows(const void* ptr, const int64_t st[3], int64_t rows, bool f32) {
  if (rows == 0) return TRINIX_OK;
  if (!ptr) return TRINIX_ERR_NULL_POINTER;
  if (st[2] != 1) return TRINIX_ERR_BAD_STRIDE;
  if (f32) return ((uintptr_t)ptr & 3) == 0 ? TRINIX_OK : TRINIX_ERR_BAD_STRIDE;
  if (((uintptr_t)ptr & 15) != 0 || st[0] % 8 != 0 || st[1] % 8 != 0) return TRINIX_ERR_BAD_STRIDE;
  return st[0] >= 0 && st[0] < kMaxKvRowStride ? TRINIX_OK : TRINIX_ERR_BAD_STRIDE;
}

}  // namespace

int validate_packed(const trinix_packed_args* a, bool backward) {
  if (!a || !a->plan) return TRINIX_ERR_NULL_POINTER;
  if (a->dtype != TRINIX_F32 && a->dtype != TRINIX_F16 && a->dtype != TRINIX_BF16) return TRINIX_ERR_BAD_DTYPE;
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return TRINIX_ERR_BAD_HEAD_DIM;
  int64_t need = 0;
  const int prc = trinix_packed_plan_bytes(a->n_seqs, a->total_q, a->total_k, &need);
  if (prc != TRINIX_OK) return prc;
  if (a->nheads_q <= 0 || a->nheads_kv <= 0 || a->nheads_q > (1 << 20) || a->nheads_q % a->nheads_kv != 0)
    return TRINIX_ERR_BAD_SHAPE;
  if (a->plan_bytes < need || ((uintptr_t)a->plan & 15) != 0) return TRINIX_ERR_BAD_ARGUMENT;
  // the largest grid: one workgroup per item of the finest list and head
  const int64_t most = lmax(packed_list_cap(a->total_q, a->n_seqs, 64), packed_list_cap(a->total_k, a->n_seqs, 64));
  if (most > INT32_MAX / (4 * a->nheads_q)) return TRINIX_ERR_BAD_SHAPE;
  const bool f32 = a->dtype == TRINIX_F32;
  const struct {
    const void* ptr;
    const int64_t* st;
    int64_t rows;
  } fwd[] = {{a->q, a->q_stride, a->total_q}, {a->k, a->k_stride, a->total_k}, {a->v, a->v_stride, a->total_k},
             {a->out, a->out_stride, a->total_q}},
    bwd[] = {{a->dout, a->dout_stride, a->total_q}, {a->dq, a->dq_stride, a->total_q}, {a->dk, a->dk_stride, a->total_k},
             {a->dv, a->dv_stride, a->total_k}};
  for (const auto& t : fwd) {
    const int rc = check_rows(t.ptr, t.st, t.rows, f32);
    if (rc != TRINIX_OK) return rc;
  }
  if (a->out_lo && !f32 && ((uintptr_t)a->out_lo & 15) != 0) return TRINIX_ERR_BAD_STRIDE;
  if (backward) {
    for (const auto& t : bwd) {
      const int rc = check_rows(t.ptr, t.st, t.rows, f32);
      if (rc != TRINIX_OK) return rc;
    }
    if (a->total_q > 0 && (!a->lse || !a->delta || (!f32 && !a->out_lo))) return TRINIX_ERR_NULL_POINTER;
  }
  if (((uintptr_t)a->lse & 3) != 0 || ((uintptr_t)a->delta & 3) != 0 || ((uintptr_t)a->alibi_slopes & 3) != 0)
    return TRINIX_ERR_BAD_STRIDE;
  return TRINIX_OK;
}

}  // namespace trinix

using namespace trinix;

extern "C" int trinix_packed_plan_bytes(int64_t n_seqs, int64_t total_q, int64_t total_k, int64_t* bytes) {
  if (!bytes) return TRINIX_ERR_NULL_POINTER;
  if (n_seqs < 1 || n_seqs >= (1ll << 24) || total_q < 0 || total_k < 0 || total_q >= (1ll << 30) ||
      total_k >= (1ll << 30))
    return TRINIX_ERR_BAD_SHAPE;
  *bytes = packed_plan_ints(total_q, total_k, n_seqs) * 4;
  return TRINIX_OK;
}
