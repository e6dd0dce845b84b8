// Host-only argument checks (declared in packed_host.h).
#include "packed_host.h"

#ifndef __host__  // plain C++: the attributes are empty
#define __host__
#define __device__
#endif
#include "packed_map.h"

#include <cstdlib>

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
  if (!packed_head_dim_ok(a->head_dim, a->dtype)) return TRINIX_ERR_BAD_HEAD_DIM;
  int64_t need = 0;
  const int prc = trinix_packed_plan_bytes(a->n_seqs, a->total_q, a->total_k, &need);
  if (prc != TRINIX_OK) return prc;
  if (a->nheads_q <= 0 || a->nheads_kv <= 0 || a->nheads_q > (1 << 20) || a->nheads_q % a->nheads_kv != 0)
    return TRINIX_ERR_BAD_SHAPE;
  if (a->plan_bytes < need || ((uintptr_t)a->plan & 15) != 0) return TRINIX_ERR_BAD_ARGUMENT;
  // the largest grid: the backward at head_dim 256, four workgroups per item of the
  // finest key list and head and two per one of the finest row list
  const int64_t most = lmax(packed_list_cap(a->total_q, a->n_seqs, 64), packed_list_cap(a->total_k, a->n_seqs, 64));
  if (most > INT32_MAX / (6 * a->nheads_q)) return TRINIX_ERR_BAD_SHAPE;
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
    const int64_t ws = packed_partial_bytes(a);
    if (ws > 0 && (!a->workspace || a->workspace_bytes < ws || ((uintptr_t)a->workspace & 15) != 0))
      return TRINIX_ERR_BAD_ARGUMENT;
    if (a->total_q > 0 && (!a->lse || !a->delta || (!f32 && !a->out_lo))) return TRINIX_ERR_NULL_POINTER;
  }
  if (((uintptr_t)a->lse & 3) != 0 || ((uintptr_t)a->delta & 3) != 0 || ((uintptr_t)a->alibi_slopes & 3) != 0)
    return TRINIX_ERR_BAD_STRIDE;
  return TRINIX_OK;
}

// dK and dV of a KV head walk the query heads of its group one after the other; with
// few key blocks that leaves CUs idle and one long chain.  Their heads then go over as
// many workgroups as give 256, whose fp32 partial sums are added in order.
int packed_head_splits(const trinix_packed_args* a) {
  const int64_t G = a->nheads_q / a->nheads_kv, blocks = lmax(1, a->total_k / 128 + lmin(a->n_seqs, a->total_k) / 2);
  int64_t n = lmin(G, 256 / (blocks * a->nheads_kv));
  if (const char* env = getenv("TRINIX_PACKED_SPLITS")) n = lmin(G, atoi(env));  // (tuning and tests)
  const int64_t per = (G + lmax(1, n) - 1) / lmax(1, n);  // heads of the longest chain
  return (int)((G + per - 1) / per);
}
int64_t packed_partial_bytes(const trinix_packed_args* a) {
  const int n = packed_head_splits(a);
  return n > 1 ? 2ll * n * a->total_k * a->nheads_kv * packed_kernel_dim(a->head_dim) * 4 : 0;
}


// A few rows behind long caches are a few long chains of tiles: their keys go over up to
// eight workgroups each, as many as the lengths in the plan ask for (packed_chunks), and a
// second launch joins them.  Measured, us whole | shared out: bf16 32/8 heads of 128, one
// token behind 4000 keys 56 | 18, 4 behind 8000 106 | 44, 64 rows behind 8000 109 | 40, 512
// 128 | 102; 12 chunks of 0 to 34 rows, two of them behind 5745 and 7929 keys, 16 heads 106 |
// 31; 8 tokens behind 3000, 16/4 heads of 64 26 | 19, of 256 103 | 63; fp32, one token behind
// 4000, 32/8 heads of 128 299 | 53, 64 rows behind 8000, 16/4 605 | 98.  It loses where the
// chains are short (30 x 30 rows behind 300 18.6 | 21) or fill the GPU (64 tokens of 32
// heads behind 600 62 | 65), and gains little on prompts (8192 rows of 4 heads 124 | 108, 2048
// of 8 33 | 35, 6 x 600 14 | 23), so those stay whole.
constexpr int kPackedChunksMost = 8;
int packed_key_chunks(const trinix_packed_args* a) {
  if (a->total_q == 0) return 1;
  if (const char* env = getenv("TRINIX_PACKED_CHUNKS")) {  // (tuning and tests)
    const int64_t grids = INT32_MAX / (packed_list_cap(a->total_q, a->n_seqs, 64) * a->nheads_q);
    return (int)lmax(1, lmin(lmin(kPackedChunksMost, atoi(env)), grids));
  }
  const int64_t block = packed_kernel_dim(a->head_dim) == 256 ? 128 : 64;
  int64_t keys = a->total_k;  // of the longest chain, at most
  if (a->has_window) {
    const int64_t right = a->causal ? 0 : clamp_window(a->window_right);
    keys = lmin(keys, lmax(0, clamp_window(a->window_left)) + lmax(0, right) + block);
  }
  const int64_t wgs = (a->total_q / block + lmin(a->n_seqs, a->total_q)) * a->nheads_q;
  return keys >= 2048 && a->total_k >= 2 * a->total_q && wgs <= 512 ? kPackedChunksMost : 1;
}
int64_t packed_chunk_bytes(const trinix_packed_args* a) {
  const int n = packed_key_chunks(a);
  return n > 1 ? (int64_t)n * a->nheads_q * a->total_q * (packed_kernel_dim(a->head_dim) + 1) * 4 : 0;
}

namespace {

// (batch, rows, heads, head_dim) or, without a batch, (rows, heads, head_dim):
// head_dim stride 1, rows on 16 bytes, a row stride that the kernels' 32-bit
// in-tile offsets reach.
int check_vec(const void* ptr, const int64_t* st, int dims, int esize) {
  if (!ptr) return TRINIX_ERR_NULL_POINTER;
  if (st[dims - 1] != 1 || ((uintptr_t)ptr & 15) != 0) return TRINIX_ERR_BAD_STRIDE;
  for (int d = 0; d < dims - 1; ++d)
    if (st[d] % (16 / esize) != 0) return TRINIX_ERR_BAD_STRIDE;
  return st[dims - 3] >= 0 && st[dims - 3] < kMaxKvRowStride ? TRINIX_OK : TRINIX_ERR_BAD_STRIDE;
}

}  // namespace

int validate_shared(const trinix_shared_prefix_args* a) {
  if (!a) return TRINIX_ERR_NULL_POINTER;
  if (a->dtype != TRINIX_F32 && a->dtype != TRINIX_F16 && a->dtype != TRINIX_BF16) return TRINIX_ERR_BAD_DTYPE;
  if (!packed_head_dim_ok(a->head_dim, a->dtype)) return TRINIX_ERR_BAD_HEAD_DIM;
  constexpr int64_t kMax = 1ll << 30;
  if (a->batch <= 0 || a->seqlen_q <= 0 || a->prefix_len < 0 || a->capacity < 0 || a->nheads_q <= 0 || a->nheads_kv <= 0 ||
      a->batch >= (1ll << 24) || a->seqlen_q >= (1ll << 24) || a->prefix_len >= kMax || a->capacity >= kMax ||
      a->nheads_q > (1 << 20) || a->nheads_q % a->nheads_kv != 0)
    return TRINIX_ERR_BAD_SHAPE;
  if (a->batch * a->seqlen_q > kMax / a->nheads_q) return TRINIX_ERR_BAD_SHAPE;
  const int esz = a->dtype == TRINIX_F32 ? 4 : 2;
  int rc = check_vec(a->q, a->q_stride, 4, esz);
  if (rc == TRINIX_OK) rc = check_vec(a->out, a->out_stride, 4, esz);
  if (rc == TRINIX_OK && a->prefix_len > 0) rc = check_vec(a->prefix_k, a->prefix_k_stride, 3, esz);
  if (rc == TRINIX_OK && a->prefix_len > 0) rc = check_vec(a->prefix_v, a->prefix_v_stride, 3, esz);
  if (rc == TRINIX_OK && a->capacity > 0) rc = check_vec(a->k, a->k_stride, 4, esz);
  if (rc == TRINIX_OK && a->capacity > 0) rc = check_vec(a->v, a->v_stride, 4, esz);
  if (rc != TRINIX_OK) return rc;
  if (((uintptr_t)a->lse & 3) != 0 || ((uintptr_t)a->seq_lens & 3) != 0) return TRINIX_ERR_BAD_STRIDE;
  return TRINIX_OK;
}

// Does one workgroup per block of `bm` whole rows walk all keys, or do workgroups share
// them out?  Whole blocks read nothing twice and need no second launch; few of them are a
// chain of all keys on few CUs, and blocks of one request's rows hold fewer than blocks of
// the batch's do (`packed`, what the prefix takes shared out).  So: from `full` blocks on,
// below that while keys are few, fewer the emptier the chip and the blocks.  Measured, us
// shared out | whole 64 (head_dim 256: 128), bf16:
//  - head_dim 128, Sq=95 16/4 heads, P=301, caches of 1001: B=15 53 | 30, 6 34 | 24, 3 29 | 23;
//    P=3000: 90 | 70, 57 | 57, 32 | 49; Sq=72 16/16 B=2 P=5335 29 | 85; Sq=60 B=8 P=500 27 | 17;
//    Sq=10 32/8 P=500 B=16 29 | 20, B=4 13 | 18; Sq=33 16/16 B=5 P=1500 21 | 30; Sq=200 32/8 B=2
//    P=6000 100 | 88;
//  - 256: Sq=95 16/4 P=301 B=15 97 | 56, 6 66 | 51, 3 42 | 47; P=3000 156 | 134, 84 | 126.
// Blocks under 32 rows are shared out (of 16, Sq=4, B=64, P=8192, 76 | 149) but for a few
// hundred keys, where one launch costs the host 4 us less and the GPU no more: 4 tokens of
// 32/8 heads of 64 behind 400 keys 8.1 | 8.5, called in turn 13.1 | 9.2; of 128 behind 150 9.0
// | 7.9, behind 400 9.4 | 11.2.
bool whole_blocks(int64_t keys, int64_t n, int64_t packed, int64_t full, int64_t limit) {
  return n >= full || keys * (full - n) * n < limit * packed;
}

int plan_shared(const trinix_shared_prefix_args* a, SharedPlan* pl) {
  const int64_t G = a->nheads_q / a->nheads_kv, own = a->seqlen_q * G, rows = a->batch * own, kv = a->nheads_kv;
  const bool f32 = a->dtype == TRINIX_F32;
  const auto blocks = [](int64_t n, int64_t per) { return (n + per - 1) / per; };
  pl->rows = (int)rows;
  const bool d256 = packed_kernel_dim(a->head_dim) == 256;
  pl->kind = f32 ? SharedKind::kRows16 : SharedKind::kSplit;
  // 128-row blocks where they fill the chip (B=8 Sq=256 G=4 P=6000 309 shared out, 246 in blocks
  // of 64, 204 in blocks of 128); head_dim 256 has no others
  const int64_t keys = a->prefix_len + a->capacity, b64 = a->batch * blocks(own, 64) * kv, b128 = a->batch * blocks(own, 128) * kv;
  if (!f32) {
    const bool few = keys * packed_kernel_dim(a->head_dim) <= 32768 && b64 <= 512;
    if (own > 64 && b128 >= 192) pl->kind = SharedKind::kWhole128;
    else if (!d256 && (own >= 32 ? whole_blocks(keys, b64, blocks(rows, 64) * kv, 225, 210000) : few)) pl->kind = SharedKind::kWhole64;
    else if (d256 && own >= 32 && whole_blocks(keys, b128, blocks(rows, 128) * kv, 192, 160000)) pl->kind = SharedKind::kWhole128;
  }
  if (const char* env = getenv("TRINIX_SHARED_KIND")) {  // 1, 2, 3: split, whole 64, whole 128 (tuning and tests)
    const int want = atoi(env);
    if (!f32 && want >= 1 && want <= 3 && !(d256 && want == 2)) pl->kind = (SharedKind)want;
  }
  if (pl->kind == SharedKind::kWhole64 || pl->kind == SharedKind::kWhole128) {
    pl->n_p = pl->n_s = 0;
    pl->chunk_p = pl->chunk_s = 0;
    pl->wg_p = 0;
    pl->wg_s = a->batch * blocks(own, pl->kind == SharedKind::kWhole64 ? 64 : 128) * kv;
    pl->ws_bytes = 0;
    return pl->wg_s > INT32_MAX ? TRINIX_ERR_BAD_SHAPE : TRINIX_OK;
  }
  const bool r16 = pl->kind == SharedKind::kRows16;
  const int64_t bm = r16 ? 16 : d256 ? 128 : 64;
  const int64_t gp = blocks(rows, bm) * kv, gs = a->batch * blocks(own, bm) * kv;
  // Chunks of whole 64 keys, at least 128, as many as give about `target`
  // workgroups.  16-bit: 256 for the prefix and 1024 for the own keys; targets of
  // 128 / 256 / 512 / 1024 for the prefix, caches warm: B=64 P=8192 40.8 | 38.9 | 49.3 |
  // 58.7 us, B=1 Sq=256 P=8192 114 | 68 | 60 | 67, B=64 Sq=4 117 | 72 | 79 | 85; of 512 / 1024 /
  // 2048 / 4096 for the own keys, caches read from memory: B=64 of 1024 54.0 | 50.2 | 52.4 |
  // 57.5.  64 keys at least: B=32 of 200 behind 500 13.3 | 17.9, B=1 9.3 | 8.9.
  const auto split = [&](int64_t keys, int64_t groups, int64_t target, int* n, int* chunk) {
    const int64_t c = lmax(kDecodeMinChunk, blocks(blocks(keys, lmax(1, target / groups)), 64) * 64);
    *n = (int)blocks(keys, c);
    *chunk = (int)c;
  };
  split(a->prefix_len, gp, r16 ? kDecodeTargetWgs : 256, &pl->n_p, &pl->chunk_p);
  split(a->capacity, gs, r16 ? 2 * kDecodeTargetWgs : 1024, &pl->n_s, &pl->chunk_s);
  if (gp >= INT32_MAX / lmax(1, pl->n_p) || gs >= INT32_MAX / lmax(1, pl->n_s)) return TRINIX_ERR_BAD_SHAPE;
  pl->wg_p = gp * pl->n_p;
  pl->wg_s = gs * pl->n_s;
  if (pl->wg_p + pl->wg_s > INT32_MAX) return TRINIX_ERR_BAD_SHAPE;
  pl->ws_bytes = kv * rows * (pl->n_p + pl->n_s) * (packed_kernel_dim(a->head_dim) + 1) * 4;
  return TRINIX_OK;
}

}  // namespace trinix

using namespace trinix;

extern "C" int trinix_packed_fwd_workspace(const trinix_packed_args* a, int64_t* bytes) {
  if (!a || !bytes) return TRINIX_ERR_NULL_POINTER;
  if (a->nheads_q <= 0 || a->nheads_kv <= 0 || a->nheads_q > (1 << 20) || a->nheads_q % a->nheads_kv != 0 || a->n_seqs < 1 ||
      a->n_seqs >= (1ll << 24) || a->total_q < 0 || a->total_q >= (1ll << 30) || a->total_k < 0 || a->total_k >= (1ll << 30) ||
      !packed_head_dim_ok(a->head_dim, a->dtype))
    return TRINIX_ERR_BAD_SHAPE;
  *bytes = packed_chunk_bytes(a);
  return TRINIX_OK;
}
extern "C" int trinix_packed_bwd_workspace(const trinix_packed_args* a, int64_t* bytes) {
  if (!a || !bytes) return TRINIX_ERR_NULL_POINTER;
  if (a->nheads_q <= 0 || a->nheads_kv <= 0 || a->nheads_q > (1 << 20) || a->nheads_q % a->nheads_kv != 0 || a->n_seqs < 1 ||
      a->total_k < 0 || a->total_k >= (1ll << 30) || !packed_head_dim_ok(a->head_dim, a->dtype))
    return TRINIX_ERR_BAD_SHAPE;
  *bytes = packed_partial_bytes(a);
  return TRINIX_OK;
}

extern "C" int trinix_shared_prefix_workspace(const trinix_shared_prefix_args* a, int64_t* bytes) {
  if (!bytes) return TRINIX_ERR_NULL_POINTER;
  int rc = validate_shared(a);
  SharedPlan pl;
  if (rc == TRINIX_OK) rc = plan_shared(a, &pl);
  if (rc == TRINIX_OK) *bytes = pl.ws_bytes;
  return rc;
}

extern "C" int trinix_packed_plan_bytes(int64_t n_seqs, int64_t total_q, int64_t total_k, int64_t* bytes) {
  if (!bytes) return TRINIX_ERR_NULL_POINTER;
  if (n_seqs < 1 || n_seqs >= (1ll << 24) || total_q < 0 || total_k < 0 || total_q >= (1ll << 30) ||
      total_k >= (1ll << 30))
    return TRINIX_ERR_BAD_SHAPE;
  *bytes = packed_plan_ints(total_q, total_k, n_seqs) * 4;
  return TRINIX_OK;
}
