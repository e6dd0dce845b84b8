// Entry points of attention over packed sequences, and the delta pass of its
// backward.
#include <cstdlib>

#include "attn_packed.h"
#include "packed_host.h"

namespace trinix {
namespace {

// delta[h, t] = sum_d dO[t, h, d] * O[t, h, d] in fp32, O with the part that its
// rounding took off (o_lo): with O as rounded, delta is off by half a step of O,
// which dZ = P (dP - delta) amplifies where a row's softmax is peaked (dQ and dK of
// bf16 then err up to 1.9 times as much as from their own rounding).
// VE elements (16 bytes) per lane, D / VE lanes per row.
template <class E, int D, bool F32>
__global__ __launch_bounds__(256) void packed_delta_kernel(const PackedParams p, int64_t rows) {
  typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
  constexpr int VE = F32 ? 4 : 8, LPR = D / VE, RPB = 256 / LPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;  // t * Hq + h
  const int c = threadIdx.x % LPR;
  float acc = 0.f;
  const int64_t t = row / p.Hq;
  const int h = (int)(row % p.Hq);
  if (row < rows && c * VE < p.d) {
    const int64_t oo = t * p.o_ss + h * p.o_sh + c * VE, od = t * p.do_ss + h * p.do_sh + c * VE;
    if constexpr (F32) {
      const f32x4_t o = *(const f32x4_any*)((const float*)p.o + oo), d = *(const f32x4_any*)((const float*)p.dout + od);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc += o[e] * d[e];
    } else {
      const u32x4_t o = *(const u32x4_t*)((const uint16_t*)p.o + oo), r = *(const u32x4_t*)((const uint16_t*)p.o_lo + oo);
      const u32x4_t d = *(const u32x4_t*)((const uint16_t*)p.dout + od);
      constexpr float f = 1.f / kLoScale<E>;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc += __builtin_fmaf(E::lo(r[e]), f, E::lo(o[e])) * E::lo(d[e]) +
               __builtin_fmaf(E::hi(r[e]), f, E::hi(o[e])) * E::hi(d[e]);
    }
  }
#pragma unroll
  for (int m = LPR / 2; m >= 1; m /= 2) acc += __shfl_xor(acc, m);
  if (c == 0 && row < rows) {
    const int64_t at = (int64_t)h * p.Tq + t;
    // a row that sees no key: P = 0 and delta = 0, whatever its dO holds
    p.delta[at] = p.lse[at] == -INFINITY ? 0.f : acc;
  }
}

// Adds the partial sums of dV (blockIdx.y = 0) and dK (1) over the splits, in order:
// four head_dim elements of a key per thread.
template <class E, bool F32>
__global__ __launch_bounds__(256) void packed_dkdv_sum(const PackedParams p, int D) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, per = (int64_t)p.Tk * p.Hkv * D;
  if (at >= per || at % D >= p.d) return;
  const int which = blockIdx.y;
  const float* x = p.part + which * per + at;
  f32x4_t s = *(const f32x4_t*)x;
  for (int k = 1; k < p.n_split; ++k) s += *(const f32x4_t*)(x + 2 * k * per);
  const int64_t row = at / D / p.Hkv;
  const int hkv = (int)(at / D % p.Hkv), d = (int)(at % D);
  void* base = which ? p.dk : p.dv;
  const int64_t to = row * (which ? p.dk_ss : p.dv_ss) + hkv * (which ? p.dk_sh : p.dv_sh) + d;
  if constexpr (F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) ((float*)base)[to + e] = s[e];
  } else {
    *(u32x2_t*)((uint16_t*)base + to) = (u32x2_t){E::pack(s[0], s[1]), E::pack(s[2], s[3])};
  }
}
template <class E, bool F32>
hipError_t launch_sum(const PackedParams& p, int D, hipStream_t st) {
  const int64_t units = (int64_t)p.Tk * p.Hkv * D / 4;
  return launch_kernel(&packed_dkdv_sum<E, F32>, dim3((unsigned)((units + 255) / 256), 2), dim3(256), 0, st, p, D);
}

template <class E, bool F32>
hipError_t launch_delta(const PackedParams& p, int D, hipStream_t st) {
  const int64_t rows = (int64_t)p.Tq * p.Hq;
  const int rpb = 256 * (F32 ? 4 : 8) / D;
  const dim3 grid((unsigned)((rows + rpb - 1) / rpb)), block(256);
  switch (D) {
    case 64: return launch_kernel(&packed_delta_kernel<E, 64, F32>, grid, block, 0, st, p, rows);
    case 128: return launch_kernel(&packed_delta_kernel<E, 128, F32>, grid, block, 0, st, p, rows);
    case 256: return launch_kernel(&packed_delta_kernel<E, 256, F32>, grid, block, 0, st, p, rows);
  }
  return hipErrorNotSupported;
}

bool rows16(const void* ptr, const int64_t st[3]) {
  const int64_t st4[4] = {0, st[0], st[1], 1};
  return rows_aligned16(ptr, st4);
}

PackedParams params(const trinix_packed_args* a) {
  PackedParams p{};
  p.q = a->q, p.k = a->k, p.v = a->v, p.o = a->out, p.o_lo = a->out_lo, p.lse = a->lse;
  p.dout = a->dout, p.delta = a->delta, p.dq = a->dq, p.dk = a->dk, p.dv = a->dv;
  p.q_ss = a->q_stride[0], p.q_sh = a->q_stride[1];
  p.k_ss = a->k_stride[0], p.k_sh = a->k_stride[1];
  p.v_ss = a->v_stride[0], p.v_sh = a->v_stride[1];
  p.o_ss = a->out_stride[0], p.o_sh = a->out_stride[1];
  p.do_ss = a->dout_stride[0], p.do_sh = a->dout_stride[1];
  p.dq_ss = a->dq_stride[0], p.dq_sh = a->dq_stride[1];
  p.dk_ss = a->dk_stride[0], p.dk_sh = a->dk_stride[1];
  p.dv_ss = a->dv_stride[0], p.dv_sh = a->dv_stride[1];
  p.Tq = (int)a->total_q;
  p.Hq = (int)a->nheads_q;
  p.Hkv = (int)a->nheads_kv;
  p.G = p.Hq / p.Hkv;
  p.d = (int)a->head_dim;
  p.scale = a->softmax_scale;
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.causal = a->causal ? 1 : 0;
  p.has_window = a->has_window ? 1 : 0;
  p.wl = clamp_window(a->window_left);
  p.wr = clamp_window(a->window_right);
  p.alibi = a->alibi_slopes;
  p.al_sh = a->alibi_stride;
  return p;
}

// Points p at a list of the plan; returns its items.
int64_t use_list(PackedParams& p, const trinix_packed_args* a, int list) {
  p.items = a->plan + packed_list_offset(list, a->total_q, a->total_k, a->n_seqs);
  return packed_list_cap(packed_list_is_keys(list) ? a->total_k : a->total_q, a->n_seqs, packed_list_block(list));
}
constexpr int kRows64 = 0, kRows128 = 1, kRows256 = 2, kKeys64 = 3, kKeys128 = 4;
constexpr int kListOf[3] = {kRows64, kRows128, kRows256};  // of a PackedShape

// Shape of the 16-bit forward.  The host knows the totals and the number of
// sequences, not their lengths.  Measured, bf16 causal, graph-timed, us pair |
// plain | wide:
//  - pair where 128-row blocks leave CUs idle and the average sequence is worth
//    halving: D=128 8192 rows x 4 heads 116 | 134 | 176; 1024 x 32 21.4 | 22.3 |
//    28.8; 512 x 32 12.6 | 13.3; D=64 2 x 1024 x 12 13.1 | 16.6.  It loses on short
//    sequences (1 + 17 + 64 x 32: 6.4 | 5.5; D=64 20 x 200 x 16 16.6 | 10.5) and on more
//    blocks (2048 x 32 52.4 | 47.8 | 54.3);
//  - wide (D=128) on long sequences that fill the chip with 256-row blocks: 4096 x 32
//    170 | 141 | 131, 8192 x 16 317 | 269 | 246, 1814 rows behind 34000 keys, window
//    4096, 143 | 119 | 112; even at an average of 4096 (8192 + 4099 + 2500 + 1593: 703 |
//    703), it loses below (4096 + 2047 + 1000 + ..., average 1365: 183 | 191; 8 x 1000
//    90 | 103; 40 x 300 85 | 121).
// TRINIX_PACKED_FWD = 0, 1, 2 forces pair, plain, wide (tuning and tests).
PackedShape packed_shape(const trinix_packed_args* a) {
  const int64_t n = a->n_seqs, blocks = (a->total_q / 128 + lmin(n, a->total_q) / 2) * a->nheads_q;
  const int D = packed_kernel_dim(a->head_dim);
  PackedShape s = PackedShape::kPlain;
  if (blocks <= 256 && a->total_k / n >= 256) s = PackedShape::kPair;
  else if (a->total_k / n >= 4096 && a->total_q * a->nheads_q / 256 >= 192) s = PackedShape::kWide;
  if (const char* env = getenv("TRINIX_PACKED_FWD")) {
    const int want = atoi(env);
    if (want >= 0 && want <= 2) s = (PackedShape)want;
  }
  if ((D == 256 && s == PackedShape::kPair) || (D != 128 && s == PackedShape::kWide)) s = PackedShape::kPlain;
  return s;
}

// Wavefronts per 32 rows (keys) of the fp32 kernels.  Measured, forward | forward with
// backward, us one, two: two wins wherever blocks are few or sequences short (8 heads of
// 128, 1090 rows 78, 44 | 219, 131; 12 heads of 64, 4 x 1024 109, 73 | 354, 302, 24 x 100
// 23, 18 | 83, 72; 16/4 heads of 128, 200 x 40 160, 124 | 616, 441) and loses where long
// sequences fill the chip (8 x 2048, 2112 blocks, 16 heads of 64 555, 580 | 2491, 2601, 16/4
// of 96 886, 1072 | 3928, 4289; even at 1560).
// TRINIX_PACKED_PAIRS = 1, 2 forces either (tuning and tests).
int fp32_wavefronts(const trinix_packed_args* a) {
  if (packed_kernel_dim(a->head_dim) == 256) return 1;
  if (const char* env = getenv("TRINIX_PACKED_PAIRS")) return atoi(env) == 1 ? 1 : 2;
  const int64_t blocks = (a->total_q / 128 + lmin(a->n_seqs, a->total_q) / 2) * a->nheads_q;
  return blocks > 1536 && a->total_k / a->n_seqs >= 1024 ? 1 : 2;
}

}  // namespace
}  // namespace trinix

using namespace trinix;

extern "C" int trinix_packed_fwd(const trinix_packed_args* a, void* stream) {
  const int rc = validate_packed(a, false);
  if (rc != TRINIX_OK) return rc;
  if (a->total_q == 0) return TRINIX_OK;
  PackedParams p = params(a);
  hipStream_t st = (hipStream_t)stream;
  const int C = packed_columns(a->head_dim);
  hipError_t e;
  p.rows16 = a->dtype == TRINIX_F32 && rows16(a->k, a->k_stride) && rows16(a->v, a->v_stride);
  const int64_t bytes = packed_chunk_bytes(a);
  if (bytes > 0 && a->workspace && a->workspace_bytes >= bytes && ((uintptr_t)a->workspace & 15) == 0) {
    p.n_chunks = packed_key_chunks(a);
    p.part = (float*)a->workspace;
    p.part_lse = p.part + (int64_t)p.n_chunks * p.Hq * p.Tq * packed_lds_dim(C);
    const int grid = (int)(use_list(p, a, C == 256 ? kRows128 : kRows64) * p.Hq);
    e = a->dtype == TRINIX_F32    ? launch_packed_chunks_f32(p, C, grid, st)
        : a->dtype == TRINIX_BF16 ? launch_packed_chunks_bf16(p, C, grid, st)
                                  : launch_packed_chunks_f16(p, C, grid, st);
  } else if (a->dtype == TRINIX_F32) {
    const int ks = fp32_wavefronts(a);
    e = launch_packed_fwd_f32(p, C, ks, (int)(use_list(p, a, ks == 2 ? kRows64 : kRows128) * p.Hq), st);
  } else {
    const PackedShape shape = packed_shape(a);
    const int grid = (int)(use_list(p, a, kListOf[(int)shape]) * p.Hq);
    e = a->dtype == TRINIX_BF16 ? launch_packed_fwd_bf16(p, C, shape, grid, st) : launch_packed_fwd_f16(p, C, shape, grid, st);
  }
  return e == hipSuccess ? TRINIX_OK : TRINIX_ERR_LAUNCH;
}

extern "C" int trinix_packed_bwd(const trinix_packed_args* a, void* stream) {
  const int rc = validate_packed(a, true);
  if (rc != TRINIX_OK) return rc;
  PackedParams p = params(a);
  hipStream_t st = (hipStream_t)stream;
  const int C = packed_columns(a->head_dim), D = packed_lds_dim(C);
  const bool f32 = a->dtype == TRINIX_F32, bf = a->dtype == TRINIX_BF16;
  hipError_t e = hipSuccess;
  p.rows16 = f32 && rows16(a->q, a->q_stride) && rows16(a->dout, a->dout_stride);
  p.rows16_q = f32 && rows16(a->k, a->k_stride) && rows16(a->v, a->v_stride);
  if (a->total_q > 0) {
    e = f32 ? launch_delta<BF16, true>(p, D, st) : bf ? launch_delta<BF16, false>(p, D, st) : launch_delta<F16, false>(p, D, st);
    if (e != hipSuccess) return TRINIX_ERR_LAUNCH;
  }
  p.Tk = (int)a->total_k;
  p.n_split = packed_head_splits(a);
  p.part = (float*)a->workspace;
  const int ks = f32 ? fp32_wavefronts(a) : 1;
  const bool pairs = f32 ? ks == 2 : C != 256;  // (16-bit: of keys only)
  const int n_q = (int)(use_list(p, a, ks == 2 ? kRows64 : kRows128) * p.Hq);
  p.items_q = p.items;
  const int n_kv = (int)(use_list(p, a, pairs ? kKeys64 : kKeys128) * p.Hkv * p.n_split);
  if (n_kv + n_q > 0)
    e = f32  ? launch_packed_bwd_f32(p, C, ks, n_kv, n_q, st)
        : bf ? launch_packed_bwd_bf16(p, C, n_kv, n_q, st)
             : launch_packed_bwd_f16(p, C, n_kv, n_q, st);
  if (e == hipSuccess && p.n_split > 1 && a->total_k > 0)
    e = f32 ? launch_sum<BF16, true>(p, D, st) : bf ? launch_sum<BF16, false>(p, D, st) : launch_sum<F16, false>(p, D, st);
  return e == hipSuccess ? TRINIX_OK : TRINIX_ERR_LAUNCH;
}
