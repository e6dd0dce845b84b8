// Packed-sequence attention on the operand policies of attn_ops.h: fp32 on fp32
// matrix products, the gradients of 16-bit types at head_dim 256 with their
// coefficients in two terms:
//   packed_fwd_f32      128 query rows of one sequence and head, 32 per wavefront,
//                       over 32-key tiles: S^T = K Q^T, online softmax, O^T += V^T P^T;
//   packed_bwd_generic  in one launch (no atomics)
//     dK, dV  128 keys of one sequence and KV head, 32 per wavefront, over 32-row
//             tiles of Q and dO of every head of the group: dV += P^T dO,
//             dZ = P (dO V^T - delta), dK += dZ^T Q;
//     dQ      128 query rows as in the forward: dQ += dZ K.
// KS = 2: 64 of them, two wavefronts per 32 taking alternate tiles, joined through LDS
// at the end: half the chain of tiles, which bounds small batches.  The dQ items come
// behind those of dK and dV and fill the CUs that these leave idle (us, forward with
// backward, launches of their own | one: fp32, 8 heads of 80, 1090 rows 143 | 103, of 128
// 183 | 131; bf16 of 256, 16/4 heads 4 x 1000 413 | 359, 8/4 2048 + 1000 340 | 294; two
// wavefronts per 32 at 256 then give nothing).  Tiles go global -> LDS asynchronously
// into two slots, one barrier per step.
// What bounds it: the fp32 products, 64 cycles for each 32x32x2.  8 x 2048 rows, 16/4
// heads of 96: forward 116, all 118 TFLOP/s of 2 and 2 + 7 products, where the library's
// large fp32 product reaches 154 on the same card.
#pragma once
#include <cfloat>

#include "attn_bwd_generic.h"
#include "attn_ops.h"
#include "attn_packed.h"

namespace trinix {

// SPLIT: p.n_chunks workgroups share the block's keys (see packed_fwd16).
template <class O, int OCC, int KS, bool SPLIT>
__global__ __launch_bounds__(256, OCC) void packed_fwd_f32(const PackedParams p) {
  using Store = typename O::Store;
  constexpr int NW = 4, BM = NW * 32 / KS, D = O::kD, DB = O::DB, TILE = kTileRows * D * (int)sizeof(Store);
  __shared__ __attribute__((aligned(1024))) char lds_k[2][KS * TILE];
  __shared__ __attribute__((aligned(1024))) char lds_v[2][KS * TILE];
  const int per_chunk = SPLIT ? (int)gridDim.x / p.n_chunks : 1, chunk = SPLIT ? (int)blockIdx.x / per_chunk : 0;
  const PackedBlock w(p, p.items, SPLIT ? packed_chunk_block((int)blockIdx.x, chunk, per_chunk) : (int)blockIdx.x, p.Hkv, p.G);
  if (w.blk < 0) return;
  const int m0 = w.blk * BM;
  int t_lo, t_hi;
  bwd_key_tiles(m0, BM, w.lq, w.lk, w.dlo, w.dhi, kTileRows, t_lo, t_hi);
  PackedChunks chunks{0, 1};
  if constexpr (SPLIT) {
    chunks = packed_chunks(t_hi - t_lo, kTileRows, p.n_chunks, w.total, p.Hq, kPackedF32Slots<D>);
    if (chunk >= chunks.n) return;
    t_lo += chunk * chunks.per;
    t_hi = min(t_hi, t_lo + chunks.per);
  }
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hq = w.h, hkv = hq / p.G, kp = wave % KS, iw0 = m0 + wave / KS * 32, i = iw0 + r, ic = min(i, w.lq - 1);
  const PackedRange kseen = w.keys();
  const bool wide = p.rows16 != 0;

  const O ops(lane, 0);
  const typename O::Frag qf = load_frag_cols<O>((const Store*)p.q + (int64_t)(w.q0 + ic) * p.q_ss + hq * p.q_sh, g, p.d);
  const float slope_l2 = p.alibi ? -p.alibi[hq * p.al_sh] * kLog2e : 0.f;
  const int off = w.lk - w.lq;
  f32x16_t acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = (f32x16_t){};
  float m_run = -INFINITY, l_run = 0.f;

  const Store* kbase = (const Store*)p.k + (int64_t)w.k0 * p.k_ss + hkv * p.k_sh;
  const Store* vbase = (const Store*)p.v + (int64_t)w.k0 * p.v_ss + hkv * p.v_sh;
  const PackedCopy<O, NW> copy_k(p.k_ss, wave, lane, p.d), copy_v(p.v_ss, wave, lane, p.d);
  auto load = [&](int t, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < KS; ++u)
      if (t + u < t_hi) {
        copy_k(kbase, (t + u) * kTileRows, kseen, lds_k[slot] + u * TILE, wide);
        copy_v(vbase, (t + u) * kTileRows, kseen, lds_v[slot] + u * TILE, wide);
      }
  };
  auto block = [&](int t, int slot) __attribute__((always_inline)) {
    const int n0 = t * kTileRows;
    if (!w.live(iw0, 32, n0, 32)) return;
    const f32x16_t s = ops.scores(lds_k[slot] + kp * TILE, qf);
    float x[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) x[v] = s[v] * p.scale_log2;
    if (p.alibi) {
      const float fi = (float)(i + off - n0 - 4 * g);
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = __builtin_fmaf(fabsf(fi - (float)((v >> 2) * 8 + (v & 3))), slope_l2, x[v]);
    }
    if (!w.full(iw0, 32, n0, 32)) {
      const Span ks = w.keys_of(i);
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = ks.ok(n0 + (v >> 2) * 8 + g * 4 + (v & 3)) ? x[v] : -INFINITY;
    }
    float mx = x[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) mx = fmaxf(mx, x[v]);
    mx = xlane_max(mx);
    if (wave_any(mx > m_run)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[db] *= alpha;
      m_run = m_new;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;  // all keys so far hidden: exp2(-inf - 0) = 0
    float sum = 0.f;  // within the tile first: one rounding of the running sum per tile
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      x[v] = __builtin_amdgcn_exp2f(x[v] - m_use);
      sum += x[v];
    }
    l_run += sum;
    ops.accum(acc, lds_v[slot] + kp * TILE, x);
  };

  if (t_lo < t_hi) load(t_lo, 0);
  auto step = [&](auto slot_c, int t) __attribute__((always_inline)) {
    constexpr int SL = decltype(slot_c)::value;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (t + KS < t_hi) load(t + KS, 1 - SL);
    if (t + kp < t_hi) block(t + kp, SL);
  };
  for (int t = t_lo; t < t_hi; t += 2 * KS) {
    step(std::integral_constant<int, 0>{}, t);
    if (t + KS < t_hi) step(std::integral_constant<int, 1>{}, t + KS);
  }

  float l = xlane_sum(l_run);
  if constexpr (KS == 2) {
    // the second wavefront's (max, sum, O) merge into the first's
    constexpr int WORDS = DB * 16 + 2;
    static_assert(2 * WORDS * 64 * 4 <= 2 * KS * TILE, "exchange fits the K tiles");
    float* x = (float*)&lds_k[0][0] + wave / KS * WORDS * 64 + lane;
    __syncthreads();
    if (kp == 1) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) x[(db * 16 + v) * 64] = acc[db][v];
      x[DB * 16 * 64] = m_run;
      x[(DB * 16 + 1) * 64] = l;
    }
    __syncthreads();
    if (kp == 1) return;
    const float m1 = x[DB * 16 * 64], l1 = x[(DB * 16 + 1) * 64];
    const float m_new = fmaxf(m_run, m1), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float a0 = __builtin_amdgcn_exp2f(m_run - m_use), a1 = __builtin_amdgcn_exp2f(m1 - m_use);
    l = l * a0 + l1 * a1;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[db][v] = acc[db][v] * a0 + x[(db * 16 + v) * 64] * a1;
    m_run = m_new;
  }
  if (i >= w.lq) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;  // a row that sees no key: 0
  const int64_t row = w.q0 + i;
  if (SPLIT && chunks.n > 1) {
    const int64_t at = ((int64_t)chunk * p.Hq + hq) * p.Tq + row;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int vq = 0; vq < 4; ++vq)
        *(f32x4_t*)(p.part + at * D + db * 32 + vq * 8 + g * 4) =
            (f32x4_t){acc[db][vq * 4] * inv, acc[db][vq * 4 + 1] * inv, acc[db][vq * 4 + 2] * inv, acc[db][vq * 4 + 3] * inv};
    if (g == 0) p.part_lse[at] = l > 0.f ? m_run + log2f(l) : -INFINITY;
    return;
  }
  Store* orow = (Store*)p.o + row * p.o_ss + hq * p.o_sh;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int vq = 0; vq < 4; ++vq)
      if (db * 32 + vq * 8 + g * 4 < p.d)
        O::store4(orow, db * 32 + vq * 8 + g * 4, acc[db][vq * 4] * inv, acc[db][vq * 4 + 1] * inv, acc[db][vq * 4 + 2] * inv,
                  acc[db][vq * 4 + 3] * inv);
  if (p.lse && g == 0) p.lse[(int64_t)hq * p.Tq + row] = l > 0.f ? (m_run + log2f(l)) * kLn2 : -INFINITY;
}

// LDS of either part, in bytes: two slots of two KS-tile operands, and rows of two floats.
template <class O, int KS>
constexpr int kGenericTiles = KS * kTileRows * O::kD * (int)sizeof(typename O::Store);
template <class O, int KS>
constexpr int kGenericLds = 4 * kGenericTiles<O, KS> + 4 * KS * kTileRows * 4;

// dK and dV.  HS workgroups share a key block, each summing D / HS of the columns.
template <class O, int HS, int KS>
__device__ __forceinline__ void generic_dkdv_body(const PackedParams& p, int wg, char* pool) {
  using Store = typename O::Store;
  constexpr int NW = 4, BK = NW * 32 / KS, D = O::kD, DB = O::DB / HS, TILE = kTileRows * D * (int)sizeof(Store);
  char(*const lds_q)[KS * TILE] = (char(*)[KS * TILE]) pool;
  char(*const lds_o)[KS * TILE] = lds_q + 2;
  float(*const lds_l)[KS * kTileRows] = (float(*)[KS * kTileRows])(lds_o + 2);
  float(*const lds_d)[KS * kTileRows] = lds_l + 2;
  const PackedBlock w(p, p.items, wg / HS, p.Hkv * p.n_split, 1);
  if (w.blk < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const PackedHeads hd(p, w.h);
  const int hkv = hd.hkv, kb0 = w.blk * BK, db0 = (wg % HS) * DB;
  const int kp = wave % KS, j0 = kb0 + wave / KS * 32, j = j0 + (lane & 31);
  const PackedRange kseen = w.keys(), qseen = w.rows();
  const int jc = min(max(j, kseen.lo), kseen.hi);
  const bool wide = p.rows16 != 0;
  const int off = w.lk - w.lq;

  int qt_lo, qt_hi;
  bwd_query_tiles(kb0, BK, w.lq, w.lk, w.dlo, w.dhi, kTileRows, qt_lo, qt_hi);
  const int nqt = qt_hi - qt_lo;
  const int n_items = nqt > 0 ? (hd.gh1 - hd.gh0) * nqt : 0;  // item = (q-head of the group, query tile)

  const O ops(lane, db0);
  const typename O::Frag kf = load_frag_cols<O>((const Store*)p.k + (int64_t)(w.k0 + jc) * p.k_ss + hkv * p.k_sh, g, p.d);
  const typename O::Frag vf = load_frag_cols<O>((const Store*)p.v + (int64_t)(w.k0 + jc) * p.v_ss + hkv * p.v_sh, g, p.d);
  f32x16_t dk[DB], dv[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dk[db] = dv[db] = (f32x16_t){};
  ZScale<O> zs;

  const PackedCopy<O, NW> copy_q(p.q_ss, wave, lane, p.d), copy_o(p.do_ss, wave, lane, p.d);
  float lse_next = 0.f, del_next = 0.f;
  auto load_step = [&](int it, int slot) __attribute__((always_inline)) {  // items it .. it + KS - 1
#pragma unroll
    for (int u = 0; u < KS; ++u) {
      if (it + u >= n_items) break;
      const int hq = hkv * p.G + hd.gh0 + (it + u) / nqt, i0 = (qt_lo + (it + u) % nqt) * kTileRows;
      copy_q((const Store*)p.q + (int64_t)w.q0 * p.q_ss + hq * p.q_sh, i0, qseen, lds_q[slot] + u * TILE, wide);
      copy_o((const Store*)p.dout + (int64_t)w.q0 * p.do_ss + hq * p.do_sh, i0, qseen, lds_o[slot] + u * TILE, wide);
      if (tid / kTileRows == u) {
        const int64_t ro = (int64_t)hq * p.Tq + w.q0 + min(i0 + tid % kTileRows, w.lq - 1);
        lse_next = p.lse[ro];
        del_next = p.delta[ro];
      }
    }
  };
  // a row that sees no key has lse -inf and every score -inf: the finite floor
  // keeps exp2(score - lse) at 0 instead of exp2(-inf + inf) = NaN
  auto write_rows = [&](int slot) __attribute__((always_inline)) {
    if (tid < KS * kTileRows) {
      lds_l[slot][tid] = fmaxf(lse_next * kLog2e, -0.5f * FLT_MAX) - O::kPShift;
      lds_d[slot][tid] = del_next;
    }
  };
  auto block = [&](int it, int slot) __attribute__((always_inline)) {
    const int hq = hkv * p.G + hd.gh0 + it / nqt, i0 = (qt_lo + it % nqt) * kTileRows;
    if (!w.live(i0, 32, j0, 32)) return;
    const char *q_lds = lds_q[slot] + kp * TILE, *o_lds = lds_o[slot] + kp * TILE;
    const f32x16_t s = ops.scores(q_lds, kf);
    float x[16];
#pragma unroll
    for (int vq = 0; vq < 4; ++vq) {
      const f32x4_t l4 = *(const f32x4_t*)(&lds_l[slot][kp * kTileRows + vq * 8 + g * 4]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[vq * 4 + e] = __builtin_fmaf(s[vq * 4 + e], p.scale_log2, -l4[e]);
    }
    if (p.alibi) {
      const float slope_l2 = -p.alibi[hq * p.al_sh] * kLog2e;
      const float fj = (float)(j - off - (i0 + g * 4));
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = __builtin_fmaf(fabsf(fj - (float)((v >> 2) * 8 + (v & 3))), slope_l2, x[v]);
    }
    if (!w.full(i0, 32, j0, 32)) {
      int jo = j;  // (not held across the loop)
      asm volatile("" : "+v"(jo));
      const Span qs = w.rows_of(jo);
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = qs.ok(i0 + (v >> 2) * 8 + g * 4 + (v & 3)) ? x[v] : -INFINITY;
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) x[v] = __builtin_amdgcn_exp2f(x[v]);
    ops.accum(dv, o_lds, x);
    const f32x16_t dp = ops.scores(o_lds, vf);
#pragma unroll
    for (int vq = 0; vq < 4; ++vq) {
      const f32x4_t d4 = *(const f32x4_t*)(&lds_d[slot][kp * kTileRows + vq * 8 + g * 4]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[vq * 4 + e] *= dp[vq * 4 + e] - d4[e];
    }
    zs.apply(x, dk);
    ops.accum(dk, q_lds, x);
  };

  if (n_items > 0) {
    load_step(0, 0);
    write_rows(0);
  }
  auto step = [&](auto slot_c, int it) __attribute__((always_inline)) {
    constexpr int SL = decltype(slot_c)::value;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (it + KS < n_items) load_step(it + KS, 1 - SL);
    if (it + kp < n_items) block(it + kp, SL);
    if (it + KS < n_items) write_rows(1 - SL);
  };
  for (int it = 0; it < n_items; it += 2 * KS) {
    step(std::integral_constant<int, 0>{}, it);
    if (it + KS < n_items) step(std::integral_constant<int, 1>{}, it + KS);
  }

  float fv = exp2f(-O::kPShift), fk = p.scale * fv * zs.undo();
  if constexpr (KS == 2) {
    merge_pair<2 * KS * TILE>(dv, fv, (float*)&lds_q[0][0], wave / KS, kp, lane);
    merge_pair<2 * KS * TILE>(dk, fk, (float*)&lds_q[0][0], wave / KS, kp, lane);
    if (kp == 1) return;
    fv = fk = 1.f;
  }
  if (j >= w.lk) return;
  if (p.n_split > 1) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int vq = 0; vq < 4; ++vq) {
        const int d0 = (db0 + db) * 32 + vq * 8 + g * 4;
        *(f32x4_t*)(packed_partial(p, hd.split, 0, w.k0 + j, hkv, D) + d0) =
            (f32x4_t){dv[db][vq * 4] * fv, dv[db][vq * 4 + 1] * fv, dv[db][vq * 4 + 2] * fv, dv[db][vq * 4 + 3] * fv};
        *(f32x4_t*)(packed_partial(p, hd.split, 1, w.k0 + j, hkv, D) + d0) =
            (f32x4_t){dk[db][vq * 4] * fk, dk[db][vq * 4 + 1] * fk, dk[db][vq * 4 + 2] * fk, dk[db][vq * 4 + 3] * fk};
      }
    return;
  }
  Store* krow = (Store*)p.dk + (int64_t)(w.k0 + j) * p.dk_ss + hkv * p.dk_sh;
  Store* vrow = (Store*)p.dv + (int64_t)(w.k0 + j) * p.dv_ss + hkv * p.dv_sh;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int vq = 0; vq < 4; ++vq) {
      const int d0 = (db0 + db) * 32 + vq * 8 + g * 4;
      if (d0 >= p.d) continue;
      O::store4(vrow, d0, dv[db][vq * 4] * fv, dv[db][vq * 4 + 1] * fv, dv[db][vq * 4 + 2] * fv, dv[db][vq * 4 + 3] * fv);
      O::store4(krow, d0, dk[db][vq * 4] * fk, dk[db][vq * 4 + 1] * fk, dk[db][vq * 4 + 2] * fk, dk[db][vq * 4 + 3] * fk);
    }
}

template <class O, int HS, int KS>
__device__ __forceinline__ void generic_dq_body(const PackedParams& p, int wg, char* pool) {
  using Store = typename O::Store;
  constexpr int NW = 4, BM = NW * 32 / KS, D = O::kD, DB = O::DB / HS, TILE = kTileRows * D * (int)sizeof(Store);
  char(*const lds_k)[KS * TILE] = (char(*)[KS * TILE]) pool;
  char(*const lds_v)[KS * TILE] = lds_k + 2;
  const PackedBlock w(p, p.items_q, wg / HS, p.Hkv, p.G);
  if (w.blk < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hq = w.h, hkv = hq / p.G, m0 = w.blk * BM, kp = wave % KS, iw0 = m0 + wave / KS * 32, i = iw0 + r;
  const PackedRange kseen = w.keys(), qseen = w.rows();
  const int ic = min(max(i, qseen.lo), qseen.hi);
  const int db0 = (wg % HS) * DB, off = w.lk - w.lq;
  const bool wide = p.rows16_q != 0;

  const O ops(lane, db0);
  const typename O::Frag qf = load_frag_cols<O>((const Store*)p.q + (int64_t)(w.q0 + ic) * p.q_ss + hq * p.q_sh, g, p.d);
  const typename O::Frag of = load_frag_cols<O>((const Store*)p.dout + (int64_t)(w.q0 + ic) * p.do_ss + hq * p.do_sh, g, p.d);
  const int64_t ro = (int64_t)hq * p.Tq + w.q0 + min(i, w.lq - 1);
  const float lse2 = fmaxf(p.lse[ro] * kLog2e, -0.5f * FLT_MAX), dlt = p.delta[ro];  // (finite: see above)
  const float slope_l2 = p.alibi ? -p.alibi[hq * p.al_sh] * kLog2e : 0.f;
  f32x16_t acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = (f32x16_t){};
  ZScale<O> zs;

  int t_lo, t_hi;
  bwd_key_tiles(m0, BM, w.lq, w.lk, w.dlo, w.dhi, kTileRows, t_lo, t_hi);
  const Store* kbase = (const Store*)p.k + (int64_t)w.k0 * p.k_ss + hkv * p.k_sh;
  const Store* vbase = (const Store*)p.v + (int64_t)w.k0 * p.v_ss + hkv * p.v_sh;
  const PackedCopy<O, NW> copy_k(p.k_ss, wave, lane, p.d), copy_v(p.v_ss, wave, lane, p.d);
  auto load = [&](int t, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < KS; ++u)
      if (t + u < t_hi) {
        copy_k(kbase, (t + u) * kTileRows, kseen, lds_k[slot] + u * TILE, wide);
        copy_v(vbase, (t + u) * kTileRows, kseen, lds_v[slot] + u * TILE, wide);
      }
  };
  auto block = [&](int t, int slot) __attribute__((always_inline)) {
    const int n0 = t * kTileRows;
    if (!w.live(iw0, 32, n0, 32)) return;
    const f32x16_t s = ops.scores(lds_k[slot] + kp * TILE, qf);
    const f32x16_t dp = ops.scores(lds_v[slot] + kp * TILE, of);
    float x[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) x[v] = __builtin_fmaf(s[v], p.scale_log2, -lse2);
    if (p.alibi) {
      const float fi = (float)(i + off - n0 - 4 * g);
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = __builtin_fmaf(fabsf(fi - (float)((v >> 2) * 8 + (v & 3))), slope_l2, x[v]);
    }
    if (!w.full(iw0, 32, n0, 32)) {
      int io = i;
      asm volatile("" : "+v"(io));
      const Span ks = w.keys_of(io);
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = ks.ok(n0 + (v >> 2) * 8 + g * 4 + (v & 3)) ? x[v] : -INFINITY;
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) x[v] = __builtin_amdgcn_exp2f(x[v]) * (dp[v] - dlt);
    zs.apply(x, acc);
    ops.accum(acc, lds_k[slot] + kp * TILE, x);
  };

  if (t_lo < t_hi) load(t_lo, 0);
  auto step = [&](auto slot_c, int t) __attribute__((always_inline)) {
    constexpr int SL = decltype(slot_c)::value;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (t + KS < t_hi) load(t + KS, 1 - SL);
    if (t + kp < t_hi) block(t + kp, SL);
  };
  for (int t = t_lo; t < t_hi; t += 2 * KS) {
    step(std::integral_constant<int, 0>{}, t);
    if (t + KS < t_hi) step(std::integral_constant<int, 1>{}, t + KS);
  }

  float f = p.scale * zs.undo();
  if constexpr (KS == 2) {
    merge_pair<2 * KS * TILE>(acc, f, (float*)&lds_k[0][0], wave / KS, kp, lane);
    if (kp == 1) return;
    f = 1.f;
  }
  if (i >= w.lq) return;
  Store* row = (Store*)p.dq + (int64_t)(w.q0 + i) * p.dq_ss + hq * p.dq_sh;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int vq = 0; vq < 4; ++vq) {
      const int d0 = (db0 + db) * 32 + vq * 8 + g * 4;
      if (d0 < p.d)
        O::store4(row, d0, acc[db][vq * 4] * f, acc[db][vq * 4 + 1] * f, acc[db][vq * 4 + 2] * f, acc[db][vq * 4 + 3] * f);
    }
}

// Workgroups [0, n_kv * HSK): dK and dV of p.items; behind them dQ of p.items_q.
template <class O, int OCC, int HSK, int HSQ, int KS>
__global__ __launch_bounds__(256, OCC) void packed_bwd_generic(const PackedParams p, int n_kv) {
  __shared__ __attribute__((aligned(1024))) char pool[kGenericLds<O, KS>];
  const int wg = (int)blockIdx.x;
  if (wg < n_kv * HSK) generic_dkdv_body<O, HSK, KS>(p, wg, pool);
  else generic_dq_body<O, HSQ, KS>(p, wg - n_kv * HSK, pool);
}
template <class O, int OCC, int HSK, int HSQ, int KS>
hipError_t launch_packed_bwd_g(const PackedParams& p, int n_kv, int n_q, hipStream_t st) {
  return launch_kernel(&packed_bwd_generic<O, OCC, HSK, HSQ, KS>, dim3((unsigned)(n_kv * HSK + n_q * HSQ)), dim3(256), 0, st, p,
                       n_kv);
}

}  // namespace trinix
