// Gradients of packed-sequence attention, 16-bit types at head_dims up to 128, in one
// launch (no atomics) of 4-wavefront workgroups, two per CU:
//   dK, dV  64 keys of one sequence and KV head, a pair of wavefronts per 32 keys: the
//           first computes S = Q K^T, P = exp(scale S - lse) and dV^T += dO^T P, hands P in
//           fp32 to the second through LDS, which runs a step behind on dP = dO V^T, dZ = P
//           (dP - delta) and dK^T += Q^T dZ.  Both walk every head of the group and
//           every query tile of the band; a pair shares a SIMD, so that one's exponentials
//           run beside the other's products.  Q, dO tiles rotate through three LDS slots, P
//           through two; one barrier per tile;
//   dQ      128 query rows of one sequence and head, 32 per wavefront, over 32-key
//           tiles: S^T, dP^T, dZ^T in registers, dQ^T += K^T dZ^T.
// The dK, dV items come first, longest first, and the dQ items, whose chains are
// shorter by the heads of a group, fill the CUs that these leave idle: the longest key
// block of a 4096-row sequence in a batch of 8192 rows has 1.4 times the work of an
// average CU.  Forward and backward, bf16 causal, us with 4-wavefront | 8-wavefront
// workgroups: 4096 + 2047 + 1000 + 3 short, 32/8 heads of 128 1065 | 1089; 40 x 300 434 |
// 497; 8 documents of 4096 rows, 12 heads of 64 72 | 88; 8192 rows 2880 | 2933 (dK, dV and
// dQ in kernels of their own, one wavefront per 32 keys, 3290).  A 32x32 block of pairs
// takes 5 + 4 products of D; 8192 rows run at 1041 TFLOP/s of them, where the library's
// large bf16 product reaches 1240 on the same card.
//
// Roundings: P enters dV in one 16-bit term (the error of dV: 1.2 to 1.4 times that of
// rounding dV alone); dZ is formed from the fp32 P and enters dK and dQ in two terms x =
// hi + lo, 16 (bf16) or 21 (fp16) significant bits: with one they err 1.45 to 1.65 times
// as much as from their own rounding, as dZ cancels over a row.
#pragma once
#include <cfloat>

#include "attn_bwd_generic.h"
#include "attn_ops.h"
#include "attn_packed.h"

namespace trinix {

// LDS of the launch, in bytes: the larger of the two parts.
template <int D>
struct PackedBwdLds {
  static constexpr int NG = 2, NSL = 3;  // dK, dV: pairs, tile slots
  static constexpr int kTile = kTileRows * D * 2, kP = NG * 64 * 64;
  static constexpr int kKv = NSL * 2 * kTile + 2 * kP + NSL * 2 * kTileRows * 4;
  static constexpr int KT = D == 64 ? 2 : 1, kDq = 2 * 2 * KT * kTile;  // dQ: tiles per step
  static constexpr int kBytes = kKv > kDq ? kKv : kDq;
};

template <class E, int D, int C>
__device__ __forceinline__ void packed_dkdv_body(const PackedParams& p, const PackedBlock& w, char* pool) {
  using O = Ops16<E, D, C>;
  using L = PackedBwdLds<D>;
  constexpr int NG = L::NG, NW = 2 * NG, BK = NG * 32, BQ = kTileRows, NSL = L::NSL;
  constexpr int DS = C / 16, DB = C / 32, UPR = D / 8, LPW = BQ * UPR / (64 * NW);
  constexpr int RPF = 4, TPF = 2;  // row and transpose reads ahead of their MFMA
  static_assert(LPW >= 1 && BQ * UPR % (64 * NW) == 0, "tile shape");
  char* const lds_q = pool;
  char* const lds_o = lds_q + NSL * L::kTile;
  char* const lds_p = lds_o + NSL * L::kTile;
  float* const lds_l = (float*)(lds_p + 2 * L::kP);
  float* const lds_d = lds_l + NSL * BQ;

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave % NG;
  const PackedHeads hd(p, w.h);
  const int hkv = hd.hkv, kb0 = w.blk * BK, j0 = kb0 + kg * 32, j = j0 + (lane & 31);
  const PackedRange kseen = w.keys(), qseen = w.rows();
  const int jc = min(max(j, kseen.lo), kseen.hi);
  const int off = w.lk - w.lq;
  const Span qspan = w.rows_of(j);

  int qt_lo, qt_hi;
  bwd_query_tiles(kb0, BK, w.lq, w.lk, w.dlo, w.dhi, BQ, qt_lo, qt_hi);
  qt_lo = __builtin_amdgcn_readfirstlane(qt_lo), qt_hi = __builtin_amdgcn_readfirstlane(qt_hi);
  const int n_items = qt_hi > qt_lo ? (hd.gh1 - hd.gh0) * (qt_hi - qt_lo) : 0;
  struct Item {
    int gh, qt;  // head of the group, query tile
  };
  auto next_item = [&](Item it) __attribute__((always_inline)) {
    return it.qt + 1 < qt_hi ? Item{it.gh, it.qt + 1} : Item{it.gh + 1, qt_lo};
  };

  // copies of an item: Q and dO rows (16-byte units, swizzled); wave 0 carries lse and
  // delta through registers and writes them at the step's end
  const uint32_t wave_lds = __builtin_amdgcn_readfirstlane((uint32_t)(wave * LPW * 1024));
  auto load_rows = [&](const uint16_t* base, int64_t ss, char* tile, int i0) __attribute__((always_inline)) {
    const uint64_t gb = uniform_ptr((const char*)base + (int64_t)i0 * ss * 2);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)tile + wave_lds;
    const PackedRange t = packed_tile_range(qseen, i0);
#pragma unroll
    for (int l = 0; l < LPW; ++l) {
      const int row = tile_copy_row(wave, LPW, l, lane, UPR);
      const uint32_t src = (uint32_t)min(max(row, t.lo), t.hi), unit = (uint32_t)min((lane % UPR) ^ swz_kt<D>(row), p.d / 8 - 1);
      dma_16b_s(tile_copy_offset(src, ss, unit), gb, __builtin_amdgcn_readfirstlane(lds0 + l * 1024));
    }
  };
  float lse_pend = 0.f, del_pend = 0.f;
  int row_dst = -1;
  auto load_item = [&](Item it, auto slot_c) __attribute__((always_inline)) {
    constexpr int SL = decltype(slot_c)::value;
    const int hq = hkv * p.G + it.gh, i0 = it.qt * BQ;
    load_rows((const uint16_t*)p.q + (int64_t)w.q0 * p.q_ss + hq * p.q_sh, p.q_ss, lds_q + SL * L::kTile, i0);
    load_rows((const uint16_t*)p.dout + (int64_t)w.q0 * p.do_ss + hq * p.do_sh, p.do_ss, lds_o + SL * L::kTile, i0);
    if (wave == 0 && lane < BQ) {
      const int64_t at = (int64_t)hq * p.Tq + w.q0 + min(i0 + lane, w.lq - 1);
      lse_pend = p.lse[at];
      del_pend = p.delta[at];
      row_dst = SL * BQ + lane;
    }
  };
  // (a row that sees no key has lse -inf and every score -inf: the finite floor keeps
  // exp2(score - lse) at 0 instead of exp2(-inf + inf) = NaN)
  auto write_rows = [&]() __attribute__((always_inline)) {
    if (wave == 0 && row_dst >= 0) {
      lds_l[row_dst] = fmaxf(lse_pend * kLog2e, -0.5f * FLT_MAX) - O::kPShift;
      lds_d[row_dst] = del_pend;
      row_dst = -1;
    }
  };
  const Tile16Reader<D> rd(lane, 0);
  auto p_slot = [&](int ps, int vq) __attribute__((always_inline)) {
    return (f32x4_t*)(lds_p + ps * L::kP) + (kg * 4 + vq) * 64 + lane;
  };

  // One of the pair: operand rows, the step loop, the epilogue.  Both run the same
  // steps and so the same barriers.
  auto run = [&](auto second_c) __attribute__((always_inline)) {
    constexpr bool SB = decltype(second_c)::value;  // dK
    const typename O::Frag br =
        SB ? load_frag_cols<O>((const uint16_t*)p.v + (int64_t)(w.k0 + jc) * p.v_ss + hkv * p.v_sh, g, p.d)
           : load_frag_cols<O>((const uint16_t*)p.k + (int64_t)(w.k0 + jc) * p.k_ss + hkv * p.k_sh, g, p.d);
    f32x16_t acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = (f32x16_t){};
    ZScale<O> zs;
    auto scores = [&](const char* tile) __attribute__((always_inline)) {
      f32x16_t s = {};
      u32x4_t a[DS];
#pragma unroll
      for (int k = 0; k < RPF; ++k) a[k] = rd.row(tile, k);
#pragma unroll
      for (int k = 0; k < DS; ++k) {
        if (k + RPF < DS) a[k + RPF] = rd.row(tile, k + RPF);
        s = E::mfma(a[k], br.r[k], s);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, RPF, 0);
#pragma unroll
      for (int k = 0; k < DS; ++k) {
        if (k + RPF < DS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      return s;
    };
    // acc += tile^T x, x in NT 16-bit terms; the first transpose reads (t0) were issued ahead
    auto grad = [&](const char* tile, const float(&x)[16], const u32x4_t(&t0)[TPF]) __attribute__((always_inline)) {
      constexpr int NT = SB ? 2 : 1, NM = 2 * DB;
      u32x4_t b[NT][2];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float x0 = x[kk * 8 + 2 * c], x1 = x[kk * 8 + 2 * c + 1];
          const uint32_t h = E::pack(x0, x1);
          b[0][kk][c] = h;
          if constexpr (NT == 2) b[1][kk][c] = E::pack(x0 - E::lo(h), x1 - E::hi(h));
        }
      __builtin_amdgcn_s_setprio(1);
      u32x4_t a[NM];
#pragma unroll
      for (int m = 0; m < TPF; ++m) a[m] = t0[m];
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        if (m + TPF < NM) a[m + TPF] = rd.tr(tile, (m + TPF) / 2, (m + TPF) % 2);
#pragma unroll
        for (int t = NT - 1; t >= 0; --t) acc[m / 2] = E::mfma(a[m], b[t][m % 2], acc[m / 2]);
      }
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        if (m + TPF < NM) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, NT, 0);
      }
      __builtin_amdgcn_s_setprio(0);
    };
    auto stage_a = [&](Item it, auto sl_c, auto ps_c) __attribute__((always_inline)) {
      constexpr int SL = decltype(sl_c)::value, PS = decltype(ps_c)::value;
      const int hq = hkv * p.G + it.gh;
      const int i0 = it.qt * BQ;
      if (!w.live(i0, 32, j0, 32)) return;
      const char *q = lds_q + SL * L::kTile, *o = lds_o + SL * L::kTile;
      const float* l = lds_l + SL * BQ;
      __builtin_amdgcn_s_setprio(1);
      const f32x16_t s = scores(q);
      u32x4_t t0[TPF];
#pragma unroll
      for (int m = 0; m < TPF; ++m) t0[m] = rd.tr(o, m / 2, m % 2);
      __builtin_amdgcn_s_setprio(0);
      float x[16];
#pragma unroll
      for (int vq = 0; vq < 4; ++vq) {
        const f32x4_t l4 = *(const f32x4_t*)(l + vq * 8 + g * 4);
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
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = qspan.ok(i0 + (v >> 2) * 8 + g * 4 + (v & 3)) ? x[v] : -INFINITY;
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = __builtin_amdgcn_exp2f(x[v]);
#pragma unroll
      for (int vq = 0; vq < 4; ++vq) *p_slot(PS, vq) = (f32x4_t){x[vq * 4], x[vq * 4 + 1], x[vq * 4 + 2], x[vq * 4 + 3]};
      grad(o, x, t0);
    };
    auto stage_b = [&](Item it, auto sl_c, auto ps_c) __attribute__((always_inline)) {
      constexpr int SL = decltype(sl_c)::value, PS = decltype(ps_c)::value;
      const int i0 = it.qt * BQ;
      if (!w.live(i0, 32, j0, 32)) return;  // (as the first of the pair: P was written)
      const char *q = lds_q + SL * L::kTile, *o = lds_o + SL * L::kTile;
      const float* dl = lds_d + SL * BQ;
      __builtin_amdgcn_s_setprio(1);
      const f32x16_t dp = scores(o);
      u32x4_t t0[TPF];
#pragma unroll
      for (int m = 0; m < TPF; ++m) t0[m] = rd.tr(q, m / 2, m % 2);
      __builtin_amdgcn_s_setprio(0);
      float z[16];
#pragma unroll
      for (int vq = 0; vq < 4; ++vq) {
        const f32x4_t p4 = *p_slot(PS, vq), d4 = *(const f32x4_t*)(dl + vq * 8 + g * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[vq * 4 + e] = p4[e] * (dp[vq * 4 + e] - d4[e]);
      }
      zs.apply(z, acc);
      grad(q, z, t0);
    };
    // Step s: the first on item s (tile slot s % 3, P slot s % 2), the second on item s
    // - 1, item s + 1 loading into slot (s + 1) % 3.  The barrier at its top is where
    // item s has landed, P of item s - 1 is written and slot (s + 1) % 3 is free.
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    Item ia{hd.gh0, qt_lo}, ib = ia;
    if (n_items > 0) load_item(ia, I0{});
    write_rows();
    auto step = [&](auto sa_c, auto pa_c, int s) __attribute__((always_inline)) {
      constexpr int SA = decltype(sa_c)::value, PA = decltype(pa_c)::value;
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      const Item in = next_item(ia);
      if (s + 1 < n_items) load_item(in, std::integral_constant<int, (SA + 1) % NSL>{});
      if constexpr (!SB) {
        if (s < n_items) stage_a(ia, sa_c, pa_c);
        write_rows();
      } else {
        if (s > 0) stage_b(ib, std::integral_constant<int, (SA + NSL - 1) % NSL>{}, std::integral_constant<int, 1 - PA>{});
      }
      ib = ia;
      ia = in;
    };
    for (int s = 0; s <= n_items; s += 6) {
      step(I0{}, I0{}, s);
      if (s + 1 <= n_items) step(I1{}, I1{}, s + 1);
      if (s + 2 <= n_items) step(I2{}, I0{}, s + 2);
      if (s + 3 <= n_items) step(I0{}, I1{}, s + 3);
      if (s + 4 <= n_items) step(I1{}, I0{}, s + 4);
      if (s + 5 <= n_items) step(I2{}, I1{}, s + 5);
    }
    if (j >= w.lk) return;
    uint16_t* row = SB ? (uint16_t*)p.dk + (int64_t)(w.k0 + j) * p.dk_ss + hkv * p.dk_sh
                       : (uint16_t*)p.dv + (int64_t)(w.k0 + j) * p.dv_ss + hkv * p.dv_sh;
    const float f = exp2f(-O::kPShift) * (SB ? p.scale * zs.undo() : 1.f);
    if (p.n_split > 1) {
      float* part = packed_partial(p, hd.split, SB ? 1 : 0, w.k0 + j, hkv, D);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int vq = 0; vq < 4; ++vq)
          *(f32x4_t*)(part + db * 32 + vq * 8 + g * 4) =
              (f32x4_t){acc[db][vq * 4] * f, acc[db][vq * 4 + 1] * f, acc[db][vq * 4 + 2] * f, acc[db][vq * 4 + 3] * f};
      return;
    }
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int vq = 0; vq < 4; ++vq)
        if (db * 32 + vq * 8 < p.d)
          O::store4(row, db * 32 + vq * 8 + g * 4, acc[db][vq * 4] * f, acc[db][vq * 4 + 1] * f, acc[db][vq * 4 + 2] * f,
                    acc[db][vq * 4 + 3] * f);
  };
  if (wave >= NG) run(std::true_type{});
  else run(std::false_type{});
}

template <class E, int D, int C>
__device__ __forceinline__ void packed_dq_body(const PackedParams& p, const PackedBlock& w, char* pool) {
  using O = Ops16<E, D, C>;
  using L = PackedBwdLds<D>;
  constexpr int NG = L::NG, BM = NG * 64, DB = C / 32, TILE = kTileRows * D * 2, NT = L::KT;  // tiles per step
  char* const lds_k = pool;
  char* const lds_v = pool + 2 * NT * TILE;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hq = w.h, hkv = hq / p.G, m0 = w.blk * BM, iw0 = m0 + wave * 32, i = iw0 + r;
  const PackedRange kseen = w.keys(), qseen = w.rows();
  const int ic = min(max(i, qseen.lo), qseen.hi);
  const int off = w.lk - w.lq;

  const O ops(lane, 0);
  const typename O::Frag qf = load_frag_cols<O>((const uint16_t*)p.q + (int64_t)(w.q0 + ic) * p.q_ss + hq * p.q_sh, g, p.d);
  const typename O::Frag of = load_frag_cols<O>((const uint16_t*)p.dout + (int64_t)(w.q0 + ic) * p.do_ss + hq * p.do_sh, g, p.d);
  const int64_t ro = (int64_t)hq * p.Tq + w.q0 + min(i, w.lq - 1);
  const float lse2 = fmaxf(p.lse[ro] * kLog2e, -0.5f * FLT_MAX), dlt = p.delta[ro];  // (finite: see write_rows)
  const float slope_l2 = p.alibi ? -p.alibi[hq * p.al_sh] * kLog2e : 0.f;
  f32x16_t acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = (f32x16_t){};
  ZScale<O> zs;

  int t_lo, t_hi;
  bwd_key_tiles(m0, BM, w.lq, w.lk, w.dlo, w.dhi, kTileRows, t_lo, t_hi);
  t_lo = __builtin_amdgcn_readfirstlane(t_lo), t_hi = __builtin_amdgcn_readfirstlane(t_hi);
  // half of the wavefronts copy K, the others V
  const bool cv = wave >= NG;
  const int64_t css = cv ? p.v_ss : p.k_ss;
  const uint16_t* cbase = cv ? (const uint16_t*)p.v + (int64_t)w.k0 * p.v_ss + hkv * p.v_sh
                             : (const uint16_t*)p.k + (int64_t)w.k0 * p.k_ss + hkv * p.k_sh;
  const PackedCopy<O, NG> copy(css, wave % NG, lane, p.d);
  auto load = [&](int t, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NT; ++u)
      if (t + u < t_hi) copy(cbase, (t + u) * kTileRows, kseen, (cv ? lds_v : lds_k) + (slot * NT + u) * TILE, true);
  };
  auto block = [&](int t, const char* kt, const char* vt) __attribute__((always_inline)) {
    const int n0 = t * kTileRows;
    if (!w.live(iw0, 32, n0, 32)) return;
    __builtin_amdgcn_s_setprio(1);
    const f32x16_t s = ops.scores(kt, qf);
    const f32x16_t dp = ops.scores(vt, of);
    __builtin_amdgcn_s_setprio(0);
    float x[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) x[v] = __builtin_fmaf(s[v], p.scale_log2, -lse2);
    if (p.alibi) {
      const float fi = (float)(i + off - n0 - 4 * g);
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = __builtin_fmaf(fabsf(fi - (float)((v >> 2) * 8 + (v & 3))), slope_l2, x[v]);
    }
    if (!w.full(iw0, 32, n0, 32)) {
      int io = i;  // (not held across the loop)
      asm volatile("" : "+v"(io));
      const Span ks = w.keys_of(io);
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = ks.ok(n0 + (v >> 2) * 8 + g * 4 + (v & 3)) ? x[v] : -INFINITY;
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) x[v] = __builtin_amdgcn_exp2f(x[v]) * (dp[v] - dlt);
    zs.apply(x, acc);
    __builtin_amdgcn_s_setprio(1);
    ops.accum(acc, kt, x);
    __builtin_amdgcn_s_setprio(0);
  };
  if (t_lo < t_hi) load(t_lo, 0);
  // step: NT tiles from one slot while the next land in the other
  auto step = [&](auto slot_c, int t) __attribute__((always_inline)) {
    constexpr int SL = decltype(slot_c)::value;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (t + NT < t_hi) load(t + NT, 1 - SL);
#pragma unroll
    for (int u = 0; u < NT; ++u)
      if (t + u < t_hi) block(t + u, lds_k + (SL * NT + u) * TILE, lds_v + (SL * NT + u) * TILE);
  };
  for (int t = t_lo; t < t_hi; t += 2 * NT) {
    step(std::integral_constant<int, 0>{}, t);
    if (t + NT < t_hi) step(std::integral_constant<int, 1>{}, t + NT);
  }
  const float f = p.scale * zs.undo();
  if (i >= w.lq) return;
  uint16_t* row = (uint16_t*)p.dq + (int64_t)(w.q0 + i) * p.dq_ss + hq * p.dq_sh;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int vq = 0; vq < 4; ++vq)
      if (db * 32 + vq * 8 < p.d)
        O::store4(row, db * 32 + vq * 8 + g * 4, acc[db][vq * 4] * f, acc[db][vq * 4 + 1] * f, acc[db][vq * 4 + 2] * f,
                  acc[db][vq * 4 + 3] * f);
}

// Workgroups [0, n_kv): dK and dV of p.items; behind them dQ of p.items_q.
template <class E, int C>
__global__ __launch_bounds__(256, 2) void packed_bwd16(const PackedParams p, int n_kv) {
  constexpr int D = packed_lds_dim(C);
  __shared__ __attribute__((aligned(1024))) char pool[PackedBwdLds<D>::kBytes];
  const int wg = (int)blockIdx.x;
  if (wg < n_kv) {
    const PackedBlock w(p, p.items, wg, p.Hkv * p.n_split, 1);
    if (w.blk >= 0) packed_dkdv_body<E, D, C>(p, w, pool);
  } else {
    const PackedBlock w(p, p.items_q, wg - n_kv, p.Hkv, p.G);
    if (w.blk >= 0) packed_dq_body<E, D, C>(p, w, pool);
  }
}

template <class E>
hipError_t launch_packed_bwd16(const PackedParams& p, int C, int n_kv, int n_q, hipStream_t st) {
  const dim3 grid((unsigned)(n_kv + n_q)), block(256);
  switch (C) {
    case 64: return launch_kernel(&packed_bwd16<E, 64>, grid, block, 0, st, p, n_kv);
    case 96: return launch_kernel(&packed_bwd16<E, 96>, grid, block, 0, st, p, n_kv);
    case 128: return launch_kernel(&packed_bwd16<E, 128>, grid, block, 0, st, p, n_kv);
  }
  return hipErrorNotSupported;
}

}  // namespace trinix
