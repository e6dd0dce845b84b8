// Packed-sequence attention forward of the 16-bit types on Tile16.
#pragma once
#include "attn_packed.h"
#include "attn_packed_merge.h"
#include "attn_tile16.h"

namespace trinix {

// NW * 32 / KS query rows of one sequence and head (the list's block).  SPLIT: p.n_chunks
// workgroups share the block's keys (those of a short range leave at once), and
// packed_fwd_merge joins what they leave; where one does it all it writes the result.
template <class E, int C, int BN, int NW, int OCC, int KS, int ALIBI, bool SPLIT>
__global__ __launch_bounds__(NW * 64, OCC) void packed_fwd16(const PackedParams p) {
  constexpr int BM = NW * 32 / KS, D = packed_lds_dim(C), DB = C / 32;
  TRINIX_TILE16_LDS(D, BN, KS);
  const int per_chunk = SPLIT ? (int)gridDim.x / p.n_chunks : 1, chunk = SPLIT ? (int)blockIdx.x / per_chunk : 0;
  const PackedBlock w(p, p.items, SPLIT ? packed_chunk_block((int)blockIdx.x, chunk, per_chunk) : (int)blockIdx.x, p.Hkv, p.G);
  if (w.blk < 0) return;
  KeyRun kr;
  PackedChunks chunks{0, 1};
  const int m0 = w.blk * BM, mlast = min(m0 + BM, w.lq) - 1;
  bwd_key_tiles(m0, BM, w.lq, w.lk, w.dlo, w.dhi, BN, kr.t_lo, kr.t_hi);
  packed_full_tiles(m0, mlast, w.lk, w.dlo, w.dhi, BN, kr.t_lo, kr.t_hi, kr.t_flo, kr.t_fhi);
  if constexpr (SPLIT) {
    chunks = packed_chunks(kr.t_hi - kr.t_lo, BN, p.n_chunks, w.total, p.Hq, C == 256 ? 256 : 512);
    if (chunk >= chunks.n) return;
    kr.t_lo += chunk * chunks.per;
    kr.t_hi = min(kr.t_hi, kr.t_lo + chunks.per);
    kr.t_flo = min(max(kr.t_flo, kr.t_lo), kr.t_hi);
    kr.t_fhi = min(max(kr.t_fhi, kr.t_flo), kr.t_hi);
  }
  Tile16<E, D, C, BN, NW, KS, ALIBI> T(lds_k0, lds_k1, lds_v0, lds_v1);
  const int hq = w.h, hkv = hq / p.G, iw0 = m0 + (T.wave / KS) * 32, i = iw0 + T.r;
  T.load_q((const uint16_t*)p.q + (int64_t)(w.q0 + min(i, w.lq - 1)) * p.q_ss + hq * p.q_sh, p.d, p.scale_log2,
           ALIBI ? p.alibi[hq * p.al_sh] : 0.f);
  const Span ks = w.keys_of(i);
  kr.k = (const uint16_t*)p.k + (int64_t)w.k0 * p.k_ss + hkv * p.k_sh;
  kr.v = (const uint16_t*)p.v + (int64_t)w.k0 * p.v_ss + hkv * p.v_sh;
  const PackedRange seen = w.keys();
  kr.k_ss = p.k_ss, kr.v_ss = p.v_ss, kr.lo = seen.lo, kr.n = seen.hi + 1, kr.d = p.d;
  kr.jlo = ks.lo, kr.jspan = ks.span;
  // (a wavefront whose rows all lie behind the sequence sees nothing)
  kr.wlo = iw0 < w.lq ? iw0 + w.dlo : INT_MAX;
  kr.whi = iw0 < w.lq ? min(min(iw0 + 31, w.lq - 1) + w.dhi, w.lk - 1) : -1;
  kr.pos = i + w.lk - w.lq;
  T.run(kr);
  const float l = T.finish();
  if (i >= w.lq || T.kp != 0) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;  // a row that sees no key: 0
  const int64_t row = w.q0 + i;
  if (SPLIT && chunks.n > 1) {
    const int64_t at = ((int64_t)chunk * p.Hq + hq) * p.Tq + row;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int vq = 0; vq < 4; ++vq)
        *(f32x4_t*)(p.part + at * D + db * 32 + vq * 8 + T.g * 4) =
            (f32x4_t){T.acc[db][vq * 4] * inv, T.acc[db][vq * 4 + 1] * inv, T.acc[db][vq * 4 + 2] * inv, T.acc[db][vq * 4 + 3] * inv};
    if (T.g == 0) p.part_lse[at] = l > 0.f ? T.m_run + __log2f(l) : -INFINITY;
    return;
  }
  uint16_t* orow = (uint16_t*)p.o + row * p.o_ss + hq * p.o_sh;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int vq = 0; vq < 4; ++vq) {
      const int d0 = db * 32 + vq * 8 + T.g * 4;
      if (db * 32 + vq * 8 >= p.d) continue;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = T.acc[db][vq * 4 + e] * inv;
      const u32x2_t hi = {E::pack(x[0], x[1]), E::pack(x[2], x[3])};
      *(u32x2_t*)(orow + d0) = hi;
      if (p.o_lo) {
        constexpr float f = kLoScale<E>;
        *(u32x2_t*)((uint16_t*)p.o_lo + row * p.o_ss + hq * p.o_sh + d0) =
            (u32x2_t){E::pack((x[0] - E::lo(hi[0])) * f, (x[1] - E::hi(hi[0])) * f),
                      E::pack((x[2] - E::lo(hi[1])) * f, (x[3] - E::hi(hi[1])) * f)};
      }
    }
  if (p.lse && T.g == 0) p.lse[(int64_t)hq * p.Tq + row] = l > 0.f ? (T.m_run + __log2f(l)) * kLn2 : -INFINITY;
}

template <class E, int C, int BN, int NW, int OCC, int KS, bool SPLIT = false>
hipError_t launch_packed_fwd16(const PackedParams& p, int grid, hipStream_t st) {
  const dim3 g((unsigned)grid), b(NW * 64);
  if (!p.alibi) return launch_kernel(&packed_fwd16<E, C, BN, NW, OCC, KS, 0, SPLIT>, g, b, 0, st, p);
  // (a causal row sees no key behind it; 128-key tiles and head_dim 256 have no registers for 2)
  if constexpr (BN <= 64 && C <= 128)
    if (p.causal) return launch_kernel(&packed_fwd16<E, C, BN, NW, OCC, KS, 2, SPLIT>, g, b, 0, st, p);
  return launch_kernel(&packed_fwd16<E, C, BN, NW, OCC, KS, 1, SPLIT>, g, b, 0, st, p);
}

template <class E, int C>
hipError_t launch_packed_fwd16_128(const PackedParams& p, PackedShape shape, int grid, hipStream_t st) {
  switch (shape) {
    case PackedShape::kPair: return launch_packed_fwd16<E, C, 32, 4, 2, 2>(p, grid, st);
    case PackedShape::kPlain: return launch_packed_fwd16<E, C, 64, 4, 2, 1>(p, grid, st);
    case PackedShape::kWide: return launch_packed_fwd16<E, C, 128, 8, 2, 1>(p, grid, st);
  }
  return hipErrorNotSupported;
}

// 64-key tiles of 4 wavefronts, two per SIMD (head_dim 256: one); kPair at
// head_dim 128 on 32-key tiles, in the same LDS (at 256 it would spill); kWide
// 128-key tiles of 8.
template <class E>
hipError_t launch_packed_fwd16(const PackedParams& p, int C, PackedShape shape, int grid, hipStream_t st) {
  const bool pair = shape == PackedShape::kPair;
  switch (C) {
    case 64: return pair ? launch_packed_fwd16<E, 64, 64, 4, 2, 2>(p, grid, st) : launch_packed_fwd16<E, 64, 64, 4, 2, 1>(p, grid, st);
    case 96: return launch_packed_fwd16_128<E, 96>(p, shape, grid, st);
    case 128: return launch_packed_fwd16_128<E, 128>(p, shape, grid, st);
    case 256: return launch_packed_fwd16<E, 256, 64, 4, 1, 1>(p, grid, st);
  }
  return hipErrorNotSupported;
}

// grid: blocks times heads.
template <class E, int C, int BN, int OCC, int KS>
hipError_t launch_packed_chunks16(const PackedParams& p, int grid, hipStream_t st) {
  const hipError_t e = launch_packed_fwd16<E, C, BN, 4, OCC, KS, true>(p, grid * p.n_chunks, st);
  if (e != hipSuccess) return e;
  return launch_kernel(&packed_fwd_merge<E, packed_lds_dim(C), 128 / KS, BN, C == 256 ? 256 : 512>, dim3((unsigned)grid), dim3(256), 0, st, p);
}
template <class E>
hipError_t launch_packed_chunks16(const PackedParams& p, int C, int grid, hipStream_t st) {
  switch (C) {
    case 64: return launch_packed_chunks16<E, 64, 64, 2, 2>(p, grid, st);
    case 96: return launch_packed_chunks16<E, 96, 32, 2, 2>(p, grid, st);
    case 128: return launch_packed_chunks16<E, 128, 32, 2, 2>(p, grid, st);
    case 256: return launch_packed_chunks16<E, 256, 64, 1, 1>(p, grid, st);
  }
  return hipErrorNotSupported;
}

}  // namespace trinix
