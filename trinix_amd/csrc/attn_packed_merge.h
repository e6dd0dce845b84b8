// Second launch of a packed forward whose keys are shared out.
#pragma once
#include "attn_packed.h"

namespace trinix {

// Joins the chunks' results (E: the 16-bit type, or float): the blocks of the launch
// before, with its BM, BN and slots, D / 4 threads a row, four columns each; blocks that
// one workgroup did leave at once.
template <class E, int D, int BM, int BN, int SLOTS>
__global__ __launch_bounds__(256) void packed_fwd_merge(const PackedParams p) {
  constexpr int TPR = D / 4, UNR = 4;
  const PackedBlock w(p, p.items, (int)blockIdx.x, p.Hkv, p.G);
  if (w.blk < 0) return;
  const int m0 = w.blk * BM, hq = w.h, c = (int)threadIdx.x % TPR;
  int t_lo, t_hi;
  bwd_key_tiles(m0, BM, w.lq, w.lk, w.dlo, w.dhi, BN, t_lo, t_hi);
  const int n = packed_chunks(t_hi - t_lo, BN, p.n_chunks, w.total, p.Hq, SLOTS).n;
  if (n <= 1) return;
  const int64_t step = (int64_t)p.Hq * p.Tq;
  for (int i = m0 + (int)threadIdx.x / TPR; i < min(m0 + BM, w.lq); i += 256 / TPR) {
    const int64_t row = w.q0 + i, at = hq * (int64_t)p.Tq + row;
    const float* pl = p.part_lse + at;
    const float* po = p.part + at * D + c * 4;
    float m = -INFINITY, L = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < n; s0 += UNR) {
      float ls[UNR], mn = m;
      f32x4_t ov[UNR];
#pragma unroll
      for (int u = 0; u < UNR; ++u) {
        const int64_t s = min(s0 + u, n - 1) * step;
        ls[u] = s0 + u < n ? pl[s] : -INFINITY;
        ov[u] = *(const f32x4_t*)(po + s * D);
        mn = fmaxf(mn, ls[u]);
      }
      const float m_use = mn == -INFINITY ? 0.f : mn, a = __builtin_amdgcn_exp2f(m - m_use);
      L *= a;
      o *= a;
#pragma unroll
      for (int u = 0; u < UNR; ++u) {
        const float f = __builtin_amdgcn_exp2f(ls[u] - m_use);
        L += f;
        o += f * ov[u];
      }
      m = mn;
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;  // a row that sees no key: 0
    if (c * 4 < p.d) {
      o *= inv;
      const int64_t to = row * p.o_ss + hq * p.o_sh + c * 4;
      if constexpr (std::is_same<E, float>::value) {
#pragma unroll
        for (int e = 0; e < 4; ++e) ((float*)p.o)[to + e] = o[e];
      } else {
        const u32x2_t hi = {E::pack(o[0], o[1]), E::pack(o[2], o[3])};
        *(u32x2_t*)((uint16_t*)p.o + to) = hi;
        if (p.o_lo) {
          constexpr float f = kLoScale<E>;
          *(u32x2_t*)((uint16_t*)p.o_lo + to) = (u32x2_t){E::pack((o[0] - E::lo(hi[0])) * f, (o[1] - E::hi(hi[0])) * f),
                                                          E::pack((o[2] - E::lo(hi[1])) * f, (o[3] - E::hi(hi[1])) * f)};
        }
      }
    }
    if (p.lse && c == 0) p.lse[at] = L > 0.f ? (m + (std::is_same<E, float>::value ? log2f(L) : __log2f(L))) * kLn2 : -INFINITY;
  }
}

}  // namespace trinix
