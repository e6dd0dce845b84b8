// The 16-bit attention forward over key tiles that packed sequences and shared
// prefixes run on: NW wavefronts, 32 query rows each (KS = 2: each pair of
// wavefronts shares 32 rows and takes alternate tiles), BN-key tiles.
//
// Per tile a wavefront computes S^T = K Q^T on v_mfma_f32_32x32x16 with keys on
// the matrix rows and its queries on the columns, so that a lane owns one row
// (row maximum: one lane ^ 32 exchange); O^T += V^T P^T takes P^T straight from the
// score registers, V^T from LDS transpose reads.  K and V tiles go global -> LDS
// asynchronously into two buffers each, one barrier per tile; operand reads run
// ahead of their MFMAs, pinned with sched_group_barrier.  Scores stay raw, the
// scale (times log2 e) folds into the FMA before the exponential, and the running
// maximum is raised only past TAU = 8, so that most tiles skip the rescale of O.
//
// Roundings: P is rounded to 16 bits for its product with V (half a step per
// weight, independent over the keys: the error of O, 1.05 to 1.35 times that of
// rounding O alone; two terms per P cost a third of the speed).  The row sum is of
// the unrounded P in fp32, so the log-sum-exp is an fp32 one.
#pragma once
#include <climits>
#include <type_traits>

#include "attn_params.h"
#include "lds_tile.h"

namespace trinix {

// LDS of a workgroup: four objects of tile16_words, so that the compiler can tell
// the buffer being read from the one that a copy fills.
template <int D, int BN, int KS>
constexpr int kTile16Words = KS * BN * D;
#define TRINIX_TILE16_LDS(D, BN, KS)                                            \
  __shared__ __attribute__((aligned(1024))) uint16_t lds_k0[kTile16Words<D, BN, KS>]; \
  __shared__ __attribute__((aligned(1024))) uint16_t lds_k1[kTile16Words<D, BN, KS>]; \
  __shared__ __attribute__((aligned(1024))) uint16_t lds_v0[kTile16Words<D, BN, KS>]; \
  __shared__ __attribute__((aligned(1024))) uint16_t lds_v1[kTile16Words<D, BN, KS>]

// A run of key tiles: keys [lo, n) at k and v (row strides in elements; rows outside
// are read as the nearest of them), tiles [t_lo, t_hi) of which [t_flo, t_fhi)
// hold only pairs that every row of the workgroup may see.  A lane's row sees
// keys jlo .. jlo + jspan (jlo = INT_MAX: none); keys outside [wlo, whi] are seen
// by no row of the wavefront.  pos: position of the lane's row among the keys (ALiBi).
// Rows hold d <= C columns (a multiple of 8): q is zero from there on in registers, and
// K and V units from there on are copies of the row's last one.
struct KeyRun {
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_ss, v_ss;
  int lo, n, d, t_lo, t_hi, t_flo, t_fhi;
  int jlo;
  uint32_t jspan;
  int wlo, whi;
  int pos;
};

// ALIBI: 0 none; 1 -slope * |distance|, three instructions per score; 2 the same where
// no key of a full tile lies behind a row (causal runs): linear in the key there, so
// that the accumulators start at its part within the tile, which stays in registers (an
// operand of the first product, no instruction of its own), and its part of the whole
// tile joins the maximum in the exponential's FMA (32 heads of 128, ten ragged prompts of
// 8326 rows: 144 us with 1, 135 with 2, 126 without ALiBi).
// The products take the first C of a tile's D columns.
template <class E, int D, int C, int BN, int NW, int KS, int ALIBI>
struct Tile16 {
  static constexpr int DS = C / 16;    // MFMA k-steps over head_dim
  static constexpr int NB = BN / 32;   // 32-key blocks per tile
  static constexpr int DB = C / 32;    // 32-wide head_dim blocks of O^T
  static constexpr int UPR = D / 8;    // 16-byte units per row
  static constexpr int LPW = BN * UPR / (64 * NW);  // copies per wavefront and tile (K or V)
  static constexpr float TAU = 8.f;
  static_assert(D % 64 == 0 && BN % 32 == 0 && BN * UPR % (64 * NW) == 0, "tile shape");
  static constexpr int NQK = NB * DS, NPV = DB * NB * 2;  // MFMAs of a tile
  // operand reads ahead of their MFMA
  static constexpr int KPF = D == 256 ? 2 : (NQK < 6 ? NQK : 6), VPF = D == 256 ? 2 : 4;
  static_assert(KPF <= NQK && VPF <= NPV, "reads ahead");

  uint16_t *k0, *k1, *v0, *v1;
  int lane, wave, r, g, kp;
  uint32_t k_lane;
  int tr_off[DB];
  u32x4_t qr[DS];
  f32x16_t acc[DB];  // O^T: element (db, 4 vq + e) is d = 32 db + 8 vq + 4 g + e of the lane's row
  float m_run, l_run, c, alibi_mul;
  f32x16_t lin[ALIBI == 2 ? NB : 1];

  __device__ __forceinline__ Tile16(uint16_t* k0_, uint16_t* k1_, uint16_t* v0_, uint16_t* v1_)
      : k0(k0_), k1(k1_), v0(v0_), v1(v1_) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    r = lane & 31, g = lane >> 5;
    kp = wave % KS;
    // K fragment (nb, ds) of this lane: byte nb*32*D*2 + (k_lane ^ 32*ds)
    k_lane = (uint32_t)(r * D * 2 + 16 * (g ^ swz_k<D>(r)));
    // transpose reads of V: 16-lane group G of the wavefront covers head_dim
    // db*32 + 16*(G&1) + 0..15 for k-group G>>1.  The empty asm keeps each offset
    // one opaque value (LDS buffer + offset + constant)
    const int tr_G = lane >> 4, tr_s = lane & 15, tr_g = tr_G >> 1, tr_dh = tr_G & 1;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int row0 = tr_g * 4 + (tr_s >> 2), u = db * 4 + tr_dh * 2 + ((tr_s & 3) >> 1);
      tr_off[db] = (row0 * D + (u ^ swz_v<D>(row0)) * 8 + (tr_s & 1) * 4) * 2;
      asm volatile("" : "+v"(tr_off[db]));
      acc[db] = (f32x16_t){};
    }
    m_run = -INFINITY, l_run = 0.f, alibi_mul = 0.f;
  }

  // The lane's query row and the scale: the maximum of raw scores is that of the
  // scaled ones for a positive scale, so a negative one negates q, a zero one clears it.
  __device__ __forceinline__ void load_q(const uint16_t* row, int d, float scale_log2, float slope) {
    const bool neg = scale_log2 < 0.f, zero = scale_log2 == 0.f;
    c = neg ? -scale_log2 : (zero ? 1.f : scale_log2);
    if constexpr (ALIBI != 0) alibi_mul = -slope * kLog2e / c;
    if constexpr (ALIBI == 2) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int v = 0; v < 16; ++v) lin[nb][v] = -alibi_mul * (float)(nb * 32 + (v >> 2) * 8 + (v & 3));
        asm volatile("" : "+v"(lin[nb]));
      }
    }
    const uint32_t flip = neg ? 0x80008000u : 0u, keep = zero ? 0u : 0xffffffffu;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) {
      const int d0 = ds * 16 + g * 8;
      qr[ds] = *(const u32x4_t*)(row + min(d0, d - 8));
      const uint32_t mask = d0 < d ? keep : 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) qr[ds][e] = (qr[ds][e] ^ flip) & mask;
    }
  }

  template <class S>
  __device__ __forceinline__ uint16_t* kbuf(S slot) const {
    if constexpr (std::is_integral_v<S>) return slot ? k1 : k0;
    else return S::value ? k1 : k0;
  }
  template <class S>
  __device__ __forceinline__ uint16_t* vbuf(S slot) const {
    if constexpr (std::is_integral_v<S>) return slot ? v1 : v0;
    else return S::value ? v1 : v0;
  }
  __device__ __forceinline__ u32x4_t kread(const uint16_t* kt, int k) const {
    const int nb = k / DS, ds = k % DS;
    return *(const u32x4_t*)((const char*)kt + nb * 32 * D * 2 + (k_lane ^ (uint32_t)(ds << 5)));
  }
  __device__ __forceinline__ u32x4_t vread(const uint16_t* vt, int m) const {
    const int db = m / (NB * 2), nb = (m / 2) % NB, kk = m % 2;
    const char* base = (const char*)vt + tr_off[db] + (nb * 32 + kk * 16) * D * 2;
    const s16x4_t lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)base);
    const s16x4_t hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(base + 8 * D * 2));
    const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo4), h2 = __builtin_bit_cast(u32x2_t, hi4);
    return (u32x4_t){l2[0], l2[1], h2[0], h2[1]};
  }
  __device__ __forceinline__ void pin_acc() {
    // head_dim 256 keeps O in accumulation registers across the tile
    if constexpr (D == 256) {
#pragma unroll
      for (int db = 0; db < DB; ++db) asm volatile("" : "+a"(acc[db]));
    }
  }

  __device__ __forceinline__ void run(KeyRun kr) {
    // (uniform by construction; 64-bit comparisons leave them in vector registers)
    for (int* x : {&kr.lo, &kr.n, &kr.t_lo, &kr.t_hi, &kr.t_flo, &kr.t_fhi, &kr.wlo, &kr.whi}) *x = __builtin_amdgcn_readfirstlane(*x);
    auto ld_row = [&](int l) __attribute__((always_inline)) { return tile_copy_row(wave, LPW, l, lane, UPR); };
    auto ld_unit_k = [&](int l) __attribute__((always_inline)) { return min((lane % UPR) ^ swz_k<D>(ld_row(l)), kr.d / 8 - 1); };
    auto ld_unit_v = [&](int l) __attribute__((always_inline)) { return min((lane % UPR) ^ swz_v<D>(ld_row(l)), kr.d / 8 - 1); };
    uint32_t ld_koff[LPW], ld_voff[LPW];
#pragma unroll
    for (int l = 0; l < LPW; ++l) {
      ld_koff[l] = tile_copy_offset((uint32_t)ld_row(l), kr.k_ss, (uint32_t)ld_unit_k(l));
      ld_voff[l] = tile_copy_offset((uint32_t)ld_row(l), kr.v_ss, (uint32_t)ld_unit_v(l));
    }
    const uint64_t kbase_s = uniform_ptr(kr.k), vbase_s = uniform_ptr(kr.v);
    const uint32_t wave_lds = __builtin_amdgcn_readfirstlane((uint32_t)(wave * LPW * 1024));
    auto load_tile = [&](auto is_k, uint64_t base_s, int64_t ss, const uint32_t* offs, uint16_t* lds_tile, int tile)
                         __attribute__((always_inline)) {
      const int n0 = tile * BN;
      const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)lds_tile + wave_lds;
      const uint64_t gb = base_s + (uint64_t)n0 * (uint64_t)(ss * 2);
      if (n0 >= kr.lo && n0 + BN <= kr.n) {
#pragma unroll
        for (int l = 0; l < LPW; ++l) dma_16b_s(offs[l], gb, __builtin_amdgcn_readfirstlane(lds0 + l * 1024));
      } else {
        const int last = kr.n - 1 - n0, first = max(kr.lo - n0, 0);  // last >= first: a tile holds keys of the run
#pragma unroll
        for (int l = 0; l < LPW; ++l) {
          const uint32_t row = (uint32_t)min(max(ld_row(l), first), last);
          const uint32_t unit = (uint32_t)(decltype(is_k)::value ? ld_unit_k(l) : ld_unit_v(l));
          dma_16b_s(tile_copy_offset(row, ss, unit), gb, __builtin_amdgcn_readfirstlane(lds0 + l * 1024));
        }
      }
    };
    auto load_k = [&](uint16_t* t, int tile) __attribute__((always_inline)) {
      load_tile(std::true_type{}, kbase_s, kr.k_ss, ld_koff, t, tile);
    };
    auto load_v = [&](uint16_t* t, int tile) __attribute__((always_inline)) {
      load_tile(std::false_type{}, vbase_s, kr.v_ss, ld_voff, t, tile);
    };

    // S^T of one tile; ALiBi starts the accumulators at bias / c
    auto qk = [&](auto edge, const uint16_t* kt, int n0, f32x16_t(&s)[NB]) __attribute__((always_inline)) {
      constexpr bool LIN = ALIBI == 2 && !decltype(edge)::value;
      u32x4_t kf[NQK];
#pragma unroll
      for (int k = 0; k < KPF; ++k) kf[k] = kread(kt, k);
      const float fi = (float)(kr.pos - n0 - 4 * g);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if constexpr (!LIN) s[nb][v] = ALIBI ? fabsf(fi - (float)(nb * 32 + (v >> 2) * 8 + (v & 3))) * alibi_mul : 0.f;
#pragma unroll
      for (int k = 0; k < NQK; ++k) {
        if (k + KPF < NQK) kf[k + KPF] = kread(kt, k + KPF);
        s[k / DS] = E::mfma(kf[k], qr[k % DS], LIN && k % DS == 0 ? lin[ALIBI == 2 ? k / DS : 0] : s[k / DS]);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, KPF, 0);
#pragma unroll
      for (int k = 0; k < NQK; ++k) {
        if (k + KPF < NQK) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
    };
    auto softmax = [&](auto edge, f32x16_t(&s)[NB], int n0, u32x4_t(&pb)[NB][2]) __attribute__((always_inline)) {
      if constexpr (decltype(edge)::value) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int j = n0 + nb * 32 + (v >> 2) * 8 + g * 4 + (v & 3);
            s[nb][v] = (uint32_t)(j - kr.jlo) <= kr.jspan ? s[nb][v] : -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int v = 0; v < 16; ++v) mx = fmaxf(mx, s[nb][v]);
      constexpr bool LIN = ALIBI == 2 && !decltype(edge)::value;
      const float tile_bias = LIN ? alibi_mul * (float)(kr.pos - n0 - 4 * g) : 0.f;
      mx = xlane_max(mx + tile_bias) * c;
      pin_acc();
      if (__builtin_expect(wave_any(mx > m_run + TAU), 0)) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] *= alpha;
        m_run = m_new;
      }
      pin_acc();
      // a row that has seen no key yet: exp2(-inf) = 0
      const float mneg = __builtin_fmaf(tile_bias, c, m_run == -INFINITY ? 0.f : -m_run);
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          s[nb][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nb][v], c, mneg));
          sum[v & 1] += s[nb][v];
        }
      l_run += sum[0] + sum[1];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
          pb[nb][kk] = (u32x4_t){E::pack(s[nb][kk * 8 + 0], s[nb][kk * 8 + 1]), E::pack(s[nb][kk * 8 + 2], s[nb][kk * 8 + 3]),
                                 E::pack(s[nb][kk * 8 + 4], s[nb][kk * 8 + 5]), E::pack(s[nb][kk * 8 + 6], s[nb][kk * 8 + 7])};
    };
    auto pv = [&](const uint16_t* vt, const u32x4_t(&pb)[NB][2], const u32x4_t(&vpre)[VPF]) __attribute__((always_inline)) {
      u32x4_t vf[NPV];
#pragma unroll
      for (int m = 0; m < VPF; ++m) vf[m] = vpre[m];
#pragma unroll
      for (int m = 0; m < NPV; ++m) {
        if (m + VPF < NPV) vf[m + VPF] = vread(vt, m + VPF);
        acc[m / (NB * 2)] = E::mfma(vf[m], pb[(m / 2) % NB][m % 2], acc[m / (NB * 2)]);
      }
#pragma unroll
      for (int m = 0; m < NPV; ++m) {
        if (m + VPF < NPV) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
    };

    // Step s covers tiles T = t_lo + KS*s .. T + KS - 1 in buffer slot s & 1 (this
    // wavefront's tile: T + kp): wait for them; barrier (every wavefront has left
    // the other slot, which now takes the next step's); scores, softmax, O.
    auto step = [&](auto edge, auto slot, int T) __attribute__((always_inline)) {
      auto other = [&]() {
        if constexpr (std::is_integral_v<decltype(slot)>) return 1 - slot;
        else return std::integral_constant<int, 1 - decltype(slot)::value>{};
      }();
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
#pragma unroll
      for (int u = 0; u < KS; ++u)
        if (T + KS + u < kr.t_hi) {
          load_k(kbuf(other) + u * BN * D, T + KS + u);
          load_v(vbuf(other) + u * BN * D, T + KS + u);
        }
      const int t = T + kp, n0 = t * BN;
      if (t < kr.t_hi && n0 <= kr.whi && n0 + BN > kr.wlo) {
        const uint16_t* kt = kbuf(slot) + kp * BN * D;
        const uint16_t* vt = vbuf(slot) + kp * BN * D;
        f32x16_t sc[NB];
        u32x4_t vpre[VPF], pb[NB][2];
        // matrix sections at raised priority: the other wavefront of the SIMD
        // fills the gaps with its softmax
        __builtin_amdgcn_s_setprio(1);
        qk(edge, kt, n0, sc);
#pragma unroll
        for (int m = 0; m < VPF; ++m) vpre[m] = vread(vt, m);
        __builtin_amdgcn_s_setprio(0);
        softmax(edge, sc, n0, pb);
        __builtin_amdgcn_s_setprio(1);
        pv(vt, pb, vpre);
        __builtin_amdgcn_s_setprio(0);
      }
    };
    if (kr.t_lo >= kr.t_hi) return;  // (wave-uniform over the workgroup)
#pragma unroll
    for (int u = 0; u < KS; ++u)
      if (kr.t_lo + u < kr.t_hi) {
        load_k(k0 + u * BN * D, kr.t_lo + u);
        load_v(v0 + u * BN * D, kr.t_lo + u);
      }
    // steps of full tiles only run in pairs without predicates, from an even step
    // (static buffer slots); the others test every element, which is always exact
    const int s_hi = (kr.t_hi - kr.t_lo + KS - 1) / KS;
    int s_flo = (kr.t_flo - kr.t_lo + KS - 1) / KS;
    int s_fhi = max(s_flo, (kr.t_fhi - kr.t_lo) / KS);
    if ((s_flo & 1) && s_flo < s_fhi) ++s_flo;
    s_fhi -= (s_fhi - s_flo) & 1;
    int si = 0;
    for (; si < s_flo; ++si) step(std::true_type{}, si & 1, kr.t_lo + KS * si);
    for (; si < s_fhi; si += 2) {
      step(std::false_type{}, std::integral_constant<int, 0>{}, kr.t_lo + KS * si);
      step(std::false_type{}, std::integral_constant<int, 1>{}, kr.t_lo + KS * (si + 1));
    }
    for (; si < s_hi; ++si) step(std::true_type{}, si & 1, kr.t_lo + KS * si);
  }

  // Ends the runs: the row's sum (KS = 2: and the partner's half, through LDS;
  // afterwards kp == 0 holds the row).  Every wavefront of the workgroup calls it.
  __device__ __forceinline__ float finish() {
    if constexpr (KS == 2) {
      constexpr int HB = BN == 32 ? (DB + 1) / 2 : DB;  // head_dim blocks per K buffer
      static_assert(NW / 2 * HB * 16 * 64 * 4 <= KS * BN * D * 2, "exchange fits the K buffers");
      const int rg = wave / 2;
      auto mo = [&](int db, int v) __attribute__((always_inline)) -> float* {
        return (float*)(db < HB ? k0 : k1) + ((rg * HB + db % HB) * 16 + v) * 64 + lane;
      };
      float* ml = (float*)v0;
      __syncthreads();
      if (kp == 1) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int v = 0; v < 16; ++v) *mo(db, v) = acc[db][v];
        ml[(rg * 2 + 0) * 64 + lane] = m_run;
        ml[(rg * 2 + 1) * 64 + lane] = l_run;
      }
      __syncthreads();
      if (kp == 0) {
        const float m1 = ml[(rg * 2 + 0) * 64 + lane], l1 = ml[(rg * 2 + 1) * 64 + lane];
        const float m = fmaxf(m_run, m1);
        const float a0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m);
        const float a1 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - m);
        l_run = l_run * a0 + l1 * a1;
        m_run = m;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[db][v] = acc[db][v] * a0 + *mo(db, v) * a1;
      }
    }
    return xlane_sum(l_run);
  }
};

}  // namespace trinix
