// Attention over packed sequences: parameters, the work item of a workgroup and
// the pieces that its kernels share (semantics: trinix_attn.h, trinix_packed_args).
#pragma once
#include "attn_ops.h"
#include "attn_params.h"
#include "lds_tile.h"
#include "packed_map.h"

namespace trinix {

struct PackedParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  void* o_lo;  // what o lost by rounding (16-bit), or null
  float* lse;
  const void* dout;
  float* delta;
  void* dq;
  void* dk;
  void* dv;
  int64_t q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, o_ss, o_sh;
  int64_t do_ss, do_sh, dq_ss, dq_sh, dk_ss, dk_sh, dv_ss, dv_sh;
  int Tq, Hq, Hkv, G;
  int d;  // columns of every tensor: head_dim, at most the kernel's C
  float scale, scale_log2;
  int causal, has_window;
  int64_t wl, wr;  // clamped to +-2^30
  const float* alibi;
  int64_t al_sh;
  // dK and dV: a group's heads over n_split workgroups, fp32 partial sums (split, dV
  // and dK, key, KV head, head_dim), or 1 and null
  int n_split, Tk;
  float* part;
  // forward: at most n_chunks workgroups share the keys of a block of rows, each leaving
  // its normalised O in part (chunk, head, row, D) and its log-sum-exp (log2) in part_lse
  int n_chunks;
  float* part_lse;
  int rows16;             // fp32: the tiles' tensors take 16-byte copies (of dK, dV: q and dout)
  int rows16_q;           // the same of the backward's dQ: k and v
  const int32_t* items;   // of the launch's list
  const int32_t* items_q; // of its second one (packed_bwd16)
};

// The block of rows or keys that a workgroup runs: its sequence (first row and
// rows, first key and keys), block number (-1: none) and head, all wave-uniform.
struct PackedBlock {
  int q0, lq, k0, lk, blk, h, dlo, dhi;
  int total;  // of the list
  __device__ PackedBlock(const PackedParams& p, const int32_t* items, int wg, int heads_kv, int G) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const PackedWork w = packed_work(wg, heads_kv, G);
    const i32x4* it = (const i32x4*)(items + (int64_t)w.item * kPackedItemInts);
    const i32x4 a = it[0];
    q0 = __builtin_amdgcn_readfirstlane(a[0]);
    lq = __builtin_amdgcn_readfirstlane(a[1]);
    k0 = __builtin_amdgcn_readfirstlane(a[2]);
    lk = __builtin_amdgcn_readfirstlane(a[3]);
    const i32x4 b = it[1];
    blk = __builtin_amdgcn_readfirstlane(b[0]);
    total = __builtin_amdgcn_readfirstlane(b[2]);
    h = w.h;
    packed_band(lq, lk, p.causal != 0, p.has_window != 0, p.wl, p.wr, dlo, dhi);
  }
  // keys that query row i sees, and rows that see key j (empty outside the sequence)
  __device__ Span keys_of(int i) const {
    return i < lq ? Span(max((int64_t)0, (int64_t)i + dlo), min((int64_t)lk - 1, (int64_t)i + dhi)) : Span(1, 0);
  }
  __device__ Span rows_of(int j) const {
    return j < lk ? Span(max((int64_t)0, (int64_t)j - dhi), min((int64_t)lq - 1, (int64_t)j - dlo)) : Span(1, 0);
  }
  __device__ PackedRange keys() const { return packed_seen_keys(lq, lk, dlo, dhi); }
  __device__ PackedRange rows() const { return packed_seeing_rows(lq, lk, dlo, dhi); }
  // Block of rows [ia, ia + ni) and keys [ja, ja + nj): does it hold allowed
  // pairs; are all of its pairs allowed?
  __device__ bool live(int ia, int ni, int ja, int nj) const {
    if (ia >= lq || ja >= lk) return false;
    const int ib = min(ia + ni, lq) - 1, jb = min(ja + nj, lk) - 1;
    return ja - ib <= dhi && jb - ia >= dlo;
  }
  __device__ bool full(int ia, int ni, int ja, int nj) const {
    return ia + ni <= lq && ja + nj <= lk && ja + nj - 1 - ia <= dhi && ja - (ia + ni - 1) >= dlo;
  }
};

// KV head, heads of its group [gh0, gh1) and split of a dK, dV workgroup.
struct PackedHeads {
  int hkv, split, gh0, gh1;
  __device__ PackedHeads(const PackedParams& p, int h) {
    hkv = h / p.n_split, split = h % p.n_split;
    gh0 = p.G * split / p.n_split, gh1 = p.G * (split + 1) / p.n_split;
  }
};
// Partial sums of key row `row` (which = 0: dV, 1: dK).
__device__ inline float* packed_partial(const PackedParams& p, int split, int which, int64_t row, int hkv, int D) {
  return p.part + ((((int64_t)split * 2 + which) * p.Tk + row) * p.Hkv + hkv) * D;
}

// Rows of d columns in kernels of C >= d: the operand in registers is zero from column
// d on, so what the other one holds there (a copy of a real unit) adds nothing, and
// output columns from d on are not written.
template <class O>
__device__ inline typename O::Frag load_frag_cols(const typename O::Store* row, int g, int d) {
  typename O::Frag f;
  constexpr int N = sizeof(f.r) / sizeof(f.r[0]), PER = O::kC / N, HALF = PER / 2;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int d0 = k * PER + g * HALF;
    if constexpr (sizeof(typename O::Store) == 2) {
      const u32x4_t x = *(const u32x4_t*)(row + min(d0, d - 8));
      f.r[k] = d0 < d ? x : (u32x4_t){0u, 0u, 0u, 0u};
    } else {
      typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // any 4-byte aligned row
      const f32x4_t x = *(const f32x4_any*)(row + min(d0, d - 4));
      f.r[k] = d0 < d ? x : (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
  }
  return f;
}

// TileCopy (attn_ops.h) of such rows: units from d on read the row's last one.
template <class O, int NW>
struct PackedCopy {
  using Store = typename O::Store;
  static constexpr int ESZ = (int)sizeof(Store), UPR = O::kD * ESZ / 16, PER = kTileRows * UPR / (64 * NW);
  static_assert(PER >= 1 && kTileRows * UPR % (64 * NW) == 0, "tile shape");
  int64_t ss;
  int wave, lane, units;
  uint32_t off[PER];
  __device__ PackedCopy(int64_t ss_, int wave_, int lane_, int d) : ss(ss_), wave(wave_), lane(lane_), units(d * ESZ / 16) {
#pragma unroll
    for (int l = 0; l < PER; ++l) off[l] = offset(l, PackedRange{0, kTileRows - 1});
  }
  __device__ uint32_t offset(int l, const PackedRange& t) const {
    const int row = tile_copy_row(wave, PER, l, lane, UPR);
    return tile32_offset(max(row, t.lo), t.hi, ss, ESZ, min(O::swz(((wave * PER + l) * 64 + lane) % UPR, row), units - 1));
  }
  // rows [i0, i0 + 32), those outside [of.lo, of.hi] as the nearest within; `wide`: 16
  // bytes a lane from 32-bit offsets (always for 16-bit types)
  __device__ void operator()(const Store* base, int i0, const PackedRange& of, char* lds_tile, bool wide) const {
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)lds_tile;
    const PackedRange t = packed_tile_range(of, i0);
    if (ESZ == 2 || wide) {
      const uint64_t gb = uniform_ptr(base + (int64_t)i0 * ss);
      if (t.lo == 0 && t.hi >= kTileRows - 1) {
#pragma unroll
        for (int l = 0; l < PER; ++l) dma_16b_s(off[l], gb, __builtin_amdgcn_readfirstlane(lds0 + (wave * PER + l) * 1024));
      } else {
#pragma unroll 1
        for (int l = 0; l < PER; ++l)
          dma_16b_s(offset(l, t), gb, __builtin_amdgcn_readfirstlane(lds0 + (wave * PER + l) * 1024));
      }
    } else {
#pragma unroll 1
      for (int l = 0; l < PER * 4; ++l) {
        const int c = wave * PER * 4 + l, word = c * 64 + lane, unit = word / 4, row = unit / UPR;
        dma_4b(base + (int64_t)(i0 + min(max(row, t.lo), t.hi)) * ss + min(O::swz(unit % UPR, row), units - 1) * 4 + (word & 3),
               __builtin_amdgcn_readfirstlane(lds0 + c * 256));
      }
    }
  }
};

// Workgroups that the fp32 forward has on the GPU at once.
template <int D>
constexpr int kPackedF32Slots = D == 64 ? 512 : 256;

// fp16 keeps its output's rounding residue times 2^11 (half a step of the
// largest fp16 number is 2^4; unscaled, the residue of 2^-10 would be denormal).
template <class E>
constexpr float kLoScale = std::is_same<E, F16>::value ? 2048.f : 1.f;

// Tile shape of a 16-bit forward: kPair 64 rows, two wavefronts per 32 of them
// taking alternate key tiles; kPlain 128 rows; kWide 256 rows (head_dim 128).
enum class PackedShape { kPair, kPlain, kWide };

// Columns C that a kernel computes, 64, 96, 128 or 256, and its rows in LDS: those of
// 96 are 128 wide (the swizzles permute the units of a power of two).
constexpr int packed_lds_dim(int C) { return C == 96 ? 128 : C; }

// Launchers, one translation unit per type (attn_packed_*.hip); grid: the items of the
// list at p.items times the heads.  ks: wavefronts per 32 rows (keys).
hipError_t launch_packed_fwd_bf16(const PackedParams& p, int C, PackedShape shape, int grid, hipStream_t st);
hipError_t launch_packed_fwd_f16(const PackedParams& p, int C, PackedShape shape, int grid, hipStream_t st);
// The same with the keys shared out (blocks of 64 rows; head_dim 256: 128), grid per chunk.
hipError_t launch_packed_chunks_bf16(const PackedParams& p, int C, int grid, hipStream_t st);
hipError_t launch_packed_chunks_f16(const PackedParams& p, int C, int grid, hipStream_t st);
hipError_t launch_packed_chunks_f32(const PackedParams& p, int C, int grid, hipStream_t st);
hipError_t launch_packed_fwd_f32(const PackedParams& p, int C, int ks, int grid, hipStream_t st);
// Backward, one launch: n_kv workgroups of dK and dV, n_q of dQ.
hipError_t launch_packed_bwd_f32(const PackedParams& p, int C, int ks, int n_kv, int n_q, hipStream_t st);
hipError_t launch_packed_bwd_bf16(const PackedParams& p, int C, int n_kv, int n_q, hipStream_t st);
hipError_t launch_packed_bwd_f16(const PackedParams& p, int C, int n_kv, int n_q, hipStream_t st);

}  // namespace trinix
