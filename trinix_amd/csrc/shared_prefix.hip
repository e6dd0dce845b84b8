// Attention of a batch behind one shared prefix (trinix_attn.h,
// trinix_shared_prefix_args): softmax over the prefix's keys, which all
// requests read together, and every request's own.
//
// A row is a (request, query, head of the KV group) of one KV head.  Kinds of launch
// (plan_shared, packed_host.cpp):
//  - shared_split, 16-bit types: 64 rows (head_dim 256: 128) by a chunk of keys per
//    workgroup on Tile16, of the prefix (rows of any requests) or of one request's
//    cache.  Leaves (O, lse) of each row and chunk in fp32 in the workspace;
//    shared_merge adds them up, one workgroup per row.  64 requests behind 8192 keys,
//    caches of 1..1024, 32/8 heads of 128, 156 MB: 49 us with caches read from memory
//    (the copy rate gives 30; chunks that wait for a whole tile, the last items' tail
//    and the merge, 5 us, the rest), 39 with caches that the last level still holds;
//    there 95 with the 16-row kernel below (the prefix's products on fp32 matrix
//    instructions), 45 with it for the own keys alone.  Own rows loaded straight into
//    registers, three steps ahead: 54 from memory;
//  - shared_whole, 16-bit types: 64 or 128 rows of one request by all its keys, where
//    there are enough such blocks.  8 turns of 256 rows behind 6000 keys: 204 us
//    (1060 TFLOP/s), 309 in chunks;
//  - shared_rows16, fp32: 16 rows by a chunk of keys: per wavefront and step of 16 keys
//    S^T = K Q^T, K rows loaded straight into operand registers, an online softmax
//    and O^T += V^T P^T, all on fp32 matrix products; then shared_merge.
#include "attn_params.h"
#include "attn_tile16.h"
#include "packed_host.h"

namespace trinix {
namespace {

struct SharedParams {
  const void* q;
  const void* pk;
  const void* pv;
  const void* k;
  const void* v;
  void* o;
  float* lse;
  const int32_t* lens;
  int64_t q_sb, q_ss, q_sh, pk_ss, pk_sh, pv_ss, pv_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, o_sb, o_ss, o_sh;
  int B, Sq, P, cap, Hq, Hkv, G;
  int d;  // columns of every tensor: head_dim, at most the kernel's D
  int rows, n_p, chunk_p, n_s, chunk_s, wg_p;
  float scale_log2;
  float* part_o;    // (Hkv, rows, n_p + n_s, D) normalised O of a chunk
  float* part_lse;  // (Hkv, rows, n_p + n_s) its log-sum-exp, log2
};

// Output rows: four consecutive head_dim elements.
template <class E>
struct Row {
  using Store = uint16_t;
  __device__ static void store4(Store* row, float a, float b, float c, float d) {
    *(u32x2_t*)row = (u32x2_t){E::pack(a, b), E::pack(c, d)};
  }
};
struct F32 {};
template <>
struct Row<F32> {
  using Store = float;
  __device__ static void store4(Store* row, float a, float b, float c, float d) { *(f32x4_t*)row = (f32x4_t){a, b, c, d}; }
};

__device__ inline int own_len(const SharedParams& p, int b) {
  return p.lens ? min(max(p.lens[b], 0), p.cap) : p.cap;
}

// Rows [r0, r1) of KV head hkv (one request's for own keys), keys [c0, c1) of the
// prefix or of request b's cache, and where the partial result goes.
struct Item {
  int r0, r1, hkv, c0, c1, slot, b;
  bool prefix;
};
// `blk`-th of p.wg_p prefix items of `rows` rows; row blocks of a chunk next to
// each other on one XCD, which reads the chunk once into its L2.
__device__ inline Item prefix_item(const SharedParams& p, int blk, int rows) {
  Item it;
  const int groups = (p.rows + rows - 1) / rows;
  int w = xcd_remap(blk, p.wg_p);
  it.r0 = w % groups * rows;
  it.r1 = min(p.rows, it.r0 + rows);
  w /= groups;
  it.slot = w % p.n_p;
  it.hkv = w / p.n_p;
  it.c0 = it.slot * p.chunk_p;
  it.c1 = min(p.P, it.c0 + p.chunk_p);
  it.b = 0;
  it.prefix = true;
  return it;
}
// The same of the own keys, first chunks first.  c0 >= c1 behind the request's
// last key: nothing to do, the merge does not read the slot.
__device__ inline Item own_item(const SharedParams& p, int blk, int rows) {
  Item it;
  const int per = p.Sq * p.G, groups = (per + rows - 1) / rows;
  it.hkv = blk % p.Hkv;
  blk /= p.Hkv;
  const int rg = blk % groups;
  blk /= groups;
  it.b = blk % p.B;
  const int c = blk / p.B;
  it.r0 = it.b * per + rg * rows;
  it.r1 = min(it.r0 + rows, (it.b + 1) * per);
  it.slot = p.n_p + c;
  it.c0 = c * p.chunk_s;
  it.c1 = min(own_len(p, it.b), it.c0 + p.chunk_s);
  it.prefix = false;
  return it;
}
__device__ inline int64_t partial_at(const SharedParams& p, int hkv, int r, int slot) {
  return ((int64_t)hkv * p.rows + r) * (p.n_p + p.n_s) + slot;
}

// 16 rows against a chunk of keys.  A lane holds key (or row) lr = lane % 16 and
// part lg = lane / 16 of head_dim: d = 16 t + 4 lg + e of a K or Q row, VC
// consecutive d from lr * VC of the V rows of keys 4 lg .. 4 lg + 3.
template <int D>
__device__ __forceinline__ void rows16_body(const SharedParams& p, const Item it, float (*lds_o)[16][D + 4],
                                            float (*lds_m)[16], float (*lds_l)[16]) {
  constexpr int VC = D / 16;
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r0 = it.r0, r1 = it.r1, hkv = it.hkv, c0 = it.c0, c1 = it.c1, b = it.b;
  const bool prefix = it.prefix;
  const int r = r0 + lr;
  const bool row_ok = r < r1;
  const int rc = row_ok ? r : r0, qi = rc / p.G, rb = qi / p.Sq, ri = qi % p.Sq, hq = hkv * p.G + rc % p.G;
  // last key that the row sees
  int jhi = c1 - 1;
  if (!prefix) jhi = min(jhi, own_len(p, b) - p.Sq + ri);
  if (!row_ok) jhi = -1;

  struct Seg {
    f32x4_t w[VC];
  };
  struct V4 {
    f32x4_t w[4][VC / 4];
  };
  auto load_row = [&](const float* row) {  // (columns from d on: the last ones again)
    Seg x;
#pragma unroll
    for (int t = 0; t < VC; ++t) x.w[t] = *(const f32x4_t*)(row + min(t * 16 + lg * 4, p.d - 4));
    return x;
  };
  Seg qv = load_row((const float*)p.q + rb * p.q_sb + (int64_t)ri * p.q_ss + hq * p.q_sh);
#pragma unroll
  for (int t = 0; t < VC; ++t)
    if (t * 16 + lg * 4 >= p.d) qv.w[t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  const int64_t kss = prefix ? p.pk_ss : p.k_ss, vss = prefix ? p.pv_ss : p.v_ss;
  const float* kbase = prefix ? (const float*)p.pk + hkv * p.pk_sh : (const float*)p.k + b * p.k_sb + hkv * p.k_sh;
  const float* vbase = prefix ? (const float*)p.pv + hkv * p.pv_sh : (const float*)p.v + b * p.v_sb + hkv * p.v_sh;
  auto load_k = [&](int j0) { return load_row(kbase + (int64_t)min(j0 + lr, c1 - 1) * kss); };
  auto load_v = [&](int j0) {
    V4 x;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < VC / 4; ++k)
        x.w[u][k] = *(const f32x4_t*)(vbase + (int64_t)min(j0 + lg * 4 + u, c1 - 1) * vss + min(lr * VC + k * 4, p.d - 4));
    return x;
  };

  float m_run = -INFINITY, l_run = 0.f;
  f32x4_t acc[VC];  // acc[e][u]: row lr, d = (lg * 4 + u) * VC + e
#pragma unroll
  for (int e = 0; e < VC; ++e) acc[e] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  auto step = [&](int j0, const Seg& kv, const V4& vv) {
    f32x4_t s = {0.f, 0.f, 0.f, 0.f};  // s[u]: key j0 + lg * 4 + u, row lr
#pragma unroll
    for (int t = 0; t < VC; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(kv.w[t][e], qv.w[t][e], s, 0, 0, 0);
    float x[4], mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      x[u] = j0 + lg * 4 + u <= jhi ? s[u] * p.scale_log2 : -INFINITY;
      mx = fmaxf(mx, x[u]);
    }
    mx = xlane_max(fmaxf(mx, __shfl_xor(mx, 16)));
    const float m_new = fmaxf(m_run, mx), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      x[u] = __builtin_amdgcn_exp2f(x[u] - m_use);
      sum += x[u];
    }
    l_run = l_run * alpha + sum;
    m_run = m_new;
#pragma unroll
    for (int e = 0; e < VC; ++e) acc[e] *= alpha;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < VC; ++e)
        acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv.w[u][e / 4][e % 4], x[u], acc[e], 0, 0, 0);
  };
  // Wavefront w takes the steps c0 + 16w + 64t, each loaded one step ahead.
  // Loads are unconditional (a condition would make the compiler wait at its
  // join): behind the last step they read the chunk's last key again, and the
  // step they feed is not run.
  const int jw = c0 + 16 * wave;
  const int n_steps = jw < c1 ? (c1 - jw + 63) / 64 : 0;
  // (Head_dim 256 has no registers to load ahead.)
  if constexpr (D == 256) {
    for (int t = 0; t < n_steps; ++t) step(jw + 64 * t, load_k(jw + 64 * t), load_v(jw + 64 * t));
  } else if (n_steps > 0) {
    auto ka = load_k(jw);
    auto va = load_v(jw);
    for (int t = 0; t < n_steps; t += 2) {
      const int ja = jw + 64 * t;
      auto kb = load_k(ja + 64);
      auto vb = load_v(ja + 64);
      __builtin_amdgcn_sched_barrier(0);
      step(ja, ka, va);
      ka = load_k(ja + 128);
      va = load_v(ja + 128);
      __builtin_amdgcn_sched_barrier(0);
      if (t + 1 < n_steps) step(ja + 64, kb, vb);
    }
  }

  const float l_row = xlane_sum(l_run + __shfl_xor(l_run, 16));
  if (lg == 0) {
    lds_m[wave][lr] = m_run;
    lds_l[wave][lr] = l_row;
  }
#pragma unroll
  for (int e = 0; e < VC; ++e)
#pragma unroll
    for (int u = 0; u < 4; ++u) lds_o[wave][lr][(lg * 4 + u) * VC + e] = acc[e][u];
  __syncthreads();
  const int rr = tid >> 4, dc = (tid & 15) * VC;
  if (r0 + rr >= r1) return;
  float mw[4], m = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) m = fmaxf(m, mw[w] = lds_m[w][rr]);
  const float m_use = m == -INFINITY ? 0.f : m;
  float L = 0.f, o[VC];
#pragma unroll
  for (int e = 0; e < VC; ++e) o[e] = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = __builtin_amdgcn_exp2f(mw[w] - m_use);
    L += lds_l[w][rr] * f;
#pragma unroll
    for (int e = 0; e < VC; ++e) o[e] += lds_o[w][rr][dc + e] * f;
  }
  const int64_t at = partial_at(p, hkv, r0 + rr, it.slot);
  const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
  for (int e = 0; e < VC; e += 4)
    *(f32x4_t*)(p.part_o + at * D + dc + e) = (f32x4_t){o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv};
  if ((tid & 15) == 0) p.part_lse[at] = L > 0.f ? m + __log2f(L) : -INFINITY;
}

template <int D>
__global__ __launch_bounds__(256) void shared_rows16(const SharedParams p) {
  __shared__ float lds_o[4][16][D + 4];
  __shared__ float lds_m[4][16];
  __shared__ float lds_l[4][16];
  const int blk = (int)blockIdx.x;
  if (blk < p.wg_p) {
    rows16_body<D>(p, prefix_item(p, blk, 16), lds_o, lds_m, lds_l);
  } else {
    const Item it = own_item(p, blk - p.wg_p, 16);
    if (it.c0 < it.c1) rows16_body<D>(p, it, lds_o, lds_m, lds_l);
  }
}

// The lane's query of a block of 32 rows from rw of KV head hkv, below r1.
struct TileRow {
  int r, b, i, h;
  bool ok;
  __device__ TileRow(const SharedParams& p, int rw, int r1, int lane, int hkv) {
    r = rw + (lane & 31);
    ok = r < r1;
    const int rc = min(r, r1 - 1), qi = rc / p.G;
    b = qi / p.Sq, i = qi % p.Sq, h = hkv * p.G + rc % p.G;
  }
  __device__ const uint16_t* q(const SharedParams& p) const {
    return (const uint16_t*)p.q + b * p.q_sb + (int64_t)i * p.q_ss + h * p.q_sh;
  }
};
// Keys [c0, c1) of the prefix: every row sees all of them.
template <int BN>
__device__ inline KeyRun prefix_run(const SharedParams& p, int hkv, int c0, int c1, bool ok, bool wave_ok) {
  KeyRun kr;
  kr.k_ss = p.pk_ss, kr.v_ss = p.pv_ss;
  kr.k = (const uint16_t*)p.pk + hkv * p.pk_sh + (int64_t)c0 * p.pk_ss;
  kr.v = (const uint16_t*)p.pv + hkv * p.pv_sh + (int64_t)c0 * p.pv_ss;
  kr.lo = 0, kr.n = c1 - c0, kr.d = p.d;
  kr.t_lo = kr.t_flo = 0;
  kr.t_hi = (kr.n + BN - 1) / BN;
  kr.t_fhi = kr.n / BN;
  kr.jlo = ok ? 0 : INT_MAX;
  kr.jspan = (uint32_t)(kr.n - 1);
  kr.wlo = 0;
  kr.whi = wave_ok ? kr.n - 1 : -1;
  kr.pos = 0;
  return kr;
}
// Keys [c0, c1) of request b's cache: query i sees those up to len - Sq + i.
// Queries of the workgroup: ib .. ie, of the wavefront: up to iw (-1: none).
template <int BN>
__device__ inline KeyRun own_run(const SharedParams& p, int b, int hkv, int c0, int c1, int len, int ib, int ie, int iw,
                                 int i, bool ok) {
  KeyRun kr;
  kr.k_ss = p.k_ss, kr.v_ss = p.v_ss;
  kr.k = (const uint16_t*)p.k + b * p.k_sb + hkv * p.k_sh + (int64_t)c0 * p.k_ss;
  kr.v = (const uint16_t*)p.v + b * p.v_sb + hkv * p.v_sh + (int64_t)c0 * p.v_ss;
  kr.lo = 0, kr.n = c1 - c0, kr.d = p.d;
  const int at0 = len - p.Sq - c0;  // last key of query 0, from c0
  kr.t_lo = kr.t_flo = 0;
  kr.t_hi = (min(kr.n, max(at0 + ie + 1, 0)) + BN - 1) / BN;
  kr.t_fhi = min(kr.t_hi, min(kr.n, max(at0 + ib + 1, 0)) / BN);
  const int last = min(at0 + i, kr.n - 1);
  kr.jlo = ok && last >= 0 ? 0 : INT_MAX;
  kr.jspan = (uint32_t)max(last, 0);
  kr.wlo = 0;
  kr.whi = iw >= 0 ? min(at0 + iw, kr.n - 1) : -1;
  kr.pos = 0;
  return kr;
}

// 128 / KS rows by a chunk of keys on Tile16 (KS = 2: two wavefronts per 32 rows):
// the prefix's items, then the own keys'.  In one launch: the prefix items are
// bound by the matrix cores, the own keys' by memory, and one of each shares a CU
// (64 KiB of LDS each; head_dim 256: 128).
template <class E, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void shared_split(const SharedParams p) {
  constexpr int KS = D == 256 ? 1 : 2, BN = D == 128 ? 32 : 64, BM = 128 / KS;
  TRINIX_TILE16_LDS(D, BN, KS);
  const int blk = (int)blockIdx.x;
  const Item it = blk < p.wg_p ? prefix_item(p, blk, BM) : own_item(p, blk - p.wg_p, BM);
  if (it.c0 >= it.c1) return;
  Tile16<E, D, D, BN, 4, KS, 0> T(lds_k0, lds_k1, lds_v0, lds_v1);
  const int rw = it.r0 + (T.wave / KS) * 32;
  const TileRow row(p, rw, it.r1, T.lane, it.hkv);
  T.load_q(row.q(p), p.d, p.scale_log2, 0.f);
  if (it.prefix) {
    T.run(prefix_run<BN>(p, it.hkv, it.c0, it.c1, row.ok, rw < it.r1));
  } else {
    const int base = it.b * p.Sq, ib = it.r0 / p.G - base, ie = (it.r1 - 1) / p.G - base;
    const int iw = rw < it.r1 ? min(rw + 31, it.r1 - 1) / p.G - base : -1;
    T.run(own_run<BN>(p, it.b, it.hkv, it.c0, it.c1, own_len(p, it.b), ib, ie, iw, row.i, row.ok));
  }
  const float l = T.finish();
  if (!row.ok || T.kp != 0) return;
  const int64_t at = partial_at(p, it.hkv, row.r, it.slot);
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int vq = 0; vq < 4; ++vq)
      *(f32x4_t*)(p.part_o + at * D + db * 32 + vq * 8 + T.g * 4) =
          (f32x4_t){T.acc[db][vq * 4] * inv, T.acc[db][vq * 4 + 1] * inv, T.acc[db][vq * 4 + 2] * inv, T.acc[db][vq * 4 + 3] * inv};
  if (T.g == 0) p.part_lse[at] = l > 0.f ? T.m_run + __log2f(l) : -INFINITY;
}

// Whole rows: 128 / KS rows of one request and KV head against the prefix and then
// its own keys, in one softmax; no partial results.  For requests of many rows.
template <class E, int D, int KS>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void shared_whole(const SharedParams p) {
  constexpr int BN = KS == 2 && D == 128 ? 32 : 64, BM = 128 / KS;
  TRINIX_TILE16_LDS(D, BN, KS);
  // an XCD runs whole KV heads where they divide evenly: their prefix is in its L2
  const int per = p.Sq * p.G, groups = (per + BM - 1) / BM;
  const int w = xcd_remap((int)blockIdx.x, p.Hkv * p.B * groups);
  const int hkv = w / (p.B * groups), b = w / groups % p.B, r0 = b * per + w % groups * BM, r1 = min(r0 + BM, (b + 1) * per);
  Tile16<E, D, D, BN, 4, KS, 0> T(lds_k0, lds_k1, lds_v0, lds_v1);
  const int rw = r0 + (T.wave / KS) * 32;
  const TileRow row(p, rw, r1, T.lane, hkv);
  T.load_q(row.q(p), p.d, p.scale_log2, 0.f);
  if (p.P > 0) {
    T.run(prefix_run<BN>(p, hkv, 0, p.P, row.ok, rw < r1));
    __syncthreads();  // the buffers are free for the second run
  }
  const int len = own_len(p, b);
  if (len > 0) {
    const int base = b * p.Sq, iw = rw < r1 ? min(rw + 31, r1 - 1) / p.G - base : -1;
    T.run(own_run<BN>(p, b, hkv, 0, len, len, r0 / p.G - base, (r1 - 1) / p.G - base, iw, row.i, row.ok));
  }
  const float l = T.finish();
  if (!row.ok || T.kp != 0) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;  // a row that sees no key: 0
  uint16_t* o = (uint16_t*)p.o + b * p.o_sb + (int64_t)row.i * p.o_ss + row.h * p.o_sh;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int vq = 0; vq < 4; ++vq)
      if (db * 32 + vq * 8 < p.d)
        Row<E>::store4(o + db * 32 + vq * 8 + T.g * 4, T.acc[db][vq * 4] * inv, T.acc[db][vq * 4 + 1] * inv,
                       T.acc[db][vq * 4 + 2] * inv, T.acc[db][vq * 4 + 3] * inv);
  if (p.lse && T.g == 0)
    p.lse[((int64_t)b * p.Hq + row.h) * p.Sq + row.i] = l > 0.f ? (T.m_run + __log2f(l)) * kLn2 : -INFINITY;
}

// One row: D / 4 threads share the columns, four each; 256 / (D / 4) groups of
// them take the chunks in turn and are merged through LDS.
template <class E, int D>
__global__ __launch_bounds__(256) void shared_merge(const SharedParams p) {
  using Store = typename Row<E>::Store;
  constexpr int TPS = D / 4, NG = 256 / TPS, UNR = 4;
  __shared__ f32x4_t s_o[NG][TPS];
  __shared__ float s_m[NG], s_l[NG];
  const int hkv = (int)blockIdx.x / p.rows, r = (int)blockIdx.x % p.rows;
  const int qi = r / p.G, b = qi / p.Sq, i = qi % p.Sq, hq = hkv * p.G + r % p.G;
  const int t = threadIdx.x, g = t / TPS, c = t % TPS;
  // chunks of the own keys that were written
  const int n = p.n_p + (p.n_s ? (own_len(p, b) + p.chunk_s - 1) / p.chunk_s : 0);
  const int64_t at = (int64_t)blockIdx.x * (p.n_p + p.n_s);
  const float* pl = p.part_lse + at;
  const float* po = p.part_o + at * D + c * 4;
  float m = -INFINITY, L = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = g; s0 < n; s0 += NG * UNR) {
    float ls[UNR];
    f32x4_t ov[UNR];
    float mn = m;
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const int s = s0 + u * NG, sc = min(s, n - 1);
      ls[u] = s < n ? pl[sc] : -INFINITY;
      ov[u] = *(const f32x4_t*)(po + (int64_t)sc * D);
      mn = fmaxf(mn, ls[u]);
    }
    const float m_use = mn == -INFINITY ? 0.f : mn, a = __builtin_amdgcn_exp2f(m - m_use);
    L *= a;
    o *= a;
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const float w = __builtin_amdgcn_exp2f(ls[u] - m_use);
      L += w;
      o += w * ov[u];
    }
    m = mn;
  }
  s_o[g][c] = o;
  if (c == 0) {
    s_m[g] = m;
    s_l[g] = L;
  }
  __syncthreads();
  if (t >= TPS) return;
  float mm = -INFINITY;
#pragma unroll
  for (int k = 0; k < NG; ++k) mm = fmaxf(mm, s_m[k]);
  const float m_use = mm == -INFINITY ? 0.f : mm;
  float LL = 0.f;
  f32x4_t oo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < NG; ++k) {
    const float w = __builtin_amdgcn_exp2f(s_m[k] - m_use);
    LL += w * s_l[k];
    oo += w * s_o[k][t];
  }
  const float inv = LL > 0.f ? 1.f / LL : 0.f;  // a row that sees no key: 0
  if (t * 4 < p.d)
    Row<E>::store4((Store*)p.o + b * p.o_sb + (int64_t)i * p.o_ss + hq * p.o_sh + t * 4, oo[0] * inv, oo[1] * inv, oo[2] * inv,
                   oo[3] * inv);
  if (p.lse && t == 0) p.lse[((int64_t)b * p.Hq + hq) * p.Sq + i] = LL > 0.f ? (mm + __log2f(LL)) * kLn2 : -INFINITY;
}

template <class E, int D>
hipError_t launch(const SharedParams& p, const SharedPlan& pl, hipStream_t st) {
  const dim3 grid((unsigned)(pl.wg_p + pl.wg_s)), block(256);
  hipError_t e = hipSuccess;
  if constexpr (std::is_same<E, F32>::value) {
    if (grid.x) e = launch_kernel(&shared_rows16<D>, grid, block, 0, st, p);
  } else {
    if (pl.kind == SharedKind::kWhole128) return launch_kernel(&shared_whole<E, D, 1>, grid, block, 0, st, p);
    if constexpr (D != 256)
      if (pl.kind == SharedKind::kWhole64) return launch_kernel(&shared_whole<E, D, 2>, grid, block, 0, st, p);
    if (grid.x) e = launch_kernel(&shared_split<E, D>, grid, block, 0, st, p);
  }
  if (e != hipSuccess) return e;
  return launch_kernel(&shared_merge<E, D>, dim3((unsigned)(p.rows * p.Hkv)), block, 0, st, p);
}
template <class E>
hipError_t launch(const SharedParams& p, int D, const SharedPlan& pl, hipStream_t st) {
  return D == 64 ? launch<E, 64>(p, pl, st) : D == 128 ? launch<E, 128>(p, pl, st) : launch<E, 256>(p, pl, st);
}

}  // namespace
}  // namespace trinix

using namespace trinix;

extern "C" int trinix_shared_prefix_fwd(const trinix_shared_prefix_args* a, void* workspace, int64_t workspace_bytes,
                                        void* stream) {
  int rc = validate_shared(a);
  SharedPlan pl;
  if (rc == TRINIX_OK) rc = plan_shared(a, &pl);
  if (rc != TRINIX_OK) return rc;
  if (pl.ws_bytes > 0 && (!workspace || workspace_bytes < pl.ws_bytes || ((uintptr_t)workspace & 15) != 0))
    return TRINIX_ERR_BAD_ARGUMENT;
  SharedParams p{};
  p.q = a->q, p.pk = a->prefix_k, p.pv = a->prefix_v, p.k = a->k, p.v = a->v, p.o = a->out;
  p.lse = a->lse;
  p.lens = a->seq_lens;
  p.q_sb = a->q_stride[0], p.q_ss = a->q_stride[1], p.q_sh = a->q_stride[2];
  p.pk_ss = a->prefix_k_stride[0], p.pk_sh = a->prefix_k_stride[1];
  p.pv_ss = a->prefix_v_stride[0], p.pv_sh = a->prefix_v_stride[1];
  p.k_sb = a->k_stride[0], p.k_ss = a->k_stride[1], p.k_sh = a->k_stride[2];
  p.v_sb = a->v_stride[0], p.v_ss = a->v_stride[1], p.v_sh = a->v_stride[2];
  p.o_sb = a->out_stride[0], p.o_ss = a->out_stride[1], p.o_sh = a->out_stride[2];
  p.B = (int)a->batch, p.Sq = (int)a->seqlen_q, p.P = (int)a->prefix_len, p.cap = (int)a->capacity;
  p.Hq = (int)a->nheads_q, p.Hkv = (int)a->nheads_kv, p.G = p.Hq / p.Hkv;
  p.d = (int)a->head_dim;
  p.rows = pl.rows;
  p.n_p = pl.n_p, p.chunk_p = pl.chunk_p, p.n_s = pl.n_s, p.chunk_s = pl.chunk_s;
  p.wg_p = (int)pl.wg_p;
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.part_o = (float*)workspace;
  p.part_lse = p.part_o + (int64_t)p.Hkv * p.rows * (p.n_p + p.n_s) * packed_kernel_dim(a->head_dim);
  const int D = packed_kernel_dim(a->head_dim);
  hipStream_t st = (hipStream_t)stream;
  const hipError_t e = a->dtype == TRINIX_F32 ? launch<F32>(p, D, pl, st)
                       : a->dtype == TRINIX_BF16 ? launch<BF16>(p, D, pl, st) : launch<F16>(p, D, pl, st);
  return e == hipSuccess ? TRINIX_OK : TRINIX_ERR_LAUNCH;
}
