// Attention of a batch behind one shared prefix (trinix_attn.h,
// trinix_shared_prefix_args): softmax over the prefix's keys, which all
// requests read together, and every request's own.
//
// shared_rows16: a workgroup of 4 wavefronts owns 16 rows of one KV head (a row:
// request, query, head of the group) and a chunk of keys, either of the prefix
// (rows of any requests) or of one request's cache.  Per wavefront and step of 16
// keys S^T = K Q^T (K rows loaded straight into operand registers), an online
// softmax in fp32 and O^T += V^T P^T on fp32 matrix products, P unrounded.  The 4
// wavefronts take steps in turn and are merged through LDS; the chunk's (O, lse)
// goes to the workspace.
// shared_merge: one workgroup per row adds up its chunks.
#include "attn_params.h"
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
  int rows, rgp, rgs, n_p, chunk_p, n_s, chunk_s, wg_p;
  float scale_log2;
  float* part_o;    // (Hkv, rows, n_p + n_s, D) normalised O of a chunk
  float* part_lse;  // (Hkv, rows, n_p + n_s) its log-sum-exp, log2
};

struct F32 {};

// How 16 keys' scores form and V enters its product, per type.  A lane holds
// key (or row) lr = lane % 16, part lg = lane / 16 of head_dim.
template <class E, int D>
struct Vec {
  using Store = uint16_t;
  static constexpr int KK = D / 32, VC = D / 16, VW = VC / 2;  // V words per row segment
  struct K {
    u32x4_t w[KK];
  };
  struct V {
    uint32_t w[VW];
  };
  __device__ static K load_k(const Store* row, int lg) {
    K x;
#pragma unroll
    for (int k = 0; k < KK; ++k) x.w[k] = *(const u32x4_t*)(row + k * 32 + lg * 8);
    return x;
  }
  __device__ static V load_v(const Store* row, int lr) {
    V x;
    if constexpr (VW == 2) *(u32x2_t*)x.w = *(const u32x2_t*)(row + lr * VC);
    else
#pragma unroll
      for (int k = 0; k < VW; k += 4) *(u32x4_t*)(x.w + k) = *(const u32x4_t*)(row + lr * VC + k * 2);
    return x;
  }
  __device__ static float v_at(const V& x, int e) { return (e & 1) ? E::hi(x.w[e / 2]) : E::lo(x.w[e / 2]); }
  __device__ static f32x4_t scores(const K& k, const K& q) {
    f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < KK; ++t) s = E::mfma16(k.w[t], q.w[t], s);
    return s;
  }
  __device__ static void store4(Store* row, float a, float b, float c, float d) {
    *(u32x2_t*)row = (u32x2_t){E::pack(a, b), E::pack(c, d)};
  }
};
template <int D>
struct Vec<F32, D> {
  using Store = float;
  static constexpr int KT = D / 16, VC = D / 16;
  struct K {
    f32x4_t w[KT];
  };
  struct V {
    float w[VC];
  };
  __device__ static K load_k(const Store* row, int lg) {
    K x;
#pragma unroll
    for (int k = 0; k < KT; ++k) x.w[k] = *(const f32x4_t*)(row + k * 16 + lg * 4);
    return x;
  }
  __device__ static V load_v(const Store* row, int lr) {
    V x;
#pragma unroll
    for (int k = 0; k < VC; k += 4) *(f32x4_t*)(x.w + k) = *(const f32x4_t*)(row + lr * VC + k);
    return x;
  }
  __device__ static float v_at(const V& x, int e) { return x.w[e]; }
  __device__ static f32x4_t scores(const K& k, const K& q) {
    f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k.w[t][e], q.w[t][e], s, 0, 0, 0);
    return s;
  }
  __device__ static void store4(Store* row, float a, float b, float c, float d) { *(f32x4_t*)row = (f32x4_t){a, b, c, d}; }
};

__device__ inline int own_len(const SharedParams& p, int b) {
  return p.lens ? min(max(p.lens[b], 0), p.cap) : p.cap;
}

template <class E, int D>
__global__ __launch_bounds__(256) void shared_rows16(const SharedParams p) {
  using X = Vec<E, D>;
  using Store = typename X::Store;
  constexpr int VC = X::VC, LDO = D + 4;
  __shared__ float lds_o[4][16][LDO];
  __shared__ float lds_m[4][16];
  __shared__ float lds_l[4][16];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // work item: rows [r0, r0 + 16) below r1 of KV head hkv, keys [c0, c1), slot
  int r0, r1, hkv, c0, c1, slot, b = 0;
  const bool prefix = (int)blockIdx.x < p.wg_p;
  if (prefix) {
    // row groups of one chunk next to each other on one XCD
    int w = xcd_remap((int)blockIdx.x, p.wg_p);
    r0 = w % p.rgp * 16;
    r1 = p.rows;
    w /= p.rgp;
    slot = w % p.n_p;
    hkv = w / p.n_p;
    c0 = slot * p.chunk_p;
    c1 = min(p.P, c0 + p.chunk_p);
  } else {
    int w = (int)blockIdx.x - p.wg_p;
    hkv = w % p.Hkv;
    w /= p.Hkv;
    const int rg = w % p.rgs;
    w /= p.rgs;
    b = w % p.B;
    const int c = w / p.B;
    r0 = b * p.Sq * p.G + rg * 16;
    r1 = (b + 1) * p.Sq * p.G;
    slot = p.n_p + c;
    c0 = c * p.chunk_s;
    c1 = min(own_len(p, b), c0 + p.chunk_s);
    if (c0 >= c1) return;  // behind the request's last key: the merge does not read the slot
  }

  const int r = r0 + lr;
  const bool row_ok = r < r1;
  const int rc = row_ok ? r : r0, qi = rc / p.G, rb = qi / p.Sq, ri = qi % p.Sq, hq = hkv * p.G + rc % p.G;
  // last key that the row sees
  int jhi = c1 - 1;
  if (!prefix) jhi = min(jhi, own_len(p, b) - p.Sq + ri);
  if (!row_ok) jhi = -1;

  const auto qv = X::load_k((const Store*)p.q + rb * p.q_sb + (int64_t)ri * p.q_ss + hq * p.q_sh, lg);
  const int64_t kss = prefix ? p.pk_ss : p.k_ss, vss = prefix ? p.pv_ss : p.v_ss;
  const Store* kbase = prefix ? (const Store*)p.pk + hkv * p.pk_sh : (const Store*)p.k + b * p.k_sb + hkv * p.k_sh;
  const Store* vbase = prefix ? (const Store*)p.pv + hkv * p.pv_sh : (const Store*)p.v + b * p.v_sb + hkv * p.v_sh;
  auto load_k = [&](int j0) { return X::load_k(kbase + (int64_t)min(j0 + lr, c1 - 1) * kss, lg); };
  struct V4 {
    typename X::V v[4];
  };
  auto load_v = [&](int j0) {
    V4 x;
#pragma unroll
    for (int u = 0; u < 4; ++u) x.v[u] = X::load_v(vbase + (int64_t)min(j0 + lg * 4 + u, c1 - 1) * vss, lr);
    return x;
  };

  float m_run = -INFINITY, l_run = 0.f;
  f32x4_t acc[VC];  // acc[e][u]: row lr, d = (lg * 4 + u) * VC + e
#pragma unroll
  for (int e = 0; e < VC; ++e) acc[e] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  auto step = [&](int j0, const typename X::K& kv, const V4& vv) {
    const f32x4_t s = X::scores(kv, qv);  // s[u]: key j0 + lg * 4 + u, row lr
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
        acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(X::v_at(vv.v[u], e), x[u], acc[e], 0, 0, 0);
  };
  // Wavefront w takes the steps c0 + 16w + 64t, each loaded one step ahead.
  // Loads are unconditional (a condition would make the compiler wait at its
  // join): behind the last step they read the chunk's last key again, and the
  // step they feed is not run.
  const int jw = c0 + 16 * wave;
  const int n_steps = jw < c1 ? (c1 - jw + 63) / 64 : 0;
  // (fp32 at head_dim 256 has no registers to load ahead.)
  if constexpr (std::is_same<E, F32>::value && D == 256) {
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
  const int64_t at = ((int64_t)hkv * p.rows + r0 + rr) * (p.n_p + p.n_s) + slot;
  const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
  for (int e = 0; e < VC; e += 4)
    *(f32x4_t*)(p.part_o + at * D + dc + e) = (f32x4_t){o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv};
  if ((tid & 15) == 0) p.part_lse[at] = L > 0.f ? m + __log2f(L) : -INFINITY;
}

// One row: D / 4 threads share the columns, four each; 256 / (D / 4) groups of
// them take the chunks in turn and are merged through LDS.
template <class E, int D>
__global__ __launch_bounds__(256) void shared_merge(const SharedParams p) {
  using X = Vec<E, D>;
  using Store = typename X::Store;
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
  X::store4((Store*)p.o + b * p.o_sb + (int64_t)i * p.o_ss + hq * p.o_sh + t * 4, oo[0] * inv, oo[1] * inv, oo[2] * inv,
            oo[3] * inv);
  if (p.lse && t == 0) p.lse[((int64_t)b * p.Hq + hq) * p.Sq + i] = LL > 0.f ? (mm + __log2f(LL)) * kLn2 : -INFINITY;
}

template <class E, int D>
hipError_t launch(const SharedParams& p, int64_t wgs, hipStream_t st) {
  hipError_t e = hipSuccess;
  if (wgs > 0) e = launch_kernel(&shared_rows16<E, D>, dim3((unsigned)wgs), dim3(256), 0, st, p);
  if (e != hipSuccess) return e;
  return launch_kernel(&shared_merge<E, D>, dim3((unsigned)(p.rows * p.Hkv)), dim3(256), 0, st, p);
}
template <class E>
hipError_t launch(const SharedParams& p, int D, int64_t wgs, hipStream_t st) {
  return D == 64 ? launch<E, 64>(p, wgs, st) : D == 128 ? launch<E, 128>(p, wgs, st) : launch<E, 256>(p, wgs, st);
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
  p.rows = pl.rows, p.rgp = pl.rgp, p.rgs = pl.rgs;
  p.n_p = pl.n_p, p.chunk_p = pl.chunk_p, p.n_s = pl.n_s, p.chunk_s = pl.chunk_s;
  p.wg_p = (int)pl.wg_p;
  p.scale_log2 = a->softmax_scale * kLog2e;
  p.part_o = (float*)workspace;
  p.part_lse = p.part_o + (int64_t)p.Hkv * p.rows * (p.n_p + p.n_s) * a->head_dim;
  const int D = (int)a->head_dim;
  const int64_t wgs = pl.wg_p + pl.wg_s;
  hipStream_t st = (hipStream_t)stream;
  const hipError_t e = a->dtype == TRINIX_F32 ? launch<F32>(p, D, wgs, st)
                       : a->dtype == TRINIX_BF16 ? launch<BF16>(p, D, wgs, st) : launch<F16>(p, D, wgs, st);
  return e == hipSuccess ? TRINIX_OK : TRINIX_ERR_LAUNCH;
}
