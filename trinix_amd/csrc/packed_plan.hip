// trinix_packed_plan: the work items of a packed batch from its cumulative
// lengths, on the GPU (nothing is read back to the host, so it can be captured
// into a graph and replayed with new lengths).
//
// One workgroup per list (packed_map.h).  Boundaries are clamped into [0, total]
// and made non-decreasing (a prefix maximum), so that no content of the arrays
// leads outside the tensors; block counts are summed over the sequences; every
// item then finds its sequence by bisection and is placed by a counting sort on
// its cost, 1024 classes, the longest first (items of one class in any order:
// it changes when an item runs, not its result).
// Latency bound, once per batch: 9 us for ten sequences of 8326 rows, 42 us for 4000 of 3.
#include "common.h"
#include "packed_map.h"
#include "trinix_attn.h"

namespace trinix {
namespace {

constexpr int kPlanThreads = 1024;

struct PlanParams {
  const int32_t* cu_q;
  const int32_t* cu_k;
  int32_t* plan;
  int n_seqs, total_q, total_k;
};

// Inclusive scan over the workgroup, and the result of all of it; every thread calls
// it.  Within the wavefronts first, then over their results.
template <class F>
__device__ inline int block_scan(int x, int* lds, F op, int& all) {
  constexpr int NW = kPlanThreads / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x = op(y, x);
  }
  __syncthreads();  // the last call's results are read
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int sum = lds[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    if (w == wave) x = op(sum, x);
    sum = op(sum, lds[w]);
  }
  all = sum;
  return x;
}

__global__ __launch_bounds__(kPlanThreads) void packed_plan_kernel(const PlanParams p) {
  __shared__ int scan[kPlanThreads / 64];
  __shared__ int hist[kPlanThreads];
  __shared__ int most;
  __shared__ unsigned long long total;
  const int list = blockIdx.x, t = threadIdx.x, n = p.n_seqs;
  int32_t* const items = p.plan + packed_list_offset(list, p.total_q, p.total_k, n);
  int32_t* const cq = p.plan + packed_list_offset(kPackedLists, p.total_q, p.total_k, n) + list * packed_scratch_ints(n);
  int32_t* const ck = cq + n + 3;
  int32_t* const first = ck + n + 3;
  const auto larger = [](int a, int b) { return a > b ? a : b; };
  const auto plus = [](int a, int b) { return a + b; };

  int top_q = 0, top_k = 0;
  for (int base = 0; base <= n; base += kPlanThreads) {
    const int i = base + t;
    int q = top_q, k = top_k;
    if (i > 0 && i <= n) {
      q = larger(q, imin(p.cu_q[i], p.total_q));
      k = larger(k, imin(p.cu_k[i], p.total_k));
    }
    q = block_scan(q, scan, larger, top_q);
    k = block_scan(k, scan, larger, top_k);
    if (i <= n) cq[i] = q, ck[i] = k;
  }
  __syncthreads();

  int count = 0;  // items of the sequences so far
  for (int base = 0; base < n + 2; base += kPlanThreads) {
    const int s = base + t;
    const int nb = s < n + 2 ? packed_blocks(packed_seq(s, n, cq, ck, p.total_q, p.total_k), list) : 0;
    int all;
    const int end = count + block_scan(nb, scan, plus, all);
    count += all;
    if (s < n + 2) first[s] = end - nb;
  }
  if (t == 0) most = 1, total = 0;
  hist[t] = 0;
  __syncthreads();

  // sequence and cost of item x
  auto find = [&](int x, PackedSeq& q, int& blk, int& cost) {
    int lo = 0, hi = n + 1;  // the last sequence whose first item is at or before x
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (first[mid] <= x) lo = mid;
      else hi = mid - 1;
    }
    q = packed_seq(lo, n, cq, ck, p.total_q, p.total_k);
    blk = x - first[lo];
    cost = packed_cost(q, list, blk);
    return lo;
  };
  PackedSeq q;
  int blk, cost, top = 0;
  unsigned long long sum = 0;
  for (int x = t; x < count; x += kPlanThreads) {
    find(x, q, blk, cost);
    top = larger(top, cost);
    sum += (unsigned long long)cost;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    top = larger(top, __shfl_xor(top, d));
    sum += __shfl_xor(sum, d);
  }
  if ((t & 63) == 0 && sum > 0) {
    atomicMax(&most, top);
    atomicAdd(&total, sum);
  }
  __syncthreads();
  const auto bucket = [&](int c) { return kPlanThreads - 1 - (int)((int64_t)c * (kPlanThreads - 1) / most); };
  for (int x = t; x < count; x += kPlanThreads) {
    find(x, q, blk, cost);
    atomicAdd(&hist[bucket(cost)], 1);
  }
  __syncthreads();
  const int mine = hist[t];
  int all;
  const int upto = block_scan(mine, scan, plus, all);
  hist[t] = upto - mine;
  __syncthreads();
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  const int sum64 = (int)lmin((int64_t)(total / 64), INT32_MAX);
  for (int x = t; x < count; x += kPlanThreads) {
    const int s = find(x, q, blk, cost);
    i32x4* dst = (i32x4*)(items + (int64_t)atomicAdd(&hist[bucket(cost)], 1) * kPackedItemInts);
    dst[0] = (i32x4){q.q0, q.lq, q.k0, q.lk};
    dst[1] = (i32x4){blk, s, sum64, 0};
  }
  const int cap = (int)packed_list_cap(packed_list_is_keys(list) ? p.total_k : p.total_q, n, packed_list_block(list));
  for (int x = count + t; x < cap; x += kPlanThreads) {
    i32x4* dst = (i32x4*)(items + (int64_t)x * kPackedItemInts);
    dst[0] = (i32x4){0, 0, 0, 0};
    dst[1] = (i32x4){-1, 0, 0, 0};
  }
}

}  // namespace
}  // namespace trinix

using namespace trinix;

extern "C" int trinix_packed_plan(const int32_t* cu_q, const int32_t* cu_k, int64_t n_seqs, int64_t total_q,
                                  int64_t total_k, int32_t* plan, int64_t plan_bytes, void* stream) {
  if (!cu_q || !cu_k || !plan) return TRINIX_ERR_NULL_POINTER;
  int64_t need = 0;
  const int rc = trinix_packed_plan_bytes(n_seqs, total_q, total_k, &need);
  if (rc != TRINIX_OK) return rc;
  if (plan_bytes < need || ((uintptr_t)plan & 15) != 0 || (((uintptr_t)cu_q | (uintptr_t)cu_k) & 3) != 0)
    return TRINIX_ERR_BAD_ARGUMENT;
  PlanParams p{cu_q, cu_k, plan, (int)n_seqs, (int)total_q, (int)total_k};
  const hipError_t e =
      launch_kernel(&packed_plan_kernel, dim3(kPackedLists), dim3(kPlanThreads), 0, (hipStream_t)stream, p);
  return e == hipSuccess ? TRINIX_OK : TRINIX_ERR_LAUNCH;
}
