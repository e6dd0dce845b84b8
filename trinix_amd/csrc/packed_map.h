// Index maps of attention over packed sequences: the plan (work items of every
// block size, built on the GPU from the cumulative lengths), which item and
// head a workgroup runs, and the band of allowed pairs.  Plain integer code
// with no HIP dependency (host and device; see index_map.h).
#pragma once
#include <stdint.h>

#include "index_map.h"

namespace trinix {

// A plan holds five lists of work items: blocks of 64, 128 and 256 query rows
// (lists 0..2) and of 64 and 128 keys (lists 3, 4) of one sequence each, the
// longest first.  An item is eight int32:
//   first query row, query rows, first key, keys of its sequence; block number
//   (-1: no item); sequence; the sum of the costs (packed_cost) of the list's items, in
//   64s; zero.
// Rows behind the last sequence form a sequence of their own without keys
// (their output is 0), keys behind it one without rows (their gradients are 0).
constexpr int kPackedLists = 5;
constexpr int kPackedItemInts = 8;
__host__ __device__ inline int packed_list_block(int list) { return 64 << (list % 3); }
__host__ __device__ inline bool packed_list_is_keys(int list) { return list >= 3; }

// Most items of a list: every sequence (the one behind the last included) ends
// in at most one block that is not whole; rounded up to whole rounds of the XCDs.
__host__ __device__ inline int64_t packed_list_cap(int64_t total, int64_t n_seqs, int block) {
  const int64_t n = total / block + lmin(n_seqs + 1, total);
  return (n + kXcds - 1) / kXcds * kXcds;
}
// First int32 of list `list` in a plan; of the scratch behind the lists for list = kPackedLists.
__host__ __device__ inline int64_t packed_list_offset(int list, int64_t total_q, int64_t total_k, int64_t n_seqs) {
  int64_t at = 0;
  for (int l = 0; l < list; ++l)
    at += packed_list_cap(packed_list_is_keys(l) ? total_k : total_q, n_seqs, packed_list_block(l)) * kPackedItemInts;
  return at;
}
// Scratch of one list: clamped boundaries of the queries and of the keys, and
// the first item of every sequence (n_seqs + 3 each).
__host__ __device__ inline int64_t packed_scratch_ints(int64_t n_seqs) { return 3 * (n_seqs + 3); }
__host__ __device__ inline int64_t packed_plan_ints(int64_t total_q, int64_t total_k, int64_t n_seqs) {
  return packed_list_offset(kPackedLists, total_q, total_k, n_seqs) + kPackedLists * packed_scratch_ints(n_seqs);
}

// Sequence s of n_seqs + 2 from the clamped boundaries.
struct PackedSeq {
  int q0, lq, k0, lk;
};
__host__ __device__ inline PackedSeq packed_seq(int s, int n_seqs, const int* cq, const int* ck, int total_q, int total_k) {
  PackedSeq r{0, 0, 0, 0};
  if (s < n_seqs) {
    r.q0 = cq[s], r.lq = cq[s + 1] - cq[s];
    r.k0 = ck[s], r.lk = ck[s + 1] - ck[s];
  } else if (s == n_seqs) {
    r.q0 = cq[n_seqs], r.lq = total_q - cq[n_seqs];
  } else {
    r.k0 = ck[n_seqs], r.lk = total_k - ck[n_seqs];
  }
  return r;
}
__host__ __device__ inline int packed_blocks(const PackedSeq& s, int list) {
  const int bs = packed_list_block(list);
  return ((packed_list_is_keys(list) ? s.lk : s.lq) + bs - 1) / bs;
}
// What orders the items: the keys that a block of rows sees, or the rows that
// see a block of keys, in a causal call.
__host__ __device__ inline int packed_cost(const PackedSeq& s, int list, int blk) {
  const int bs = packed_list_block(list), off = s.lk - s.lq;
  if (packed_list_is_keys(list)) return s.lq - imin(imax(blk * bs - off, 0), s.lq);
  return imin(imax(off + imin((blk + 1) * bs, s.lq), 0), s.lk);
}

// Item and head of workgroup `blk` of n_items * heads; G heads share keys.
// With the KV heads dealt evenly to the XCDs an XCD runs whole groups, item by
// item, so that the blocks of a sequence find its keys in one L2; otherwise the
// items are dealt to the XCDs (n_items is a multiple of kXcds), all heads of an
// item on one.  Either way every XCD meets the longest items first.
struct PackedWork {
  int item, h;
};
__host__ __device__ inline PackedWork packed_work(int blk, int heads_kv, int G) {
  PackedWork w;
  const int xcd = blk % kXcds, j = blk / kXcds;
  if (heads_kv % kXcds == 0) {
    const int per = heads_kv / kXcds * G;
    w.item = j / per;
    w.h = xcd * per + j % per;
  } else {
    const int heads = heads_kv * G;
    w.item = j / heads * kXcds + xcd;
    w.h = j % heads;
  }
  return w;
}

// Allowed pairs of a sequence: j - i in [dlo, dhi] for query row i and key j of
// it, the queries being its last lq positions: causal j <= i + off, window
// -wl <= j - i - off <= wr, off = lk - lq.
__host__ __device__ inline void packed_band(int lq, int lk, bool causal, bool has_window, int64_t wl, int64_t wr,
                                            int& dlo, int& dhi) {
  constexpr int64_t kFar = 1ll << 30;
  const int64_t off = (int64_t)lk - lq;
  int64_t lo = -kFar, hi = kFar;
  if (causal) hi = off;
  if (has_window) {
    lo = lmax(lo, off - wl);
    hi = lmin(hi, off + wr);
  }
  dlo = (int)lmin(lmax(lo, -kFar), kFar);
  dhi = (int)lmin(lmax(hi, -kFar), kFar);
}

// First and last key of a sequence that any of its rows sees, and row that sees any key
// (inside the sequence; anything there where no pair is allowed).  Tiles read nothing
// outside, so what the others hold, NaN too, reaches no result.
struct PackedRange {
  int lo, hi;
};
__host__ __device__ inline PackedRange packed_range(int64_t lo, int64_t hi, int n) {
  PackedRange r;
  r.hi = (int)lmin(lmax(hi, 0), (int64_t)n - 1);
  r.lo = (int)lmin(lmax(lo, 0), (int64_t)r.hi);
  return r;
}
__host__ __device__ inline PackedRange packed_seen_keys(int lq, int lk, int dlo, int dhi) {
  return packed_range(dlo, (int64_t)lq - 1 + dhi, lk);
}
__host__ __device__ inline PackedRange packed_seeing_rows(int lq, int lk, int dlo, int dhi) {
  return packed_range(-(int64_t)dhi, (int64_t)lk - 1 - dlo, lq);
}
// First and last row of the tile at n0 of such a range; the rows before and behind read these.
__host__ __device__ inline PackedRange packed_tile_range(const PackedRange& r, int n0) {
  PackedRange t;
  t.hi = imax(r.hi - n0, 0);
  t.lo = imin(imax(r.lo - n0, 0), t.hi);
  return t;
}

// A block's `tiles` tiles of BN keys over at most `most` workgroups: tiles per chunk and
// chunks (1 for no tiles).  A chunk is at least kPackedChunkKeys keys and at least what
// each of `slots` workgroups would take of all items' keys (`total`, in 64s) and heads.
constexpr int kPackedChunkKeys = 512;
struct PackedChunks {
  int per, n;
};
__host__ __device__ inline PackedChunks packed_chunks(int tiles, int BN, int most, int total, int heads, int slots) {
  const int64_t share = (int64_t)total * heads / slots * (64 / BN);
  PackedChunks c;
  c.per = (int)lmin(lmax(lmax(kPackedChunkKeys / BN, share), (tiles + most - 1) / most), INT32_MAX);
  c.n = imax(1, (int)(((int64_t)tiles + c.per - 1) / c.per));
  return c;
}
// Workgroup of a grid of `per_chunk` (whole rounds of the XCDs) per chunk: a block's
// chunks on different XCDs.
__host__ __device__ inline int packed_chunk_block(int blk, int chunk, int per_chunk) {
  const int b = blk - chunk * per_chunk;
  return b / kXcds * kXcds + (b + chunk * (kXcds - 1)) % kXcds;
}

// Tiles of BN keys, within [t_lo, t_hi), whose keys all of rows m0 .. mlast see.
__host__ __device__ inline void packed_full_tiles(int m0, int mlast, int lk, int dlo, int dhi, int BN, int t_lo, int t_hi,
                                                  int& t_flo, int& t_fhi) {
  const int64_t flo = lmax(0, (int64_t)mlast + dlo), fhi = lmin((int64_t)lk, (int64_t)m0 + dhi + 1);
  t_flo = (int)lmin(lmax((flo + BN - 1) / BN, t_lo), t_hi);
  t_fhi = (int)lmin(lmax(fhi > 0 ? fhi / BN : 0, t_flo), t_hi);
}

}  // namespace trinix
