"""CPU: argument checks of the packed-sequence entry points (status codes, no
launch), the layout of ``trinix_packed_args``, and the index maps of the plan
(``csrc/packed_map.h``) driven over random batches by a small C++ program."""
import ctypes
import os
import subprocess

import pytest
import torch

import trinix_amd as tx
from trinix_amd import _native as nat
from trinix_amd.build import CSRC_DIR, INCLUDE_DIR, LIB_PATH, build


@pytest.fixture(scope="module")
def lib():
    if not LIB_PATH.exists():
        build()
    return nat.load_library()


def layout(cname, cls, tmp_path):
    fields = [f for f, _ in cls._fields_]
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join(["#include <stdio.h>", "#include <stddef.h>", '#include "trinix_attn.h"', "int main(void){",
                              f'printf("%zu\\n", sizeof({cname}));',
                              *[f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields], "return 0;}"]))
    subprocess.run(["gcc", "-std=c99", "-I", str(INCLUDE_DIR), str(src), "-o", str(exe)], check=True)
    vals = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(cls)
    assert [getattr(cls, f).offset for f in fields] == vals[1:]


def test_packed_args_layout(tmp_path):
    layout("trinix_packed_args", nat.PackedArgs, tmp_path)


def test_shared_prefix_args_layout(tmp_path):
    layout("trinix_shared_prefix_args", nat.SharedPrefixArgs, tmp_path)


def shared_args(**kw):
    a = nat.SharedPrefixArgs()
    for f in ("q", "prefix_k", "prefix_v", "k", "v", "out"):
        setattr(a, f, 4096)
    a.q_stride = a.out_stride = nat.Int64x4(8 * 128, 8 * 128, 128, 1)
    a.k_stride = a.v_stride = nat.Int64x4(500 * 256, 256, 128, 1)
    a.prefix_k_stride = a.prefix_v_stride = nat.Int64x3(256, 128, 1)
    a.batch, a.seqlen_q, a.prefix_len, a.capacity, a.nheads_q, a.nheads_kv, a.head_dim = 4, 1, 1000, 500, 8, 2, 128
    a.dtype, a.softmax_scale = nat.TRINIX_BF16, 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=nat.TRINIX_U8), nat.TRINIX_ERR_BAD_DTYPE),
    (dict(head_dim=84), nat.TRINIX_ERR_BAD_HEAD_DIM),
    (dict(head_dim=264), nat.TRINIX_ERR_BAD_HEAD_DIM),
    (dict(batch=0), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(seqlen_q=0), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(prefix_len=-1), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(capacity=1 << 30), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(nheads_kv=3), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(batch=1 << 23, seqlen_q=1 << 23), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(q=None), nat.TRINIX_ERR_NULL_POINTER),
    (dict(prefix_v=None), nat.TRINIX_ERR_NULL_POINTER),
    (dict(k=None), nat.TRINIX_ERR_NULL_POINTER),
    (dict(out=4104), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(k_stride=nat.Int64x4(500 * 256, 256, 132, 1)), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(prefix_k_stride=nat.Int64x3(256, 128, 2)), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(prefix_v_stride=nat.Int64x3(1 << 22, 128, 1)), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(v_stride=nat.Int64x4(500 * 256, -256, 128, 1)), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(seq_lens=4098), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(lse=4098), nat.TRINIX_ERR_BAD_STRIDE),
])
def test_shared_prefix_status_codes(lib, kw, code):
    a, n = shared_args(**kw), ctypes.c_int64(0)
    assert lib.trinix_shared_prefix_workspace(ctypes.byref(a), ctypes.byref(n)) == code
    assert lib.trinix_shared_prefix_fwd(ctypes.byref(a), 4096, 1 << 40, None) == code


def test_shared_prefix_workspace(lib):
    n = ctypes.c_int64(0)
    a = shared_args()
    assert lib.trinix_shared_prefix_workspace(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value > 0
    for ws, size in ((None, n.value), (4096, n.value - 1), (4100, n.value)):
        assert lib.trinix_shared_prefix_fwd(ctypes.byref(a), ws, size, None) == nat.TRINIX_ERR_BAD_ARGUMENT
    assert lib.trinix_shared_prefix_workspace(None, ctypes.byref(n)) == nat.TRINIX_ERR_NULL_POINTER
    assert lib.trinix_shared_prefix_workspace(ctypes.byref(a), None) == nat.TRINIX_ERR_NULL_POINTER
    assert lib.trinix_shared_prefix_fwd(None, None, 0, None) == nat.TRINIX_ERR_NULL_POINTER
    # absent prefix or caches: their pointers are not looked at
    for kw in (dict(prefix_len=0, prefix_k=None, prefix_v=None), dict(capacity=0, k=None, v=None)):
        a = shared_args(**kw)
        assert lib.trinix_shared_prefix_workspace(ctypes.byref(a), ctypes.byref(n)) == 0


def plan_bytes(lib, n, tq, tk):
    out = ctypes.c_int64(0)
    return lib.trinix_packed_plan_bytes(n, tq, tk, ctypes.byref(out)), out.value


def test_plan_bytes(lib):
    rc, n = plan_bytes(lib, 3, 1000, 2000)
    assert rc == 0 and n > 0
    for bad in ((0, 1, 1), (1 << 24, 1, 1), (1, -1, 1), (1, 1, -1), (1, 1 << 30, 1), (1, 1, 1 << 30)):
        assert plan_bytes(lib, *bad)[0] == nat.TRINIX_ERR_BAD_SHAPE, bad
    assert lib.trinix_packed_plan_bytes(1, 1, 1, None) == nat.TRINIX_ERR_NULL_POINTER
    args = (4096, 4096, 3, 1000, 2000, 4096, n, None)
    for at, value, code in ((0, None, nat.TRINIX_ERR_NULL_POINTER), (5, None, nat.TRINIX_ERR_NULL_POINTER),
                            (5, 4104, nat.TRINIX_ERR_BAD_ARGUMENT), (0, 4098, nat.TRINIX_ERR_BAD_ARGUMENT),
                            (6, n - 1, nat.TRINIX_ERR_BAD_ARGUMENT), (2, 0, nat.TRINIX_ERR_BAD_SHAPE)):
        a = list(args)
        a[at] = value
        assert lib.trinix_packed_plan(*a) == code, (at, value)


def args(lib, **kw):
    a = nat.PackedArgs()
    for f in ("q", "k", "v", "out", "out_lo", "lse", "dout", "delta", "dq", "dk", "dv", "plan"):
        setattr(a, f, 4096)
    for f in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        setattr(a, f + "_stride", nat.Int64x3(8 * 128, 128, 1))
    a.n_seqs, a.total_q, a.total_k, a.nheads_q, a.nheads_kv, a.head_dim = 3, 1000, 1000, 8, 8, 128
    a.plan_bytes = plan_bytes(lib, 3, 1000, 1000)[1]
    a.dtype, a.softmax_scale = nat.TRINIX_BF16, 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=nat.TRINIX_U8), nat.TRINIX_ERR_BAD_DTYPE),
    (dict(head_dim=92), nat.TRINIX_ERR_BAD_HEAD_DIM),
    (dict(head_dim=264), nat.TRINIX_ERR_BAD_HEAD_DIM),
    (dict(head_dim=0), nat.TRINIX_ERR_BAD_HEAD_DIM),
    (dict(nheads_kv=3), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(nheads_q=0), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(nheads_kv=0), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(n_seqs=0), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(total_q=-1), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(total_q=1 << 30), nat.TRINIX_ERR_BAD_SHAPE),
    (dict(plan=None), nat.TRINIX_ERR_NULL_POINTER),
    (dict(plan=4100), nat.TRINIX_ERR_BAD_ARGUMENT),
    (dict(plan_bytes=64), nat.TRINIX_ERR_BAD_ARGUMENT),
    (dict(total_q=2000), nat.TRINIX_ERR_BAD_ARGUMENT),  # the plan is of a smaller batch
    (dict(q=None), nat.TRINIX_ERR_NULL_POINTER),
    (dict(v=None), nat.TRINIX_ERR_NULL_POINTER),
    (dict(out=4104), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(q_stride=nat.Int64x3(1024, 128, 2)), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(k_stride=nat.Int64x3(1024, 130, 1)), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(k_stride=nat.Int64x3(1 << 22, 128, 1)), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(q_stride=nat.Int64x3(-1024, 128, 1)), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(lse=4098), nat.TRINIX_ERR_BAD_STRIDE),
    (dict(alibi_slopes=4097), nat.TRINIX_ERR_BAD_STRIDE),
])
def test_packed_status_codes(lib, kw, code):
    for fn in (lib.trinix_packed_fwd, lib.trinix_packed_bwd):
        a = args(lib, **kw)
        assert fn(ctypes.byref(a), None) == code
        assert fn(None, None) == nat.TRINIX_ERR_NULL_POINTER


@pytest.mark.parametrize("field", ["lse", "delta", "out_lo", "dout", "dq", "dk", "dv"])
def test_packed_backward_needs_its_tensors(lib, field):
    a = args(lib, **{field: None})
    assert lib.trinix_packed_bwd(ctypes.byref(a), None) == nat.TRINIX_ERR_NULL_POINTER


def test_packed_forward_workspace(lib, monkeypatch):
    monkeypatch.delenv("TRINIX_PACKED_CHUNKS", raising=False)
    n = ctypes.c_int64(0)

    def need(**kw):
        a = args(lib)
        for k, v in kw.items():
            setattr(a, k, v)
        assert lib.trinix_packed_fwd_workspace(ctypes.byref(a), ctypes.byref(n)) == 0
        return n.value

    long = dict(total_q=8, total_k=16384, n_seqs=4, nheads_q=8, nheads_kv=2, head_dim=128, dtype=nat.TRINIX_BF16)
    assert need(**long) == 8 * 8 * 8 * 129 * 4
    assert need(**{**long, "dtype": nat.TRINIX_F32, "head_dim": 40}) == 8 * 8 * 8 * 65 * 4
    assert need(**{**long, "total_k": 1000}) == 0
    assert need(**{**long, "has_window": 1, "window_left": 500, "causal": 1}) == 0
    assert need(**{**long, "has_window": 1, "window_left": 1 << 62, "window_right": 1 << 62}) == n.value > 0
    assert need(**{**long, "total_q": 16384, "n_seqs": 64}) == 0  # the rows fill the GPU
    assert need(**{**long, "total_q": 0}) == 0
    monkeypatch.setenv("TRINIX_PACKED_CHUNKS", "3")
    assert need(**long) == 3 * 8 * 8 * 129 * 4
    monkeypatch.setenv("TRINIX_PACKED_CHUNKS", "-1")
    assert need(**long) == 0
    assert lib.trinix_packed_fwd_workspace(None, ctypes.byref(n)) == nat.TRINIX_ERR_NULL_POINTER
    assert lib.trinix_packed_fwd_workspace(ctypes.byref(args(lib)), None) == nat.TRINIX_ERR_NULL_POINTER
    for bad in (dict(nheads_q=0), dict(nheads_kv=3), dict(n_seqs=0), dict(n_seqs=(1 << 63) - 1), dict(total_q=-1),
                dict(total_q=1 << 30), dict(total_k=1 << 30), dict(head_dim=12, dtype=nat.TRINIX_BF16), dict(head_dim=264)):
        a = args(lib)
        for k, v in bad.items():
            setattr(a, k, v)
        assert lib.trinix_packed_fwd_workspace(ctypes.byref(a), ctypes.byref(n)) == nat.TRINIX_ERR_BAD_SHAPE


def test_packed_backward_workspace(lib):
    n = ctypes.c_int64(-1)
    a = args(lib)  # 8 heads of their own: no head to share out
    assert lib.trinix_packed_bwd_workspace(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value == 0
    a = args(lib, nheads_kv=1)
    assert lib.trinix_packed_bwd_workspace(ctypes.byref(a), ctypes.byref(n)) == 0
    assert n.value % (2 * 1000 * 128 * 4) == 0 and n.value > 0
    for ws, size in ((None, n.value), (4096, n.value - 1), (4104, n.value)):
        a.workspace, a.workspace_bytes = ws, size
        assert lib.trinix_packed_bwd(ctypes.byref(a), None) == nat.TRINIX_ERR_BAD_ARGUMENT
    assert lib.trinix_packed_bwd_workspace(None, ctypes.byref(n)) == nat.TRINIX_ERR_NULL_POINTER
    assert lib.trinix_packed_bwd_workspace(ctypes.byref(a), None) == nat.TRINIX_ERR_NULL_POINTER
    for bad in (dict(nheads_kv=0), dict(nheads_kv=3), dict(head_dim=92), dict(total_k=-1), dict(n_seqs=0)):
        assert lib.trinix_packed_bwd_workspace(ctypes.byref(args(lib, **bad)), ctypes.byref(n)) == nat.TRINIX_ERR_BAD_SHAPE


def test_python_layer_without_a_gpu():
    x = torch.zeros(4, 2, 64)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError):
            tx.PackedSequences([0, 4])
    with pytest.raises(ValueError):
        tx.packed_attn_func(x, x, x, None)


CHECK = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include <set>
#include <algorithm>
#define __host__
#define __device__
#include "packed_map.h"
using namespace trinix;
static long fails = 0;
#define EXPECT(c) do { if (!(c)) { if (++fails < 10) std::printf("line %d: %s\n", __LINE__, #c); } } while (0)
int main() {
  std::srand(7);
  for (int round = 0; round < 400; ++round) {
    const int n = 1 + std::rand() % (round % 4 == 0 ? 300 : 8), far = round % 5 == 0 ? 3000 : 200;
    std::vector<int> cq(n + 1, 0), ck(n + 1, 0);
    for (int s = 0; s < n; ++s) {
      cq[s + 1] = cq[s] + (std::rand() % 4 ? std::rand() % far : 0);
      ck[s + 1] = ck[s] + (std::rand() % 4 ? std::rand() % far : 0);
    }
    const int tq = cq[n] + (std::rand() % 2 ? std::rand() % 300 : 0), tk = ck[n] + (std::rand() % 2 ? std::rand() % 300 : 0);
    int64_t end = 0;
    for (int list = 0; list < kPackedLists; ++list) {
      const int total = packed_list_is_keys(list) ? tk : tq, bs = packed_list_block(list);
      const int64_t cap = packed_list_cap(total, n, bs);
      EXPECT(packed_list_offset(list, tq, tk, n) == end);
      end += cap * kPackedItemInts;
      // every row (key) of the tensors in exactly one block of one sequence, inside the list
      std::vector<int> seen(total, 0);
      int64_t items = 0;
      for (int s = 0; s < n + 2; ++s) {
        const PackedSeq q = packed_seq(s, n, cq.data(), ck.data(), tq, tk);
        EXPECT(q.q0 >= 0 && q.k0 >= 0 && q.lq >= 0 && q.lk >= 0 && q.q0 + q.lq <= tq && q.k0 + q.lk <= tk);
        const int nb = packed_blocks(q, list);
        items += nb;
        for (int b = 0; b < nb; ++b) {
          const int lo = b * bs, len = packed_list_is_keys(list) ? q.lk : q.lq, base = packed_list_is_keys(list) ? q.k0 : q.q0;
          EXPECT(lo < len);
          for (int x = lo; x < std::min(len, lo + bs); ++x) ++seen[base + x];
          const int c = packed_cost(q, list, b);
          EXPECT(c >= 0 && c <= std::max(q.lq, q.lk));
        }
      }
      for (int x : seen) EXPECT(x == 1);
      EXPECT(items <= cap && cap % kXcds == 0);
      // workgroups cover items x heads once
      for (int hkv : {1, 3, 8, 16}) for (int G : {1, 4}) {
        if (cap * hkv * G > 20000) continue;
        std::set<std::pair<int, int>> work;
        for (int b = 0; b < cap * hkv * G; ++b) {
          const PackedWork w = packed_work(b, hkv, G);
          EXPECT(w.item >= 0 && w.item < cap && w.h >= 0 && w.h < hkv * G);
          work.insert({w.item, w.h});
        }
        EXPECT((int64_t)work.size() == cap * hkv * G);
      }
    }
    EXPECT(packed_plan_ints(tq, tk, n) == end + kPackedLists * packed_scratch_ints(n));
    // chunks of a run of tiles: every tile in one; which workgroup runs which block of which chunk
    for (int t = 0; t < 50; ++t) {
      const int tiles = std::rand() % 300, most = 1 + std::rand() % 8, BN = std::rand() % 2 ? 32 : 64;
      const int total = std::rand() % 3 ? std::rand() % 4000 : INT32_MAX, heads = 1 + std::rand() % 64;
      const PackedChunks c = packed_chunks(tiles, BN, most, total, heads, 512);
      EXPECT(c.n >= 1 && c.n <= most && c.per * (int64_t)BN >= kPackedChunkKeys && (int64_t)c.n * c.per >= tiles);
      EXPECT(c.n == 1 || (c.n - 1) * c.per < tiles);
      // every block of every chunk once
      const int per = kXcds * (1 + std::rand() % 20);
      std::set<std::pair<int, int>> seen;
      for (int b = 0; b < per * most; ++b) {
        const int x = packed_chunk_block(b, b / per, per);
        EXPECT(x >= 0 && x < per);
        seen.insert({b / per, x});
      }
      EXPECT((int)seen.size() == per * most);
    }
    // the band against its definition, tile ranges around it
    for (int t = 0; t < 20; ++t) {
      const int lq = 1 + std::rand() % 300, lk = 1 + std::rand() % 300;
      const bool causal = std::rand() % 2, win = std::rand() % 2;
      const int64_t wl = std::rand() % 200 - 50, wr = std::rand() % 200 - 50;
      int dlo, dhi;
      packed_band(lq, lk, causal, win, wl, wr, dlo, dhi);
      const int off = lk - lq;
      // keys that any row sees, rows that see any key, and what a tile reads of them
      int k_lo = lk, k_hi = -1, r_lo = lq, r_hi = -1;
      for (int i = 0; i < lq; ++i) for (int j = std::max(0, i + dlo); j <= std::min(lk - 1, i + dhi); ++j) {
        k_lo = std::min(k_lo, j), k_hi = std::max(k_hi, j), r_lo = std::min(r_lo, i), r_hi = std::max(r_hi, i);
      }
      const PackedRange ks = packed_seen_keys(lq, lk, dlo, dhi), rs = packed_seeing_rows(lq, lk, dlo, dhi);
      EXPECT(0 <= ks.lo && ks.lo <= ks.hi && ks.hi < lk && 0 <= rs.lo && rs.lo <= rs.hi && rs.hi < lq);
      if (k_hi >= 0) EXPECT(ks.lo == k_lo && ks.hi == k_hi && rs.lo == r_lo && rs.hi == r_hi);
      for (int n0 = 0; n0 < lk; n0 += 32) {
        const PackedRange t = packed_tile_range(ks, n0);
        EXPECT(0 <= t.lo && t.lo <= t.hi && n0 + t.hi < lk);
        if (n0 <= ks.hi && n0 + 32 > ks.lo)
          for (int r = 0; r < 32; ++r) EXPECT(n0 + std::min(std::max(r, t.lo), t.hi) == std::min(std::max(n0 + r, ks.lo), ks.hi));
      }
      for (int BM : {64, 128}) for (int m0 = 0; m0 < lq; m0 += BM) {
        int lo, hi;
        bwd_key_tiles(m0, BM, lq, lk, dlo, dhi, 32, lo, hi);
        EXPECT(lo >= hi || (lo >= 0 && (hi - 1) * 32 < lk));
        int flo, fhi;
        packed_full_tiles(m0, std::min(m0 + BM, lq) - 1, lk, dlo, dhi, 32, lo, hi, flo, fhi);
        EXPECT(lo <= flo && flo <= fhi && fhi <= std::max(lo, hi));
        for (int i = m0; i < std::min(lq, m0 + BM); ++i) for (int j = flo * 32; j < fhi * 32; ++j)
          EXPECT(j < lk && j - i >= dlo && j - i <= dhi);
        for (int i = m0; i < std::min(lq, m0 + BM); ++i) for (int j = 0; j < lk; ++j) {
          const bool ok = (!causal || j <= i + off) && (!win || (j - i - off >= -wl && j - i - off <= wr));
          EXPECT(ok == (j - i >= dlo && j - i <= dhi));
          if (ok) EXPECT(j / 32 >= lo && j / 32 < hi);
        }
      }
      for (int k0 = 0; k0 < lk; k0 += 128) {
        int lo, hi;
        bwd_query_tiles(k0, 128, lq, lk, dlo, dhi, 32, lo, hi);
        EXPECT(lo >= hi || (lo >= 0 && (hi - 1) * 32 < lq));
        for (int j = k0; j < std::min(lk, k0 + 128); ++j) for (int i = 0; i < lq; ++i)
          if (j - i >= dlo && j - i <= dhi) EXPECT(i / 32 >= lo && i / 32 < hi);
      }
    }
  }
  std::printf("%ld failures\n", fails);
  return fails != 0;
}
"""


def test_index_maps(tmp_path):
    src, exe = tmp_path / "c.cpp", tmp_path / "c"
    src.write_text(CHECK)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    f"-I{CSRC_DIR}", str(src), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
