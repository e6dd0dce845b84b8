"""Attention over packed sequences against plain 64-bit attention of every
sequence (``packed_oracle``): types, head layouts, lengths from nothing to
several tiles, odd sizes, strides, rows that see no key, padding, and gradients."""
import math

import pytest
import torch

import trinix_amd as tx
from packed_oracle import close, packed

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def cumulative(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def make(Tq, Tk, H, Hkv, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g).to(dtype)
    return r(Tq, H, D), r(Tk, Hkv, D), r(Tk, Hkv, D), r(Tq, H, D)


def check(lens_q, lens_k=None, H=4, Hkv=2, D=64, dtype=BF, causal=True, window=None, alibi=False, pad=0, scale=None,
          seed=0, grad=True, gpu_lengths=True):
    cu_q = cumulative(lens_q)
    cu_k = cumulative(lens_k) if lens_k is not None else cu_q
    Tq, Tk = cu_q[-1] + pad, cu_k[-1] + pad
    q, k, v, do = make(Tq, Tk, H, Hkv, D, dtype, seed)
    slopes = torch.tensor([2.0 ** -(h % 8 + 1) for h in range(H)]) if alibi else None
    if gpu_lengths:
        seqs = tx.PackedSequences(torch.tensor(cu_q, device=DEV), None if lens_k is None else torch.tensor(cu_k, device=DEV),
                                  total_q=Tq, total_k=Tk)
    else:
        seqs = tx.PackedSequences(cu_q, None if lens_k is None else cu_k, total_q=Tq, total_k=Tk)
    dq, dk, dv = (t.to(DEV).requires_grad_(grad) for t in (q, k, v))
    out, lse = tx.packed_attn_func(dq, dk, dv, seqs, scale, causal, window, None if slopes is None else slopes.to(DEV),
                                   return_lse=True)
    val, tol = packed(q, k, v, do if grad else None, cu_q, cu_k, D ** -0.5 if scale is None else scale, causal, window, slopes)
    got = dict(out=out, lse=lse)
    if grad:
        got.update(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (dq, dk, dv), do.to(DEV))))
    for n, t in got.items():
        close(n, t, val[n], tol[n], F32 if n == "lse" else dtype)


RAGGED = [3, 1, 64, 130, 0, 65, 33, 257]


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("D", [64, 128, 256, 8, 30, 40, 80, 96, 129, 200])
def test_ragged_causal(dtype, D):
    check(RAGGED, D=D, dtype=dtype, pad=5, seed=D)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 8), (8, 1), (16, 8), (6, 3), (24, 8)])
def test_head_layouts(H, Hkv):
    check([70, 1, 190], H=H, Hkv=Hkv, D=128, seed=H)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("kw", [dict(causal=False), dict(window=(40, 0)), dict(causal=False, window=(17, 5)),
                                dict(alibi=True), dict(causal=False, alibi=True, window=(100, 100)), dict(scale=-0.2),
                                dict(scale=0.0)])
def test_masks_and_biases(kw, dtype):
    check([129, 5, 320, 64], dtype=dtype, D=64, seed=3, **kw)
    check([129, 5, 320, 64], dtype=dtype, D=128, seed=4, **kw)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64), (F32, 64), (BF, 256)])
@pytest.mark.parametrize("causal,window", [(True, None), (True, (100, 0)), (False, None), (False, (30, 10))])
def test_queries_are_the_last_positions(dtype, D, causal, window):
    # caches before the chunk, more queries than keys (rows that see nothing), no keys, no queries
    check([5, 64, 100, 7, 0, 130], [300, 64, 33, 0, 20, 515], D=D, dtype=dtype, causal=causal, window=window, seed=9)


@pytest.mark.parametrize("window", [(-3, 10), (5, -8), (1 << 40, 1 << 40), (-200, 100)])
def test_windows_beside_the_diagonal(window):
    check([90, 200, 3], causal=False, window=window, D=64, seed=1)


@pytest.mark.parametrize("shape", ["0", "1", "2"])
@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (BF, 256), (BF, 96), (HF, 80)])
def test_forced_tile_shapes(shape, dtype, D, monkeypatch):
    # 64, 128 and 256 rows per workgroup (where the head_dim has that shape)
    monkeypatch.setenv("TRINIX_PACKED_FWD", shape)
    kw = dict(D=D, dtype=dtype, grad=False)
    check([1, 257, 33, 0, 700, 128], pad=9, **kw)
    check([200, 64, 3], [900, 64, 33], window=(150, 0), **kw)
    check([300, 40], [10, 555], causal=False, alibi=True, **kw)
    check([100, 513], window=(-2, 40), causal=False, **kw)


@pytest.mark.parametrize("chunks", ["1", "2", "3", "8"])
@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (BF, 256), (HF, 40), (BF, 96), (F32, 64), (F32, 80), (F32, 128),
                                     (F32, 256)])
def test_keys_shared_out(chunks, dtype, D, monkeypatch):
    # the keys of a block of rows over several workgroups, joined by a second launch
    monkeypatch.setenv("TRINIX_PACKED_CHUNKS", chunks)
    kw = dict(D=D, dtype=dtype, pad=3)
    check([1, 5, 0, 70, 3], [1500, 900, 300, 1100, 0], **kw)  # some blocks in one chunk, rows without keys
    check([700, 1], causal=False, alibi=True, **kw)
    check([40, 130], [2000, 1000], alibi=True, grad=False, **kw)
    check([9, 300], [1700, 40], window=(700, 0), grad=False, **kw)
    check([64, 1], [1200, 1], causal=False, window=(600, -20), grad=False, **kw)


def test_single_tokens_behind_long_caches():
    check([1] * 6, [9000, 1, 3000, 257, 256, 4100], H=8, Hkv=2, D=128, grad=False)
    check([1, 2], [6000, 70], H=4, Hkv=1, D=64, dtype=HF, alibi=True, grad=False)
    check([1, 2], [6000, 70], H=4, Hkv=1, D=64, dtype=F32, grad=False)


@pytest.mark.parametrize("splits", ["1", "2", "3", "16"])
@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (BF, 256), (F32, 64), (BF, 80), (F32, 96)])
def test_heads_shared_out(splits, dtype, D, monkeypatch):
    # the query heads of a KV head over several workgroups, summed in order
    monkeypatch.setenv("TRINIX_PACKED_SPLITS", splits)
    check([70, 1, 0, 190], [90, 1, 7, 190], H=5, Hkv=1, D=D, dtype=dtype, pad=4)


@pytest.mark.parametrize("pairs", ["1", "2"])
@pytest.mark.parametrize("dtype,D", [(F32, 64), (F32, 128), (F32, 256), (BF, 256), (HF, 256), (F32, 80), (F32, 96)])
def test_forced_pairs(pairs, dtype, D, monkeypatch):
    # one or two wavefronts per 32 rows
    monkeypatch.setenv("TRINIX_PACKED_PAIRS", pairs)
    check([1, 257, 33, 0, 300, 128], D=D, dtype=dtype, pad=9)
    check([200, 64, 3], [500, 64, 33], D=D, dtype=dtype, window=(150, 0))
    check([300, 40], [10, 255], D=D, dtype=dtype, causal=False, alibi=True)


def test_single_tokens_and_many_sequences():
    check([1] * 300, D=64, seed=2)
    check([(7 * i) % 23 for i in range(1500)], H=2, Hkv=1, D=64, seed=2)


@pytest.mark.parametrize("n", [1, 31, 32, 33, 63, 127, 128, 129, 255, 256, 257, 1025])
def test_lengths_around_the_tiles(n):
    check([n, 2], D=64, seed=n)
    check([n], D=128, seed=n, causal=False)


def test_long_sequence_beside_short_ones():
    check([1, 3000, 17], H=2, Hkv=1, D=128, seed=5)


def test_host_lengths_and_padding():
    check([33, 65], pad=70, gpu_lengths=False)
    check([40], [90], pad=3, gpu_lengths=False)


def test_padding_rows_are_zero_and_poison_there_is_not_read():
    q, k, v, do = make(300, 300, 4, 2, 64, BF, 0)
    for t in (q, k, v, do):
        t[200:] = float("nan")
    seqs = tx.PackedSequences([0, 150, 200], total_q=300)
    x = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    out = tx.packed_attn_func(*x, seqs, causal=True)
    grads = torch.autograd.grad(out, x, do.to(DEV))
    for t in (out, *grads):
        assert bool(torch.isfinite(t[:200]).all()) and bool((t[200:] == 0).all())


@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (F32, 96), (BF, 256), (F32, 64), (BF, 96)])
@pytest.mark.parametrize("causal,window", [(True, (40, 0)), (False, (30, -5)), (True, None), (False, (-20, 60))])
def test_what_no_row_sees_holds_anything(dtype, D, causal, window):
    """Keys before every row's window, keys behind, and rows that see no key: NaN there changes no bit."""
    lens_q, lens_k, H, Hkv = [50, 200, 3, 140, 1], [300, 70, 500, 140, 33], 4, 2
    cu_q, cu_k = cumulative(lens_q), cumulative(lens_k)
    q, k, v, do = (t.to(DEV) for t in make(cu_q[-1], cu_k[-1], H, Hkv, D, dtype, 5))
    seqs = tx.PackedSequences(cu_q, cu_k)

    def run(*ts):
        a, b, c, do = ts
        a, b, c = (t.detach().clone().requires_grad_(True) for t in (a, b, c))
        out, lse = tx.packed_attn_func(a, b, c, seqs, causal=causal, window_size=window, return_lse=True)
        return (out.detach(), lse, *torch.autograd.grad(out, (a, b, c), do))

    want = run(q, k, v, do)
    for s, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        i, j = torch.arange(lq)[:, None] + (lk - lq), torch.arange(lk)[None]
        ok = torch.ones(lq, lk, dtype=torch.bool)
        if causal:
            ok &= j <= i
        if window is not None:
            ok &= (j - i >= -window[0]) & (j - i <= window[1])
        rows, keys = (~ok.any(1)).to(DEV), (~ok.any(0)).to(DEV)
        for t in (q, do):
            t[cu_q[s]:cu_q[s + 1]][rows] = float("nan")
        k[cu_k[s]:cu_k[s + 1]][keys] = float("nan")
        v[cu_k[s]:cu_k[s + 1]][keys] = float("inf")
    for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), run(q, k, v, do), want):
        assert torch.equal(a, b), name


def test_strided_operands():
    # q, k and v as slices of one projection, a KV head expanded without a copy, dout with a stride of 0
    g = torch.Generator().manual_seed(4)
    cu, H, D = [0, 50, 117, 260], 4, 64
    qkv = torch.randn(260, 3 * H, D, generator=g).to(HF)
    x = qkv.to(DEV).requires_grad_(True)
    seqs = tx.PackedSequences(cu)
    out = tx.packed_attn_func(x[:, :H], x[:, H:2 * H], x[:, 2 * H:], seqs, causal=True)
    d, = torch.autograd.grad(out.sum(), x)
    val, tol = packed(qkv[:, :H], qkv[:, H:2 * H], qkv[:, 2 * H:], torch.ones(260, H, D, dtype=HF), cu, cu, D ** -0.5, True)
    close("out", out, val["out"], tol["out"], HF)
    close("grad", d, torch.cat([val["dq"], val["dk"], val["dv"]], 1), torch.cat([tol["dq"], tol["dk"], tol["dv"]], 1), HF)
    kv = torch.randn(260, 1, D, generator=g).to(HF)
    e = kv.to(DEV).expand(260, H, D)
    got = tx.packed_attn_func(x[:, :H].detach(), e, e, seqs, causal=True)
    val, tol = packed(qkv[:, :H], kv.expand(260, H, D), kv.expand(260, H, D), None, cu, cu, D ** -0.5, True)
    close("out", got, val["out"], tol["out"], HF)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_offsets_beyond_32_bits(dtype):
    """Rows 8192 elements apart, the last ones more than 2^32 bytes and 2^31 elements behind the first: as a copy."""
    n, D = 300_000, 64
    cu_q, cu_k = [0, 1, 101, 164], [0, 298_500, 299_500, n]
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)
    wide = torch.empty(n, 2, 4096, dtype=dtype, device=DEV)
    k, v = wide[:, :, :D], wide[:, :, 100 * 8:100 * 8 + D]
    k.copy_(r(n, 2, D)), v.copy_(r(n, 2, D))
    q, do = r(164, 4, D), r(164, 4, D)
    seqs = tx.PackedSequences(cu_q, cu_k)

    def run(k, v):
        a, b, c = q.clone().requires_grad_(True), k.detach().requires_grad_(True), v.detach().requires_grad_(True)
        out = tx.packed_attn_func(a, b, c, seqs, causal=True)
        return (out.detach(), *torch.autograd.grad(out, (a, b, c), do))

    for a, b in zip(run(k, v), run(k.contiguous(), v.contiguous())):
        assert torch.equal(a, b)
    # queries that far behind, of a few keys
    wide[-164:, :, :D] = q.view(164, 2, 2, D)[:, :, 0]
    few = tx.PackedSequences([0, n - 164, n], [0, 10, 40])
    got = tx.packed_attn_func(wide[:, :, :D], k[:40], v[:40], few, causal=False)
    want = tx.packed_attn_func(wide[-164:, :, :D].contiguous(), k[10:40], v[10:40], tx.PackedSequences([0, 164], [0, 30]))
    assert torch.equal(got[-164:], want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_unaligned_operands(dtype):
    base = torch.randn(200 * 2 * 64 + 3, generator=torch.Generator().manual_seed(1)).to(dtype)
    t = base[3:].view(200, 2, 64)
    seqs = tx.PackedSequences([0, 77, 200])
    x = base.to(DEV)[3:].view(200, 2, 64)
    out = tx.packed_attn_func(x, x, x, seqs, causal=True)
    val, tol = packed(t, t, t, None, [0, 77, 200], [0, 77, 200], 0.125, True)
    close("out", out, val["out"], tol["out"], dtype)


def test_peaked_softmax_keeps_its_gradients():
    # scores of +-50: delta has to come from more than the rounded output
    q, k, v, do = make(256, 256, 2, 2, 64, BF, 7)
    q = (q.float() * 6).to(BF)
    cu = [0, 100, 256]
    x = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    out = tx.packed_attn_func(*x, tx.PackedSequences(cu), causal=True)
    grads = torch.autograd.grad(out, x, do.to(DEV))
    val, tol = packed(q, k, v, do, cu, cu, 0.125, True)
    for n, t in zip(("dq", "dk", "dv"), grads):
        close(n, t, val[n], tol[n], BF)


def test_gradient_against_differences():
    q, k, v, do = make(40, 40, 2, 1, 64, F32, 11)
    cu = [0, 13, 40]
    seqs = tx.PackedSequences(cu)
    x = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(tx.packed_attn_func(*x, seqs, causal=True), x, do.to(DEV))
    g = torch.Generator().manual_seed(5)
    for n, (t, d) in enumerate(zip((q, k, v), grads)):
        step = torch.randn(t.shape, generator=g)
        eps = 1e-5
        f = [sum((packed(*[(y.double() + (s * eps * step.double() if m == n else 0)) for m, y in enumerate((q, k, v))], None,
                         cu, cu, 0.125, True)[0]["out"] * do.double()).flatten()) for s in (1, -1)]
        want = ((f[0] - f[1]) / (2 * eps)).item()
        got = (d.cpu().double() * step.double()).sum().item()
        # differences in 64 bits: eps^2 of the third derivative, far below the fp32 gradient's error
        assert abs(got - want) <= 1e-4 * (d.cpu().double() * step.double()).abs().sum().item(), (n, got, want)


def test_as_one_padded_batch():
    """Equal lengths: the framework's batched attention on the same rows."""
    B, S, H, D = 3, 200, 4, 128
    q, k, v, _ = make(B * S, B * S, H, 2, D, BF, 0)
    q, k, v = (t.to(DEV) for t in (q, k, v))
    got = tx.packed_attn_func(q, k, v, tx.PackedSequences([0, S, 2 * S, 3 * S]), causal=True)
    want = tx.triton_attn_func(q.view(B, S, H, D), k.view(B, S, 2, D), v.view(B, S, 2, D), causal=True)
    # both within the rounding of P and of the output: 4 half steps of values up to max |v|
    assert (got - want.view_as(got)).abs().max().item() <= 4 * 2.0 ** -9 * v.abs().max().item()


def test_boundaries_on_the_gpu_are_clamped():
    q, k, v, _ = make(128, 128, 2, 2, 64, BF, 0)
    q, k, v = (t.to(DEV) for t in (q, k, v))
    bad = torch.tensor([7, 50, 20, 10 ** 6, -5, 128], device=DEV)  # -> 0, 50, 50, 128, 128, 128
    got = tx.packed_attn_func(q, k, v, tx.PackedSequences(bad, total_q=128), causal=True)
    want = tx.packed_attn_func(q, k, v, tx.PackedSequences([0, 50, 50, 128, 128, 128]), causal=True)
    assert torch.equal(got, want)


def test_empty_tensors():
    e = torch.empty(0, 2, 64, device=DEV, dtype=BF)
    x = torch.randn(5, 2, 64, device=DEV).to(BF).requires_grad_(True)
    assert tx.packed_attn_func(e, e, e, tx.PackedSequences([0, 0])).shape == (0, 2, 64)
    out = tx.packed_attn_func(x, e, e, tx.PackedSequences([0, 5], [0, 0]))
    assert bool((out == 0).all())
    assert bool((torch.autograd.grad(out.sum(), x)[0] == 0).all())
    out = tx.packed_attn_func(e, x, x, tx.PackedSequences([0, 0], [0, 5]))
    dk, = torch.autograd.grad(out.sum(), x)
    assert out.shape[0] == 0 and bool((dk == 0).all())


def test_same_bits_every_run_and_other_streams():
    q, k, v, do = make(900, 900, 8, 2, 128, BF, 3)
    x = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    do = do.to(DEV)
    seqs = tx.PackedSequences([0, 500, 501, 900])

    def run():
        out = tx.packed_attn_func(*x, seqs, causal=True)
        return (out, *torch.autograd.grad(out, x, do))

    ref = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    res = []
    for s in streams * 2:
        with torch.cuda.stream(s):
            res.append(run())
    torch.cuda.synchronize()
    for r in res:
        assert all(torch.equal(a, b) for a, b in zip(r, ref))


def test_a_plan_and_its_calls_on_different_streams():
    """Calls wait for the plan, and a rebuild waits for the calls, whichever streams they run on."""
    q, k, v, _ = (t.to(DEV) for t in make(900, 900, 4, 2, 64, BF, 3))
    bounds = [torch.tensor(b, dtype=torch.int32, device=DEV) for b in ([0, 500, 501, 900], [0, 0, 33, 700])]
    want = [tx.packed_attn_func(q, k, v, tx.PackedSequences(b, total_q=900), causal=True) for b in bounds]
    cu = bounds[0].clone()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        torch.cuda._sleep(20_000_000)
        seqs = tx.PackedSequences(cu, total_q=900)
    with torch.cuda.stream(b):
        torch.cuda._sleep(20_000_000)
        first = tx.packed_attn_func(q, k, v, seqs, causal=True)
    with torch.cuda.stream(a):
        cu.copy_(bounds[1])
        seqs.rebuild()
    second = tx.packed_attn_func(q, k, v, seqs, causal=True)
    with torch.cuda.stream(b):
        third = tx.packed_attn_func(q, k, v, seqs, causal=True)
        del seqs
    torch.cuda.synchronize()
    for got, ref in zip((first, second, third), (want[0], want[1], want[1])):
        assert torch.equal(got, ref)


def test_a_scale_in_a_tensor_is_read_at_every_call():
    q, k, v, _ = (t.to(DEV) for t in make(50, 50, 2, 2, 64, BF, 3))
    seqs, scale = tx.PackedSequences([0, 50]), torch.tensor(0.125)
    first = tx.packed_attn_func(q, k, v, seqs, scale)
    scale.fill_(0.5)
    assert torch.equal(tx.packed_attn_func(q, k, v, seqs, scale), tx.packed_attn_func(q, k, v, seqs, 0.5))
    assert torch.equal(first, tx.packed_attn_func(q, k, v, seqs, 0.125))


def test_window_bounds_beyond_64_bits():
    q, k, v, _ = (t.to(DEV) for t in make(150, 150, 2, 2, 64, BF, 3))
    seqs = tx.PackedSequences([0, 150])
    for wide, same in (((1 << 70, 0), (150, 0)), ((3, 1 << 64), (3, 150)), ((-(1 << 70), 5), (-150, 5))):
        assert torch.equal(tx.packed_attn_func(q, k, v, seqs, window_size=wide), tx.packed_attn_func(q, k, v, seqs, window_size=same))


def test_captured_step_with_new_lengths():
    """Plan, forward and backward in one graph; the boundaries change between replays."""
    H, Hkv, D, T = 4, 2, 64, 400
    cu = torch.tensor([0, 100, 400], dtype=torch.int32, device=DEV)
    q, k, v, do = (torch.zeros(s, device=DEV, dtype=BF) for s in ((T, H, D), (T, Hkv, D), (T, Hkv, D), (T, H, D)))
    seqs = tx.PackedSequences(cu, total_q=T)

    def step():
        seqs.rebuild()
        x = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = tx.packed_attn_func(*x, seqs, causal=True)
        return (out.detach(), *torch.autograd.grad(out, x, do))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(), step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        static = step()
    for n, bounds in enumerate(([0, 1, 400], [0, 399, 400], [0, 128, 256], [0, 0, 33])):
        data = make(T, T, H, Hkv, D, BF, n)
        for t, src in zip((q, k, v, do), data):
            t.copy_(src)
        cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        torch.cuda.synchronize()
        g.replay()
        _ = torch.randn(64, 64, device=DEV) @ torch.randn(64, 64, device=DEV)
        torch.cuda.synchronize()
        for a, b in zip(static, step()):
            assert torch.equal(a, b), n
        val, tol = packed(*data, bounds, bounds, D ** -0.5, True)
        for name, t in zip(("out", "dq", "dk", "dv"), static):
            close(name, t, val[name], tol[name], BF)


def test_rebuild_between_forward_and_backward_is_refused():
    x = torch.randn(20, 2, 64, device=DEV).to(BF).requires_grad_(True)
    seqs = tx.PackedSequences(torch.tensor([0, 9, 20], device=DEV), total_q=20)
    out = tx.packed_attn_func(x, x, x, seqs, causal=True)
    seqs.rebuild()
    with pytest.raises(RuntimeError, match="rebuilt"):
        out.sum().backward()


def test_second_derivatives_and_gradients_of_slopes_are_refused():
    q, k, v = (torch.randn(20, 2, 64, device=DEV).to(BF).requires_grad_(True) for _ in range(3))
    seqs = tx.PackedSequences([0, 9, 20])
    slopes = torch.tensor([0.5, 0.25], device=DEV, requires_grad=True)
    for _ in range(2):  # (the second call finds the first one's arguments)
        with pytest.raises(ValueError):
            tx.packed_attn_func(q, k, v, seqs, causal=True, alibi_slopes=slopes)
        tx.packed_attn_func(q, k, v, seqs, causal=True, alibi_slopes=slopes.detach())
    with torch.no_grad():
        tx.packed_attn_func(q, k, v, seqs, causal=True, alibi_slopes=slopes)
    (dq,) = torch.autograd.grad(tx.packed_attn_func(q, k, v, seqs).float().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.float().sum().backward()


def test_refusals():
    x = torch.randn(20, 4, 64, device=DEV).to(BF)
    seqs = tx.PackedSequences([0, 9, 20])
    f = tx.packed_attn_func
    for bad in (lambda: f(x.cpu(), x, x, seqs), lambda: f(x, x, x, [0, 20]), lambda: f(x[None], x, x, seqs),
                lambda: f(x, x.half(), x.half(), seqs), lambda: f(x.double(), x.double(), x.double(), seqs),
                lambda: f(x, x[:, :3], x[:, :3], seqs), lambda: f(x[:19], x, x, seqs), lambda: f(x, x[:, :2], x, seqs),
                lambda: f(x, x[..., :32], x[..., :32], seqs), lambda: f(x, x, x, seqs, alibi_slopes=torch.ones(3, device=DEV)),
                lambda: f(*[torch.randn(20, 2, 264, device=DEV)] * 3, seqs),
                lambda: tx.PackedSequences([0, 5, 3]), lambda: tx.PackedSequences([1, 5]), lambda: tx.PackedSequences([0]),
                lambda: tx.PackedSequences([0, 9], total_q=8), lambda: tx.PackedSequences([0, 9], [0, 4, 9]),
                lambda: tx.PackedSequences(torch.tensor([0, 9], device=DEV)), lambda: tx.PackedSequences([0, 9], total_k=7),
                lambda: tx.PackedSequences(torch.tensor([0.0, 9.0])), lambda: tx.PackedSequences([0, 9], device="cpu")):
        with pytest.raises(ValueError):
            bad()
