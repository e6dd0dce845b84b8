"""Attention behind a shared prefix against plain 64-bit attention of every
request: types, head layouts, one query to many, lengths from nothing to several
chunks, cache layouts, and rows that see no key."""
import math

import pytest
import torch

import trinix_amd as tx
from packed_oracle import close

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def oracle(q, pk, pv, k, v, lens, scale):
    """Values and bounds (packed_oracle; here one more merge of fp32 partial sums, inside its Lk w)."""
    f = torch.float64
    B, Sq, H, D = q.shape
    P, G = pk.shape[0], H // k.shape[2]
    u, w = torch.finfo(q.dtype).eps / 2, 2.0 ** -24
    out, tol = torch.zeros(B, Sq, H, D, dtype=f), torch.zeros(B, Sq, H, D, dtype=f)
    lse, ltol = torch.full((B, H, Sq), -math.inf, dtype=f), torch.zeros(B, H, Sq, dtype=f)
    for b in range(B):
        n = min(max(int(lens[b]), 0), k.shape[1])
        for h in range(H):
            x = q[b, :, h].to(f)
            kk = torch.cat([pk[:, h // G], k[b, :n, h // G]]).to(f)
            vv = torch.cat([pv[:, h // G], v[b, :n, h // G]]).to(f)
            if not kk.shape[0]:
                continue
            z = scale * x @ kk.T
            T = abs(scale) * (x.abs() @ kk.abs().T).max().item()
            last = P + n - Sq + torch.arange(Sq)
            hide = (torch.arange(P + n)[None, :] > last[:, None]) & (torch.arange(P + n)[None, :] >= P)
            z = z.masked_fill(hide, -math.inf)
            live = (~hide).any(-1)
            p = torch.zeros_like(z)
            p[live] = torch.softmax(z[live], -1)
            rp = 2 * (D + 4) * w * T + (P + n + 16) * w
            out[b, :, h] = p @ vv
            tol[b, :, h] = u * out[b, :, h].abs() + (u + rp) * (p @ vv.abs())
            lse[b, h, live] = torch.logsumexp(z[live], -1)
            ltol[b, h] = rp + 4 * w * lse[b, h].abs().nan_to_num(0, 0, 0)
    return out, tol, lse, ltol


def check(B, Sq, P, cap, lens, H=8, Hkv=2, D=64, dtype=BF, seed=0, layout="bhsd", scale=None, poison=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g).to(dtype)
    q, pk, pv = r(B, Sq, H, D), r(P, Hkv, D), r(P, Hkv, D)
    if layout == "bhsd":
        k, v = r(B, Hkv, cap, D).transpose(1, 2), r(B, Hkv, cap, D).transpose(1, 2)
    else:
        k, v = r(B, cap, Hkv, D), r(B, cap, Hkv, D)
    lens = [cap] * B if lens is None else lens
    kd, vd = k.to(DEV), v.to(DEV)
    if poison:  # nothing behind a request's keys is read
        for b, n in enumerate(lens):
            kd[b, max(0, n):] = float("nan")
            vd[b, max(0, n):] = float("inf")
    got, lse = tx.shared_prefix_attn_func(q.to(DEV), pk.to(DEV), pv.to(DEV), kd, vd,
                                          torch.tensor(lens, device=DEV, dtype=torch.int32), scale, return_lse=True)
    out, tol, ref, ltol = oracle(q, pk, pv, k, v, lens, D ** -0.5 if scale is None else scale)
    close("out", got, out, tol, dtype)
    close("lse", lse, ref, ltol, F32)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("D", [64, 128, 256, 8, 30, 40, 80, 96, 129, 200])
def test_decode(dtype, D):
    check(5, 1, 300, 200, [1, 200, 64, 17, 129], D=D, dtype=dtype, seed=D)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 8), (16, 1), (32, 8), (6, 3), (40, 2)])
def test_head_layouts(H, Hkv):
    check(3, 2, 150, 90, [2, 90, 33], H=H, Hkv=Hkv, seed=H)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("Sq", [2, 5, 16, 33, 128])
def test_several_queries(Sq, dtype):
    check(3, Sq, 257, 300, [Sq, 300, Sq + 40], Sq and 8, 2, 128, dtype, seed=Sq)


@pytest.mark.parametrize("P", [0, 1, 15, 64, 127, 129, 1000, 5000])
def test_prefix_lengths(P):
    check(4, 1, P, 70, [1, 70, 16, 31], D=128, seed=P)
    check(20, 3, P, 70, [3 + 3 * b for b in range(20)], D=64, seed=P)


def test_rows_without_keys():
    # no prefix; requests without own keys, and queries before the first own key
    check(4, 3, 0, 40, [0, 2, 3, 40], D=64)
    check(4, 3, 20, 40, [0, 1, 3, 40], D=64)
    check(2, 1, 50, 0, [0, 0], D=64)
    check(2, 2, 0, 0, [0, 0], D=128)


@pytest.mark.parametrize("B", [1, 2, 16, 70])
def test_batches(B):
    check(B, 1, 700, 130, [1 + (41 * b) % 130 for b in range(B)], D=128, seed=B)


def test_long_prefix_and_long_caches():
    check(2, 1, 20000, 9000, [9000, 4001], H=4, Hkv=1, D=128)


@pytest.mark.parametrize("dtype,Sq", [(BF, 1), (BF, 70), (F32, 1)])
def test_offsets_beyond_32_bits(dtype, Sq):
    """Caches and a prefix that end more than 2^32 bytes and 2^31 elements behind their start: as copies."""
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)
    B, P, S, D = 3, 270_000, 90_000, 64
    wide = torch.empty(B * S, 2, 4096, dtype=dtype, device=DEV)
    wide[:, :, :2 * D] = r(B * S, 2, 2 * D)
    cache = wide.view(B, S, 2, 4096)
    args = (wide[:, :, :D], wide[:, :, D:2 * D], cache[..., :D], cache[..., D:2 * D])
    q, lens = r(B, Sq, 4, D), torch.tensor([S, 100, S - 3], device=DEV)
    assert args[0].shape[0] == P
    got = tx.shared_prefix_attn_func(q, *args, lens)
    assert torch.equal(got, tx.shared_prefix_attn_func(q, *(t.contiguous() for t in args), lens))


def test_layouts_and_scales():
    check(3, 2, 100, 64, [64, 5, 33], layout="bshd")
    check(3, 2, 100, 64, None, poison=False)
    check(3, 2, 100, 64, [64, 5, 33], scale=-0.3)
    check(3, 2, 100, 64, [64, 5, 33], scale=0.0)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strided_and_unaligned_operands(dtype):
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(s, generator=g).to(dtype)
    base, pk, pv, kv = r(3 * 2 * 8 * 64 + 1), r(90, 4, 64), r(90, 2, 64 + 4), r(3, 50, 2, 130)
    dev = [t.to(DEV) for t in (base, pk, pv, kv)]

    def args(base, pk, pv, kv):  # start off 16 bytes; every second head; odd row strides; a slice
        return base[1:].view(3, 2, 8, 64), pk[:, ::2], pv[..., 2:66], kv[..., :64], kv[..., 65:129]

    lens = [50, 2, 31]
    got = tx.shared_prefix_attn_func(*args(*dev), torch.tensor(lens, device=DEV))
    out, tol, _, _ = oracle(*args(base, pk, pv, kv), lens, 0.125)
    close("out", got, out, tol, dtype)


@pytest.mark.parametrize("kind", ["1", "2", "3"])
@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (BF, 256)])
def test_forced_kinds(kind, dtype, D, monkeypatch):
    # 64 or 128 rows by a chunk of keys, whole rows of 64 and of 128
    monkeypatch.setenv("TRINIX_SHARED_KIND", kind)
    check(5, 1, 300, 200, [1, 200, 64, 0, 129], D=D, dtype=dtype)
    check(3, 40, 1000, 500, [500, 3, 97], D=D, dtype=dtype)
    check(2, 100, 0, 260, [260, 0], H=6, Hkv=3, D=D, dtype=dtype)
    check(2, 7, 65, 0, [0, 0], H=6, Hkv=3, D=D, dtype=dtype)


@pytest.mark.parametrize("kind", ["1", "2", "3"])
def test_small_calls_by_every_kind(kind, monkeypatch):
    # (the rule takes whole rows for most of these sizes)
    monkeypatch.setenv("TRINIX_SHARED_KIND", kind)
    for H, Hkv in ((1, 1), (16, 1), (6, 3), (40, 2)):
        check(3, 2, 150, 90, [2, 90, 33], H=H, Hkv=Hkv, seed=H)
    check(4, 3, 0, 40, [0, 2, 3, 40], D=64)
    check(4, 3, 20, 40, [0, 1, 3, 40], D=64)
    check(2, 1, 50, 0, [0, 0], D=64)
    check(2, 2, 0, 0, [0, 0], D=128)
    check(20, 3, 129, 70, [3 + 3 * b for b in range(20)], D=64)
    check(3, 2, 100, 64, [64, 5, 33], layout="bshd", scale=-0.3, dtype=HF, D=80)
    check(3, 2, 100, 64, None, poison=False, scale=0.0)
    check(4, 1, 60, 64, [-5, 1000, 64, 0], poison=False)


def test_another_kind_for_a_call_seen_before(monkeypatch):
    # its workspace was sized for the first one
    for kind in ("3", "1", "2", "1"):
        monkeypatch.setenv("TRINIX_SHARED_KIND", kind)
        check(3, 2, 150, 90, [2, 90, 33], seed=3)


def test_lengths_outside_the_cache_are_clamped():
    check(4, 1, 60, 64, [-5, 1000, 64, 0], poison=False)


def test_as_one_sequence_per_request():
    """The framework's decode over prefix and own keys side by side."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g).to(BF).to(DEV)
    B, P, S = 3, 500, 77
    q, pk, pv, k, v = r(B, 1, 16, 128), r(P, 4, 128), r(P, 4, 128), r(B, S, 4, 128), r(B, S, 4, 128)
    got = tx.shared_prefix_attn_func(q, pk, pv, k, v)
    kk, vv = (torch.cat([a.expand(B, P, 4, 128), b], 1) for a, b in ((pk, k), (pv, v)))
    want = tx.triton_attn_func(q, kk, vv)
    assert (got - want).abs().max().item() <= 4 * 2.0 ** -9 * vv.abs().max().item()


def test_captured_step_with_new_lengths_and_two_streams():
    B, P, cap, H, Hkv, D = 4, 400, 200, 8, 2, 128
    z = lambda *s: torch.zeros(s, device=DEV, dtype=BF)
    q, pk, pv, k, v = z(B, 1, H, D), z(P, Hkv, D), z(P, Hkv, D), z(B, cap, Hkv, D), z(B, cap, Hkv, D)
    lens = torch.ones(B, dtype=torch.int32, device=DEV)

    def step():
        return tx.shared_prefix_attn_func(q, pk, pv, k, v, lens, return_lse=True)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(), step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for n in range(4):
        for t in (q, pk, pv, k, v):
            t.copy_(torch.randn(t.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(n)))
        lens.copy_(torch.tensor([1 + n, 200 - n, 64 * (n % 2), 130]))
        torch.cuda.synchronize()
        for (g, _), st in zip(graphs, streams):  # both at once
            with torch.cuda.stream(st):
                g.replay()
        _ = torch.randn(64, 64, device=DEV) @ torch.randn(64, 64, device=DEV)
        torch.cuda.synchronize()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), n


def test_with_packed_prompts():
    """A system prompt and user turns prefilled as packed sequences, the turns
    behind the prompt's keys, then a decode step: against each whole conversation
    as one packed sequence."""
    g = torch.Generator().manual_seed(3)
    H, Hkv, D, P, turns = 8, 2, 64, 333, [20, 1, 97]
    r = lambda *s: torch.randn(s, generator=g).to(F32).to(DEV)
    pq, pk, pv = r(P, H, D), r(P, Hkv, D), r(P, Hkv, D)
    own = [(r(n + 1, H, D), r(n + 1, Hkv, D), r(n + 1, Hkv, D)) for n in turns]
    cap, B = 128, len(turns)
    kc, vc = torch.full((B, Hkv, cap, D), float("nan"), device=DEV), torch.full((B, Hkv, cap, D), float("nan"), device=DEV)
    for b, (_, k, v) in enumerate(own):
        kc[b, :, :k.shape[0]], vc[b, :, :v.shape[0]] = k.transpose(0, 1), v.transpose(0, 1)
    decode = tx.shared_prefix_attn_func(torch.stack([o[0][-1:] for o in own]), pk, pv, kc.transpose(1, 2), vc.transpose(1, 2),
                                        torch.tensor([n + 1 for n in turns], device=DEV))
    lens = [P + n + 1 for n in turns]
    cu = [0, *torch.tensor(lens).cumsum(0).tolist()]
    cat = lambda a, i: torch.cat([torch.cat([a, o[i]]) for o in own])
    whole = tx.packed_attn_func(cat(pq, 0), cat(pk, 1), cat(pv, 2), tx.PackedSequences(cu), causal=True)
    for b in range(B):
        # fp32 on both sides: sums of up to 431 terms in another order
        assert (decode[b, 0] - whole[cu[b + 1] - 1]).abs().max().item() <= 2e-5
    # the turns as chunks behind the prompt
    ck = [0, *torch.tensor([P + n for n in turns]).cumsum(0).tolist()]
    cq = [0, *torch.tensor(turns).cumsum(0).tolist()]
    chunk = tx.packed_attn_func(torch.cat([o[0][:-1] for o in own]), torch.cat([torch.cat([pk, o[1][:-1]]) for o in own]),
                                torch.cat([torch.cat([pv, o[2][:-1]]) for o in own]), tx.PackedSequences(cq, ck), causal=True)
    for b in range(B):
        want = whole[cu[b] + P:cu[b + 1] - 1]
        assert (chunk[cq[b]:cq[b + 1]] - want).abs().max().item() <= 2e-5


def test_refusals():
    z = lambda *s, t=BF: torch.zeros(s, device=DEV, dtype=t)
    q, p, k = z(2, 1, 4, 64), z(9, 2, 64), z(2, 7, 2, 64)
    f = tx.shared_prefix_attn_func
    n = torch.ones(2, dtype=torch.int32, device=DEV)
    for bad in (lambda: f(q.cpu(), p, p, k, k), lambda: f(q[0], p, p, k, k), lambda: f(q, p[None], p[None], k, k),
                lambda: f(q, p.half(), p.half(), k, k), lambda: f(q, p, p[:8], k, k), lambda: f(q, p, p, k, k[:, :6]),
                lambda: f(q, p[:, :1], p[:, :1], k, k), lambda: f(q, p, p, k[:1], k[:1]), lambda: f(z(2, 1, 3, 64), p, p, k, k),
                lambda: f(q, p, p, k, k, n[:1]), lambda: f(q, p, p, k, k, n.float()), lambda: f(q, p, p, k, k, n.cpu()),
                lambda: f(q.requires_grad_(True), p, p, k, k),
                lambda: f(*[z(*s, t=torch.float64) for s in ((2, 1, 4, 64), (9, 2, 64), (9, 2, 64), (2, 7, 2, 64), (2, 7, 2, 64))]),
                lambda: f(*[z(*s) for s in ((2, 1, 4, 264), (9, 2, 264), (9, 2, 264), (2, 7, 2, 264), (2, 7, 2, 264))])):
        with pytest.raises(ValueError):
            bad()
    q = q.detach()
    assert f(z(0, 1, 4, 64), p, p, z(0, 7, 2, 64), z(0, 7, 2, 64)).shape == (0, 1, 4, 64)
    with torch.no_grad():
        assert f(q.requires_grad_(True), p, p, k, k).shape == q.shape


def test_a_scale_in_a_tensor_is_read_at_every_call():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV, torch.bfloat16)
    ts = (r(2, 1, 4, 64), r(70, 2, 64), r(70, 2, 64), r(2, 40, 2, 64), r(2, 40, 2, 64))
    scale = torch.tensor(0.125)
    first = tx.shared_prefix_attn_func(*ts, None, scale)
    scale.fill_(0.5)
    assert torch.equal(tx.shared_prefix_attn_func(*ts, None, scale), tx.shared_prefix_attn_func(*ts, None, 0.5))
    assert torch.equal(first, tx.shared_prefix_attn_func(*ts, None, 0.125))
