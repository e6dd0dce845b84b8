"""Attention over ragged batches, as measured cases: packed sequences of
different lengths (forward, and forward with backward), and a batch of requests
behind one shared prefix.

A case is a dict of plain values.  ``listed()`` names the fixed ones,
``draw(rng)`` makes one more of the same ranges; ``prepare`` builds what a
program holds before the call, ``run`` is one pass, ``exact`` the same pass from
the operators' definitions in 64 bits, ``work`` the bytes and operations that a
pass cannot do without.

``own`` false: ``run`` computes the operators in elementary torch operations in
32 bits.  ``own`` true: it calls the framework's ``packed_attn_func`` and
``shared_prefix_attn_func``.

Packed attention: sequence s holds the rows q_start[s] .. of q and k_start[s] ..
of k and v; with Lq and Lk of them and off = Lk - Lq (the queries are the
sequence's last positions)
    s[i, j] = scale * <q_i, k_j> - slope * |i + off - j|
    s[i, j] = -inf  where j > i + off (causal) or j < i + off - window
    out_i   = sum_j softmax_j(s[i, :]) v_j,   0 for a row that sees no key
Shared prefix: every query sees the whole prefix; query i of request b (the last
Sq of its ``len`` own positions) also sees the own keys j <= len - Sq + i.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _packed(name, lens, H, Hkv, D, dtype, past=None, pad=0, window=0, alibi=False, grad=False, lse=False):
    """Sequences of ``lens`` query rows, each behind ``past`` keys of its own (a
    chunk of a longer prompt), ``pad`` rows of padding behind the last one."""
    c = dict(kind="packed", lens=",".join(map(str, lens)), past=",".join(map(str, past)) if past else "", pad=pad, H=H,
             Hkv=Hkv, D=D, dtype=dtype, causal=True, window=window, alibi=alibi, grad=grad, lse=lse)
    return dict(name=name, **c) if name else c


def _shared(name, P, lens, cap, Sq, H, Hkv, D, dtype):
    """One request per entry of ``lens`` (own keys, the ``Sq`` new ones among
    them) in caches of ``cap`` rows, behind a prefix of ``P`` keys."""
    c = dict(kind="shared", P=P, lens=",".join(map(str, lens)), cap=cap, Sq=Sq, H=H, Hkv=Hkv, D=D, dtype=dtype)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # three short prompts that arrive together: launches and latency count
        _packed("prompts_short", [1, 17, 64], 32, 8, 128, "bf16"),
        # an ordinary prefill batch of a GQA model, ragged and odd lengths
        _packed("prompts_ragged", [2048, 1, 977, 1531, 64, 300, 2047, 5, 1224, 129], 32, 8, 128, "bf16"),
        # long prompts, the longest of 8192 tokens
        _packed("prompts_long", [8192, 4099, 2500, 1593], 32, 8, 128, "bf16"),
        # prompts of an ALiBi model with heads of 64, fp16, the batch padded to a fixed row count
        _packed("prompts_alibi_fp16", [1024, 333, 2048, 700, 1, 1300, 512, 90], 16, 16, 64, "fp16", pad=136, alibi=True),
        # the next chunk of long prompts against their caches through a sliding window
        _packed("chunk_window", [512, 512, 200, 512, 1, 77], 32, 8, 128, "bf16", past=[7000, 3584, 0, 16000, 9000, 1],
                window=4096, lse=True),
        # training on packed documents, GPT-2-small heads
        _packed("train_documents", [1024, 37, 700, 255, 512, 1, 900, 667], 12, 12, 64, "bf16", grad=True),
        # training of a GQA model on packed documents
        _packed("train_gqa", [4096, 1000, 2047, 49, 500, 500], 32, 8, 128, "bf16", grad=True),
        # training in torch's default dtype, a head_dim between the kernels'
        _packed("train_fp32", [200, 512, 77, 300, 1], 8, 8, 80, "fp32", pad=14, grad=True),
        # one prompt sampled four times: small and latency bound
        _shared("samples_four", 1024, [1, 1, 1, 1], 256, 1, 32, 8, 128, "bf16"),
        # a serving batch behind one long system prompt
        _shared("serve_prefix", 8192, [1 + 37 * i % 1024 for i in range(64)], 1024, 1, 32, 8, 128, "bf16"),
        # the same for a model without grouped heads, a few draft tokens verified at once
        _shared("verify_drafts", 4000, [5 + 53 * i % 700 for i in range(16)], 1024, 5, 16, 16, 64, "fp16"),
        # user turns of up to 256 tokens appended behind the prefix
        _shared("extend_turns", 6000, [256 + 91 * i for i in range(8)], 1024, 256, 32, 8, 128, "bf16"),
    ]


def draw(rng):
    def size(lo, hi):  # spread over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    half = rng.choice(["bf16", "bf16", "fp16"])
    while True:
        pick = rng.randrange(6)
        if pick < 4:
            grad = pick >= 2
            n = size(1, 24)
            top = size(8, 4096 if grad else 8192)
            lens = [size(1, top) for _ in range(n)]
            if n > 1 and rng.random() < 0.2:
                lens[rng.randrange(n)] = 0
            H, Hkv = rng.choice([(32, 8), (16, 4), (16, 16), (12, 12), (16, 1)])
            D = rng.choice([64, 128, 128, 128, 256, 80, 96])
            dtype = half if pick != 3 or rng.random() < 0.5 else "fp32"
            past, window = None, 0
            if pick == 1:
                past = [rng.choice([0, size(1, 8192)]) for _ in range(n)]
                window = rng.choice([0, 0, size(16, 4096)])
            c = _packed(None, lens, H, Hkv, D, dtype, past, rng.choice([0, 0, size(1, 200)]), window,
                        rng.random() < 0.25, grad, pick == 1)
            cost = work(c)["flops"] * (8 if dtype == "fp32" else 2 if D == 256 else 1)
            least = 2e5
        else:
            B, Sq = size(1, 64), rng.choice([1, 1, 1, size(2, 16), size(16, 256)])
            cap = max(size(16, 2048), Sq)
            lens = [rng.randint(Sq, cap) for _ in range(B)]
            H, Hkv = rng.choice([(32, 8), (16, 4), (16, 16), (16, 1)])
            c = _shared(None, size(100, 8192), lens, cap, Sq, H, Hkv, rng.choice([64, 128, 128, 256]),
                        half if rng.random() < 0.85 else "fp32")
            cost = work(c)["flops"] * (8 if c["dtype"] == "fp32" else 2 if c["D"] == 256 else 1)
            least = 2e5
        if least < cost < 6e11 and work(c)["bytes"] < 1.2e9:
            return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _ints(text):
    return [int(x) for x in text.split(",")] if text else []


def _seqs(case):
    """(q_start, Lq, k_start, Lk) of every sequence, and the rows of q and k."""
    lens = _ints(case["lens"])
    past = _ints(case["past"]) or [0] * len(lens)
    out, q0, k0 = [], 0, 0
    for n, p in zip(lens, past):
        out.append((q0, n, k0, n + p))
        q0, k0 = q0 + n, k0 + n + p
    return out, q0 + case["pad"], k0 + (case["pad"] if not case["past"] else 0)


def _slopes(H):
    n = 2 ** math.floor(math.log2(H))
    s = [2.0 ** (-8.0 * (i + 1) / n) for i in range(n)] + [2.0 ** (-4.0 * (2 * i + 1) / n) for i in range(H - n)]
    return torch.tensor(s, dtype=torch.float32, device=DEV)


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dt)

    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    if case["kind"] == "packed":
        _, tq, tk = _seqs(case)
        d = dict(q=rand(tq, H, D), k=rand(tk, Hkv, D), v=rand(tk, Hkv, D))
        if case["grad"]:
            d["dout"] = rand(tq, H, D)
        return d
    B, cap = len(_ints(case["lens"])), case["cap"]
    # caches as the layers keep them: (batch, kv head, position, head_dim)
    return dict(q=rand(B, case["Sq"], H, D), pk=rand(case["P"], Hkv, D), pv=rand(case["P"], Hkv, D),
                k=rand(B, Hkv, cap, D).transpose(1, 2), v=rand(B, Hkv, cap, D).transpose(1, 2))


def prepare(case, seed):
    st = dict(case=case, **_inputs(case, seed))
    if case["kind"] == "packed":
        seqs, tq, tk = _seqs(case)
        st["seqs"] = seqs
        st["slopes"] = _slopes(case["H"]) if case["alibi"] else None
        if case["grad"]:
            for n in ("q", "k", "v"):
                st[n].requires_grad_(True)
        if own:
            from trinix_amd import PackedSequences

            cu_q = torch.tensor([s[0] for s in seqs] + [seqs[-1][0] + seqs[-1][1]], dtype=torch.int32, device=DEV)
            cu_k = torch.tensor([s[2] for s in seqs] + [seqs[-1][2] + seqs[-1][3]], dtype=torch.int32, device=DEV)
            st["plan"] = PackedSequences(cu_q, cu_k if case["past"] else None, total_q=tq, total_k=tk)
    else:
        st["lens"] = torch.tensor(_ints(case["lens"]), dtype=torch.int32, device=DEV)
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if case["kind"] == "packed":
        if own:
            return _own_packed(st, case)
        return _plain_packed(st, case)
    if own:
        from trinix_amd import shared_prefix_attn_func

        return shared_prefix_attn_func(st["q"], st["pk"], st["pv"], st["k"], st["v"], st["lens"])
    return _plain_shared(st, case)


def _own_packed(st, case):
    from trinix_amd import packed_attn_func

    out = packed_attn_func(st["q"], st["k"], st["v"], st["plan"], causal=True,
                           window_size=(case["window"], 0) if case["window"] else None, alibi_slopes=st["slopes"],
                           return_lse=case["lse"])
    if not case["grad"]:
        return out
    dq, dk, dv = torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["dout"])
    return out.detach(), dq, dk, dv


def _plain_packed(st, case):
    """Every sequence by itself, 2048 query rows at a time, the heads of a group as rows."""
    dt, H, Hkv, D, grad = DTYPES[case["dtype"]], case["H"], case["Hkv"], case["D"], case["grad"]
    G, scale = H // Hkv, D ** -0.5
    with torch.no_grad():
        q, k, v = (st[n].float() for n in ("q", "k", "v"))
        out = torch.zeros_like(q)
        lse = torch.full((H, q.shape[0]), -math.inf, device=DEV)
        if grad:
            do = st["dout"].float()
            dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        for q0, lq, k0, lk in st["seqs"]:
            if not lq or not lk:
                continue
            ks = k[k0:k0 + lk].permute(1, 0, 2).contiguous()
            vs = v[k0:k0 + lk].permute(1, 0, 2).contiguous()
            kt = ks.transpose(1, 2).contiguous()
            vt = vs.transpose(1, 2).contiguous()
            for i0 in range(0, lq, 2048):
                n = min(2048, lq - i0)

                def rows(x):  # (n, H, D) rows to (Hkv, G * n, D)
                    x = x[q0 + i0:q0 + i0 + n].reshape(n, Hkv, G, D).permute(1, 2, 0, 3)
                    return x.reshape(Hkv, G * n, D)

                def back(x):
                    return x.reshape(Hkv, G, n, D).permute(2, 0, 1, 3).reshape(n, H, D)

                qs = rows(q)
                s = (torch.matmul(qs, kt) * scale).view(Hkv, G, n, lk)
                i = torch.arange(i0, i0 + n, device=DEV)[:, None] + (lk - lq)
                j = torch.arange(lk, device=DEV)[None, :]
                if st["slopes"] is not None:
                    s -= st["slopes"].view(Hkv, G, 1, 1) * (i - j).abs().float()
                hide = j > i
                if case["window"]:
                    hide = hide | (j < i - case["window"])
                s.masked_fill_(hide, -math.inf)
                m = s.amax(-1, keepdim=True)
                m = torch.where(m == -math.inf, torch.zeros_like(m), m)
                p = torch.exp(s - m)
                total = p.sum(-1, keepdim=True)
                p = p / torch.where(total == 0, torch.ones_like(total), total)
                lse[:, q0 + i0:q0 + i0 + n] = (torch.log(total) + m).reshape(H, n)
                p = p.view(Hkv, G * n, lk)
                o = torch.matmul(p, vs)
                out[q0 + i0:q0 + i0 + n] = back(o)
                if grad:
                    ds = rows(do)
                    dv[k0:k0 + lk] += torch.matmul(p.transpose(1, 2), ds).permute(1, 0, 2)
                    dz = p * (torch.matmul(ds, vt) - (ds * o).sum(-1, keepdim=True))
                    dq[q0 + i0:q0 + i0 + n] = back(torch.matmul(dz, ks) * scale)
                    dk[k0:k0 + lk] += torch.matmul(dz.transpose(1, 2), qs).permute(1, 0, 2) * scale
        if grad:
            return out.to(dt), dq.to(dt), dk.to(dt), dv.to(dt)
        return (out.to(dt), lse) if case["lse"] else out.to(dt)


def _plain_shared(st, case):
    """Scores against the prefix and against the own keys side by side, one softmax over both."""
    H, Hkv, D, P, Sq = case["H"], case["Hkv"], case["D"], case["P"], case["Sq"]
    B, cap, G, scale = st["q"].shape[0], case["cap"], H // Hkv, D ** -0.5
    q = st["q"].float().view(B, Sq, Hkv, G, D).permute(2, 0, 3, 1, 4).contiguous()  # (Hkv, B, G, Sq, D)
    pk, pv = (st[n].float().permute(1, 0, 2).contiguous() for n in ("pk", "pv"))     # (Hkv, P, D)
    k, v = (st[n].float().permute(2, 0, 1, 3).contiguous() for n in ("k", "v"))      # (Hkv, B, cap, D)
    s = torch.empty((Hkv, B, G * Sq, P + cap), device=DEV)
    s[..., :P] = torch.matmul(q.view(Hkv, B * G * Sq, D), pk.transpose(1, 2).contiguous()).view(Hkv, B, G * Sq, P)
    s[..., P:] = torch.matmul(q.view(Hkv, B, G * Sq, D), k.transpose(2, 3).contiguous())
    s *= scale
    j = torch.arange(cap, device=DEV)
    last = st["lens"].view(B, 1) - Sq + torch.arange(Sq, device=DEV)  # the last own key that a query sees
    hide = (j > last[..., None])[:, None].expand(B, G, Sq, cap).reshape(B, G * Sq, cap)
    s[..., P:].masked_fill_(hide, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p[..., :P].reshape(Hkv, B * G * Sq, P), pv).view(Hkv, B, G * Sq, D) + torch.matmul(p[..., P:], v)
    return o.view(Hkv, B, G, Sq, D).permute(1, 3, 0, 2, 4).reshape(B, Sq, H, D).to(DTYPES[case["dtype"]])


# ---------------------------------------------------------------------------
# The same in 64 bits, head by head, gradients by autograd
# ---------------------------------------------------------------------------
def exact(case, seed):
    x = {n: t.double() for n, t in _inputs(case, seed).items()}
    return _exact_packed(case, x) if case["kind"] == "packed" else _exact_shared(case, x)


def _exact_packed(case, x):
    H, G = case["H"], case["H"] // case["Hkv"]
    slopes = _slopes(H).double() if case["alibi"] else None
    out = torch.zeros_like(x["q"])
    lse = torch.full((H, out.shape[0]), -math.inf, device=DEV, dtype=torch.float64)
    grads = [torch.zeros_like(x[n]) for n in ("q", "k", "v")]
    for q0, lq, k0, lk in _seqs(case)[0]:
        if not lq or not lk:
            continue
        dist = torch.arange(lk, device=DEV)[None, :] - torch.arange(lk - lq, lk, device=DEV)[:, None]  # j - i
        seen = dist <= 0
        if case["window"]:
            seen &= dist >= -case["window"]
        empty = ~seen.any(-1)
        for h in range(H):
            parts = [x["q"][q0:q0 + lq, h], x["k"][k0:k0 + lk, h // G], x["v"][k0:k0 + lk, h // G]]
            if case["grad"]:
                parts = [t.detach().clone().requires_grad_(True) for t in parts]
            z = parts[0] @ parts[1].T / math.sqrt(case["D"])
            if slopes is not None:
                z = z + slopes[h] * -dist.abs()
            z = z.masked_fill(~seen, -math.inf)
            z = z.masked_fill(empty[:, None], 0.0)  # rows without a key: put right below
            o = (torch.softmax(z, -1) @ parts[2]).masked_fill(empty[:, None], 0.0)
            out[q0:q0 + lq, h] = o.detach()
            lse[h, q0:q0 + lq] = torch.logsumexp(z.detach(), -1).masked_fill(empty, -math.inf)
            if case["grad"]:
                d = torch.autograd.grad(o, parts, x["dout"][q0:q0 + lq, h])
                grads[0][q0:q0 + lq, h] = d[0]
                grads[1][k0:k0 + lk, h // G] += d[1]
                grads[2][k0:k0 + lk, h // G] += d[2]
    if case["grad"]:
        return (out, *grads)
    return (out, lse) if case["lse"] else out


def _exact_shared(case, x):
    Sq, G = case["Sq"], case["H"] // case["Hkv"]
    out = torch.empty_like(x["q"])
    for b, n in enumerate(_ints(case["lens"])):
        # keys of the prefix, then the request's own, as one sequence
        k = torch.cat([x["pk"], x["k"][b, :n]]).permute(1, 2, 0).repeat_interleave(G, 0).contiguous()
        v = torch.cat([x["pv"], x["v"][b, :n]]).permute(1, 0, 2).repeat_interleave(G, 0).contiguous()
        z = x["q"][b].permute(1, 0, 2).contiguous() @ k / math.sqrt(case["D"])
        at = torch.arange(z.shape[-1], device=DEV)[None, :]
        z = z.masked_fill(at > case["P"] + n - Sq + torch.arange(Sq, device=DEV)[:, None], -math.inf)
        out[b] = (torch.softmax(z, -1) @ v).permute(1, 0, 2)
    return out


# ---------------------------------------------------------------------------
# What a pass has to move and compute
# ---------------------------------------------------------------------------
def work(case):
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "shared":
        lens, Sq = _ints(case["lens"]), case["Sq"]
        B = len(lens)
        pairs = sum(case["P"] * Sq + sum(n - Sq + i + 1 for i in range(Sq)) for n in lens)
        return {"bytes": size * D * (2 * B * Sq * H + 2 * Hkv * (case["P"] + sum(lens))) + 4 * B,
                "flops": 4 * D * H * pairs}
    seqs, tq, tk = _seqs(case)
    pairs, seen = 0, 0
    for _, lq, _, lk in seqs:
        w = case["window"] or lk
        pairs += sum(min(i + 1, w + 1) for i in range(lk - lq, lk))
        seen += min(lk, lq + w) if lq else 0
    q_bytes, k_bytes = size * D * H * tq, size * D * Hkv * (seen + (case["pad"] if not case["past"] else 0))
    if not case["grad"]:
        return {"bytes": 2 * q_bytes + 2 * k_bytes + (4 * H * tq if case["lse"] else 0), "flops": 4 * D * H * pairs}
    # forward: q, k, v -> out; backward: dout as well -> dq, dk, dv (two products forward, five more backward)
    return {"bytes": 4 * q_bytes + 4 * k_bytes, "flops": 14 * D * H * pairs}
