"""Plain 64-bit attention over packed sequences, with the error that a correct
kernel may show against it.

Bounds (u = finfo(t).eps / 2, half a step of the tensors' type; w = 2^-24, half a
step of fp32; |.| of matrices elementwise):
  scores     a product of D terms in fp32 errs by at most (D + 4) w T, with T the
             largest scale * sum_d |q_d k_d| plus the largest bias; a probability
             then by the relative rp = 2 (D + 4) w T + (Lk + 16) w (its own score and
             the row's sum), and by u more where it enters a product in the type;
  out        |out - ref| <= u |ref| + (u + rp) P |V|
  dV         <= u |dV| + (u + rp) P^T |dO|
  delta      the kernel's own out enters it with 2 u^2 of its size:
             ed = sum_d |dO| ((u + rp) P |V| + 2 u^2 |O|) + D w sum_d |dO| |O|
  dZ         ez = (rp + 4 u^2) |dZ| + P (D w |dO| |V|^T + ed)
  dQ, dK     <= u |dQ| + scale (ez + (Lk w) |dZ|) |K|, the same with Q for dK
fp32 calls have u = w.  The bounds are of the worst case; ``close`` also holds the
2-norm of the error under that of independent roundings, two half steps.
"""
import math

import torch


def band(lq, lk, causal, window):
    d = torch.arange(lk)[None, :] - torch.arange(lk - lq, lk)[:, None]
    ok = torch.ones(lq, lk, dtype=torch.bool)
    if causal:
        ok &= d <= 0
    if window is not None:
        ok &= (d >= -window[0]) & (d <= window[1])
    return ok, d


def one(q, k, v, do, scale, causal, window, slope, dtype):
    """One head of one sequence in 64 bits: values and their bounds, as dicts."""
    f = torch.float64
    q, k, v = q.to(f), k.to(f), v.to(f)
    (lq, D), lk = q.shape, k.shape[0]
    u, w = torch.finfo(dtype).eps / 2, 2.0 ** -24
    ok, d = band(lq, lk, causal, window)
    z = scale * q @ k.T
    T = abs(scale) * (q.abs() @ k.abs().T).max().item() if lq and lk else 0.0
    if slope is not None:
        z = z - slope * d.abs()
        T += abs(slope) * max(lk, lq)
    z = z.masked_fill(~ok, -math.inf)
    live = ok.any(-1) if lk else torch.zeros(lq, dtype=torch.bool)
    lse = torch.full((lq,), -math.inf, dtype=f)
    P = torch.zeros(lq, lk, dtype=f)
    if live.any():
        lse[live] = torch.logsumexp(z[live], -1)
        P[live] = torch.softmax(z[live], -1)
    rp = 2 * (D + 4) * w * T + (lk + 16) * w
    out, A = P @ v, P @ v.abs()
    val, tol = dict(out=out, lse=lse), dict(out=u * out.abs() + (u + rp) * A, lse=torch.full((lq,), rp, dtype=f) + 4 * w * lse.abs().nan_to_num(0, 0, 0))
    if do is not None:
        do = do.to(f)
        do = torch.where(live[:, None], do, torch.zeros_like(do))
        dP = do @ v.T
        dZ = P * (dP - (do * out).sum(-1, keepdim=True))
        ed = (do.abs() * ((u + rp) * A + 2 * u * u * out.abs())).sum(-1, keepdim=True) + D * w * (do.abs() * out.abs()).sum(-1, keepdim=True)
        ez = (rp + 4 * u * u) * dZ.abs() + P * (D * w * (do.abs() @ v.abs().T) + ed) + max(lk, lq) * w * dZ.abs()
        val.update(dq=scale * dZ @ k, dk=scale * dZ.T @ q, dv=P.T @ do)
        tol.update(dq=u * val["dq"].abs() + abs(scale) * ez @ k.abs(), dk=u * val["dk"].abs() + abs(scale) * ez.T @ q.abs(),
                   dv=u * val["dv"].abs() + (u + rp) * (P.T @ do.abs()))
    return val, tol


def packed(q, k, v, do, cu_q, cu_k, scale, causal=False, window=None, slopes=None):
    """(values, bounds) of a packed batch on CPU tensors of the call's type."""
    f = torch.float64
    Tq, H, D = q.shape
    G = H // k.shape[1]
    names = dict(out=(Tq, H, D), lse=(H, Tq))
    if do is not None:
        names.update(dq=(Tq, H, D), dk=tuple(k.shape), dv=tuple(v.shape))
    val = {n: torch.full(s, -math.inf if n == "lse" else 0.0, dtype=f) for n, s in names.items()}
    tol = {n: torch.zeros(s, dtype=f) for n, s in names.items()}
    for s in range(len(cu_q) - 1):
        a, b, c, e = cu_q[s], cu_q[s + 1], cu_k[s], cu_k[s + 1]
        if a == b and c == e:
            continue
        for h in range(H):
            x, t = one(q[a:b, h], k[c:e, h // G], v[c:e, h // G], None if do is None else do[a:b, h], scale, causal, window,
                       None if slopes is None else float(slopes[h]), q.dtype)
            for d, r in ((val, x), (tol, t)):
                d["out"][a:b, h], d["lse"][h, a:b] = r["out"], r["lse"]
                if do is not None:
                    d["dq"][a:b, h] = r["dq"]
                    d["dk"][c:e, h // G] += r["dk"]
                    d["dv"][c:e, h // G] += r["dv"]
    return val, tol


def close(name, got, val, tol, dtype):
    got = got.detach().double().cpu()
    assert got.shape == val.shape, (name, got.shape, val.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(val)), f"{name}: finite where the oracle is not, or the reverse"
    fin = torch.isfinite(val)
    assert torch.equal(got[~fin], val[~fin]), name
    err = (got - val)[fin].abs()
    over = err - tol[fin] - 2.0 ** -100
    # results below the type's smallest normal number are off by half its smallest step
    over -= torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert not (over > 0).any(), f"{name}: off by {err[over.argmax()]:.3e}, bound {tol[fin][over.argmax()]:.3e}"
    if err.numel() > 256 and val[fin].norm() > 0:
        u = torch.finfo(dtype).eps / 2
        rel = (err.norm() / val[fin].norm()).item()
        assert rel <= 2 * u + (3e-6 if dtype == torch.float32 else 0), f"{name}: 2-norm {rel:.3e}"
