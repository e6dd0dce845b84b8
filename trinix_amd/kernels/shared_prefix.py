"""Attention of a batch of requests behind one shared prefix through
``libtrinix_attn.so`` (semantics: ``trinix_shared_prefix_args`` in
``include/trinix_attn.h``).  The prefix's keys and values are read once for the
whole batch instead of once per request; no counterpart in the reference.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from .. import _native as nat
from .attention_kernel import _DTYPE_CODE, KERNEL_HEAD_DIMS, TritonAttentionKernel, current_stream_ptr, kernel_head_dim


def _strides(t: torch.Tensor):
    """Element strides; of a dimension of one element, which torch leaves open,
    the contiguous one."""
    st, inner = list(t.stride()), 1
    for d in range(t.dim() - 1, -1, -1):
        if t.shape[d] <= 1:
            st[d] = inner
        inner *= t.shape[d]
    return st


def _operand(t: torch.Tensor, d_kernel: int) -> torch.Tensor:
    """t as the kernels read it: at their head_dim, rows on 16 bytes."""
    if t.shape[-1] != d_kernel:
        t = torch.nn.functional.pad(t, (0, d_kernel - t.shape[-1]))
    per = 16 // t.element_size()

    def ready(x):
        st = _strides(x)
        return (st[-1] == 1 and x.data_ptr() % 16 == 0 and all(s % per == 0 for s in st[:-1]) and st[-3] < 1 << 22)

    if not ready(t):
        t = t.contiguous()
        if not ready(t):
            t = t.clone(memory_format=torch.contiguous_format)
    return t


# Launch cache (see attention_kernel.py): a call whose operands the kernels read
# in place is described, apart from its pointers, by shapes, strides, types and
# scalars.  The first one goes through every check and leaves its arguments here.
class _Launch:
    __slots__ = ("args", "lse_shape", "ws_bytes")

    def __init__(self, args, lse_shape, ws_bytes):
        self.args, self.lse_shape, self.ws_bytes = args, lse_shape, ws_bytes


_LAUNCHES: dict = {}
_MAX_LAUNCHES = 256


def _key(q, pk, pv, k, v, lens, scale, return_lse):
    return (q.shape, q.stride(), pk.shape, pk.stride(), pv.shape, pv.stride(), k.shape, k.stride(), v.shape, v.stride(),
            q.dtype, pk.dtype, pv.dtype, k.dtype, v.dtype, q.device, pk.device, pv.device, k.device, v.device,
            None if lens is None else (lens.shape, lens.stride(), lens.dtype, lens.device), scale, return_lse)


def shared_prefix_attention(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k: torch.Tensor,
                            v: torch.Tensor, seq_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                            return_lse: bool = False):
    """``shared_prefix_attn_func`` (``layers/attention/functional.py``)."""
    ts = (q, prefix_k, prefix_v, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or prefix_k.requires_grad or prefix_v.requires_grad or k.requires_grad
                                    or v.requires_grad):
        raise ValueError("shared_prefix_attention has no backward; call it under torch.no_grad()")
    if scale is not None:
        scale = float(scale)
    key = _key(*ts, seq_lens, scale, return_lse)
    ent = _LAUNCHES.get(key)
    if ent is not None:
        ptrs = [t.data_ptr() for t in ts]
        if not (ptrs[0] | ptrs[1] | ptrs[2] | ptrs[3] | ptrs[4]) % 16:
            a = nat.SharedPrefixArgs.from_buffer_copy(ent.args)
            a.q, a.prefix_k, a.prefix_v, a.k, a.v = ptrs
            if seq_lens is not None:
                a.seq_lens = seq_lens.data_ptr()
            return _run(a, ent, q)
    return _full(key, ts, seq_lens, scale, return_lse)


def _full(key, ts, seq_lens, scale, return_lse):
    q, prefix_k, prefix_v, k, v = ts
    if not all(t.is_cuda for t in ts):
        raise ValueError("shared_prefix_attention requires GPU tensors")
    if any(t.device != q.device for t in ts):
        raise ValueError(f"the tensors are on different devices: {[str(t.device) for t in ts]}")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or prefix_k.dim() != 3 or prefix_v.dim() != 3:
        raise ValueError("Expected q, k, v (batch, seqlen, nheads, headdim) and prefix_k, prefix_v (seqlen, nheads, headdim), "
                         f"got {[tuple(t.shape) for t in ts]}")
    if q.dtype not in _DTYPE_CODE or any(t.dtype != q.dtype for t in ts):
        raise ValueError(f"the tensors must share one type of float32, float16 and bfloat16, got {[t.dtype for t in ts]}")
    B, Sq, H, D = q.shape
    S, Hkv = k.shape[1], k.shape[2]
    if k.shape != (B, S, Hkv, D) or v.shape != k.shape or prefix_k.shape[1:] != (Hkv, D) or prefix_v.shape != prefix_k.shape:
        raise ValueError(f"shapes don't match: q, prefix_k, prefix_v, k, v are {[tuple(t.shape) for t in ts]}")
    if Hkv <= 0 or H <= 0 or D <= 0 or H % Hkv != 0:
        raise ValueError(f"num_heads ({H}) must be a multiple of the KV heads ({Hkv})")
    per = 16 // q.element_size()
    d_kernel = -(-D // per) * per  # rows of whole 16 bytes
    if kernel_head_dim(D) is None:
        raise ValueError(f"head_dim {D} > {KERNEL_HEAD_DIMS[-1]} is not supported")
    if seq_lens is not None and (seq_lens.shape != (B,) or seq_lens.device != q.device
                                 or seq_lens.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"seq_lens must be {B} int32 or int64 lengths on {q.device}, got {tuple(seq_lens.shape)} "
                         f"{seq_lens.dtype} on {seq_lens.device}")
    if not TritonAttentionKernel.is_available():
        raise RuntimeError("HIP attention kernel not available (build trinix_amd; needs a gfx950 GPU)")
    lse_shape = (B, H, Sq) if return_lse else None
    if not (B and Sq):
        out = torch.empty((B, Sq, H, D), dtype=q.dtype, device=q.device)
        return (out, torch.empty(lse_shape, dtype=torch.float32, device=q.device)) if return_lse else out
    ops = [_operand(t, d_kernel) for t in ts]
    a = nat.SharedPrefixArgs()
    a.q_stride, a.k_stride, a.v_stride = (nat.Int64x4(*_strides(ops[n])) for n in (0, 3, 4))
    a.prefix_k_stride, a.prefix_v_stride = (nat.Int64x3(*_strides(ops[n])) for n in (1, 2))
    a.out_stride = nat.Int64x4(Sq * H * d_kernel, H * d_kernel, d_kernel, 1)
    a.batch, a.seqlen_q, a.prefix_len, a.capacity = B, Sq, prefix_k.shape[0], S
    a.nheads_q, a.nheads_kv, a.head_dim, a.dtype = H, Hkv, d_kernel, _DTYPE_CODE[q.dtype]
    a.softmax_scale = float(D ** -0.5 if scale is None else scale)
    ent = _Launch(nat.SharedPrefixArgs.from_buffer_copy(a), lse_shape, None)
    lens = None
    if seq_lens is not None:
        lens = seq_lens.to(torch.int32).contiguous()
        a.seq_lens = lens.data_ptr()
    a.q, a.prefix_k, a.prefix_v, a.k, a.v = (t.data_ptr() for t in ops)
    res = _run(a, ent, ops[0])
    if all(x is y for x, y in zip(ops, ts)) and lens is seq_lens:  # read in place
        if len(_LAUNCHES) >= _MAX_LAUNCHES:
            _LAUNCHES.clear()
        _LAUNCHES[key] = ent
    if d_kernel != D:
        out = res[0] if return_lse else res
        out = out[..., :D].contiguous()
        return (out, res[1]) if return_lse else out
    return res


def _run(a: nat.SharedPrefixArgs, ent: _Launch, q: torch.Tensor):
    """Allocates out (shaped as q), lse and the workspace and launches; ent.ws_bytes None:
    asks for it first."""
    device = q.device
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _run(a, ent, q)
    lib = nat.load_library()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    a.out = out.data_ptr()
    lse = None
    if ent.lse_shape is not None:
        lse = torch.empty(ent.lse_shape, dtype=torch.float32, device=device)
        a.lse = lse.data_ptr()
    kept = ent.ws_bytes is not None
    if not kept:
        n = ctypes.c_int64(0)
        nat.check(lib.trinix_shared_prefix_workspace(ctypes.byref(a), ctypes.byref(n)), "trinix_shared_prefix_workspace")
        ent.ws_bytes = n.value
    ws = torch.empty(ent.ws_bytes, dtype=torch.uint8, device=device) if ent.ws_bytes else None
    rc = lib.trinix_shared_prefix_fwd(ctypes.byref(a), None if ws is None else ws.data_ptr(), ent.ws_bytes,
                                      current_stream_ptr(device))
    if rc == nat.TRINIX_ERR_BAD_ARGUMENT and kept:  # another kind than when the size was asked for (TRINIX_SHARED_KIND)
        ent.ws_bytes = None
        return _run(a, ent, q)
    nat.check(rc, "trinix_shared_prefix_fwd")
    return out if lse is None else (out, lse)
