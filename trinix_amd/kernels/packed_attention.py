"""Attention over packed sequences through ``libtrinix_attn.so``.

Sequences of different lengths lie one behind the other in the rows of q, k and
v, without padding between them (semantics: ``trinix_packed_args`` in
``include/trinix_attn.h``).  ``PackedSequences`` holds their boundaries and the
kernels' table of work items, built on the GPU once per batch and used by every
layer's ``packed_attention`` call.  No counterpart in the reference, whose
attention takes sequences of one length
(``trinix/kernels/attention_kernel.py:497-517``).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from .. import _native as nat
from .attention_kernel import _DTYPE_CODE, KERNEL_HEAD_DIMS, TritonAttentionKernel, current_stream_ptr, kernel_head_dim

Boundaries = Union[torch.Tensor, Sequence[int]]


class PackedSequences:
    """The sequences of a packed batch.

    Args:
        cu_seqlens_q: the N + 1 cumulative lengths of the queries, starting
            with 0: sequence s holds rows ``cu[s]`` to ``cu[s + 1] - 1``.  A list
            or a CPU tensor is checked (ValueError).  A GPU tensor (int32 or
            int64) is not read back: boundaries outside ``[0, total]`` or out of
            order are clamped, so that they never lead outside the tensors.
        cu_seqlens_k: the same for keys and values; by default the queries'.
            A sequence of Lk keys and Lq queries: the queries are its last Lq
            positions.
        total_q, total_k: rows of q, and of k and v; by default the last
            boundary, which a GPU tensor does not tell (required there).  Rows
            behind the last sequence are padding: their output is 0 and they
            take no part in any gradient.
        device: of the plan; by default the boundaries' GPU or the current one.

    The plan is built on the stream that is current then.  Calls on another
    stream wait for it, and ``rebuild`` waits for the calls, outside of graph
    captures; inside one the order is the caller's.
    """

    def __init__(self, cu_seqlens_q: Boundaries, cu_seqlens_k: Optional[Boundaries] = None, *,
                 total_q: Optional[int] = None, total_k: Optional[int] = None, device=None):
        if not TritonAttentionKernel.is_available():
            raise RuntimeError("HIP attention kernel not available (build trinix_amd; needs a gfx950 GPU)")
        if device is None:
            device = next((c.device for c in (cu_seqlens_q, cu_seqlens_k)
                           if isinstance(c, torch.Tensor) and c.is_cuda), torch.device("cuda"))
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("PackedSequences requires a GPU device")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if cu_seqlens_k is None and total_k is None:
            total_k = total_q
        self.device = device
        self._source_q, self.total_q = self._boundaries(cu_seqlens_q, total_q, "q")
        if cu_seqlens_k is None:
            self._source_k, self.total_k = self._source_q, self.total_q
            if total_k is not None and total_k != self.total_q:
                raise ValueError("total_k differs from total_q, but there is no cu_seqlens_k")
        else:
            self._source_k, self.total_k = self._boundaries(cu_seqlens_k, total_k, "k")
        if self._source_q.shape != self._source_k.shape:
            raise ValueError(f"cu_seqlens_q and cu_seqlens_k differ in length: {self._source_q.numel()}, "
                             f"{self._source_k.numel()}")
        self.n_seqs = self._source_q.numel() - 1
        n = ctypes.c_int64(0)
        nat.check(nat.load_library().trinix_packed_plan_bytes(self.n_seqs, self.total_q, self.total_k, ctypes.byref(n)),
                  "trinix_packed_plan_bytes")
        self._bytes = n.value
        self._launches: dict = {}  # of calls with these sequences (_Launch)
        self.plan = torch.empty(n.value // 4, dtype=torch.int32, device=device)
        self.generation = 0
        self._stream = self._built = None  # where the plan was built, and when
        self._used: dict = {}  # calls on other streams since then
        self.rebuild()

    def _boundaries(self, cu, total, what) -> Tuple[torch.Tensor, int]:
        if not isinstance(cu, torch.Tensor):
            cu = torch.tensor(list(cu), dtype=torch.int64)
        if cu.dim() != 1 or cu.numel() < 2 or cu.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"cu_seqlens_{what} must be a 1-D int32 or int64 tensor of at least two entries, got "
                             f"{tuple(cu.shape)} {cu.dtype}")
        if cu.is_cuda:
            if cu.device != self.device:
                raise ValueError(f"cu_seqlens_{what} is on {cu.device}, the plan on {self.device}")
            if total is None:
                raise ValueError(f"total_{what} is required with cu_seqlens_{what} on the GPU")
        else:
            last = int(cu[-1])
            total = last if total is None else int(total)
            if int(cu[0]) != 0 or bool((cu[1:] < cu[:-1]).any()) or last > total:
                raise ValueError(f"cu_seqlens_{what} must start with 0, not decrease and end within {total} rows")
            if total >= 1 << 30:
                raise ValueError(f"total_{what} ({total}) must be below 2**30")
            cu = cu.to(device=self.device, dtype=torch.int32)
        if int(total) < 0:
            raise ValueError(f"total_{what} must not be negative, got {total}")
        return cu, int(total)

    def rebuild(self) -> None:
        """Builds the plan from the present contents of the boundary tensors, on
        the current stream: for boundaries that are written anew in place, and
        inside a captured graph."""
        with torch.cuda.device(self.device):
            capturing = torch.cuda.is_current_stream_capturing()
            stream = torch.cuda.current_stream(self.device)
            if not capturing:
                if self._built is not None and self._stream != stream:
                    stream.wait_stream(self._stream)
                for ev in self._used.values():
                    stream.wait_event(ev)
            cq = self._source_q.to(torch.int32).contiguous()
            ck = cq if self._source_k is self._source_q else self._source_k.to(torch.int32).contiguous()
            nat.check(nat.load_library().trinix_packed_plan(
                cq.data_ptr(), ck.data_ptr(), self.n_seqs, self.total_q, self.total_k, self.plan.data_ptr(), self._bytes,
                current_stream_ptr(self.device)), "trinix_packed_plan")
            self._used.clear()
            self._stream, self._stream_ptr = stream, current_stream_ptr(self.device)
            self._built = None if capturing else stream.record_event()
        self.generation += 1

    def _enter(self, ptr: int) -> None:
        """A call on another stream than the plan's: waits for the plan, and keeps its memory."""
        stream = torch.cuda.current_stream(self.device)
        if self._built is not None:
            stream.wait_event(self._built)
        if ptr not in self._used:
            self._used[ptr] = torch.cuda.Event()
            self.plan.record_stream(stream)

    def _leave(self, ptr: int) -> None:
        self._used[ptr].record(torch.cuda.current_stream(self.device))


def _strides(t: torch.Tensor):
    """Element strides of a (rows, heads, head_dim) tensor; of a dimension of one
    element, which torch leaves open, the contiguous one."""
    s, h, d = t.stride()
    if t.shape[1] <= 1:
        h = t.shape[2]
    if t.shape[0] <= 1:
        s = t.shape[1] * t.shape[2]
    return s, h, d


def _ready(t: torch.Tensor) -> bool:
    s, h, d = _strides(t)
    if d != 1 and t.shape[2] > 1:
        return False
    return t.element_size() == 4 or (t.data_ptr() % 16 == 0 and s % 8 == 0 and h % 8 == 0 and s < 1 << 22)


def _columns(t: torch.Tensor) -> int:
    """Columns that the kernels take t at: its head_dim rounded up to 16 bytes."""
    per = 16 // t.element_size()
    return -(-t.shape[-1] // per) * per


def _operand(t: torch.Tensor, d: int) -> torch.Tensor:
    if t.shape[-1] != d:
        t = torch.nn.functional.pad(t, (0, d - t.shape[-1]))
    if not _ready(t):
        t = t.contiguous()
        if not _ready(t):
            t = t.clone(memory_format=torch.contiguous_format)
    return t


def _check(q, k, v, seqs: PackedSequences, alibi_slopes) -> None:
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise ValueError("packed_attention requires GPU tensors")
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"Expected 3D tensors (rows, heads, head_dim), got q: {tuple(q.shape)}, k: {tuple(k.shape)}, "
                         f"v: {tuple(v.shape)}")
    if q.dtype not in _DTYPE_CODE:
        raise ValueError(f"Unsupported dtype {q.dtype}; use float32, float16 or bfloat16")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k, v dtypes differ: {q.dtype}, {k.dtype}, {v.dtype}")
    if not (q.device == k.device == v.device == seqs.device):
        raise ValueError(f"q, k, v and the sequences are on different devices: {q.device}, {k.device}, {v.device}, "
                         f"{seqs.device}")
    Tq, H, D = q.shape
    Tk, Hkv, _ = k.shape
    if k.shape != v.shape or k.shape[2] != D or D == 0:
        raise ValueError(f"k/v shapes {tuple(k.shape)}, {tuple(v.shape)} don't match q {tuple(q.shape)}")
    if Tq != seqs.total_q or Tk != seqs.total_k:
        raise ValueError(f"q and k have {Tq} and {Tk} rows, the packed sequences {seqs.total_q} and {seqs.total_k}")
    if Hkv <= 0 or H <= 0 or H % Hkv != 0:
        raise ValueError(f"num_heads ({H}) must be a multiple of the KV heads ({Hkv})")
    if kernel_head_dim(D) is None:
        raise ValueError(f"head_dim {D} > {KERNEL_HEAD_DIMS[-1]} is not supported")
    if alibi_slopes is not None and tuple(alibi_slopes.shape) not in ((H,), (1, H)):
        raise ValueError(f"alibi_slopes shape {tuple(alibi_slopes.shape)} must be (H,) or (1, H)")


# Launch cache (see attention_kernel.py), kept with the sequences: a call whose
# operands the kernels read in place is described, apart from its pointers, by
# shapes, strides, types and scalars.  The first one goes through every check and
# leaves its arguments; the first backward leaves its own, per strides of dout.
class _Launch:
    __slots__ = ("fwd", "bwd", "slopes_as_given", "ws_bytes")

    def __init__(self, fwd, slopes_as_given, ws_bytes):
        self.fwd, self.bwd, self.slopes_as_given, self.ws_bytes = fwd, {}, slopes_as_given, ws_bytes


def _fwd_workspace(a) -> int:
    n = ctypes.c_int64(0)
    nat.check(nat.load_library().trinix_packed_fwd_workspace(ctypes.byref(a), ctypes.byref(n)), "trinix_packed_fwd_workspace")
    return n.value


_MAX_LAUNCHES = 64


def _launch(fn: str, a: nat.PackedArgs, seqs: PackedSequences) -> None:
    device = seqs.device
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _launch(fn, a, seqs)
    stream = current_stream_ptr(device)
    other = stream != seqs._stream_ptr and not torch.cuda.is_current_stream_capturing()
    if other:
        seqs._enter(stream)
    nat.check(getattr(nat.load_library(), fn)(ctypes.byref(a), stream), fn)
    if other:
        seqs._leave(stream)


def _run(a, ent, q, seqs, slopes, want_lse, keep):
    """Allocates the outputs of a forward (arguments a, operands set) and launches
    it: (out at the kernel's head_dim, out_lo, lse)."""
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    a.out = out.data_ptr()
    out_lo = lse = None
    if keep and q.dtype != torch.float32:
        out_lo = torch.empty_like(out)
        a.out_lo = out_lo.data_ptr()
    if want_lse or keep:
        lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device)
        a.lse = lse.data_ptr()
    if slopes is not None:
        a.alibi_slopes = slopes.data_ptr()
    n = _fwd_workspace(a) if ent is None else ent.ws_bytes
    if n:
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), n
    _launch("trinix_packed_fwd", a, seqs)
    return out, out_lo, lse


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, ent, a, seqs, slopes, return_lse):
        D, d_kernel = q.shape[-1], int(a.head_dim)
        if ent is None:
            q, k, v = _set_operands(a, q, k, v, d_kernel)
        out, out_lo, lse = _run(a, ent, q, seqs, slopes, True, True)
        ctx.save_for_backward(q, k, v, out, out_lo, lse, slopes)
        ctx.call = (ent, a, seqs, seqs.generation, D)
        res = out if d_kernel == D else out[..., :D].contiguous()
        if return_lse:
            ctx.mark_non_differentiable(lse)
            return res, lse
        return res

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, *unused):
        q, k, v, out, out_lo, lse, slopes = ctx.saved_tensors
        ent, fwd, seqs, generation, D = ctx.call
        if seqs.generation != generation:
            raise RuntimeError("the packed sequences were rebuilt between the forward and its backward")
        dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
        delta = torch.empty_like(lse)
        tpl = None
        if ent is not None and dout.dtype == q.dtype and not dout.data_ptr() % 16:
            tpl = ent.bwd.get(dout.stride())
        if tpl is not None:
            a, do = nat.PackedArgs.from_buffer_copy(tpl), dout
        else:
            a, do = nat.PackedArgs.from_buffer_copy(fwd), _operand(dout.to(q.dtype), q.shape[-1])
            for name, t in (("out", out), ("dout", do), ("dq", dq), ("dk", dk), ("dv", dv)):
                setattr(a, name + "_stride", nat.Int64x3(*_strides(t)))
            if ent is not None and do is dout and len(ent.bwd) < _MAX_LAUNCHES:
                ent.bwd[dout.stride()] = nat.PackedArgs.from_buffer_copy(a)
        a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
        a.out, a.dout, a.lse, a.delta = out.data_ptr(), do.data_ptr(), lse.data_ptr(), delta.data_ptr()
        a.out_lo = None if out_lo is None else out_lo.data_ptr()
        a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        if slopes is not None:
            a.alibi_slopes = slopes.data_ptr()
        a.workspace, a.workspace_bytes = None, 0  # (fwd may hold the forward's)
        n = ctypes.c_int64(0)
        nat.check(nat.load_library().trinix_packed_bwd_workspace(ctypes.byref(a), ctypes.byref(n)),
                  "trinix_packed_bwd_workspace")
        if n.value:
            ws = torch.empty(n.value, dtype=torch.uint8, device=q.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), n.value
        _launch("trinix_packed_bwd", a, seqs)
        if q.shape[-1] != D:
            dq, dk, dv = dq[..., :D], dk[..., :D], dv[..., :D]
        return dq, dk, dv, None, None, None, None, None


def _set_operands(a, q, k, v, d_kernel):
    """The operands as the kernels read them, entered into a."""
    q, k, v = (_operand(t, d_kernel) for t in (q, k, v))
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_stride, a.k_stride, a.v_stride = (nat.Int64x3(*_strides(t)) for t in (q, k, v))
    H = q.shape[1]
    a.out_stride = nat.Int64x3(H * d_kernel, d_kernel, 1)
    return q, k, v


def _args(q, k, seqs, scale, causal, window_size, slopes, d_kernel) -> nat.PackedArgs:
    a = nat.PackedArgs()
    a.plan, a.plan_bytes = seqs.plan.data_ptr(), seqs._bytes
    a.n_seqs, a.total_q, a.total_k = seqs.n_seqs, seqs.total_q, seqs.total_k
    a.nheads_q, a.nheads_kv, a.head_dim = q.shape[1], k.shape[1], d_kernel
    a.dtype = _DTYPE_CODE[q.dtype]
    a.softmax_scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    a.causal = 1 if causal else 0
    if window_size is not None:
        a.has_window = 1
        a.window_left, a.window_right = (min(max(w, -1 << 62), 1 << 62) for w in window_size)
    if slopes is not None:
        a.alibi_stride = 1
    return a


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, sequences: PackedSequences,
                     scale: Optional[float] = None, causal: bool = False,
                     window_size: Optional[Tuple[int, int]] = None, alibi_slopes: Optional[torch.Tensor] = None,
                     return_lse: bool = False):
    """``packed_attn_func`` (``layers/attention/functional.py``), with gradients
    when q, k or v require them."""
    if not isinstance(sequences, PackedSequences):
        raise ValueError(f"sequences must be PackedSequences, got {type(sequences)}")
    if window_size is not None:
        window_size = (int(window_size[0]), int(window_size[1]))
    if scale is not None:
        scale = float(scale)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if alibi_slopes is not None and alibi_slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError("alibi_slopes are constants without a gradient; pass alibi_slopes.detach()")
    key = (q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), q.dtype, k.dtype, v.dtype, q.device, k.device,
           v.device, scale, bool(causal), window_size,
           None if alibi_slopes is None else (alibi_slopes.shape, alibi_slopes.dtype, alibi_slopes.stride(), alibi_slopes.device))
    ent = sequences._launches.get(key)
    if ent is not None and (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        ent = None
    if ent is None:
        _check(q, k, v, sequences, alibi_slopes)
    slopes = alibi_slopes
    if slopes is not None and (ent is None or not ent.slopes_as_given):
        slopes = alibi_slopes.detach().reshape(-1).to(device=q.device, dtype=torch.float32).contiguous()
    elif slopes is not None:
        slopes = slopes.detach()
    if ent is not None:
        a = nat.PackedArgs.from_buffer_copy(ent.fwd)
        a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    else:
        d_kernel = _columns(q)
        a = _args(q, k, sequences, scale, causal, window_size, slopes, d_kernel)
        if d_kernel == q.shape[-1] and _ready(q) and _ready(k) and _ready(v):
            _set_operands(a, q, k, v, d_kernel)
            as_given = alibi_slopes is not None and (alibi_slopes.dim() == 1 and alibi_slopes.dtype == torch.float32
                                                     and alibi_slopes.device == q.device and alibi_slopes.is_contiguous())
            ent = _Launch(nat.PackedArgs.from_buffer_copy(a), as_given, _fwd_workspace(a))
            ent.fwd.q = ent.fwd.k = ent.fwd.v = None
            if not (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
                if len(sequences._launches) >= _MAX_LAUNCHES:
                    sequences._launches.clear()
                sequences._launches[key] = ent
    if grad:
        return _PackedAttention.apply(q, k, v, ent, a, sequences, slopes, return_lse)
    D = q.shape[-1]
    ops = (q, k, v) if ent is not None else _set_operands(a, q, k, v, int(a.head_dim))  # held until the launch returns
    out, _, lse = _run(a, ent, ops[0], sequences, slopes, return_lse, False)
    if out.shape[-1] != D:
        out = out[..., :D].contiguous()
    return (out, lse) if return_lse else out
