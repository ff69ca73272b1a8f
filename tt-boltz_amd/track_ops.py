"""Operators between tracks in the caller's own element type, with their gradients.

``embedding`` (token -> atom broadcasts, residue types, vocabularies) with ``embedding_grad`` (its
transpose: sums by token) and ``dropout_add`` (the pair updates' residual dropout) take fp32, fp16 or
bf16 device tensors and return the same type; sums and statistics are fp32.  They differentiate like
torch's own operators (first derivatives).  The ``launch_*`` functions enqueue the kernels on the
current stream, for programs that write their own backward pass or capture one: they take contiguous
device tensors and allocate nothing.

Under ``torch.cuda.graph`` the same care is due as with torch's operators: ``backward()`` captured
while an eager graph of the same leaves still lives ends the process, whichever operators the graph
holds (the leaves' accumulation belongs to the stream of the eager graph): drop the eager results
first, use ``torch.autograd.grad``, or call the ``launch_*`` functions.
"""
from __future__ import annotations

import contextlib
import ctypes
import operator
from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops

DTYPE_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # PF_FP32 ...
SHARED_CODE = {None: 0, "row": 1, "column": 2}                         # PF_DROP_ELEMENT ...


# --------------------------------------------------------------------------------------
# plumbing
# --------------------------------------------------------------------------------------
def _device(what: str, *ts: Optional[torch.Tensor]) -> torch.device:
    """The one device of the given tensors, RuntimeError where they are on several or not on a GPU."""
    devices = {t.device for t in ts if t is not None}
    if len(devices) > 1:
        raise RuntimeError(f"{what}: tensors on different devices ({', '.join(sorted(map(str, devices)))})")
    return ops._require_gpu(*ts)


def _on(device: torch.device):
    """The device made current for a launch (its current stream is the one used), where it is not."""
    if device.type != "cuda" or device.index == torch._C._cuda_getDevice():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _code(what: str, t: torch.Tensor) -> int:
    code = DTYPE_CODE.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: element type {t.dtype} (fp32, fp16 or bf16 is needed)")
    return code


def _dense(t: torch.Tensor) -> torch.Tensor:
    """Contiguous values of ``t``, without its graph."""
    t = t.detach()
    return (t.resolve_neg() if t.is_neg() else t).contiguous()


def _wants_grad(*ts: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# --------------------------------------------------------------------------------------
# table lookup
# --------------------------------------------------------------------------------------
def launch_embedding(index: torch.Tensor, weight: torch.Tensor, out: torch.Tensor, scale: float = 1.0) -> None:
    """out [n, C] = scale * weight[index] (pf_embedding_fwd); index int32 or int64 [n], weight [V, C]
    with contiguous rows."""
    V, C = weight.shape
    _lib.check(_lib.load().pf_embedding_fwd(ops._ptr(index), int(index.dtype == torch.int64), weight.data_ptr(),
                                            max(weight.stride(0), C) if V > 1 else C, ops._ptr(out), index.numel(), V, C,
                                            DTYPE_CODE[weight.dtype], float(scale), ops._stream()), "pf_embedding_fwd")


def embedding_grad_workspace_bytes(n: int, V: int, C: int) -> int:
    return _lib.load().pf_embedding_grad_workspace_size(n, V, C)


def launch_embedding_grad(index: torch.Tensor, grad: torch.Tensor, dw: torch.Tensor, ws: torch.Tensor,
                          scale: float = 1.0) -> None:
    """dw [V, C] = scale * sums of grad [n, C] by index (pf_embedding_grad)."""
    V, C = dw.shape
    _lib.check(_lib.load().pf_embedding_grad(ops._ptr(index), int(index.dtype == torch.int64), ops._ptr(grad), ops._ptr(dw),
                                             index.numel(), V, C, DTYPE_CODE[dw.dtype], float(scale), ops._ptr(ws),
                                             ws.numel(), ops._stream()), "pf_embedding_grad")


def _index(what: str, index: torch.Tensor) -> torch.Tensor:
    if index.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: index type {index.dtype} (int32 or int64 is needed)")
    return index.contiguous()


def _embedding(index: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    C = weight.shape[1]
    w = weight.detach()
    # rows are read where they are; other strides through a copy
    if w.is_neg() or (C > 1 and w.stride(1) != 1) or (w.shape[0] > 1 and w.stride(0) < C):
        w = _dense(w)
    out = torch.empty((*index.shape, C), dtype=w.dtype, device=w.device)
    with _on(w.device):
        launch_embedding(index, w, out, scale)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, index, weight, scale):
        ctx.save_for_backward(index)
        ctx.rows, ctx.scale = weight.shape[0], scale
        return _embedding(index, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        index, = ctx.saved_tensors
        return None, embedding_grad(grad, index, ctx.rows, ctx.scale), None


def embedding(index: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[index]``: index int32 or int64 of any shape, weight [V, C] fp32, fp16 or bf16;
    [*index.shape, C] in weight's type.  An index outside [0, V), such as the -1 of padding, gives a
    row of zeros and takes no part in the gradient (nothing is raised: that would wait for the GPU).

    Differentiable in ``weight``; see :func:`embedding_grad`.  The lookup in place of a one-hot
    product, as ``MSA`` embeds its alignment (``tt_bio/reference.py:1253-1276``) and the atom
    transformer broadcasts token states."""
    dev = _device("embedding", index, weight)
    if weight.dim() != 2:
        raise ValueError(f"embedding expects weight [V, C], got {tuple(weight.shape)}")
    _code("embedding", weight)
    index = _index("embedding", index)
    if _wants_grad(weight):
        return _Embedding.apply(index, weight, float(scale))
    return _embedding(index, weight, float(scale))


def embedding_grad(grad: torch.Tensor, index: torch.Tensor, num_rows: int, scale: float = 1.0) -> torch.Tensor:
    """The gradient of :func:`embedding` in its table, [num_rows, C] in grad's type: row v is
    ``scale`` times the sum of the rows of ``grad`` [*index.shape, C] whose index is v, zeros where
    there is none.  The sum of atoms by their token is the same operator.

    fp32 sums, rounded once, whose order depends on the indexes alone: equal calls give equal bits."""
    dev = _device("embedding_grad", grad, index)
    if grad.dim() < 1 or grad.shape[:-1] != index.shape:
        raise ValueError(f"embedding_grad expects grad [*index.shape, C], got {tuple(grad.shape)} for index "
                         f"{tuple(index.shape)}")
    _code("embedding_grad", grad)
    num_rows = operator.index(num_rows)
    if num_rows < 0:
        raise ValueError(f"embedding_grad: num_rows is negative ({num_rows})")
    index, grad = _index("embedding_grad", index), _dense(grad)
    C = grad.shape[-1]
    dw = torch.empty((num_rows, C), dtype=grad.dtype, device=dev)
    with _on(dev):
        ws = ops.workspace(embedding_grad_workspace_bytes(index.numel(), num_rows, C), dev)
        launch_embedding_grad(index, grad, dw, ws, scale)
    return dw


# --------------------------------------------------------------------------------------
# residual dropout
# --------------------------------------------------------------------------------------
def launch_dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor], out: torch.Tensor, p: float,
                       seed: Union[int, torch.Tensor], offset: int = 0, shared: Optional[str] = None) -> None:
    """out = residual + dropout(x) (pf_dropout_add_fwd) on contiguous tensors of one shape."""
    if shared is None:
        B, I, J, C = 1, 1, 1, x.numel()
    else:
        I, J, C = x.shape[-3:]
        B = x.numel() // (I * J * C) if x.numel() else 0
    on_device = isinstance(seed, torch.Tensor)
    a = _lib.DropoutArgs(B=B, I=I, J=J, C=C, dtype=DTYPE_CODE[x.dtype], shared=SHARED_CODE[shared], p=p,
                         seed=0 if on_device else seed & 0xFFFFFFFFFFFFFFFF, offset=offset,
                         seed_at=ops._ptr(seed) if on_device else None, x=ops._ptr(x), residual=ops._ptr(residual),
                         out=ops._ptr(out), stream=ops._stream())
    _lib.check(_lib.load().pf_dropout_add_fwd(ctypes.byref(a)), "pf_dropout_add_fwd")


def _dropout_add(x, residual, p, seed, offset, shared):
    x = _dense(x)
    residual = None if residual is None else _dense(residual)
    out = torch.empty_like(x)
    with _on(x.device):
        launch_dropout_add(x, residual, out, p, seed, offset, shared)
    return out


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, shared):
        on_device = isinstance(seed, torch.Tensor)
        if on_device:
            ctx.save_for_backward(seed)   # a seed that is written before the backward pass is an error there
        ctx.args = (p, None if on_device else seed, offset, shared)
        return _dropout_add(x, residual, p, seed, offset, shared)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        p, seed, offset, shared = ctx.args
        if seed is None:
            seed, = ctx.saved_tensors
        dx = _dropout_add(grad, None, p, seed, offset, shared) if ctx.needs_input_grad[0] else None
        return dx, grad if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor], p: float, seed: Union[int, torch.Tensor],
                offset: int = 0, shared: Optional[str] = None) -> torch.Tensor:
    """``residual + dropout(x)``: each element of x is kept with probability 1 - p and divided by it.

    x and residual (or None: no residual) have one shape and type (fp32, fp16 or bf16).  ``shared``:
    None draws for every element; on a pair tensor [..., I, J, C], "row" draws once per row i and
    "column" once per column j of each batch element, as ``get_dropout_mask(columnwise=...)``
    (``tt_bio/boltz2.py:293-304``).

    The mask is a function of (seed, offset) and the position alone, Philox4x32-10 at counter
    (position / 4, offset) under key ``seed``: it is drawn again in the backward pass and never
    stored.  Give every call of a step its own ``offset`` (or seed).  ``seed``: an integer (modulo
    2^64) or an int64 device tensor of one element, read when the kernel runs: a captured graph draws
    new masks when that tensor is written between replays.  Dropped elements are not used, so a NaN
    among them does not spread; p = 1 drops all."""
    dev = _device("dropout_add", x, residual, seed if isinstance(seed, torch.Tensor) else None)
    _code("dropout_add", x)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"dropout_add: residual {tuple(residual.shape)} {residual.dtype} is not like x "
                         f"{tuple(x.shape)} {x.dtype}")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout_add: p must be in [0, 1], got {p}")
    if shared not in SHARED_CODE:
        raise ValueError(f"dropout_add: shared must be None, 'row' or 'column', got {shared!r}")
    if shared is not None and x.dim() < 3:
        raise ValueError(f"dropout_add: a {shared} mask needs x [..., I, J, C], got {tuple(x.shape)}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"dropout_add: a seed tensor holds one int64, got {seed.dtype} {tuple(seed.shape)}")
    else:
        seed = operator.index(seed)
    offset = operator.index(offset)
    if not 0 <= offset < 1 << 64:
        raise ValueError(f"dropout_add: offset must be in [0, 2^64), got {offset}")
    if _wants_grad(x, residual):
        return _DropoutAdd.apply(x, residual, p, seed, offset, shared)
    return _dropout_add(x, residual, p, seed, offset, shared)
