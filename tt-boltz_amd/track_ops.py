"""Operators between tracks in the caller's own element type, with their gradients.

``cross_attention`` (queries of one track over another track's keys and values), ``embedding`` (token ->
atom broadcasts, residue types, vocabularies) with ``embedding_grad`` (its transpose: sums by token) and
``dropout_add`` (the pair updates' residual dropout) take fp32, fp16 or bf16 device tensors and return the
same type; sums and statistics are fp32.  They differentiate like torch's own operators
(``cross_attention`` once).  The ``launch_*`` functions enqueue the kernels on the current stream of the
current device, for programs that write their own backward pass or capture one: they take contiguous
device tensors and allocate nothing.

Under ``torch.cuda.graph`` the same care is due as with torch's operators: ``backward()`` captured
while an eager graph of the same leaves still lives ends the process, whichever operators the graph
holds (the leaves' accumulation belongs to the stream of the eager graph): drop the eager results
first, use ``torch.autograd.grad``, or call the ``launch_*`` functions.
"""
from __future__ import annotations

import ctypes
import operator
from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib

DTYPE_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # PF_FP32 ...
SHARED_CODE = {None: 0, "row": 1, "column": 2}                         # PF_DROP_ELEMENT ...


# --------------------------------------------------------------------------------------
# plumbing
# --------------------------------------------------------------------------------------
def _device(what: str, *ts: Optional[torch.Tensor]) -> torch.device:
    """The one device of the given tensors, RuntimeError where they are on several or not on a GPU."""
    dev = None
    for t in ts:
        if t is not None:
            d = t.device
            if dev is None:
                dev = d
                if d.type != "cuda":
                    ops._require_gpu(t)
            elif d != dev:
                raise RuntimeError(f"{what}: tensors on different devices ({dev}, {d})")
    return dev


def _elsewhere(device: torch.device) -> bool:
    """Whether ``device`` is not the current one: its own current stream is the one to launch on."""
    return device.type == "cuda" and device.index != torch._C._cuda_getDevice()


def _code(what: str, t: torch.Tensor) -> int:
    code = DTYPE_CODE.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: element type {t.dtype} (fp32, fp16 or bf16 is needed)")
    return code


# (the functions below run under autograd.Function or where nothing wants a gradient: no detach)
def _dense(t: torch.Tensor) -> torch.Tensor:
    """Contiguous values of ``t``."""
    return (t.resolve_neg() if t.is_neg() else t).contiguous()


def _wants_grad(*ts: Optional[torch.Tensor]) -> bool:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


# --------------------------------------------------------------------------------------
# cross attention
# --------------------------------------------------------------------------------------
def _strided(t: torch.Tensor) -> torch.Tensor:
    """``t`` [., ., ., D] where the kernels can read it in 16-byte pieces of its last dimension, else a copy."""
    s0, s1, s2, s3 = t.stride()
    unit = 3 if t.dtype == torch.float32 else 7
    if s3 == 1 and not (s0 | s1 | s2) & unit and not t.data_ptr() & 15 and s1 < 1 << 22 and not t.is_neg():
        return t
    if (t.is_neg() or t.data_ptr() & 15 or s3 != 1 or (s1 >= 1 << 22 and t.shape[1] > 1)
            or any(s & unit for n, s in zip(t.shape, (s0, s1, s2)) if n > 1)):
        return t.resolve_neg().clone(memory_format=torch.contiguous_format)
    return t


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = _dense(t)
    return t.clone() if t.data_ptr() & 15 else t


def _strides(t: torch.Tensor) -> tuple:
    """Strides of the leading three dimensions; those of size 1 (any number stands there) as 0."""
    s = t.stride()
    if 1 in t.shape:
        return tuple(0 if n == 1 else x for n, x in zip(t.shape[:3], s))
    return s[:3]


def _cross_args(q, k, v, bias, mask, k_lens, scale, o, o32, stats, whole=0) -> "_lib.CrossAttnArgs":
    (B, Lq, H, D), (_, Lk, Hk, _) = q.shape, k.shape
    if bias is None:
        bias_code, bias_at, bias_strides = 0, None, (0, 0, 0, 0)
    else:
        bias_code, bias_at = DTYPE_CODE[bias.dtype], bias.data_ptr()
        bias_strides = (*_strides(bias), bias.stride(3) if Lk > 1 else 1)
    return _lib.CrossAttnArgs(
        B, Lq, Lk, H, Hk, D, DTYPE_CODE[q.dtype], bias_code, scale, q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k),
        v.data_ptr(), *_strides(v), bias_at, *bias_strides, None if mask is None else mask.data_ptr(),
        0 if mask is None or B == 1 else mask.stride(0), ops._ptr(k_lens), ops._ptr(o), ops._ptr(o32), whole, ops._ptr(stats),
        None, 0, ops._stream())


def _with_workspace(a, size: str, device: torch.device):
    """The call's scratch memory (kept by the caller until the call is enqueued)."""
    nb = getattr(_lib.load(), size)(ctypes.byref(a))
    if nb:
        ws = ops.workspace(nb, device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nb
        return ws
    return None


def launch_cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                           bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                           k_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                           o32: Optional[torch.Tensor] = None, stats: Optional[torch.Tensor] = None,
                           ws: Optional[torch.Tensor] = None, o32_whole: bool = False) -> None:
    """o = cross attention (pf_cross_attn_fwd) of q [B, Lq, H, D] on k, v [B, Lk, Hk, D]; bias
    [B or 1, H or 1, Lq, Lk], mask bool or uint8 [B, Lk], k_lens int32 [B].  ``o32`` fp32 like o (16-bit
    types) and ``stats`` fp32 [2, B, H, Lq] keep what the backward pass needs; ``ws`` of
    ``cross_attention_workspace_bytes``.  ``o32_whole``: o32 from unrounded probabilities, for a bias's gradient."""
    a = _cross_args(q, k, v, bias, mask, k_lens, q.shape[-1] ** -0.5 if scale is None else scale, o, o32, stats,
                    int(o32_whole))
    if ws is not None:
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _lib.check(_lib.load().pf_cross_attn_fwd(ctypes.byref(a)), "pf_cross_attn_fwd")


def cross_attention_workspace_bytes(q: torch.Tensor, k: torch.Tensor) -> int:
    return _lib.load().pf_cross_attn_workspace_size(ctypes.byref(_cross_args(q, k, k, None, None, None, 1.0, None, None, None)))


def cross_attention_bwd_workspace_bytes(q: torch.Tensor, k: torch.Tensor, bias: Optional[torch.Tensor] = None) -> int:
    """``bias``: the bias whose gradient is wanted, or None."""
    a = _cross_args(q, k, k, bias, None, None, 1.0, None, None, None)
    if bias is not None:
        a.dbias_B, a.dbias_H = bias.shape[:2]
    return _lib.load().pf_cross_attn_bwd_workspace_size(ctypes.byref(a))


def _bwd_args(do, q, k, v, o, o32, stats, dq, dk, dv, bias, dbias, mask, k_lens, scale):
    a = _cross_args(q, k, v, bias, mask, k_lens, scale, o, o32, stats)
    a.dout, a.dq, a.dk, a.dv, a.dbias = ops._ptr(do), ops._ptr(dq), ops._ptr(dk), ops._ptr(dv), ops._ptr(dbias)
    if dbias is not None:
        a.dbias_B, a.dbias_H = dbias.shape[:2]
    return a


def launch_cross_attention_bwd(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                               o: torch.Tensor, o32: Optional[torch.Tensor], stats: torch.Tensor,
                               dq: Optional[torch.Tensor], dk: Optional[torch.Tensor], dv: Optional[torch.Tensor],
                               ws: torch.Tensor, bias: Optional[torch.Tensor] = None,
                               dbias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                               k_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> None:
    """The gradients of ``launch_cross_attention`` (pf_cross_attn_bwd) into contiguous dq, dk, dv and
    dbias (of bias's shape and type); dq alone, or dk and dv alone, where the others are None."""
    a = _bwd_args(do, q, k, v, o, o32, stats, dq, dk, dv, bias, dbias, mask, k_lens,
                  q.shape[-1] ** -0.5 if scale is None else scale)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _lib.check(_lib.load().pf_cross_attn_bwd(ctypes.byref(a)), "pf_cross_attn_bwd")


def _cross_fwd(q, k, v, bias, mask, k_lens, scale, keep: bool, whole: bool):
    """(o, o32, stats) on strided tensors; the last two only where a backward pass will read them."""
    dev = q.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _cross_fwd(q, k, v, bias, mask, k_lens, scale, keep, whole)
    shape = q.shape
    o = torch.empty(shape, dtype=q.dtype, device=dev)
    o32 = torch.empty(shape, dtype=torch.float32, device=dev) if keep and q.dtype != torch.float32 else None
    stats = torch.empty((2, shape[0], shape[2], shape[1]), dtype=torch.float32, device=dev) if keep else None
    a = _cross_args(q, k, v, bias, mask, k_lens, scale, o, o32, stats, int(whole))
    ws = _with_workspace(a, "pf_cross_attn_workspace_size", dev)  # noqa: F841
    _lib.check(_lib.load().pf_cross_attn_fwd(ctypes.byref(a)), "pf_cross_attn_fwd")
    return o, o32, stats


def _cross_bwd(do, q, k, v, bias, mask, k_lens, o32, stats, scale, want_q: bool, want_kv: bool, want_b: bool):
    dev = q.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _cross_bwd(do, q, k, v, bias, mask, k_lens, o32, stats, scale, want_q, want_kv, want_b)
    some = q.numel() > 0 and k.numel() > 0   # else nothing is launched, and what has elements is zero
    make = torch.empty if some else torch.zeros
    dq = make(q.shape, dtype=q.dtype, device=dev) if want_q or want_b else None
    dk, dv = (make(k.shape, dtype=q.dtype, device=dev) if want_kv else None for _ in range(2))
    dbias = make(bias.shape, dtype=bias.dtype, device=dev) if want_b else None
    if some:
        do = _aligned(do)   # (held by name until the launch: a pointer keeps nothing alive)
        a = _bwd_args(do, q, k, v, o32, o32, stats, dq, dk, dv, bias, dbias, mask, k_lens, scale)
        ws = _with_workspace(a, "pf_cross_attn_bwd_workspace_size", dev)  # noqa: F841
        _lib.check(_lib.load().pf_cross_attn_bwd(ctypes.byref(a)), "pf_cross_attn_bwd")
    return dq, dk, dv, dbias


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, mask, k_lens, scale):
        q, k, v = _strided(q), _strided(k), _strided(v)
        o, o32, stats = _cross_fwd(q, k, v, bias, mask, k_lens, scale, True, ctx.needs_input_grad[3])
        ctx.save_for_backward(q, k, v, bias, mask, k_lens, o if q.dtype == torch.float32 else o32, stats)
        ctx.scale = scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, bias, mask, k_lens, o32, stats = ctx.saved_tensors
        want_q, want_k, want_v, want_b = ctx.needs_input_grad[:4]
        dq, dk, dv, dbias = _cross_bwd(grad, q, k, v, bias, mask, k_lens, o32, stats, ctx.scale, want_q, want_k or want_v, want_b)
        return dq if want_q else None, dk if want_k else None, dv if want_v else None, dbias, None, None, None


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    mask: Optional[torch.Tensor] = None, k_lens: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one track's queries over another track's keys and values:
    ``softmax_j(scale q_i . k_j + bias_ij) v_j``, as ``AttentionPairBias`` with keys of another length
    (``tt_bio/boltz2.py:343-367``: atom windows, tokens against atoms) or a decoder over an encoder's
    states.  Returns [B, Lq, H, D] in q's type; differentiable in q, k, v and bias.

    q: [B, Lq, H, D]; k, v: [B, Lk, Hk, D], H a multiple of Hk (each key head serves H / Hk query heads in
    a row), all fp32, fp16 or bf16, D a multiple of 8 up to 128; views of any strides are read in place
    where 16-byte pieces allow it (a batch of beams may share states through ``expand``).
    bias: added to the logits, [B or 1, H or 1, Lq, Lk] (leading dimensions may be missing), fp32 or q's
    type; -inf hides a key from a query.  mask: [B, Lk] (or [1, Lk], [Lk]), bool or numbers, keys of 0 are
    hidden; k_lens: int32 or int64 [B], keys from k_lens[b] on are hidden (lengths outside [0, Lk] count as
    the nearer end).  Hidden keys are not used, whatever they hold; a query that sees nothing gives zeros.
    scale: D ** -0.5 by default.

    Softmax statistics and sums are fp32; 16-bit types round P (and in the backward pass dS) to their type
    for the products, fp32 runs on fp32 products throughout."""
    _device("cross_attention", q, k, v, bias, mask, k_lens)
    _code("cross_attention", q)
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"cross_attention expects q [B, Lq, H, D] and k, v [B, Lk, Hk, D], got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D or Hk == 0 or H % Hk:
        raise ValueError(f"cross_attention: k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)} "
                         "([B, Lk, Hk, D], H a multiple of Hk)")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"cross_attention: q, k and v differ in type ({q.dtype}, {k.dtype}, {v.dtype})")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"cross_attention: D must be a multiple of 8 up to 128, got {D}")
    scale = D ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= 3e38:
        raise ValueError(f"cross_attention: scale must be finite, got {scale}")
    if bias is not None:
        if bias.dim() > 4 or bias.dim() < 2:
            raise ValueError(f"cross_attention expects bias [B or 1, H or 1, Lq, Lk], got {tuple(bias.shape)}")
        bias = bias[(None,) * (4 - bias.dim())]
        if bias.shape[0] not in (1, B) or bias.shape[1] not in (1, H) or tuple(bias.shape[2:]) != (Lq, Lk):
            raise ValueError(f"cross_attention: bias {tuple(bias.shape)} does not fit [{B} or 1, {H} or 1, {Lq}, {Lk}]")
        if bias.dtype not in (torch.float32, q.dtype):
            raise ValueError(f"cross_attention: bias is {bias.dtype} (fp32 or {q.dtype} is needed)")
        if bias.is_neg():
            bias = bias.resolve_neg()
    if mask is not None:
        if mask.dtype != torch.bool:
            mask = mask.detach() != 0
        mask = ops.shaped(mask, (B, Lk))
        if Lk > 1 and mask.stride(1) != 1:
            mask = mask.contiguous()
    if k_lens is not None:
        if k_lens.dtype not in (torch.int32, torch.int64) or tuple(k_lens.shape) != (B,):
            raise ValueError(f"cross_attention expects k_lens int32 or int64 [{B}], got {k_lens.dtype} {tuple(k_lens.shape)}")
        if k_lens.dtype == torch.int64:
            k_lens = k_lens.clamp(0, Lk).to(torch.int32)
        k_lens = k_lens.contiguous()
    if _wants_grad(q, k, v, bias):
        return _CrossAttention.apply(q, k, v, bias, mask, k_lens, scale)
    return _cross_fwd(_strided(q), _strided(k), _strided(v), bias, mask, k_lens, scale, False, False)[0]


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


def _embedding(index: torch.Tensor, w: torch.Tensor, scale: float) -> torch.Tensor:
    dev = w.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _embedding(index, w, scale)
    V, C = w.shape
    # rows are read where they are; other strides through a copy
    if w.is_neg() or (C > 1 and w.stride(1) != 1) or (V > 1 and w.stride(0) < C):
        w = _dense(w)
    out = torch.empty((*index.shape, C), dtype=w.dtype, device=dev)
    launch_embedding(index, w, out, scale)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, index, weight, scale):
        ctx.save_for_backward(index)
        ctx.rows, ctx.scale = weight.shape[0], scale
        return _embedding(index, weight, scale)

    @staticmethod
    def backward(ctx, grad):
        index, = ctx.saved_tensors
        again = grad.requires_grad and torch.is_grad_enabled()   # a gradient of this gradient is wanted
        return None, (embedding_grad if again else _embedding_grad)(grad, index, ctx.rows, ctx.scale), None


def embedding(index: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[index]``: index int32 or int64 of any shape, weight [V, C] fp32, fp16 or bf16;
    [*index.shape, C] in weight's type.  An index outside [0, V), such as the -1 of padding, gives a
    row of zeros and takes no part in the gradient (nothing is raised: that would wait for the GPU).

    Differentiable in ``weight``; see :func:`embedding_grad`.  The lookup in place of a one-hot
    product, as ``MSA`` embeds its alignment (``tt_bio/reference.py:1253-1276``) and the atom
    transformer broadcasts token states."""
    _device("embedding", index, weight)
    if weight.dim() != 2:
        raise ValueError(f"embedding expects weight [V, C], got {tuple(weight.shape)}")
    _code("embedding", weight)
    index = _index("embedding", index)
    if _wants_grad(weight):
        return _Embedding.apply(index, weight, float(scale))
    return _embedding(index, weight, float(scale))


def _embedding_grad(grad: torch.Tensor, index: torch.Tensor, num_rows: int, scale: float) -> torch.Tensor:
    dev = grad.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _embedding_grad(grad, index, num_rows, scale)
    grad = _dense(grad)
    C = grad.shape[-1]
    dw = torch.empty((num_rows, C), dtype=grad.dtype, device=dev)
    ws = ops.workspace(embedding_grad_workspace_bytes(index.numel(), num_rows, C), dev)
    launch_embedding_grad(index, grad, dw, ws, scale)
    return dw


class _EmbeddingGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad, index, num_rows, scale):
        ctx.save_for_backward(index)
        ctx.rows, ctx.scale = num_rows, scale
        return _embedding_grad(grad, index, num_rows, scale)

    @staticmethod
    def backward(ctx, dw):
        index, = ctx.saved_tensors   # (an index outside the table took no part)
        return embedding(index, dw, ctx.scale), None, None, None


def embedding_grad(grad: torch.Tensor, index: torch.Tensor, num_rows: int, scale: float = 1.0) -> torch.Tensor:
    """The gradient of :func:`embedding` in its table, [num_rows, C] in grad's type: row v is
    ``scale`` times the sum of the rows of ``grad`` [*index.shape, C] whose index is v, zeros where
    there is none.  The sum of atoms by their token is the same operator.

    fp32 sums, rounded once, whose order depends on the indexes alone: equal calls give equal bits.
    Differentiable in ``grad`` (its gradient is the lookup)."""
    _device("embedding_grad", grad, index)
    if grad.dim() < 1 or grad.shape[:-1] != index.shape:
        raise ValueError(f"embedding_grad expects grad [*index.shape, C], got {tuple(grad.shape)} for index "
                         f"{tuple(index.shape)}")
    _code("embedding_grad", grad)
    num_rows = operator.index(num_rows)
    if num_rows < 0:
        raise ValueError(f"embedding_grad: num_rows is negative ({num_rows})")
    index = _index("embedding_grad", index)
    if _wants_grad(grad):
        return _EmbeddingGrad.apply(grad, index, num_rows, float(scale))
    return _embedding_grad(grad, index, num_rows, float(scale))


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
    if isinstance(seed, torch.Tensor):
        seed, seed_at = 0, seed.data_ptr()
    else:
        seed, seed_at = seed & 0xFFFFFFFFFFFFFFFF, None
    a = _lib.DropoutArgs(B, I, J, C, DTYPE_CODE[x.dtype], SHARED_CODE[shared], p, seed, offset, seed_at, x.data_ptr(),
                         ops._ptr(residual), out.data_ptr(), ops._stream())
    _lib.check(_lib.load().pf_dropout_add_fwd(ctypes.byref(a)), "pf_dropout_add_fwd")


def _dropout_add(x, residual, p, seed, offset, shared):
    dev = x.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _dropout_add(x, residual, p, seed, offset, shared)
    x = _dense(x)
    residual = None if residual is None else _dense(residual)
    out = torch.empty_like(x)
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
    def backward(ctx, grad):
        p, seed, offset, shared = ctx.args
        if seed is None:
            seed, = ctx.saved_tensors
        again = grad.requires_grad and torch.is_grad_enabled()   # a gradient of this gradient is wanted
        dx = (dropout_add if again else _dropout_add)(grad, None, p, seed, offset, shared) if ctx.needs_input_grad[0] else None
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
    _device("dropout_add", x, residual, seed if isinstance(seed, torch.Tensor) else None)
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


from . import ops  # noqa: E402  (which re-exports the names above, whichever of the two is imported first)
