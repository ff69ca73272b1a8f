"""Plain 64-bit forms of the operators between tracks, from their formulas (CPU or GPU tensors)."""
from __future__ import annotations

import torch

_LOW = 0xFFFFFFFF


def embedding(index: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * weight[index], zeros where an index is outside the table."""
    inside = (index >= 0) & (index < weight.shape[0])
    out = weight.new_zeros((*index.shape, weight.shape[1]), dtype=torch.float64)
    out[inside] = weight.double()[index[inside].long()] * scale
    return out


def embedding_grad(grad: torch.Tensor, index: torch.Tensor, rows: int, scale: float = 1.0) -> torch.Tensor:
    inside = (index >= 0) & (index < rows)
    out = grad.new_zeros((rows, grad.shape[-1]), dtype=torch.float64)
    for t, g in zip(index[inside].long().tolist(), grad[inside].double()):
        out[t] += g
    return out * scale


def philox4x32(counter, key, rounds: int = 10):
    """Philox4x32 (Salmon et al., SC 2011) on four counter words and two key words."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & _LOW, (a >> 32) ^ c[3] ^ k[1], a & _LOW]
        k = [(k[0] + 0x9E3779B9) & _LOW, (k[1] + 0xBB67AE85) & _LOW]
    return c


def dropout_words(n: int, seed: int, offset: int) -> list:
    """Words 0 .. n - 1 of (seed, offset), as whole numbers."""
    words = []
    for i in range((n + 3) // 4):
        words += philox4x32((i & _LOW, i >> 32, offset & _LOW, offset >> 32), (seed & _LOW, (seed >> 32) & _LOW))
    return words[:n]


def dropout_keep(shape, p: float, seed: int, offset: int, shared=None) -> torch.Tensor:
    """Which elements stay, as a mask of ``shape``."""
    shape = tuple(shape)
    if shared == "row":
        small = shape[:-2] + (1, 1)
    elif shared == "column":
        small = shape[:-3] + (1, shape[-2], 1)
    else:
        small = shape
    n = 1
    for s in small:
        n *= s
    t = round(p * 2 ** 32)
    keep = torch.tensor([w >= t for w in dropout_words(n, seed % 2 ** 64, offset)], dtype=torch.bool)
    return keep.view(small).expand(shape)


def cross_attention(q, k, v, bias=None, mask=None, k_lens=None, scale=None, do=None) -> dict:
    """Softmax attention of q [B, Lq, H, D] over k, v [B, Lk, Hk, D] in 64 bits, on the CPU: ``o`` and, with
    ``do``, ``dq``, ``dk``, ``dv``, ``dbias`` [B, H, Lq, Lk]; besides the probabilities ``p``, logits
    ``x`` (0 at hidden keys), ``dp``, ``delta``, ``ds`` [B, H, Lq, Lk] and which keys are ``seen`` [B, Lk]."""
    q, k, v = (t.detach().cpu().double().transpose(1, 2) for t in (q, k, v))
    (B, H, Lq, D), (Hk, Lk) = q.shape, k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    seen = torch.ones((B, Lk), dtype=torch.bool)
    if mask is not None:
        seen &= mask.detach().cpu().expand(B, Lk) != 0
    if k_lens is not None:
        seen &= torch.arange(Lk)[None] < k_lens.cpu()[:, None]
    hide = ~seen[:, None, :, None]
    k, v = (t.masked_fill(hide, 0.0).repeat_interleave(H // Hk, 1) for t in (k, v))
    x = scale * (q @ k.transpose(2, 3))
    if bias is not None:
        x = x + bias.detach().cpu().double().masked_fill(~seen[:, None, None], 0.0)
    hidden = ~seen[:, None, None].expand(B, H, Lq, Lk) | (x == -torch.inf)
    top = x.masked_fill(hidden, -torch.inf).amax(3, keepdim=True) if Lk else x.new_zeros((B, H, Lq, 1))
    e = torch.exp(x - top.masked_fill(top == -torch.inf, 0.0)).masked_fill(hidden, 0.0)
    total = e.sum(3, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    r = {"o": (p @ v).transpose(1, 2), "p": p, "x": x.masked_fill(hidden, 0.0), "seen": seen, "q": q, "k": k, "v": v,
         "scale": scale}
    if do is not None:
        do = do.detach().cpu().double().transpose(1, 2)
        dp = do @ v.transpose(2, 3)
        delta = (p * dp).sum(3, keepdim=True)
        ds = p * (dp - delta)
        r.update(do=do, dp=dp, delta=delta, ds=ds, dbias=ds, dq=(scale * (ds @ k)).transpose(1, 2))
        fold = lambda t: t.view(B, Hk, H // Hk, Lk, D).sum(2).transpose(1, 2)  # noqa: E731
        r.update(dk=fold(scale * (ds.transpose(2, 3) @ q)), dv=fold(p.transpose(2, 3) @ do))
    return r


def cross_attention_slack(r: dict, dtype: torch.dtype, bias=None) -> dict:
    """How far fp32 arithmetic on operands of ``dtype`` may take each result of ``cross_attention`` before
    its own last rounding, from u = 2^-24 per fp32 step and half a step of ``dtype`` per rounded operand."""
    u, half = 2.0 ** -24, (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
    q, k, v, p, scale = (r[n] for n in ("q", "k", "v", "p", "scale"))
    (B, H, Lq, D), Lk = q.shape, k.shape[2]
    ab = abs(scale) * (q.abs() @ k.abs().transpose(2, 3)) + r["x"].abs()
    if bias is not None:
        ab = ab + bias.detach().cpu().double().abs().expand(B, H, Lq, Lk).masked_fill(p == 0, 0.0)
    dx = (D + 8) * u * ab                                   # a logit, with the product, the bias and the exponent's rounding
    dx = dx.masked_fill(p == 0, 0.0)
    rel = 2 * (dx + dx.amax(3, keepdim=True) if Lk else dx) + (Lk + 8) * u      # a probability, relatively
    rel = rel + (Lk + D + 8) * u
    # a small P: half of fp16's smallest subnormal where it is an operand, and an exponential below fp32's
    # normal range (2^-126) is 0
    flush = 2.0 ** -126
    tiny = 2.0 ** -25 if dtype == torch.float16 else flush
    eo = (p * (rel + half) + tiny * (p > 0)) @ v.abs()      # o before its rounding
    s = {"o": eo.transpose(1, 2)}
    if "do" in r:
        do, dp, delta, ds = (r[n] for n in ("do", "dp", "delta", "ds"))
        mag = do.abs() @ v.abs().transpose(2, 3)
        # (with a bias, whose gradient is wanted, o is kept from unrounded P for delta)
        ed = eo if bias is None else (p * (rel + 2.0 ** -22) + tiny * (p > 0)) @ v.abs()
        edelta = (do.abs() * (ed + (D + 4) * u * r["o"].transpose(1, 2).abs())).sum(3, keepdim=True)
        eds = p * ((D + 4) * u * (mag + delta.abs()) + edelta) + (rel + 4 * u) * ds.abs() + flush * (mag + delta.abs())
        s["dbias"] = eds
        bound = 2 * do.norm(dim=3).amax(2)[..., None, None] * v.norm(dim=3).amax(2)[..., None, None] if Lk and Lq else 0.0
        low = bound * H * 2.0 ** -36 if dtype == torch.float16 else 0.0   # a small dS in fp16, heads of one key head scaled alike
        eds = eds + half * (ds.abs() + eds) + low * (p > 0)
        n = (Lk + 4) * u
        s["dq"] = (abs(scale) * (eds + n * ds.abs()) @ k.abs()).transpose(1, 2)
        Hk = r["dk"].shape[2]
        n = (Lq * (H // Hk) + 4) * u
        fold = lambda t: t.view(B, Hk, H // Hk, Lk, D).sum(2).transpose(1, 2)  # noqa: E731
        s["dk"] = fold(abs(scale) * (eds + n * ds.abs()).transpose(2, 3) @ q.abs())
        s["dv"] = fold((p * (rel + half + n) + max(tiny * 2.0 ** -15, flush) * (p > 0)).transpose(2, 3) @ do.abs())
    return s
