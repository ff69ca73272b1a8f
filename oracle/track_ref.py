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
