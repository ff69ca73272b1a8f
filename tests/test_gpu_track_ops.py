"""The operators between tracks on the GPU against their 64-bit forms.

Tolerances: one rounding of a value to the result's type is off by at most eps(type) / 2 of it (half of
the smallest subnormal below the normal range); an fp32 sum of m terms in any order by at most
m 2^-24 times the sum of their magnitudes; fp32 factors and products by 2^-24 each.
"""
import pytest
import torch

from oracle import track_ref as ref
from tt_boltz_amd import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U32 = 2.0 ** -24


def half_step(t, want):
    """Half a step of type t around each value."""
    info = torch.finfo(t)
    return (want.abs() * (info.eps / 2)).clamp_min(info.tiny * info.eps / 2)


def check(got, want, slack):
    """|got - want| within one rounding of ``want +- slack`` to got's type."""
    assert got.shape == want.shape
    want = want.cpu()
    tol = slack + half_step(got.dtype, want.abs() + slack)
    err = (got.double().cpu() - want).abs()
    worst = (err - tol).max().item() if err.numel() else 0.0
    assert worst <= 0, f"off by {err.max().item():.3e}, {worst:.3e} over the tolerance"


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def tokens(g, dist, n, V):
    """Indexes of a distribution, some outside the table."""
    if dist == "one":
        t = torch.full((n,), V // 2)
    elif dist == "sorted":
        t = torch.sort(torch.randint(0, V, (n,), generator=g)).values
        t[n - n // 8:] = -1
    elif dist == "few":
        t = torch.randint(0, max(1, V // 10), (n,), generator=g)
    else:
        t = torch.randint(-2, V + 2, (n,), generator=g)
    return t


# ------------------------------------------------------------------------------ lookup
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,C", [(1, 1, 1), (1, 7, 128), (5, 33, 64), (257, 100, 24), (100, 513, 130), (33, 40, 2056),
                                   (1000, 3, 8)])
def test_embedding(gpu, dtype, n, V, C):
    g = torch.Generator().manual_seed(n + V + C)
    w, t = normal(g, V, C, dtype=dtype), tokens(g, "uniform", n, V)
    for scale in (1.0, C ** 0.5):
        got = ops.embedding(t.to(gpu), w.to(gpu), scale)
        want = ref.embedding(t, w, scale)
        check(got, want, 2 * U32 * want.abs() if scale != 1.0 else 0 * want)


def test_embedding_shapes_and_strides(gpu):
    g = torch.Generator().manual_seed(1)
    w = normal(g, 20, 48).to(gpu)
    t = torch.randint(0, 10, (2, 3, 4), generator=g).to(gpu)
    for weight in (w, w[:, :24], w[:, 1:25], w[::2], w[:20, :20].t(), w[3:4].expand(20, 48), w.bfloat16()[:, 8:]):
        for index in (t, t.int(), t.transpose(0, 2), t[..., :0], t[0, 0, 0]):
            assert torch.equal(ops.embedding(index, weight), weight[index.long()])
    assert ops.embedding(t, w[:0]).abs().sum() == 0 and ops.embedding(t, w[:, :0]).shape == (2, 3, 4, 0)
    far = torch.tensor([2 ** 40, -2 ** 40, 2 ** 31, 1, 2 ** 32 + 1], device=gpu)
    got = ops.embedding(far, w)
    assert torch.equal(got[3], w[1]) and not got[:3].any() and not got[4].any()


def test_embedding_offsets_past_32_bits(gpu):
    """A table of more than 2^31 elements, its last rows named."""
    V, C = 70000, 32768
    w = torch.empty((V, C), dtype=torch.bfloat16, device=gpu)
    w[-3:] = torch.arange(3, device=gpu, dtype=torch.bfloat16)[:, None] + 1
    t = torch.tensor([V - 1, V - 3, V - 2], device=gpu)
    assert torch.equal(ops.embedding(t, w)[:, ::100], w[t][:, ::100])
    dw = ops.embedding_grad(torch.ones((3, C), dtype=torch.bfloat16, device=gpu), t, V, 2.0)
    assert (dw[-3:] == 2).all() and not dw[:-3].any()


# ------------------------------------------------------------------------------ its gradient
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,C,dist", [
    (1, 1, 1, "one"), (1, 5, 8, "uniform"), (64, 1, 16, "one"), (65, 3, 16, "one"), (129, 1, 7, "one"), (63, 100, 128, "uniform"),
    (1024, 33, 64, "uniform"), (1025, 33, 65, "few"), (3000, 700, 24, "uniform"), (4097, 200, 132, "sorted"),
    (2500, 600, 16, "few"), (700, 40, 2056, "few"), (5000, 300000, 8, "uniform"), (300, 50, 1100, "one")])
def test_embedding_grad(gpu, dtype, n, V, C, dist):
    g = torch.Generator().manual_seed(n + V + C)
    t, do = tokens(g, dist, n, V), normal(g, n, C, dtype=dtype)
    scale = 1.0 if n % 2 else 3.7
    got = ops.embedding_grad(do.to(gpu), t.to(gpu), V, scale)
    want = ref.embedding_grad(do, t, V, scale)
    size, count = ref.embedding_grad(do.abs(), t, V, scale), ref.embedding_grad(torch.ones((n, 1)), t, V)
    check(got, want, (count + 2) * U32 * size)
    assert got.cpu()[(count == 0)[:, 0]].abs().sum() == 0
    again = ops.embedding_grad(do.to(gpu), t.int().to(gpu), V, scale)
    assert torch.equal(got, again)


@pytest.mark.parametrize("n,V", [(200000, 33), (300000, 1), (262144 + 5, 70000), (140000, 513)])
def test_embedding_grad_long(gpu, n, V):
    """More tokens than the sort's workgroups hold in one tile, in whole numbers: the sums are exact."""
    g = torch.Generator().manual_seed(n)
    t, do = torch.randint(-1, V + 1, (n,), generator=g).to(gpu), torch.randint(-8, 9, (n, 12), generator=g).float().to(gpu)
    want = torch.zeros((V + 2, 12), dtype=torch.float64, device=gpu).index_add_(0, t + 1, do.double())[1:-1]
    assert torch.equal(ops.embedding_grad(do, t, V).double(), want)


def test_embedding_grad_edges(gpu):
    t = torch.zeros((0,), dtype=torch.int64, device=gpu)
    assert torch.equal(ops.embedding_grad(torch.zeros((0, 8), device=gpu), t, 5), torch.zeros((5, 8), device=gpu))
    assert ops.embedding_grad(torch.zeros((0, 8), device=gpu), t, 0).shape == (0, 8)
    assert ops.embedding_grad(torch.ones((3, 8), device=gpu), torch.full((3,), -1, device=gpu), 4).abs().sum() == 0
    wide = torch.randn((6, 16), device=gpu)
    t = torch.tensor([1, 1, 0, 3, 1, 0], device=gpu)
    for do in (wide[:, ::2], wide[:, 1:9], wide[:1].expand(6, 16), wide.t().contiguous().t()):
        assert torch.equal(ops.embedding_grad(do, t, 4), ops.embedding_grad(do.contiguous().clone(), t, 4))


@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_autograd(gpu, dtype):
    g = torch.Generator().manual_seed(5)
    w, t, do = normal(g, 50, 40, dtype=dtype), tokens(g, "uniform", 300, 50).view(3, 100), normal(g, 3, 100, 40, dtype=dtype)
    wd = w.to(gpu).requires_grad_()
    out = ops.embedding(t.to(gpu), wd, 2.0)
    out.backward(do.to(gpu))
    assert torch.equal(wd.grad, ops.embedding_grad(do.to(gpu), t.to(gpu), 50, 2.0))
    with torch.no_grad():
        assert not ops.embedding(t.to(gpu), wd).requires_grad


def test_embedding_grad_by_differences(gpu):
    """<dw, e> against (f(w + e) - f(w - e)) / 2: the lookup is linear, so only fp32 roundings differ."""
    g = torch.Generator().manual_seed(6)
    w, e, do = normal(g, 9, 16), normal(g, 9, 16), normal(g, 40, 16)
    t = tokens(g, "uniform", 40, 9)
    f = lambda x: (ops.embedding(t.to(gpu), x.to(gpu), 1.5).double().cpu() * do.double()).sum()  # noqa: E731
    got = (ops.embedding_grad(do.to(gpu), t.to(gpu), 9, 1.5).double().cpu() * e.double()).sum()
    size = (ref.embedding_grad(do.abs(), t, 9, 1.5) * (w.abs() + e.abs())).sum()
    assert abs((f(w + e) - f(w - e)) / 2 - got) <= 64 * U32 * size


# ------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,shared", [((1,), None), ((3, 5), None), ((2, 100, 16), None), ((4099,), None), ((2, 1, 24), "row"),
                                          ((2, 5, 7, 16), "row"), ((3, 6, 6, 5), "row"), ((2, 5, 7, 16), "column"),
                                          ((9, 4, 3), "column"), ((2, 2, 3, 10, 8), "column")])
def test_dropout_add(gpu, dtype, shape, shared):
    g = torch.Generator().manual_seed(len(shape))
    x, r = normal(g, *shape, dtype=dtype), normal(g, *shape, dtype=dtype)
    for p, seed, offset in ((0.3, 2 ** 63 + 5, 0), (0.0, 1, 1), (1.0, -3, 2 ** 40 + 1), (0.5, 77, 2 ** 64 - 1)):
        keep = ref.dropout_keep(shape, p, seed, offset, shared)
        factor = keep.double() / (1 - p) if p < 1 else keep.double()
        y = x.double() * factor
        got = ops.dropout_add(x.to(gpu), None, p, seed, offset, shared)
        check(got, y, 2 * U32 * y.abs())
        assert torch.equal(got.cpu() != 0, keep & (x != 0))
        got = ops.dropout_add(x.to(gpu), r.to(gpu), p, seed, offset, shared)
        check(got, r.double() + y, 3 * U32 * (y.abs() + r.double().abs()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shared", [None, "row", "column"])
def test_dropout_grad(gpu, dtype, shared):
    g = torch.Generator().manual_seed(2)
    x, r, do = (normal(g, 2, 9, 6, 24, dtype=dtype).to(gpu) for _ in range(3))
    x.requires_grad_(), r.requires_grad_()
    out = ops.dropout_add(x, r, 0.4, 11, 5, shared)
    dx, dr = torch.autograd.grad(out, (x, r), do)
    assert torch.equal(dr, do) and torch.equal(dx, ops.dropout_add(do, None, 0.4, 11, 5, shared))
    out = ops.dropout_add(x, None, 0.4, 11, 5, shared)
    dx2, = torch.autograd.grad(out, x, do.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(dx, dx2)


def test_dropout_strides_alignment_and_empties(gpu):
    x, r = torch.randn((4, 6, 6, 16), device=gpu), torch.randn((4, 6, 6, 16), device=gpu)
    for a, b in ((x.transpose(1, 2), r), (x[..., 1:9], r[..., :8]), (x[:1].expand(4, 6, 6, 16), r), (x[:, ::2], r[:, 1::2])):
        for shared in (None, "row", "column"):
            got = ops.dropout_add(a, b, 0.5, 3, shared=shared)
            assert torch.equal(got, ops.dropout_add(a.contiguous().clone(), b.contiguous().clone(), 0.5, 3, shared=shared))
    flat = torch.randn(1001, device=gpu)
    assert torch.equal(ops.dropout_add(flat[1:], None, 0.5, 9), ops.dropout_add(flat[1:].clone(), None, 0.5, 9))
    assert ops.dropout_add(x[:0], r[:0], 0.5, 1, shared="row").shape == (0, 6, 6, 16)


def test_dropout_nan_in_dropped_places(gpu):
    x = torch.full((1, 8, 8, 16), float("nan"), device=gpu)
    for shared in (None, "row", "column"):
        keep = ref.dropout_keep(x.shape, 0.5, 4, 0, shared).to(gpu)
        got = ops.dropout_add(torch.where(keep, 1.0, x), torch.ones_like(x), 0.5, 4, shared=shared)
        assert torch.equal(got, 1.0 + 2.0 * keep)


def test_dropout_rate(gpu):
    """2^22 draws: the kept share is within six standard deviations of 1 - p."""
    x = torch.ones(1 << 22, device=gpu)
    for p in (0.1, 0.5, 0.9):
        kept = (ops.dropout_add(x, None, p, 123, 4) != 0).double().mean().item()
        assert abs(kept - (1 - p)) <= 6 * (p * (1 - p) / 2 ** 22) ** 0.5
    a, b = (ops.dropout_add(x, None, 0.5, 123, o) != 0 for o in (4, 5))
    assert abs((a == b).double().mean().item() - 0.5) <= 6 * 0.5 / 2 ** 11


def test_dropout_seed_tensor_in_a_graph(gpu):
    """A captured call reads its seed at each replay; the backward pass of an eager call refuses a written one."""
    x, r = torch.randn((64, 64), device=gpu), torch.randn((64, 64), device=gpu)
    seed = torch.tensor([5], device=gpu)
    assert torch.equal(ops.dropout_add(x, r, 0.5, seed, 1), ops.dropout_add(x, r, 0.5, 5, 1))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.dropout_add(x, r, 0.5, seed, 1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.dropout_add(x, r, 0.5, seed, 1)
    for s in (9, -4, 2 ** 62):
        seed.fill_(s)
        graph.replay()
        assert torch.equal(out, ops.dropout_add(x, r, 0.5, s, 1))
        torch.cuda.synchronize()
    leaf = x.clone().requires_grad_()
    y = ops.dropout_add(leaf, r, 0.5, seed, 1)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


# ------------------------------------------------------------------------------ streams and graphs
def test_embedding_step_in_a_graph(gpu):
    """Lookup and gradient captured with the launchers; replays on new tokens, eager work between."""
    g = torch.Generator().manual_seed(8)
    V, C, n = 300, 64, 2000
    w = normal(g, V, C).to(gpu)
    t, do = tokens(g, "few", n, V).to(gpu), normal(g, n, C).to(gpu)
    out, dw = torch.empty((n, C), device=gpu), torch.empty((V, C), device=gpu)
    ws = ops.workspace(ops.embedding_grad_workspace_bytes(n, V, C), gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.launch_embedding(t, w, out, 1.5)
        ops.launch_embedding_grad(t, do, dw, ws, 1.5)
    for dist in ("one", "uniform", "sorted", "few"):
        t.copy_(tokens(g, dist, n, V))
        do.copy_(normal(g, n, C))
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.embedding(t, w, 1.5)) and torch.equal(dw, ops.embedding_grad(do, t, V, 1.5))


def test_two_streams_at_once(gpu):
    g = torch.Generator().manual_seed(9)
    t, do = tokens(g, "few", 20000, 500).to(gpu), normal(g, 20000, 64).to(gpu)
    want = ops.embedding_grad(do, t, 500)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.embedding_grad(do, t, 500))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)
