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
@pytest.mark.parametrize("n,V,C", [(300, 50, 12), (70, 9, 1100), (1, 1, 1), (1, 7, 128), (5, 33, 64), (257, 100, 24), (100, 513, 130), (33, 40, 2056),
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
    (2000, 300, 12, "uniform"), (900, 7, 1100, "uniform"), (1, 1, 1, "one"), (1, 5, 8, "uniform"), (64, 1, 16, "one"), (65, 3, 16, "one"), (129, 1, 7, "one"), (63, 100, 128, "uniform"),
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


@pytest.mark.parametrize("C", [8, 132])
def test_embedding_grad_padding_from_any_place(gpu, C):
    """The last token of the table ends anywhere in a chunk, padding follows for chunks; every row is written."""
    pad = torch.full((600,), -1, device=gpu)
    for n in range(0, 140):
        t = torch.cat([torch.arange(n, device=gpu) // 3, pad])
        do, dw = torch.ones((n + 600, C), device=gpu), torch.full((50, C), torch.nan, device=gpu)
        ws = torch.empty(ops.embedding_grad_workspace_bytes(t.numel(), 50, C), dtype=torch.uint8, device=gpu)
        ops.launch_embedding_grad(t, do, dw, ws)
        assert torch.equal(dw, torch.bincount(t[:n], minlength=50).float()[:, None].expand(50, C)), n


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
    # the sum by token is a lookup's transpose, and the other way round
    dod, dw = do.to(gpu).requires_grad_(), normal(g, 50, 40, dtype=dtype).to(gpu)
    got, = torch.autograd.grad(ops.embedding_grad(dod, t.to(gpu), 50, 2.0), dod, dw)
    assert torch.equal(got, ops.embedding(t.to(gpu), dw, 2.0))
    first, = torch.autograd.grad(ops.embedding(t.to(gpu), wd, 2.0), wd, dod, create_graph=True)
    assert torch.equal(torch.autograd.grad(first, dod, dw)[0], got)


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
                                          ((8,), None), ((7,), None), ((2047, 5), None), ((8193,), None), ((3, 1367), None),
                                          ((2, 5, 7, 12), "row"), ((2, 6, 5, 12), "column"), ((1, 9, 301, 132), "column"),
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


# ------------------------------------------------------------------------------ cross attention
def inputs(seed, dtype, B, Lq, Lk, H, Hk, D, bias=None, hide=None, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    c = {"q": normal(g, B, Lq, H, D, dtype=dtype, scale=scale), "k": normal(g, B, Lk, Hk, D, dtype=dtype),
         "v": normal(g, B, Lk, Hk, D, dtype=dtype), "bias": None, "mask": None, "k_lens": None}
    do = normal(g, B, Lq, H, D, dtype=dtype)
    if bias:
        bdt = dtype if "own" in bias else torch.float32
        c["bias"] = normal(g, 1 if "b1" in bias else B, 1 if "h1" in bias else H, Lq, Lk, dtype=bdt)
    if hide in ("mask", "both"):
        c["mask"] = torch.rand((B, Lk), generator=g) < 0.7
    if hide in ("lens", "both"):
        c["k_lens"] = torch.randint(0, Lk + 1, (B,), generator=g, dtype=torch.int32)
        c["k_lens"][0] = Lk
    return c, do


def to(c, dev):
    return {n: None if t is None else t.to(dev) for n, t in c.items()}


def run_cross(c, do, gpu, scale=None, names=("q", "k", "v", "bias")):
    d = to(c, gpu)
    leaves = [d[n].requires_grad_() for n in names if d[n] is not None]
    o = ops.cross_attention(**d, scale=scale)
    return o, dict(zip(["d" + n for n in names if d[n] is not None], torch.autograd.grad(o, leaves, do.to(gpu))))


def check_cross(c, do, gpu, scale=None):
    dtype = c["q"].dtype
    r = ref.cross_attention(**c, scale=scale, do=do)
    slack = ref.cross_attention_slack(r, dtype, c["bias"])
    plain = ops.cross_attention(**to(c, gpu), scale=scale)
    o, grads = run_cross(c, do, gpu, scale)
    if c["bias"] is None or dtype == torch.float32:   # (else a bias that wants its gradient keeps P unrounded)
        assert torch.equal(plain, o.detach())
    check(plain, r["o"], slack["o"])
    check(o.detach(), r["o"], slack["o"])
    for n, got in grads.items():
        want, s = r[n], slack[n]
        if n == "dbias":
            for d in (0, 1):
                if c["bias"].shape[d] == 1 and want.shape[d] != 1:
                    m = want.shape[d]
                    s = s.sum(d, keepdim=True) + m * U32 * want.abs().sum(d, keepdim=True)
                    want = want.sum(d, keepdim=True)
        check(got, want, s)
    return o, grads


CROSS = [  # B, Lq, Lk, H, Hk, D
    (1, 1, 1, 1, 1, 8), (2, 1, 33, 4, 4, 24), (3, 1, 300, 8, 2, 64), (2, 32, 128, 4, 4, 32), (1, 33, 127, 4, 4, 32),
    (2, 5, 129, 6, 2, 128), (1, 130, 64, 2, 2, 48), (2, 70, 200, 4, 1, 40), (1, 257, 65, 2, 1, 96), (1, 3, 1030, 2, 2, 16),
    (1, 129, 515, 1, 1, 128), (1, 40, 700, 3, 3, 56)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias,hide", [(None, None), ("full", "mask"), ("b1 own", "lens"), ("h1", "both")])
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", CROSS)
def test_cross_attention(gpu, B, Lq, Lk, H, Hk, D, bias, hide, dtype):
    c, do = inputs(Lq + Lk + D, dtype, B, Lq, Lk, H, Hk, D, bias, hide)
    check_cross(c, do, gpu)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias,hide", [(None, "both"), ("full", "lens")])
@pytest.mark.parametrize("Lq,Lk,H,Hk,D", [(1, 2300, 2, 1, 8), (2, 5000, 2, 2, 24), (1, 9000, 1, 1, 128), (40, 4200, 2, 2, 64), (35, 8200, 1, 1, 104)])
def test_cross_attention_joins_of_many_parts(gpu, Lq, Lk, H, Hk, D, bias, hide, dtype):
    """Few queries over long keys, and a batch element whose later parts see nothing."""
    c, do = inputs(Lk + D, dtype, 2, Lq, Lk, H, Hk, D, bias, hide)
    c["k_lens"][1] = 150
    check_cross(c, do, gpu)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
def test_cross_attention_scales(gpu, dtype, scale):
    c, do = inputs(3, dtype, 2, 40, 90, 2, 2, 32, "full", "mask")
    o, grads = check_cross(c, do, gpu, scale)
    if scale == 0.0:
        assert not grads["dq"].any() and not grads["dk"].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Lq", [1, 40])
def test_cross_attention_peaked(gpu, dtype, Lq):
    """Logits of some hundreds: nearly all weight on one key, and most probabilities 0."""
    c, do = inputs(4, dtype, 2, Lq, 150, 2, 2, 64, "full", "lens", scale=40.0)
    c["bias"] *= 30
    check_cross(c, do, gpu)


@pytest.mark.parametrize("factor", [2.0 ** -12, 2.0 ** 6])
def test_cross_attention_fp16_gradients_of_any_size(gpu, factor):
    """Small and large output gradients: dS lies outside fp16's range, its sums do not."""
    c, do = inputs(5, torch.float16, 1, 70, 600, 4, 2, 32)
    check_cross(c, (do.float() * factor).half(), gpu)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Lq,Lk,D", [(1, 130, 64), (50, 130, 32), (150, 70, 128)])
@pytest.mark.parametrize("bias", [None, "full"])
def test_cross_attention_rows_that_see_nothing(gpu, dtype, Lq, Lk, D, bias):
    """Batch element 0: every key masked; 1: length 0; 2: all but one key hidden; with a bias, element 3's
    queries hide all keys from themselves every third row."""
    c, do = inputs(6, dtype, 4, Lq, Lk, 2, 2, D, bias, "both")
    c["mask"][:], c["k_lens"][:] = True, Lk
    c["mask"][0], c["k_lens"][1], c["mask"][2] = False, 0, False
    c["mask"][2, Lk // 2] = True
    if bias:
        c["bias"][3, :, ::3] = -torch.inf
        c["bias"][3, :, 1::3, ::2] = -torch.inf
    o, grads = check_cross(c, do, gpu)
    for t in (o, grads["dq"], grads["dk"], grads["dv"]):
        assert not t[:2].any()
    assert torch.equal(o[2].cpu(), c["v"][2, Lk // 2].expand(Lq, 2, D))
    if bias:
        assert not grads["dbias"][:2].any() and not o[3, ::3].any() and not grads["dq"][3, ::3].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf"), None])
@pytest.mark.parametrize("Lq", [1, 60])
def test_cross_attention_ignores_what_is_hidden(gpu, dtype, junk, Lq):
    """NaN, infinities and the lowest value in hidden keys, values and biases change no bit."""
    c, do = inputs(7, dtype, 2, Lq, 140, 4, 2, 32, "full", "both")
    c["k_lens"][1] = 77
    hidden = ~ref.cross_attention(**c)["seen"]
    clean, grads = run_cross(c, do, gpu)
    bad = torch.finfo(dtype).min if junk is None else junk
    for n in "kv":
        c[n][hidden] = bad
    c["bias"] = torch.where(hidden[:, None, None], torch.full((), torch.finfo(torch.float32).min if junk is None else junk), c["bias"])
    o, dirty = run_cross(c, do, gpu)
    assert torch.equal(o, clean) and all(torch.equal(grads[n], dirty[n]) for n in grads)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_attention_lowest_value_as_a_mask(gpu, dtype):
    """A bias of fp32's lowest value hides a key as long as another is there; a row of nothing else sees all its
    keys alike, as fp32 softmax does (the logits vanish next to it)."""
    c, do = inputs(8, dtype, 1, 40, 100, 2, 2, 32, "full")
    low = torch.finfo(torch.float32).min
    c["bias"][:, :, :20, 50:] = low
    c["bias"][:, :, 20:] = low
    o, grads = run_cross(c, do, gpu)
    first = {**c, "q": c["q"][:, :20], "k": c["k"][:, :50], "v": c["v"][:, :50], "bias": c["bias"][:, :, :20, :50]}
    r = ref.cross_attention(**first)
    check(o[:, :20].detach(), r["o"], ref.cross_attention_slack(r, dtype, first["bias"])["o"])
    rest = {**c, "q": c["q"][:, 20:], "bias": None}
    r = ref.cross_attention(**rest, scale=0.0, do=do[:, 20:])
    slack = ref.cross_attention_slack(r, dtype)
    check(o[:, 20:].detach(), r["o"], slack["o"])
    check(grads["dbias"][:, :, 20:], r["dbias"], slack["dbias"])   # P is 1 / 100 there, not 1
    assert torch.isfinite(grads["dq"]).all() and grads["dv"].abs().max() < 100


def test_cross_attention_visible_nan_spreads(gpu):
    c, _ = inputs(9, torch.float32, 2, 5, 200, 2, 2, 32)
    c["q"][0, 1, 0, 3] = float("nan")
    c["k"][1, 150, 1, 3] = float("nan")
    bad = ops.cross_attention(**to(c, gpu)).isnan().all(3).cpu()
    want = torch.zeros((2, 5, 2), dtype=torch.bool)
    want[0, 1, 0] = True
    want[1, :, 1] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_attention_strides(gpu, dtype):
    """Views of a fused projection, permuted heads, shared batches, biases in [B, Lq, Lk, H], offset bases."""
    c, do = inputs(10, dtype, 2, 37, 100, 4, 4, 32, "full", "mask")
    d = to(c, gpu)
    do = do.to(gpu)

    def run(x):
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "bias")]
        o = ops.cross_attention(*leaves[:3], bias=leaves[3], mask=x["mask"])
        return [o, *torch.autograd.grad(o, leaves, do)]
    want = run(d)
    kv = torch.cat([d["k"], d["v"]], 3)                       # [B, Lk, H, 2 D]
    views = [{**d, "k": kv[..., :32], "v": kv[..., 32:]},
             {**d, "q": d["q"].transpose(1, 2).contiguous().transpose(1, 2)},
             {**d, "k": d["k"].permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3)},
             {**d, "v": d["v"].transpose(2, 3).contiguous().transpose(2, 3)},
             {**d, "q": torch.cat([d["q"].flatten()[:1], d["q"].flatten()])[1:].view(d["q"].shape)},
             {**d, "bias": d["bias"].permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)},
             {**d, "bias": torch.cat([d["bias"].flatten()[:1], d["bias"].flatten()])[1:].view(d["bias"].shape)},
             {**d, "mask": d["mask"].t().contiguous().t()}, {**d, "mask": d["mask"].float() * 3}]
    for x in views:
        assert all(torch.equal(a, b) for a, b in zip(run(x), want))
    one = {**d, "k": d["k"][:1].expand(2, -1, -1, -1), "v": d["v"][:1].expand(2, -1, -1, -1), "mask": d["mask"][:1]}
    two = {**d, "k": d["k"][:1].repeat(2, 1, 1, 1), "v": d["v"][:1].repeat(2, 1, 1, 1), "mask": d["mask"][:1].repeat(2, 1)}
    assert all(torch.equal(a, b) for a, b in zip(run(one), run(two)))
    grad = do.transpose(1, 2).contiguous().transpose(1, 2)
    q = d["q"].detach().requires_grad_()
    o = ops.cross_attention(q, d["k"], d["v"], d["bias"], d["mask"])
    assert torch.equal(*(torch.autograd.grad(o, q, g, retain_graph=True)[0] for g in (grad, do)))


@pytest.mark.parametrize("names", [("q",), ("k",), ("v",), ("bias",), ("k", "bias"), ("q", "v")])
def test_cross_attention_partial_gradients(gpu, names):
    c, do = inputs(11, torch.bfloat16, 2, 37, 100, 4, 2, 32, "b1", "mask")
    # (o is kept from unrounded P where the bias has a gradient)
    _, every = run_cross(c, do, gpu, names=("q", "k", "v", "bias")[:4 if "bias" in names else 3])
    _, some = run_cross(c, do, gpu, names=names)
    assert set(some) == {"d" + n for n in names} and all(torch.equal(some[n], every[n]) for n in some)


def test_cross_attention_empties(gpu):
    for B, Lq, Lk, H in ((2, 3, 0, 2), (2, 0, 5, 2), (0, 3, 5, 2), (1, 40, 0, 2)):
        q, k = torch.ones((B, Lq, H, 16), device=gpu), torch.ones((B, Lk, H, 16), device=gpu)
        bias = torch.ones((B, H, Lq, Lk), device=gpu)
        leaves = [t.requires_grad_() for t in (q, k, k.detach().clone(), bias)]
        o = ops.cross_attention(*leaves[:3], bias=bias)
        assert o.shape == q.shape and not o.any()
        for g, t in zip(torch.autograd.grad(o, leaves, torch.ones_like(o)), leaves):
            assert g.shape == t.shape and not g.any()


def test_cross_attention_lengths_are_clamped(gpu):
    c, _ = inputs(12, torch.float16, 4, 5, 60, 2, 2, 32)
    d = to(c, gpu)
    lens = torch.tensor([-7, 0, 60, 10 ** 6], device=gpu)
    got = ops.cross_attention(d["q"], d["k"], d["v"], k_lens=lens)
    assert not got[:2].any() and torch.equal(got[2:], ops.cross_attention(d["q"], d["k"], d["v"])[2:])
    assert torch.equal(got, ops.cross_attention(d["q"], d["k"], d["v"], k_lens=lens.int()))
    far = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32 + 1, 3], device=gpu)
    got = ops.cross_attention(d["q"], d["k"], d["v"], k_lens=far)
    assert not got[1].any() and torch.equal(got[::2], ops.cross_attention(d["q"], d["k"], d["v"])[::2])


def test_cross_attention_offsets_past_32_bits(gpu):
    """Batch elements and heads 2^31 elements apart."""
    buf = torch.empty(2 ** 32 + 2 ** 21, dtype=torch.float16, device=gpu)
    k = buf.as_strided((2, 70, 2, 32), (2 ** 31, 64, 32, 1))
    v = buf.as_strided((2, 70, 2, 32), (2 ** 20, 64, 2 ** 32, 1), 8192)
    far = buf.as_strided((2, 2040, 2, 32), (32, 2 ** 21, 64, 1))   # rows 2^21 elements apart
    far.copy_(torch.randn(far.shape, device=gpu))
    q = far[:, -40:]
    near = far.contiguous()
    p = ops.cross_attention(q.detach().contiguous().requires_grad_(), near.requires_grad_(), near)
    o = ops.cross_attention(q.detach().requires_grad_(), far.requires_grad_(), far)
    assert torch.equal(o, p)
    assert torch.equal(torch.autograd.grad(o, far, torch.ones_like(o))[0], torch.autograd.grad(p, near, torch.ones_like(p))[0])
    k.copy_(torch.randn(k.shape, device=gpu)), v.copy_(torch.randn(v.shape, device=gpu))
    for Lq in (1, 50):
        q, do = torch.randn((2, Lq, 4, 32), device=gpu).half().requires_grad_(), torch.randn((2, Lq, 4, 32), device=gpu).half()
        o, p = ops.cross_attention(q, k, v), ops.cross_attention(q, k.contiguous(), v.contiguous())
        assert torch.equal(o, p) and torch.equal(torch.autograd.grad(o, q, do)[0], torch.autograd.grad(p, q, do)[0])


def test_cross_attention_gradients_by_differences(gpu):
    """fp32, a few directions: (f(x + e) - f(x - e)) / 2 with e of size 2^-7 of x; the third derivative's part is of
    relative order e^2 / 6 (a factor of 16 is allowed for its size), fp32 roundings of f are divided by e."""
    c, do = inputs(13, torch.float32, 1, 6, 20, 2, 1, 16, "full")
    _, grads = run_cross(c, do, gpu)
    g = torch.Generator().manual_seed(14)
    for n in ("q", "k", "v", "bias"):
        e = normal(g, *c[n].shape) * 2.0 ** -7
        f = [(ops.cross_attention(**to({**c, n: c[n] + s * e}, gpu)).double().cpu() * do.double()).sum() for s in (1, -1)]
        want = (f[0] - f[1]) / 2
        got = (grads["d" + n].double().cpu() * e.double()).sum()
        size = (grads["d" + n].double().cpu().abs() * e.double().abs()).sum()
        r = ref.cross_attention(**c, do=do)
        slack = ref.cross_attention_slack(r, torch.float32, c["bias"])["o"]
        assert abs(want - got) <= 16 / 6 * 2.0 ** -14 * size + (slack * do.double().abs()).sum()


def test_cross_attention_same_bits_each_time(gpu):
    for dtype in DTYPES:
        c, do = inputs(15, dtype, 2, 300, 500, 4, 2, 64, "h1", "both")
        first = run_cross(c, do, gpu)
        again = run_cross(c, do, gpu)
        assert torch.equal(first[0], again[0]) and all(torch.equal(first[1][n], again[1][n]) for n in first[1])


# ------------------------------------------------------------------------------ a run of them together
class Block:
    """Token rows broadcast to their atoms, atoms attending over another track, a dropped-out residual update and the
    sum of atoms by token."""

    def __init__(self, gpu, dtype, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.tokens, self.atoms, self.H, self.D = 40, 150, 4, 16
        c = self.H * self.D
        self.w = normal(g, self.tokens, c, dtype=dtype).to(gpu)
        self.kv = normal(g, 1, 70, 2, self.H, self.D, dtype=dtype).to(gpu)
        self.bias = normal(g, self.H, self.atoms, 70).to(gpu)
        self.owner = tokens(g, "sorted", self.atoms, self.tokens).to(gpu)
        self.lens = torch.tensor([61], device=gpu, dtype=torch.int32)
        self.do = normal(g, self.tokens, c, dtype=dtype).to(gpu)

    def run(self, seed):
        leaves = [t.detach().requires_grad_() for t in (self.w, self.kv, self.bias)]
        w, kv, bias = leaves
        x = ops.embedding(self.owner, w, 0.5)
        q = x.view(1, self.atoms, self.H, self.D)
        a = ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1], bias=bias, k_lens=self.lens)
        y = ops.dropout_add(a.reshape(x.shape), x, 0.25, seed, 3)
        out = ops.embedding_grad(y, self.owner, self.tokens)   # sums by token; its own gradient is a lookup
        return [y.detach(), out.detach(), *torch.autograd.grad(out, leaves, self.do)]

    def plain(self, seed):
        leaves = [t.detach().cpu().double().requires_grad_() for t in (self.w, self.kv, self.bias)]
        w, kv, bias = leaves
        owner = self.owner.cpu()
        inside = (owner >= 0)[:, None]
        x = torch.where(inside, w[owner.clamp_min(0)] * 0.5, torch.zeros((), dtype=torch.float64))
        q = x.view(1, self.atoms, self.H, self.D).transpose(1, 2)
        k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        logits = q @ k.transpose(2, 3) / self.D ** 0.5 + bias
        logits = logits.masked_fill(torch.arange(70) >= self.lens.cpu(), -torch.inf)
        a = (torch.softmax(logits, 3) @ v).transpose(1, 2).reshape(x.shape)
        y = x + a * ref.dropout_keep(x.shape, 0.25, seed, 3).double() / 0.75
        out = torch.zeros((self.tokens, x.shape[1]), dtype=torch.float64).index_add(0, owner.clamp_min(0), y * inside)
        return [y.detach(), out.detach(), *torch.autograd.grad(out, leaves, self.do.cpu().double())]


@pytest.mark.parametrize("dtype", DTYPES)
def test_block(gpu, dtype):
    """Every operator rounds its result to the type once and the products' operands once: eight roundings follow
    each other on the longest way (lookup, o, residual, dS, dq, the residual's gradient, their sum, dw); each is
    at most half a step of a value, and within a gradient's row values differ by less than its largest."""
    b = Block(gpu, dtype)
    for got, want in zip(b.run(77), b.plain(77)):
        tol = (8 * torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 512 * U32) * 4 * want.abs().max()
        assert (got.double().cpu() - want).abs().max() <= tol


def test_block_in_a_graph(gpu):
    """Forward and backward captured together (torch.autograd.grad: no accumulation), replayed with new inputs, other
    eager work and synchronizations between."""
    b = Block(gpu, torch.bfloat16)
    seed = torch.tensor([5], device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.run(seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = b.run(seed)
    for s in range(4):
        new = Block(gpu, torch.bfloat16, seed=s)
        for n in ("w", "kv", "bias", "owner", "do"):
            getattr(b, n).copy_(getattr(new, n))
        b.lens.fill_(70 - 20 * s)
        seed.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, b.run(s)))


def test_cross_attention_launchers_in_two_graphs(gpu):
    """Two captured steps with workspaces of their own, replayed on two streams at once."""
    graphs = []
    for seed in (1, 2):
        c, do = inputs(seed, torch.float16, 2, 20, 900, 4, 2, 64, "b1", "both")
        d, do = to(c, gpu), do.to(gpu)
        o, o32 = torch.empty_like(d["q"]), torch.empty(d["q"].shape, device=gpu)
        stats = torch.empty((2, 2, 4, 20), device=gpu)
        dq, dk, dv, db = (torch.empty_like(d[n]) for n in ("q", "k", "v", "bias"))
        ws = ops.workspace(ops.cross_attention_workspace_bytes(d["q"], d["k"]), gpu)
        wb = ops.workspace(ops.cross_attention_bwd_workspace_bytes(d["q"], d["k"], d["bias"]), gpu)
        more = dict(bias=d["bias"], mask=d["mask"], k_lens=d["k_lens"])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.launch_cross_attention(d["q"], d["k"], d["v"], o, o32=o32, stats=stats, ws=ws, o32_whole=True, **more)
            ops.launch_cross_attention_bwd(do, d["q"], d["k"], d["v"], o, o32, stats, dq, dk, dv, wb, dbias=db, **more)
        graphs.append((graph, c, do.cpu(), (o, dq, dk, dv, db), (ws, wb), (d, do, o32, stats)))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for _, _, _, outs, ws, _ in graphs:
            for t in (*outs, *ws):
                t.fill_(float("nan") if t.is_floating_point() else 255)
        torch.cuda.synchronize()
        for (graph, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, c, do, outs, _, _ in graphs:
            o, grads = run_cross(c, do, gpu)
            assert all(torch.equal(x, y) for x, y in zip(outs, (o, grads["dq"], grads["dk"], grads["dv"], grads["dbias"])))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hide", [None, "both"])
def test_cross_attention_many_heads(gpu, dtype, hide):
    """512 workgroups of 256 rows and more: two row tiles per wave."""
    c, do = inputs(16, dtype, 64, 70, 150, 8, 8, 48, None, hide)
    check_cross(c, do, gpu)
