"""Cross attention, table lookup and residual dropout, as cases that can be prepared, run and compared.

A case is a dict of plain values.  Its ``op`` names the operator:

* ``cross``    ``ops.cross_attention``: queries of one track against keys and values of another, ``b`` batch
               elements of ``lq`` queries and ``lk`` keys, ``h`` heads (``hk`` of keys) of ``d`` channels;
               ``bias`` none, full [B, H, Lq, Lk] or shared by the batch; ``hide`` none, lens (padded
               encoder states) or mask (single keys); ``grad``: with its backward pass
* ``embed``    ``ops.embedding``: ``n`` indexes into a table of ``v`` rows of ``c`` channels; ``grad``: with
               the table's gradient
* ``dropout``  ``ops.dropout_add``: residual + dropped-out update over [``b``, ``i``, ``j``, ``c``], the mask per
               element or shared by a pair tensor's rows or columns; ``grad``: with the update's gradient

``run`` computes the plain form with elementary torch operations in fp32 (long sums in fp64) unless
``own`` is true, where it calls the framework.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
#: the costliest drawn case, in scores x channels (cross), rows x channels (embed) and elements (dropout)
MOST_CROSS, MOST_CROSS_GRAD, MOST_CROSS_FP32, MOST_EMBED, MOST_DROP = 2 << 34, 1 << 34, 1 << 30, 1 << 26, 1 << 25


def listed():
    return [
        # one decoder token of each of eight requests against its padded encoder states, shared heads
        dict(name="token_step", op="cross", dtype="fp16", b=8, lq=1, lk=1536, h=16, hk=4, d=64, bias="none", hide="lens",
             grad=False),
        # the atom transformer's windows: 32 atoms against the 128 around them, with the pair bias
        dict(name="atom_windows", op="cross", dtype="bf16", b=512, lq=32, lk=128, h=4, hk=4, d=32, bias="full", hide="mask",
             grad=False),
        # a prompt of a decoder against long encoder states
        dict(name="prompt", op="cross", dtype="bf16", b=4, lq=2048, lk=4096, h=16, hk=16, d=64, bias="none", hide="none",
             grad=False),
        # the single track's heads over another track of odd length, trained with the pair bias
        dict(name="track_train", op="cross", dtype="fp16", b=2, lq=512, lk=765, h=16, hk=16, d=24, bias="full", hide="mask",
             grad=True),
        # a decoder layer in training, heads shared by four, padded encoder states
        dict(name="decoder_train", op="cross", dtype="bf16", b=2, lq=2048, lk=2048, h=16, hk=4, d=128, bias="none",
             hide="lens", grad=True),
        # tokens against their atoms in the framework's own fp32, trained
        dict(name="tokens_atoms_fp32", op="cross", dtype="fp32", b=1, lq=384, lk=2900, h=8, hk=8, d=48, bias="none",
             hide="mask", grad=True),
        # token states broadcast to the tokens' atoms, padded at the end
        dict(name="token_to_atom", op="embed", dtype="fp32", n=4608, v=512, c=128, dist="sorted", scale=1.0, grad=False),
        # a decoder's scaled input rows
        dict(name="vocabulary", op="embed", dtype="bf16", n=16384, v=32000, c=2048, dist="zipf", scale=math.sqrt(2048.0),
             grad=False),
        # the residue types of an alignment of 1024 sequences of 512, trained: few rows, each used thousands of times
        dict(name="residues_train", op="embed", dtype="fp32", n=1024 * 512, v=33, c=64, dist="uniform", scale=1.0, grad=True),
        # a large vocabulary in training
        dict(name="vocabulary_train", op="embed", dtype="bf16", n=16384, v=128000, c=2048, dist="zipf",
             scale=math.sqrt(2048.0), grad=True),
        # a triangle update's residual, one mask value per row of the pair tensor
        dict(name="pair_row", op="dropout", dtype="fp32", b=1, i=512, j=512, c=128, shared="row", p=0.25, grad=True),
        # hidden states of a decoder, a mask value per element
        dict(name="hidden", op="dropout", dtype="bf16", b=4, i=1, j=2048, c=4096, shared="none", p=0.1, grad=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("cross", "cross", "cross", "embed", "dropout"))
    dtype = rng.choice(("fp32", "fp16", "bf16", "bf16"))
    grad = rng.random() < 0.5
    if op == "cross":
        h = rng.choice((4, 8, 16))
        hk = rng.choice((h, h, h // 2, h // 4))
        d = rng.choice((16, 24, 32, 48, 64, 96, 128))
        lq, lk = _log(rng, 1, 4096), _log(rng, 4, 8192)
        most = MOST_CROSS_FP32 if dtype == "fp32" else MOST_CROSS_GRAD if grad else MOST_CROSS
        while lq * lk * h * d > most:
            lq, lk = max(1, lq // 2), max(4, lk - lk // 3)
        b = _log(rng, 1, max(1, min(64, most // (lq * lk * h * d))))
        return dict(op="cross", dtype=dtype, b=b, lq=lq, lk=lk, h=h, hk=hk, d=d, bias=rng.choice(("none", "full", "shared")),
                    hide=rng.choice(("none", "lens", "mask")), grad=grad)
    if op == "embed":
        c = 8 * _log(rng, 2, 512)
        n = _log(rng, 1, min(1 << 19, MOST_EMBED // c // 2))
        v = _log(rng, 20, min(200000, MOST_EMBED // c))
        return dict(op="embed", dtype=dtype, n=n, v=v, c=c, dist=rng.choice(("sorted", "zipf", "uniform")),
                    scale=rng.choice((1.0, math.sqrt(c))), grad=grad)
    shared = rng.choice(("none", "none", "row", "column"))
    p = rng.choice((0.1, 0.15, 0.25, 0.5))
    if shared == "none":
        b, i, c = rng.choice((1, 1, 3)), 1, _log(rng, 1, 8192)
        j = _log(rng, 1, min(32768, MOST_DROP // c // b))
    else:
        b, c = rng.choice((1, 1, 2)), rng.choice((32, 64, 128, 132))
        i = j = _log(rng, 4, min(700, math.isqrt(MOST_DROP // c // b)))
    return dict(op="dropout", dtype=dtype, b=b, i=i, j=j, c=c, shared=shared, p=p, grad=grad)


def _shape(case):
    return [case[k] for k in ("b", "i", "j", "c")]


# ------------------------------------------------------------------------------ inputs
def _visible(case, g, dev):
    """lens [B] or mask [B, Lk] of a cross case, and which keys are seen, [B, Lk]."""
    b, lk = case["b"], case["lk"]
    if case["hide"] == "lens":
        lens = torch.randint((lk + 1) // 2, lk + 1, (b,), generator=g, device=dev, dtype=torch.int32)
        return lens, torch.arange(lk, device=dev)[None] < lens[:, None]
    mask = torch.rand((b, lk), generator=g, device=dev) < 0.85
    mask[:, 0] = True
    return mask, mask


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = {"case": case}

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)

    if case["op"] == "cross":
        b, lq, lk, h, hk, d = (case[k] for k in ("b", "lq", "lk", "h", "hk", "d"))
        st["q"], st["k"], st["v"] = normal(b, lq, h, d), normal(b, lk, hk, d), normal(b, lk, hk, d)
        st["bias"] = {"none": lambda: None, "full": lambda: normal(b, h, lq, lk, dtype=torch.float32),
                      "shared": lambda: normal(1, h, lq, lk, dtype=torch.float32)}[case["bias"]]()
        st["lens"] = st["mask"] = st["seen"] = None
        if case["hide"] != "none":
            st[case["hide"]], st["seen"] = _visible(case, g, dev)
        if case["grad"]:
            st["do"] = normal(b, lq, h, d)
            st["leaves"] = [t.requires_grad_() for t in (st["q"], st["k"], st["v"], st["bias"]) if t is not None]
    elif case["op"] == "embed":
        n, v, c = case["n"], case["v"], case["c"]
        st["w"] = normal(v, c)
        if case["dist"] == "uniform":
            t = torch.randint(0, v, (n,), generator=g, device=dev)
        elif case["dist"] == "zipf":   # token frequencies fall like 1 / rank; ranks are scattered over the table
            u = torch.rand((n,), generator=g, device=dev, dtype=torch.float64)
            t = (torch.exp(u * math.log(v)).long().clamp(1, v) * 7919) % v
        else:   # atoms in their tokens' order, the last eighth padding
            t = torch.sort(torch.randint(0, v, (n,), generator=g, device=dev)).values
            t[n - n // 8:] = -1
        st["t"] = t
        if case["grad"]:
            st["do"] = normal(n, c)
            st["w"].requires_grad_()
    else:
        shape = _shape(case)
        st["x"], st["r"] = normal(*shape), normal(*shape)
        st["seed"], st["offset"] = int(torch.randint(0, 1 << 62, (1,), generator=g, device=dev)), seed % 1000
        if case["grad"]:
            st["do"] = normal(*shape)
            st["x"].requires_grad_()
    return st


# ------------------------------------------------------------------------------ plain forms
def _plain_cross(st):
    case = st["case"]
    b, lq, lk, h, hk, d = (case[k] for k in ("b", "lq", "lk", "h", "hk", "d"))
    group, scale, dt = h // hk, d ** -0.5, st["q"].dtype
    q = st["q"].detach().float().transpose(1, 2)                                         # [B, H, Lq, D]
    k, v = (st[n].detach().float().transpose(1, 2).repeat_interleave(group, 1) for n in "kv")   # [B, H, Lk, D]
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    if st["bias"] is not None:
        x = x + st["bias"].detach()
    if st["seen"] is not None:
        x = torch.where(st["seen"][:, None, None], x, x.new_tensor(-math.inf))
    top = x.amax(3, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(3, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    o = torch.matmul(p, v).transpose(1, 2).to(dt)
    if not case["grad"]:
        return o
    do = st["do"].float().transpose(1, 2).contiguous()
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (dp - (p * dp).sum(3, keepdim=True))
    del p, dp
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    dk, dv = (t.view(b, hk, group, lk, d).sum(2).transpose(1, 2).to(dt) for t in (dk, dv))
    out = [o, dq.transpose(1, 2).to(dt), dk, dv]
    if st["bias"] is not None:
        out.append(ds if st["bias"].shape[0] == b else ds.sum(0, keepdim=True))
    return out


def _plain_embed(st):
    case, w, t = st["case"], st["w"].detach(), st["t"]
    inside = (t >= 0) & (t < case["v"])
    at = torch.where(inside, t, torch.zeros_like(t))
    out = (w[at].float() * case["scale"] * inside[:, None]).to(w.dtype)
    if not case["grad"]:
        return out
    rows = st["do"].double() * inside[:, None]
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device).index_add_(0, at, rows) * case["scale"]
    return [out, dw.to(w.dtype)]


def _words(n, seed, offset, dev):
    """The first n words of Philox4x32-10 under key ``seed``: counter i holds words 4 i to 4 i + 3, ``offset`` its upper half."""
    low = 0xFFFFFFFF
    i = torch.arange((n + 3) // 4, dtype=torch.int64, device=dev)
    c = [i & low, i >> 32, torch.full_like(i, offset & low), torch.full_like(i, (offset >> 32) & low)]
    key = [seed & low, (seed >> 32) & low]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57   # modulo 2^64
        c = [((b >> 32) & low) ^ c[1] ^ key[0], b & low, ((a >> 32) & low) ^ c[3] ^ key[1], a & low]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    return torch.stack(c, 1).view(-1)[:n]


def _keep(case, seed, offset, dev):
    """Which elements stay, in a shape that broadcasts to the case's."""
    b, i, j, _ = shape = _shape(case)
    shape = {"none": shape, "row": [b, i, 1, 1], "column": [b, 1, j, 1]}[case["shared"]]
    return (_words(math.prod(shape), seed, offset, dev) >= round(case["p"] * 2 ** 32)).view(shape)


def _plain_dropout(st):
    case, x = st["case"], st["x"].detach()
    keep = _keep(case, st["seed"], st["offset"], x.device).float() * (1.0 / (1.0 - case["p"]))
    out = (st["r"].float() + x.float() * keep).to(x.dtype)
    return [out, (st["do"].float() * keep).to(x.dtype)] if case["grad"] else out


# ------------------------------------------------------------------------------ the framework's calls
def _own_cross(st):
    from tt_boltz_amd import ops
    o = ops.cross_attention(st["q"], st["k"], st["v"], bias=st["bias"], mask=st["mask"], k_lens=st["lens"])
    return [o.detach(), *torch.autograd.grad(o, st["leaves"], st["do"])] if st["case"]["grad"] else o


def _own_embed(st):
    from tt_boltz_amd import ops
    out = ops.embedding(st["t"], st["w"], scale=st["case"]["scale"])
    return [out.detach(), *torch.autograd.grad(out, st["w"], st["do"])] if st["case"]["grad"] else out


def _own_dropout(st):
    from tt_boltz_amd import ops
    case = st["case"]
    out = ops.dropout_add(st["x"], st["r"], case["p"], st["seed"], st["offset"],
                          shared=None if case["shared"] == "none" else case["shared"])
    return [out.detach(), *torch.autograd.grad(out, st["x"], st["do"])] if case["grad"] else out


PLAIN = {"cross": _plain_cross, "embed": _plain_embed, "dropout": _plain_dropout}
OWN = {"cross": _own_cross, "embed": _own_embed, "dropout": _own_dropout}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------------------ floors
def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once, the products of the formulas."""
    e = BYTES[case["dtype"]]
    if case["op"] == "cross":
        b, lq, lk, h, hk, d = (case[k] for k in ("b", "lq", "lk", "h", "hk", "d"))
        qs, ks = b * lq * h * d * e, b * lk * hk * d * e
        bias = {"none": 0, "full": b, "shared": 1}[case["bias"]] * h * lq * lk * 4
        seen = {"none": 1.0, "lens": 0.75, "mask": 1.0}[case["hide"]]   # padded states need not be read
        pair = b * h * lq * lk * d * seen
        if not case["grad"]:
            return {"bytes": int(2 * qs + 2 * ks * seen + bias), "flops": int(4 * pair)}
        return {"bytes": int(4 * qs + 2 * ks * seen + 2 * ks + 2 * bias), "flops": int(14 * pair)}
    if case["op"] == "embed":
        n, v, c = case["n"], case["v"], case["c"]
        rows = min(n, v) * c * e + n * c * e + 8 * n
        if not case["grad"]:
            return {"bytes": rows, "flops": n * c}
        return {"bytes": rows + n * c * e + v * c * e, "flops": 2 * n * c}
    n = math.prod(_shape(case))
    return {"bytes": (5 if case["grad"] else 3) * n * e, "flops": (3 if case["grad"] else 2) * n}


# ------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_cross(st):
    case = st["case"]
    group, scale = case["h"] // case["hk"], 1.0 / math.sqrt(case["d"])
    q, k, v = (st[n].detach().double() for n in "qkv")
    o = torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    bias = None if st["bias"] is None else st["bias"].detach().double()
    dbias = None if bias is None else torch.zeros_like(bias)
    for i in range(case["b"]):
        keys = slice(None) if st["seen"] is None else st["seen"][i].nonzero()[:, 0]
        for j in range(case["h"]):
            qh, kh, vh = q[i, :, j], k[i, :, j // group][keys], v[i, :, j // group][keys]
            bi = 0 if bias is None or bias.shape[0] == 1 else i
            logits = scale * (qh @ kh.T)
            if bias is not None:
                logits = logits + bias[bi, j][:, keys]
            prob = torch.softmax(logits, 1)
            o[i, :, j] = prob @ vh
            if not case["grad"]:
                continue
            doh = st["do"][i, :, j].double()
            dlogits = prob * (doh @ vh.T - (doh * o[i, :, j]).sum(1, keepdim=True))
            grads[0][i, :, j] = scale * (dlogits @ kh)
            grads[1][i, :, j // group][keys] += scale * (dlogits.T @ qh)
            grads[2][i, :, j // group][keys] += prob.T @ doh
            if dbias is not None:
                dbias[bi, j][:, keys] += dlogits
    if not case["grad"]:
        return o
    return [o, *grads] + ([] if dbias is None else [dbias])


def _exact_embed(st):
    case, t = st["case"], st["t"]
    table = torch.cat([st["w"].detach().double() * case["scale"], torch.zeros((1, case["c"]), dtype=torch.float64, device=t.device)])
    at = torch.where((t < 0) | (t >= case["v"]), case["v"], t)
    out = table.index_select(0, at)
    if not case["grad"]:
        return out
    order = torch.argsort(at, stable=True)   # running sums over the sorted rows, differences at the tokens' ends
    sums = torch.cat([torch.zeros((1, case["c"]), dtype=torch.float64, device=t.device), st["do"].double()[order].cumsum(0)])
    ends = torch.searchsorted(at[order].contiguous(), torch.arange(case["v"] + 1, device=t.device))
    return [out, (sums[ends[1:]] - sums[ends[:-1]]) * case["scale"]]


def _exact_dropout(st):
    import numpy as np
    case = st["case"]
    shape = _shape(case)
    if case["shared"] == "row":
        shape[-2:] = [1, 1]
    elif case["shared"] == "column":
        shape[-3], shape[-1] = 1, 1
    n = math.prod(shape)
    counters = np.arange((n + 3) // 4, dtype=np.uint64)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    x0, x1 = counters & low, counters >> half
    x2, x3 = (np.full_like(counters, (st["offset"] >> s) & 0xFFFFFFFF) for s in (0, 32))
    for r in range(10):
        k0 = np.uint64((st["seed"] + r * 0x9E3779B9) & 0xFFFFFFFF)
        k1 = np.uint64(((st["seed"] >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
        m0, m1 = np.uint64(0xD2511F53) * x0, np.uint64(0xCD9E8D57) * x2
        x0, x1, x2, x3 = (m1 >> half) ^ x1 ^ k0, m1 & low, (m0 >> half) ^ x3 ^ k1, m0 & low
    words = np.stack([x0, x1, x2, x3], 1).reshape(-1)[:n]
    stays = torch.from_numpy(words >= np.uint64(round(case["p"] * 2 ** 32))).to(st["x"].device).view(shape)
    factor = stays.double() / (1.0 - case["p"])
    out = st["r"].double() + st["x"].detach().double() * factor
    return [out, st["do"].double() * factor] if case["grad"] else out


def exact(case, seed):
    st = prepare(case, seed)
    return {"cross": _exact_cross, "embed": _exact_embed, "dropout": _exact_dropout}[case["op"]](st)
