"""The operators between tracks without a GPU: their plain forms, what they hand to the library, and what they refuse."""
import ctypes
import pathlib
import subprocess
import sys

import pytest
import torch

from oracle import track_ref as ref
from tt_boltz_amd import _lib, ops, track_ops

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _err():
    return _lib.load().pf_last_error().decode()


class Recorder:
    """Stands for the library: keeps the calls and their arguments."""

    def __init__(self, monkeypatch):
        self.calls = []
        monkeypatch.setattr(ops, "_require_gpu", lambda *ts: torch.device("cpu"))
        monkeypatch.setattr(ops, "_stream", lambda: 0)
        monkeypatch.setattr(_lib, "load", lambda *a: self)

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("workspace_size"):
                return 64
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def lib(monkeypatch):
    return Recorder(monkeypatch)


# ------------------------------------------------------------------------------ the generator
@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), "d16cfe09 94fdcceb 5001e420 24126ea1"),
])
def test_philox_known_answers(counter, key, want):
    """The generator's published test vectors."""
    assert " ".join(f"{w:08x}" for w in ref.philox4x32(counter, key)) == want


def test_dropout_keep_shares():
    rows = ref.dropout_keep((2, 3, 5, 4), 0.5, 7, 0, "row")
    cols = ref.dropout_keep((2, 3, 5, 4), 0.5, 7, 0, "column")
    words = [w >= 1 << 31 for w in ref.dropout_words(10, 7, 0)]
    assert rows[..., 0, 0].reshape(-1).tolist() == words[:6] and (rows == rows[..., :1, :1]).all()
    assert cols[:, 0, :, 0].reshape(-1).tolist() == words and (cols == cols[:, :1, :, :1]).all()


# ------------------------------------------------------------------------------ refusals
def test_cpu_tensors_are_refused():
    x = torch.zeros((2, 3))
    for call in (lambda: ops.embedding(torch.zeros(2, dtype=torch.int64), x),
                 lambda: ops.embedding_grad(x, torch.zeros(2, dtype=torch.int64), 4),
                 lambda: ops.dropout_add(x, x, 0.5, 1)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


def test_embedding_refuses(lib):
    t, w = torch.zeros((2, 3), dtype=torch.int64), torch.zeros((4, 8))
    for index, weight, say in ((t.float(), w, "index type"), (t.to(torch.int16), w, "index type"), (t, w.double(), "element type"),
                               (t, w[0], r"weight \[V, C\]"), (t, w[None], r"weight \[V, C\]")):
        with pytest.raises(ValueError, match=say):
            ops.embedding(index, weight)
    for grad, index, rows, say in ((torch.zeros((2, 4, 8)), t, 4, "index"), (torch.zeros((2, 3)), t, 4, "index"),
                                   (torch.zeros((2, 3, 8)).double(), t, 4, "element type"), (torch.zeros((2, 3, 8)), t, -1, "negative")):
        with pytest.raises(ValueError, match=say):
            ops.embedding_grad(grad, index, rows)
    with pytest.raises(TypeError):
        ops.embedding_grad(torch.zeros((2, 3, 8)), t, 4.5)
    assert not lib.calls


def test_dropout_refuses(lib):
    x = torch.zeros((2, 3, 3, 8))
    for args, kw, say in (((x, x[:1], 0.5, 1), {}, "not like x"), ((x, x.half(), 0.5, 1), {}, "not like x"),
                          ((x, None, 1.5, 1), {}, r"\[0, 1\]"), ((x, None, -0.1, 1), {}, r"\[0, 1\]"),
                          ((x, None, float("nan"), 1), {}, r"\[0, 1\]"), ((x.double(), None, 0.5, 1), {}, "element type"),
                          ((x, None, 0.5, 1), {"shared": "rows"}, "shared"), ((x[0, 0], None, 0.5, 1), {"shared": "row"}, "mask needs"),
                          ((x, None, 0.5, torch.zeros(2, dtype=torch.int64)), {}, "one int64"),
                          ((x, None, 0.5, torch.zeros(1)), {}, "one int64"), ((x, None, 0.5, 1, -1), {}, "offset"),
                          ((x, None, 0.5, 1, 1 << 64), {}, "offset")):
        with pytest.raises(ValueError, match=say):
            ops.dropout_add(*args, **kw)
    with pytest.raises(TypeError):
        ops.dropout_add(x, None, 0.5, 1.5)
    assert not lib.calls


def test_embedding_reads_rows_where_they_are(lib):
    t, w = torch.zeros(5, dtype=torch.int32), torch.randn((6, 16))
    for weight, stride in ((w, 16), (w[:, :8], 16), (w[::2], 32), (w.t(), 6), (w[:1], 16), (w[:1].expand(4, 16), 16)):
        lib.calls.clear()
        ops.embedding(t, weight, 2.0)
        (name, args), = lib.calls
        assert name == "pf_embedding_fwd" and args[1] == 0 and args[3] == stride and args[5:8] == (5, *weight.shape)
        assert (args[2] == weight.data_ptr()) == (weight.stride(1) == 1 and (weight.shape[0] == 1 or weight.stride(0) > 0))


def test_dropout_shapes_and_seeds(lib):
    x = torch.zeros((2, 3, 4, 5, 8))
    for shared, shape in ((None, (1, 1, 1, 960)), ("row", (6, 4, 5, 8)), ("column", (6, 4, 5, 8))):
        lib.calls.clear()
        ops.dropout_add(x, x, 0.25, -1, 3, shared=shared)
        (name, (a,)), = lib.calls
        a = a._obj
        assert (a.B, a.I, a.J, a.C) == shape and a.seed == 2 ** 64 - 1 and a.offset == 3 and a.seed_at is None
    lib.calls.clear()
    ops.dropout_add(x, None, 0.25, torch.zeros((), dtype=torch.int64))
    a = lib.calls[0][1][0]._obj
    assert a.seed_at is not None and a.residual is None


# ------------------------------------------------------------------------------ the C entry points
def test_abi_refuses_without_launching():
    lib, d = _lib.load(), 4096
    assert lib.pf_embedding_fwd(d, 1, d, 8, d, 4, 4, 8, 3, 1.0, None) == -1 and "dtype" in _err()
    assert lib.pf_embedding_fwd(d, 2, d, 8, d, 4, 4, 8, 0, 1.0, None) == -1 and "index64" in _err()
    assert lib.pf_embedding_fwd(d, 1, d, 7, d, 4, 4, 8, 0, 1.0, None) == -1 and "stride" in _err()
    assert lib.pf_embedding_fwd(None, 1, d, 8, d, 4, 4, 8, 0, 1.0, None) == -1 and "null" in _err()
    assert lib.pf_embedding_fwd(d, 1, d, 8, None, 4, 4, 8, 0, 1.0, None) == -1 and "null" in _err()
    assert lib.pf_embedding_fwd(d, 1, d, 8, d, -1, 4, 8, 0, 1.0, None) == -1 and "bad shape" in _err()
    assert lib.pf_embedding_fwd(d, 1, d, 8, d, 1 << 31, 4, 8, 0, 1.0, None) == -1 and "bad shape" in _err()
    assert lib.pf_embedding_fwd(d, 1, d, 8, d, 0, 4, 8, 0, 1.0, None) == 0
    need = lib.pf_embedding_grad_workspace_size(100, 50, 8)
    assert need > 100 * 16 and lib.pf_embedding_grad_workspace_size(0, 50, 8) == 0
    assert lib.pf_embedding_grad(d, 1, d, d, 100, 50, 8, 0, 1.0, d, need - 1, None) == -1 and "workspace too small" in _err()
    assert lib.pf_embedding_grad(d, 1, d, d, 100, 50, 8, 0, 1.0, d + 4, need, None) == -1 and "aligned" in _err()
    assert lib.pf_embedding_grad(d, 1, None, d, 100, 50, 8, 0, 1.0, d, need, None) == -1 and "null" in _err()
    assert lib.pf_embedding_grad(d, 1, d, d, 100, 0, 8, 0, 1.0, d, need, None) == 0
    ok = dict(B=1, I=1, J=1, C=8, dtype=0, shared=0, p=0.5, x=d, out=d)
    for change, say in ((dict(dtype=3), "dtype"), (dict(shared=3), "sharing"), (dict(p=1.5), "p must"), (dict(p=float("nan")), "p must"),
                        (dict(B=-1), "bad shape"), (dict(C=1 << 33), "bad shape"), (dict(B=1 << 40, C=1 << 30), "2\\^32"),
                        (dict(x=None), "null"), (dict(out=None), "null"), (dict(C=1 << 16, J=1 << 16, x=d + 4), "aligned")):
        a = _lib.DropoutArgs(**{**ok, **change})
        assert lib.pf_dropout_add_fwd(ctypes.byref(a)) == -1
        import re
        assert re.search(say, _err()), (change, _err())
    assert lib.pf_dropout_add_fwd(None) == -1 and "null args" in _err()
    assert lib.pf_dropout_add_fwd(ctypes.byref(_lib.DropoutArgs(**{**ok, "C": 0}))) == 0


# ------------------------------------------------------------------------------ cross attention
def test_cross_attention_oracle_against_autograd():
    g = torch.Generator().manual_seed(0)
    shapes = dict(q=(2, 5, 4, 8), k=(2, 7, 2, 8), v=(2, 7, 2, 8), bias=(2, 4, 5, 7))
    t = {n: torch.randn(s, generator=g, dtype=torch.float64, requires_grad=True) for n, s in shapes.items()}
    mask, do = torch.rand((2, 7), generator=g) < 0.7, torch.randn((2, 5, 4, 8), generator=g, dtype=torch.float64)
    k, v = (t[n].transpose(1, 2).repeat_interleave(2, 1) for n in "kv")
    o = torch.nn.functional.scaled_dot_product_attention(t["q"].transpose(1, 2), k, v,
                                                         t["bias"].masked_fill(~mask[:, None, None], -torch.inf)).transpose(1, 2)
    want = [o, *torch.autograd.grad(o, list(t.values()), do)]
    r = ref.cross_attention(**t, mask=mask, do=do)
    for n, w in zip(("o", "dq", "dk", "dv", "dbias"), want):
        assert (r[n] - w).abs().max() < 1e-13


def _cross(dtype=torch.float32, B=2, Lq=5, Lk=7, H=4, Hk=2, D=16):
    return torch.zeros((B, Lq, H, D), dtype=dtype), torch.zeros((B, Lk, Hk, D), dtype=dtype), torch.zeros((B, Lk, Hk, D), dtype=dtype)


def test_cross_attention_refuses(lib):
    q, k, v = _cross()
    bias = torch.zeros((2, 4, 5, 7))
    for args, kw, say in (((q[0], k, v), {}, "expects q"), ((q, k[0], v), {}, "expects q"), ((q, k, v[:, :6]), {}, "do not fit"),
                          ((q, k[:1], v[:1]), {}, "do not fit"), ((q, k[..., :8], v[..., :8]), {}, "do not fit"),
                          ((q[:, :, :3], k, v), {}, "do not fit"), ((q, k[:, :, :0], v[:, :, :0]), {}, "do not fit"),
                          ((q, k.half(), v), {}, "differ in type"), ((q.double(), k.double(), v.double()), {}, "element type"),
                          ((q[..., :12], k[..., :12], v[..., :12]), {}, "multiple of 8"), (_cross(D=136), {}, "multiple of 8"),
                          ((q, k, v), {"scale": float("nan")}, "finite"), ((q, k, v), {"scale": float("inf")}, "finite"),
                          ((q, k, v), {"bias": bias[0, 0, 0]}, "expects bias"), ((q, k, v), {"bias": bias[..., :6]}, "does not fit"),
                          ((q, k, v), {"bias": bias[:, :, :1]}, "does not fit"), ((q, k, v), {"bias": bias[:, :3]}, "does not fit"),
                          ((q, k, v), {"bias": bias.half()}, "bias is"), ((q, k, v), {"k_lens": torch.zeros(3, dtype=torch.int32)}, "k_lens"),
                          ((q, k, v), {"k_lens": torch.zeros(2)}, "k_lens")):
        with pytest.raises(ValueError, match=say):
            ops.cross_attention(*args, **kw)
    for mask in (torch.ones((2, 6)), torch.ones((3, 7)), torch.ones((2, 1, 7))):
        with pytest.raises(RuntimeError):
            ops.cross_attention(q, k, v, mask=mask)
    assert not lib.calls


def test_cross_attention_reads_views_in_place(lib):
    kv = torch.zeros((2, 7, 2, 32))
    q, bias = torch.zeros((2, 4, 5, 16)).transpose(1, 2), torch.zeros((4, 5, 7))
    ops.cross_attention(q, kv[..., :16], kv[..., 16:], bias=bias, mask=torch.ones(7))
    (name, (a,)), = [c for c in lib.calls]
    a = a._obj
    assert name == "pf_cross_attn_fwd" and (a.B, a.Lq, a.Lk, a.H, a.Hk, a.D) == (2, 5, 7, 4, 2, 16)
    assert a.q == q.data_ptr() and (a.q_b, a.q_l, a.q_h) == (320, 16, 80)
    assert a.v == kv.data_ptr() + 64 and (a.v_b, a.v_l, a.v_h) == (448, 64, 32)
    assert a.bias == bias.data_ptr() and (a.bias_b, a.bias_h, a.bias_q, a.bias_k) == (0, 35, 7, 1) and a.mask_b == 0
    assert a.o32 is None and a.stats is None
    lib.calls.clear()
    ops.cross_attention(q, kv[..., 1:17], kv[..., :16])   # not in 16-byte pieces: a copy
    a = lib.calls[0][1][0]._obj
    assert a.k != kv.data_ptr() + 4 and (a.k_b, a.k_l, a.k_h) == (224, 32, 16)


def test_cross_attention_abi_refuses_without_launching():
    lib, d = _lib.load(), 4096
    ok = dict(B=2, Lq=5, Lk=7, H=4, Hk=2, D=16, scale=0.25, q=d, q_b=320, q_l=64, q_h=16, k=d, k_b=224, k_l=32, k_h=16, v=d,
              v_b=224, v_l=32, v_h=16, o=d)
    for change, say in ((dict(dtype=5), "dtype"), (dict(D=20), "D must"), (dict(D=136), "D must"), (dict(H=3), "bad shape"),
                        (dict(Hk=0), "bad shape"), (dict(B=-1), "bad shape"), (dict(scale=float("nan")), "finite"), (dict(q=None), "null"),
                        (dict(k=None), "null"), (dict(o=None), "null"), (dict(q=d + 4), "aligned"), (dict(k_l=34), "strides"), (dict(v_l=1 << 22), "below 2^22"),
                        (dict(o=d + 8), "aligned"), (dict(bias=d, bias_dtype=1), "bias"), (dict(Lk=1 << 30), "too long"),
                        (dict(B=1 << 20, Lq=1 << 20), "too large")):
        a = _lib.CrossAttnArgs(**{**ok, **change})
        assert lib.pf_cross_attn_fwd(ctypes.byref(a)) == -1 and say in _err(), (change, _err())
    assert lib.pf_cross_attn_fwd(None) == -1 and "null args" in _err()
    assert lib.pf_cross_attn_fwd(ctypes.byref(_lib.CrossAttnArgs(**{**ok, "Lq": 0}))) == 0
    long = _lib.CrossAttnArgs(**{**ok, "Lk": 100000})
    need = lib.pf_cross_attn_workspace_size(ctypes.byref(long))
    assert need > 0 and lib.pf_cross_attn_fwd(ctypes.byref(long)) == -1 and "workspace too small" in _err()
    long.workspace, long.workspace_bytes = d + 4, need
    assert lib.pf_cross_attn_fwd(ctypes.byref(long)) == -1 and "aligned" in _err()
    back = {**ok, "stats": d, "dout": d, "dq": d, "dk": d, "dv": d, "workspace": d, "workspace_bytes": 1 << 30}
    for change, say in ((dict(stats=None), "statistics"), (dict(dout=None), "dout"), (dict(dtype=1), "unrounded"), (dict(dv=None), "come together"),
                        (dict(dbias=d, dbias_B=2, dbias_H=4), "does not belong"), (dict(dbias_B=2, dbias_H=4), "do not agree"),
                        (dict(bias=d, dbias=d, dbias_B=1, dbias_H=4, dq=None), "comes with dq"),
                        (dict(bias=d, dbias=d, dbias_B=3, dbias_H=4), "does not belong"), (dict(workspace_bytes=16), "workspace too small"),
                        (dict(bias=d, dbias=d, dbias_B=1, dbias_H=4, Lq=65535, Lk=65537), "too large"),
                        (dict(dq=d + 4), "aligned"), (dict(Lq=0), "no queries")):
        a = _lib.CrossAttnArgs(**{**back, **change})
        assert lib.pf_cross_attn_bwd(ctypes.byref(a)) == -1 and say in _err(), (change, _err())
    assert lib.pf_cross_attn_bwd(None) == -1 and "null args" in _err()


@pytest.mark.parametrize("first", ["ops", "track_ops"])
def test_modules_import_in_either_order(first):
    code = (f"import importlib; m = importlib.import_module('tt_boltz_amd.{first}'); "
            "from tt_boltz_amd import ops, track_ops; assert ops.embedding is track_ops.embedding; m.cross_attention")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=pathlib.Path(__file__).resolve().parent.parent)
