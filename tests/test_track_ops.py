"""The operators between tracks without a GPU: their plain forms, what they hand to the library, and what they refuse."""
import ctypes

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
                        (dict(x=None), "null"), (dict(out=None), "null")):
        a = _lib.DropoutArgs(**{**ok, **change})
        assert lib.pf_dropout_add_fwd(ctypes.byref(a)) == -1
        import re
        assert re.search(say, _err()), (change, _err())
    assert lib.pf_dropout_add_fwd(None) == -1 and "null args" in _err()
    assert lib.pf_dropout_add_fwd(ctypes.byref(_lib.DropoutArgs(**{**ok, "C": 0}))) == 0
