"""CPU-only: the argument checks of the layer norm and gradient-clipping entry points, the gradient table's host layout, and the
options that switch them on (nothing here reaches a GPU)."""
import ctypes
import struct

import numpy as np
import pytest
import torch

NULL, PTR = None, ctypes.c_void_p(4096)      # (an address no check follows: every call here is refused before a launch)


@pytest.fixture(scope="module")
def L():
    from vince_amd import build
    build.build(verbose=False)
    from vince_amd import _lib
    return _lib.lib()


def test_layer_norm_refusals(L):
    fwd = lambda **k: L.vince_layer_norm_fwd(*[{**dict(dtype=0, x=PTR, w=PTR, b=PTR, out=PTR, mean=PTR, rstd=PTR, rows=4, cols=8, eps=1e-5,  # noqa: E731
                                                       relu=0, stream=NULL), **k}[n] for n in
                                               ("dtype", "x", "w", "b", "out", "mean", "rstd", "rows", "cols", "eps", "relu", "stream")])
    assert fwd(dtype=2) == -2 and b"dtype 2" in L.vince_last_error()
    assert fwd(cols=0) == -1 and fwd(rows=-1) == -1 and b"rows=-1" in L.vince_last_error()
    assert fwd(eps=-1.0) == -5 and fwd(eps=float("nan")) == -5
    assert fwd(x=NULL) == fwd(out=NULL) == fwd(mean=NULL) == fwd(rstd=NULL) == -5
    assert fwd(w=NULL) == -5 and b"bias without a weight" in L.vince_last_error()
    assert fwd(rows=0, x=NULL, out=NULL, mean=NULL, rstd=NULL) == 0           # no rows: nothing to do
    names = ("dtype", "x", "w", "mean", "rstd", "dout", "act", "dx", "dw", "db", "acc", "rows", "cols", "scratch", "nbytes", "stream")
    bwd = lambda **k: L.vince_layer_norm_bwd(*[{**dict(dtype=1, x=PTR, w=PTR, mean=PTR, rstd=PTR, dout=PTR, act=NULL, dx=PTR, dw=PTR, db=PTR,  # noqa: E731
                                                       acc=0, rows=4, cols=8, scratch=PTR, nbytes=1 << 20, stream=NULL), **k}[n] for n in names])
    assert bwd(dtype=5) == -2 and bwd(cols=-8) == -1
    for name in ("x", "mean", "rstd", "dout", "dx"):
        assert bwd(**{name: NULL}) == -5
    assert bwd(dw=NULL) == -5 and b"together" in L.vince_last_error()
    need = L.vince_layer_norm_bwd_scratch_bytes(1, 4000, 64)
    assert need > 0 and bwd(rows=4000, cols=64, nbytes=need - 1) == -5 and b"scratch" in L.vince_last_error()
    assert bwd(rows=4000, cols=64, nbytes=need, scratch=NULL) == -5
    assert L.vince_layer_norm_bwd_scratch_bytes(0, 0, 64) == 0
    assert bwd(rows=0, x=NULL, dout=NULL, dx=NULL, mean=NULL, rstd=NULL, acc=1) == 0


def test_layer_norm_bwd_refuses_gradients_that_share_memory(L):
    at = lambda bytes_off: ctypes.c_void_p(1 << 20 | bytes_off)  # noqa: E731
    for rows, cols in ((4, 8), (4000, 64), (4, 40000)):          # one launch, two, long rows
        need = L.vince_layer_norm_bwd_scratch_bytes(0, rows, cols)
        for a, b in ((0, 0), (0, 4 * cols - 4), (4, 0)):
            assert L.vince_layer_norm_bwd(0, PTR, PTR, PTR, PTR, PTR, NULL, PTR, at(a), at(b), 0, rows, cols, PTR, need, NULL) == -5
            assert b"share memory" in L.vince_last_error()


def test_longest_rows(L):
    """The partial rows of a few very long rows are no more than the rows; a length past the C interface's 32 bits is refused, not cut."""
    cols = 2 ** 31 - 1
    for rows, parts in ((1, 1), (7, 7), (8, 8), (9, 8), (32, 8), (33, 16)):
        assert L.vince_layer_norm_bwd_scratch_bytes(1, rows, cols) == parts * 2 * 4 * cols, rows
    from vince_amd import ops
    assert ops._layer_norm_shape("f", torch.empty(2, cols, device="meta"))[1] == cols
    for n in (2 ** 31, 2 ** 32 + 8):
        with pytest.raises(ValueError, match="2\\^31"):
            ops._layer_norm_shape("f", torch.empty(2, n, device="meta"))


def test_grad_entry_point_refusals(L):
    norm = lambda **k: L.vince_grad_norm(*[{**dict(table=PTR, chunks=300, limit=1.0, clip=PTR, scratch=PTR, nbytes=1 << 20, stream=NULL), **k}[n]  # noqa: E731
                                           for n in ("table", "chunks", "limit", "clip", "scratch", "nbytes", "stream")])
    assert norm(table=NULL) == norm(clip=NULL) == norm(scratch=NULL) == norm(chunks=-1) == -5
    assert norm(limit=-1.0) == -5 and norm(limit=float("nan")) == -5 and b"max_norm" in L.vince_last_error()
    assert norm(nbytes=0) == -5 and b"scratch" in L.vince_last_error()
    assert norm(chunks=3, table=NULL) == norm(chunks=3, clip=NULL) == norm(chunks=3, limit=-1.0) == -5
    assert L.vince_grad_clip(PTR, 300, -1.0, PTR, PTR, 1 << 20, NULL) == L.vince_grad_clip(PTR, 3, -1.0, PTR, PTR, 1 << 20, NULL) == -5
    assert L.vince_grad_scale(NULL, 3, PTR, NULL) == -5 and L.vince_grad_scale(PTR, 3, NULL, NULL) == -5
    assert L.vince_grad_scale(NULL, 0, PTR, NULL) == 0
    sgd = lambda **k: L.vince_sgd_flat_clip(*[{**dict(p=PTR, g=PTR, b=PTR, n=16, lr=0.1, mom=0.9, wd=0.0, gs=1.0, clip=PTR, stream=NULL), **k}[n]  # noqa: E731
                                              for n in ("p", "g", "b", "n", "lr", "mom", "wd", "gs", "clip", "stream")])
    assert sgd(clip=NULL) == sgd(p=NULL) == sgd(n=0) == -5
    assert sgd(g=ctypes.c_void_p(4100)) == -3 and b"aligned" in L.vince_last_error()


def _entries(*rows):
    from vince_amd._lib import GradTensor
    return (GradTensor * len(rows))(*[GradTensor(data=d, n=n, scale=s, dtype=t) for d, n, s, t in rows])


def test_grad_table_covers_every_element_once(L):
    """The entries' ranges are the tensors' memory, whole, in order, with each tensor's type and scale; empty tensors have none."""
    rows = [(0x10000, 1, 1.0, 0), (0x20000, 0, 2.0, 0), (0x30002, 100003, 0.5, 1), (0x100000, 3 * 16384, -1.5, 0), (0, 0, 1.0, 1)]
    e = _entries(*rows)
    chunks = L.vince_grad_table_chunks(e, len(rows))
    buf = (ctypes.c_uint8 * (16 * chunks + 16))(*([0xAB] * (16 * chunks + 16)))
    assert L.vince_grad_table_fill(e, len(rows), buf, chunks) == 0
    assert bytes(buf[16 * chunks:]) == b"\xab" * 16                            # nothing behind the last entry
    got = [struct.unpack_from("<QIf", bytes(buf), 16 * i) for i in range(chunks)]
    want = iter(got)
    for data, n, scale, dtype in rows:
        at, size = data, 4 if dtype == 0 else 2
        while n > 0:
            ptr, m, s = next(want)
            count, bf16 = m & 0x7FFFFFFF, m >> 31
            assert ptr == at and s == scale and bf16 == dtype and 0 < count <= n
            at, n = at + count * size, n - count
    assert next(want, None) is None


def test_grad_table_refusals(L):
    for row, code in [((4096, 4, 1.0, 2), -2), ((4096, -1, 1.0, 0), -5), ((0, 4, 1.0, 0), -5), ((4098, 4, 1.0, 0), -3), ((4097, 4, 1.0, 1), -3),
                      ((4096, 4, float("nan"), 0), -5), ((4096, 4, float("inf"), 0), -5)]:
        e = _entries((8192, 8, 1.0, 0), row)
        assert L.vince_grad_table_chunks(e, 2) == code, row
        assert b"tensor 1" in L.vince_last_error()
        assert L.vince_grad_table_fill(e, 2, (ctypes.c_uint8 * 64)(), 2) == code
    e = _entries((8192, 8, 1.0, 0))
    assert L.vince_grad_table_fill(e, 1, (ctypes.c_uint8 * 64)(), 2) == -5
    assert L.vince_grad_table_chunks(e, -1) == -5 and L.vince_grad_table_chunks(None, 0) == 0
    assert L.vince_grad_norm_scratch_bytes(0) == 0 and L.vince_grad_norm_scratch_bytes(1 << 40) < (1 << 20)


def test_python_entry_points_refuse_cpu_tensors():
    from vince_amd import ops
    x = torch.randn(4, 8)
    for call in (lambda: ops.layer_norm_fwd(x), lambda: ops.layer_norm_bwd(x, None, x[:, 0].contiguous(), x[:, 0].contiguous(), x),
                 lambda: ops.GradTable([x]), lambda: ops.grad_norm([x]), lambda: ops.grad_clip([x], 1.0),
                 lambda: ops.sgd_flat(x, x, x, 0.1, clip=torch.ones(2))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(ValueError):
        ops.GradTable([])


def test_dense_memory_rule():
    from vince_amd.ops import _dense
    t = torch.empty(4, 6, 3, 5)
    for yes in (t, t.permute(2, 0, 3, 1), t.to(memory_format=torch.channels_last), t[1:3], torch.empty(0, 3), torch.empty(()), torch.empty(1, 7)[:, :7],
                torch.empty(3, 1, 5).transpose(0, 1)):
        assert _dense(yes), (yes.shape, yes.stride())
    for no in (t[:, 1:], t[..., ::2], torch.empty(3, 1).expand(3, 4), torch.empty(1).expand(5), torch.empty(16).as_strided((3, 3), (1, 2))):
        assert not _dense(no), (no.shape, no.stride())


def test_options():
    from vince_amd import arg_parser
    from vince_amd.config import make_args
    from vince_amd.models.vince_model import VinceModel
    from vince_amd.optim import FlatSGD
    a = arg_parser.parse_args([])
    assert a.head_norm == "none" and a.max_grad_norm is None
    a = arg_parser.parse_args(["--head-norm", "layer", "--max-grad-norm", "1.5"])
    assert a.head_norm == "layer" and a.max_grad_norm == 1.5
    with pytest.raises(ValueError, match="head_norm"):
        VinceModel(make_args(head_norm="batch"))
    model = VinceModel(make_args())
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="max_grad_norm"):
            FlatSGD(model, lr=0.1, max_grad_norm=bad)
    assert "max_grad_norm" not in repr(FlatSGD(model, lr=0.1)) and "max_grad_norm=2" in repr(FlatSGD(model, lr=0.1, max_grad_norm=2.0))


@pytest.mark.parametrize("jigsaw", [False, True])
def test_head_norm_parameters_live_in_the_flat_buffer(jigsaw):
    """The option adds its parameters and nothing else: the reference's keys and values stay, every new parameter is a view of the flat
    buffer inside its head's range, and a checkpoint without them still loads."""
    from vince_amd.config import make_args
    from vince_amd.models.vince_model import VinceModel
    torch.manual_seed(0)
    plain = VinceModel(make_args(jigsaw=jigsaw))
    torch.manual_seed(0)
    model = VinceModel(make_args(jigsaw=jigsaw, head_norm="layer"))
    new = set(model.state_dict()) - set(plain.state_dict())
    heads = ["embedding_norm"] + (["jigsaw_embedding_norm"] if jigsaw else [])
    assert new == {h + s for h in heads for s in (".weight", ".bias")}
    for k, v in plain.state_dict().items():
        assert torch.equal(v, model.state_dict()[k]), k
    base = model._flat.data_ptr()
    for h in heads:
        a, b = model._segments["jigsaw" if h.startswith("jigsaw") else "embedding"]
        for p in getattr(model, h).parameters():
            off = (p.data_ptr() - base) // 4
            assert a <= off and off + p.numel() <= b and p.grad is not None
    assert {id(p) for h in heads for p in getattr(model, h).parameters()} <= {id(p) for p in model.vince_parameters()}
    missing, unexpected = model.load_state_dict(plain.state_dict(), strict=False)
    assert set(missing) == new and not unexpected
    ranges = sorted(model._segments.values())
    assert ranges[0][0] == 0 and all(x[1] == y[0] for x, y in zip(ranges, ranges[1:])) and ranges[-1][1] == model._n_train
    np.testing.assert_array_equal(model._flat[model._segments["embedding"][0]:][:64].numpy(), plain._flat[plain._segments["embedding"][0]:][:64].numpy())
