"""GPU tests of layer norm (forward, backward), the gradient norm with clipping and the clipped SGD step against plain 64-bit
computations of the same formulas.  Tolerances count roundings: u = 2^-24 for fp32 arithmetic, 2^-8 for a value stored as bfloat16, and a
chain of n additions is off by at most n u times the sum of the magnitudes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
STORE = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TINY = 2.0 ** -126


def _ops():
    from vince_amd import ops
    return ops


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=gen(seed), device=DEV).to(dtype)


def inside(got, want, bound, what):
    """|got - want| <= bound element by element (fp64 tensors), NaN and infinities at the same places."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), what
    d = torch.where(fine, (got - want).abs(), torch.zeros_like(want))
    over = d - torch.where(fine, bound, torch.ones_like(bound))
    assert float(over.max() if over.numel() else -1.0) <= 0.0, (what, float(d.max()), float(over.max()), int(over.argmax()))


# ------------------------------------------------------------------------------------------------ layer norm
def ln_bounds(x, w, b, eps, relu, store):
    """fp64 outputs of the forward and how far fp32 arithmetic may be from them.  Additions of a row: at most h in a chain, whatever the
    split over lanes (D / 64 in a lane, or up to 32 where a row has fewer lanes, then the tree)."""
    x = x.double()
    D = x.shape[-1]
    h = max(-(-D // 64), 32) + 10
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    var = (xc * xc).mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    dm = (h + 1) * U * x.abs().mean(-1, keepdim=True) + U * mean.abs()                    # the mean
    # centred values: own rounding and the mean's; squares: chain, rounding, twice the centred value's; the mean's part has no first order
    dvar = ((h + 4) * U * var + dm * dm + 2 * U * (xc.abs() * (xc.abs() + dm)).mean(-1, keepdim=True)) / (var + eps)
    drstd = rstd * (0.5 * dvar + 4 * U) * 1.01
    xh = xc * rstd
    dxh = (rstd * (dm + U * xc.abs()) + xc.abs() * drstd + U * xh.abs()) * 1.01
    ww = w.double() if w is not None else torch.ones(D, device=x.device, dtype=torch.float64)
    bb = b.double() if b is not None else torch.zeros_like(ww)
    y = xh * ww + bb
    dy = (dxh * ww.abs() + U * (xh * ww).abs() + U * y.abs()) * 1.01
    if relu:
        y = y.clamp(min=0.0)
    return y, mean.squeeze(-1), rstd.squeeze(-1), dy + (y.abs() + dy) * store + TINY, dm.squeeze(-1) + TINY, drstd.squeeze(-1)


def check_fwd(x, w, b, eps=1e-5, relu=False):
    out, mean, rstd = _ops().layer_norm_fwd(x, w, b, eps=eps, relu=relu)
    assert out.dtype == x.dtype and out.shape == x.shape and mean.shape == rstd.shape == x.shape[:-1] and mean.dtype == rstd.dtype == torch.float32
    y, m, r, dy, dm, dr = ln_bounds(x, w, b, eps, relu, STORE[x.dtype])
    inside(mean, m, dm, "mean")
    inside(rstd, r, dr, "rstd")
    inside(out, y, dy, "out")
    return out, mean, rstd


def check_bwd(x, w, mean, rstd, dout, act=None, **given):
    """Against the formula in 64 bits on the same mean and rstd."""
    before = {k: v.double() for k, v in given.items()}
    dx, dw, db = _ops().layer_norm_bwd(x, w, mean, rstd, dout, act=act, **given)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    D = x.shape[-1]
    rows = mean.numel()
    X, G = x.double().view(rows, D), dout.double().view(rows, D)
    m, r = mean.double().view(rows, 1), rstd.double().view(rows, 1)
    if act is not None:
        G = torch.where(act.view(rows, D) > 0, G, torch.zeros_like(G))
    xh = (X - m) * r
    g = G * w.double() if w is not None else G
    h = max(-(-D // 64), 32) + 10
    c1, c2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    a1, a2 = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    d1, d2 = (h + 2) * U * a1, (h + 5) * U * a2
    want = r * (g - c1 - xh * c2)
    bound = r * (3 * U * g.abs() + d1 + 4 * U * c1.abs() + xh.abs() * d2 + 6 * U * (xh * c2).abs()) * 1.01 + 2 * U * want.abs()
    inside(dx.view(rows, D), want, bound + (want.abs() + bound) * STORE[x.dtype] + TINY, "dx")
    if w is None:
        assert dw is None and db is None
        return dx, dw, db
    # sums over the rows: chains of at most rows / 64 rows in one place, then at most 1100 partial sums
    chain = min(rows, rows // 64 + 1100) + 6
    for name, got, terms in (("dweight", dw, G * xh), ("dbias", db, G)):
        assert got.dtype == torch.float32 and got.shape == (D,)
        total = terms.sum(0)
        bound = chain * U * terms.abs().sum(0) + 2 * U * total.abs() + TINY
        if given:
            total = total + before[name]
            bound = bound + U * total.abs()
        inside(got, total, bound, name)
    return dx, dw, db


DTYPES = [torch.float32, torch.bfloat16]
# the smallest rows, sizes around every vector width, wavefront and workgroup split, and past what a workgroup's registers hold
COLS = [1, 2, 3, 7, 8, 9, 31, 64, 65, 127, 128, 129, 255, 511, 512, 515, 1000, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4097, 8191, 8200, 16383,
        16384, 16385, 20011, 40000]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm_sizes(cols, dtype):
    """Every size with a few rows: forward with a ReLU, backward through it."""
    rows = 5 if cols > 4096 else 13
    x = (randn(rows, cols, seed=cols) * (1 + torch.arange(rows, device=DEV)[:, None]) + 0.5).to(dtype)
    w, b = 1 + 0.2 * randn(cols, seed=1), 0.3 * randn(cols, seed=2)
    act, mean, rstd = check_fwd(x, w, b, relu=True)
    check_bwd(x, w, mean, rstd, randn(rows, cols, seed=3, dtype=dtype), act=act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 2048), (2, 64), (63, 100), (64, 128), (65, 33), (257, 512), (1000, 2048), (4099, 1023), (10007, 515),
                                       (100003, 16), (70001, 3), (2049, 4100), (300, 16384), (129, 17000)])
def test_layer_norm_rows(rows, cols, dtype):
    x = randn(rows, cols, seed=rows, dtype=dtype)
    w, b = 1 + 0.2 * randn(cols, seed=1), 0.3 * randn(cols, seed=2)
    _, mean, rstd = check_fwd(x, w, b)
    check_bwd(x, w, mean, rstd, randn(rows, cols, seed=3, dtype=dtype))


# a whole and a cut length (bfloat16: an even and an odd one) for every number of threads a row and of chunks a thread that the forward and
# the backward of many rows take
MANY = {torch.float32: [5, 8, 13, 16, 21, 32, 50, 64, 99, 128, 201, 256, 400, 512, 770, 1024, 1300, 1536, 2047, 2048, 3001, 4096, 4101, 5120,
                        6656, 7003, 8192, 8197, 9216, 12001, 16384],
        torch.bfloat16: [9, 16, 17, 22, 27, 32, 40, 59, 64, 100, 123, 128, 200, 251, 256, 400, 507, 512, 900, 1019, 1024, 1500, 1536, 2043, 2048,
                         2100, 4091, 4096, 5000, 5120, 8187, 8192, 9216, 10000, 16377, 16384]}


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype,cols", [(t, c) for t in DTYPES for c in MANY[t]])
def test_layer_norm_many_rows(cols, dtype, masked):
    """More rows than one turn of the workgroups takes, and more than the backward of few rows is for: its partial rows go through
    scratch, which a call of the other kind would not ask for."""
    from vince_amd import _lib
    ops = _ops()
    w, b = 1 + 0.2 * randn(cols, seed=1), 0.3 * randn(cols, seed=2)
    for rows in (1031, 6007) if cols <= 1024 else (1031,):
        x = (randn(rows, cols, seed=rows + cols) * (0.5 + torch.arange(rows, device=DEV)[:, None] % 7) + 0.5).to(dtype)
        assert _lib.lib().vince_layer_norm_bwd_scratch_bytes(ops.dtype_code(x), rows, cols) > 0
        act, mean, rstd = check_fwd(x, w, b, relu=masked)
        check_bwd(x, w, mean, rstd, randn(rows, cols, seed=3, dtype=dtype), act=act if masked else None)


@pytest.mark.parametrize("cols", [16379, 16386, 18432, 20000, 20011, 32761, 32766, 32767, 32768])
def test_layer_norm_many_rows_of_the_forward_alone(cols):
    """bfloat16 rows that the forward's registers still hold and the backward's do not."""
    x = (randn(517, cols, seed=cols) * (0.5 + torch.arange(517, device=DEV)[:, None] % 7) + 0.5).bfloat16()
    check_fwd(x, 1 + 0.2 * randn(cols, seed=1), 0.3 * randn(cols, seed=2), relu=cols % 2 == 0)


@pytest.mark.parametrize("rows", [7, 1031])
@pytest.mark.parametrize("cols", [4099, 4352, 5000, 5120, 5121, 6143, 6144, 6145, 6400])
def test_layer_norm_rows_of_five_to_seven_wavefronts(cols, rows):
    """fp32 rows around the length from which a thread has two chunks instead of four: whole and cut ones, few and many."""
    x = randn(rows, cols, seed=cols) + 0.25
    w, b = 1 + 0.2 * randn(cols, seed=1), 0.3 * randn(cols, seed=2)
    act, mean, rstd = check_fwd(x, w, b, relu=True)
    check_bwd(x, w, mean, rstd, randn(rows, cols, seed=3), act=act)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_without_parameters_and_with_leading_axes(dtype):
    x = randn(3, 5, 7, 96, seed=4, dtype=dtype)
    w = 1 + 0.2 * randn(96, seed=1)
    _, mean, rstd = check_fwd(x, None, None)
    assert mean.shape == (3, 5, 7)
    check_bwd(x, None, mean, rstd, randn(3, 5, 7, 96, seed=5, dtype=dtype))
    check_fwd(x, w, None, eps=1e-2)
    check_bwd(x, w, mean, rstd, randn(3, 5, 7, 96, seed=5, dtype=dtype))
    check_fwd(x[0, 0, 0], w, w)                                                 # one row of no leading axis


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [33, 256, 1030])
def test_layer_norm_at_odd_addresses(cols, dtype):
    """Every tensor starts one element behind an aligned address, and the parameters too."""
    def odd(t):
        store = torch.empty(t.numel() + 1, device=DEV, dtype=t.dtype)
        store[1:].copy_(t.reshape(-1))
        return store[1:].view(t.shape)
    rows = 70
    x, w, b = odd(randn(rows, cols, seed=1, dtype=dtype)), odd(1 + 0.2 * randn(cols, seed=2)), odd(0.3 * randn(cols, seed=3))
    act, mean, rstd = check_fwd(x, w, b, relu=True)
    dw, db = odd(randn(cols, seed=7)), odd(randn(cols, seed=8))
    check_bwd(x, w, odd(mean), odd(rstd), odd(randn(rows, cols, seed=4, dtype=dtype)), act=odd(act), dweight=dw, dbias=db)


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("rows,cols", [(70, 131), (1500, 131), (1100, 2049), (1030, 3001), (600, 8201)])
def test_layer_norm_odd_rows_with_mixed_addresses(rows, cols, which):
    """bfloat16 rows of odd lengths, whose chunks follow the addresses of x: one of the tensors lies differently from the others."""
    def put(t, shift):
        store = torch.full((t.numel() + 16,), 9.0, device=DEV, dtype=t.dtype)
        store[shift:shift + t.numel()].copy_(t.reshape(-1))
        return store[shift:shift + t.numel()].view(t.shape)
    dtype = torch.bfloat16
    w, b = 1 + 0.2 * randn(cols, seed=2), 0.3 * randn(cols, seed=3)
    x = put(randn(rows, cols, seed=1, dtype=dtype), 5 if which == 0 else 0)
    act, mean, rstd = check_fwd(x, w, b, relu=which != 4)
    check_bwd(x, w, mean, rstd, put(randn(rows, cols, seed=4, dtype=dtype), 3 if which == 1 else 0), act=put(act, 7 if which == 2 else 0) if which < 4 else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [48, 2048, 17000])
def test_layer_norm_writes_its_rows_only(cols, dtype):
    """Memory behind the last row and behind the parameters' gradients stays as it was."""
    from vince_amd import _lib
    ops, L, rows = _ops(), _lib.lib(), 9
    x, dout = randn(rows, cols, seed=1, dtype=dtype), randn(rows, cols, seed=2, dtype=dtype)
    w = 1 + 0.2 * randn(cols, seed=3)
    pad = 4096
    def guard(n, t):   # noqa: E306
        return torch.full((n + pad,), 7.0, device=DEV, dtype=t)
    out, dx = guard(rows * cols, dtype), guard(rows * cols, dtype)
    mean, rstd, dw, db = guard(rows, torch.float32), guard(rows, torch.float32), guard(cols, torch.float32), guard(cols, torch.float32)
    nbytes = L.vince_layer_norm_bwd_scratch_bytes(ops.dtype_code(x), rows, cols)
    scratch = torch.full((nbytes + pad,), 7, device=DEV, dtype=torch.uint8)
    p = lambda t: t.data_ptr()   # noqa: E731
    _lib.check(L.vince_layer_norm_fwd(ops.dtype_code(x), p(x), p(w), None, p(out), p(mean), p(rstd), rows, cols, 1e-5, 0, ops.stream_ptr()))
    _lib.check(L.vince_layer_norm_bwd(ops.dtype_code(x), p(x), p(w), p(mean), p(rstd), p(dout), None, p(dx), p(dw), p(db), 0, rows, cols, p(scratch),
                                      nbytes, ops.stream_ptr()))
    torch.cuda.synchronize()
    for name, t, n in (("out", out, rows * cols), ("dx", dx, rows * cols), ("mean", mean, rows), ("rstd", rstd, rows), ("dweight", dw, cols),
                       ("dbias", db, cols), ("scratch", scratch, nbytes)):
        assert bool((t[n:] == 7).all()), name
    want = ops.layer_norm_bwd(x, w, mean[:rows].contiguous(), rstd[:rows].contiguous(), dout)
    assert torch.equal(want[0].view(-1), dx[:rows * cols]) and torch.equal(want[1], dw[:cols]) and torch.equal(want[2], db[:cols])


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_no_rows(dtype):
    ops = _ops()
    x, w = torch.empty(0, 4, 32, device=DEV, dtype=dtype), randn(32)
    out, mean, rstd = ops.layer_norm_fwd(x, w, w)
    assert out.shape == x.shape and mean.shape == (0, 4)
    dx, dw, db = ops.layer_norm_bwd(x, w, mean, rstd, x)
    assert dx.shape == x.shape and bool((dw == 0).all()) and bool((db == 0).all())     # the sum of no rows
    acc = randn(32, seed=5), randn(32, seed=6)
    kept = [t.clone() for t in acc]
    ops.layer_norm_bwd(x, w, mean, rstd, x, dweight=acc[0], dbias=acc[1])
    assert torch.equal(acc[0], kept[0]) and torch.equal(acc[1], kept[1])


@pytest.mark.parametrize("cols", [40, 600, 5000, 17000])
def test_layer_norm_values_that_are_not_finite_stay_in_their_row(cols):
    """A NaN or an infinity spoils its row's output and dx and its columns' sums; every other row has the bits it has without it.
    A gradient that is not finite at a place the ReLU masks counts as zero."""
    ops = _ops()
    rows = 11
    x, w, b, dout = randn(rows, cols, seed=1), 1 + 0.2 * randn(cols, seed=2), randn(cols, seed=3), randn(rows, cols, seed=4)
    out, mean, rstd = ops.layer_norm_fwd(x, w, b, relu=True)
    bad = x.clone()
    bad[3, cols // 2], bad[7, 1] = float("nan"), float("inf")
    out2, mean2, rstd2 = ops.layer_norm_fwd(bad, w, b, relu=True)
    rest = torch.tensor([i for i in range(rows) if i not in (3, 7)], device=DEV)
    assert torch.equal(out2[rest], out[rest]) and torch.equal(mean2[rest], mean[rest]) and torch.equal(rstd2[rest], rstd[rest])
    assert bool(out2[3].isnan().all()) and bool(out2[7].isnan().all()) and bool(mean2[3].isnan())
    dx, dw, _ = ops.layer_norm_bwd(x, w, mean, rstd, dout, act=out)
    hidden = torch.nonzero(out[5] == 0)[0, 0]
    d2 = dout.clone()
    d2[5, hidden] = float("nan")
    d2[6, torch.nonzero(out[6] == 0)[0, 0]] = float("inf")
    got = ops.layer_norm_bwd(x, w, mean, rstd, d2, act=out)
    assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
    seen = torch.nonzero(out[2] > 0)[0, 0]
    d2[2, seen] = float("nan")
    got = ops.layer_norm_bwd(x, w, mean, rstd, d2, act=out)
    keep = torch.tensor([i for i in range(rows) if i != 2], device=DEV)
    assert torch.equal(got[0][keep], dx[keep]) and bool(got[0][2].isnan().all())
    cols_kept = torch.arange(cols, device=DEV) != seen
    assert torch.equal(got[1][cols_kept], dw[cols_kept]) and bool(got[1][seen].isnan())


@pytest.mark.parametrize("cols", [5, 64, 515, 2048, 5000, 17000, 40000])
def test_layer_norm_small_variances_without_eps(cols):
    """eps = 0: rows of values down to 1e-18 (a variance of 1e-36, and one below the normal numbers) still come out normalised."""
    for scale in (1.0, 1e-10, 1e-18, 3e-20):
        x = randn(3, cols, seed=cols) * scale
        out, mean, rstd = _ops().layer_norm_fwd(x, eps=0.0)
        X = x.double()
        want = (X - X.mean(1, keepdim=True)) / X.var(1, unbiased=False, keepdim=True).sqrt()
        # (squares of 3e-20 are below 2^-126: each is off by up to 2^-150, a few 1e-6 of the variance 1e-39)
        assert float((out.double() - want).abs().max()) < (1e-4 if scale > 1e-19 else 2e-2), scale


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(7, 1), (3, 64), (4, 700), (5, 2048), (2, 4100), (3, 16384), (2, 20000), (1100, 1023)])
def test_layer_norm_of_one_value_is_the_bias(rows, cols, dtype):
    """Rows of one value whose multiples are exact in fp32: their mean is that value and the variance 0."""
    x = torch.full((rows, cols), 0.0, device=DEV)
    x += torch.tensor([0.0, 3.0, -1024.0, 0.5, 96.0], device=DEV).repeat(rows // 5 + 1)[:rows, None]
    b = randn(cols, seed=3)
    out, mean, _ = _ops().layer_norm_fwd(x.to(dtype), 1 + 0.2 * randn(cols, seed=2), b)
    assert torch.equal(out, b.to(dtype).expand(rows, cols)) and torch.equal(mean, x[:, 0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_level_and_extreme_rows(dtype):
    """Rows of one value (variance 0: the bias comes out), rows far from zero, large and small ones."""
    cols = 640
    x = torch.stack([torch.full((cols,), 0.0), torch.full((cols,), 3.0), torch.full((cols,), -1e4)]).to(DEV).to(dtype)
    w, b = 1 + 0.2 * randn(cols, seed=2), randn(cols, seed=3)
    out, mean, rstd = _ops().layer_norm_fwd(x, w, b)
    assert torch.equal(out, b.to(dtype).expand(3, cols)) and torch.equal(mean, x[:, 0].float())
    inside(rstd, torch.full((3,), 1e-5, dtype=torch.float64, device=DEV).rsqrt(), torch.full((3,), 4 * U * 317, dtype=torch.float64, device=DEV), "rstd")
    base = randn(6, cols, seed=5)
    check_fwd((base * torch.tensor([1e-3, 1.0, 1e3, 1e6, 1e15, 1.0], device=DEV)[:, None]
               + torch.tensor([0.0, 100.0, 0.0, 1e6, 0.0, -30.0], device=DEV)[:, None]).to(dtype), w, b)


def test_layer_norm_rows_past_32_bit_offsets():
    """2^31 + 4096 bfloat16 elements: rows behind the 2^31st element, against the same rows in a small call."""
    ops = _ops()
    cols, rows = 4096, (1 << 31) // 4096 + 1
    x = torch.empty(rows, cols, device=DEV, dtype=torch.bfloat16)
    step = 1 << 14
    block = randn(step, cols, seed=1, dtype=torch.bfloat16)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        x[r:r + n].copy_(block[:n])
    x[-1].copy_(randn(cols, seed=2, dtype=torch.bfloat16))
    w, b = 1 + 0.2 * randn(cols, seed=3), randn(cols, seed=4)
    out, mean, rstd = ops.layer_norm_fwd(x, w, b)
    tail = x[-3:].clone()
    o, m, r = ops.layer_norm_fwd(tail, w, b)
    assert torch.equal(out[-3:], o) and torch.equal(mean[-3:], m) and torch.equal(rstd[-3:], r) and torch.equal(out[:4], out[step:step + 4])
    del out
    dx, dw, db = ops.layer_norm_bwd(x, w, mean, rstd, x)
    d2 = ops.layer_norm_bwd(tail, w, m, r, tail)[0]
    assert torch.equal(dx[-3:], d2) and torch.equal(dx[:4], dx[step:step + 4])
    # db of a block that repeats: whole blocks times its column sums, and the last row
    want = block.double().sum(0) * ((rows - 1) // step) + x[-1].double()
    bound = (rows // 64 + 1100) * U * (block.double().abs().sum(0) * (rows // step + 1))
    inside(db, want, bound, "dbias")


@pytest.mark.parametrize("rows", [0, 1, 3])
@pytest.mark.parametrize("cols", [(1 << 25) + 1, (1 << 26) - 1, (1 << 26) + 1])
def test_layer_norm_bwd_of_very_long_rows(cols, rows):
    """dweight and dbias on both sides of the length at which a workgroup for every 32 of their columns would be 2^32 threads, which no
    launch has; no rows: their sum is 0.  mean and rstd are given, so that one row's dweight is a difference and two products."""
    dtype = torch.bfloat16
    x, dout = randn(rows, cols, seed=1, dtype=dtype), randn(rows, cols, seed=2, dtype=dtype)
    mean, rstd = torch.tensor([0.25, -0.5, 0.0], device=DEV)[:rows], torch.tensor([1.5, 0.75, 1.0], device=DEV)[:rows]
    dw, db = _ops().layer_norm_bwd(x, torch.ones(cols, device=DEV), mean, rstd, dout)[1:]
    xh = (x.float() - mean[:, None]) * rstd[:, None]
    # a difference, a product, a multiply-add a row, the partial rows' additions
    for name, got, terms in (("dweight", dw, dout.double() * xh.double()), ("dbias", db, dout.double())):
        inside(got, terms.sum(0), (rows + 4) * U * terms.abs().sum(0), name)


def test_layer_norm_bwd_of_the_longest_row():
    """2^31 - 1 columns: every column of dweight and dbias, added to what was there (128 million at a time)."""
    cols, step = (1 << 31) - 1, 1 << 27
    x = torch.empty(1, cols, device=DEV, dtype=torch.bfloat16)
    dout = torch.empty_like(x)
    for i in range(0, cols, step):
        n = min(step, cols - i)
        x[0, i:i + n] = randn(n, seed=i % 1000003, dtype=torch.bfloat16)
        dout[0, i:i + n] = randn(n, seed=i % 1000003 + 1, dtype=torch.bfloat16)
    mean, rstd = torch.tensor([0.25], device=DEV), torch.tensor([1.5], device=DEV)
    dw, db = torch.full((cols,), 2.0, device=DEV), torch.full((cols,), -3.0, device=DEV)
    _ops().layer_norm_bwd(x, torch.ones(cols, device=DEV), mean, rstd, dout, dweight=dw, dbias=db)
    for i in range(0, cols, step):
        d, xh = dout[0, i:i + step].double(), (x[0, i:i + step].double() - 0.25) * 1.5
        inside(dw[i:i + step], 2 + d * xh, 4 * U * (d * xh).abs() + U * (2 + d * xh).abs() * 1.01, "dweight")
        inside(db[i:i + step], d - 3, U * (d - 3).abs(), "dbias")


@pytest.mark.parametrize("value", [0.3, 1 / 3])
@pytest.mark.parametrize("cols", [40000, (1 << 25) + 3, 1 << 27])
def test_layer_norm_long_rows_of_one_value(cols, value):
    """Rows past a workgroup's registers, of one value that fp32 sums of a few hundred thousand of it do not hold: the mean is that value
    (chunks of four are exact, their fp64 sum has at most 24 + 25 bits, a cut chunk's one rounding is below 2^-24 / cols of the sum), the
    output the bias."""
    x = torch.full((1, cols), value, device=DEV)
    b = randn(cols, seed=3)
    out, mean, rstd = _ops().layer_norm_fwd(x, torch.ones(cols, device=DEV), b)
    assert torch.equal(mean, x[:, 0]) and torch.equal(out[0], b)
    want = torch.full((1,), float(np.float32(1e-5)), device=DEV, dtype=torch.float64).rsqrt()
    inside(rstd, want, 1.01 * U * want, "rstd")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [40001, (1 << 25) + 5])
def test_layer_norm_long_rows_are_as_good_as_short_ones(cols, dtype):
    """Bounds that do not grow with the row's length: sums of 8 values in a tree of three fp32 additions (3 u of the magnitudes), fp64
    sums of those.  Backward with a level dout, whose average c1 takes out of dx."""
    x = (randn(2, cols, seed=1) + torch.tensor([[0.5], [-2.0]], device=DEV)).to(dtype)
    w, b = 1 + 0.2 * randn(cols, seed=2), 0.3 * randn(cols, seed=3)
    out, mean, rstd = _ops().layer_norm_fwd(x, w, b)
    X, W = x.double(), w.double()
    m = X.mean(1, keepdim=True)
    xc = X - m
    var = (xc * xc).mean(1, keepdim=True)
    r = (var + float(np.float32(1e-5))).rsqrt()
    dm = 3.01 * U * X.abs().mean(1, keepdim=True) + 1.01 * U * m.abs()
    inside(mean[:, None], m, dm, "mean")
    # squares: twice the centred value's rounding and the mean's, the product's, the tree's; the mean's error has no first order in the sum
    dvar = 4.1 * U * var + dm * dm + 2.02 * U * (xc.abs() * (xc.abs() + dm)).mean(1, keepdim=True)
    dr = r * (0.5 * dvar / (var + 1e-5) * 1.01 + 1.01 * U)
    inside(rstd[:, None], r, dr, "rstd")
    xh = xc * r
    y = xh * W + b.double()
    dy = ((r * (dm + U * xc.abs()) + xc.abs() * dr + U * xh.abs()) * W.abs() + U * y.abs()) * 1.01
    inside(out, y, dy + (y.abs() + dy) * STORE[dtype] + TINY, "out")
    dout = torch.full_like(x, 0.3)
    dx, dw, db = _ops().layer_norm_bwd(x, w, mean, rstd, dout)
    G, m, r = dout.double(), mean.double()[:, None], rstd.double()[:, None]
    xh = (X - m) * r
    g = G * W
    c1, c2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    d1 = 5 * U * g.abs().mean(1, keepdim=True)                       # g's rounding, the tree, c1's own
    d2 = 8 * U * (g * xh).abs().mean(1, keepdim=True)                # xhat's two and g's, the product, the tree, c2's own
    want = r * (g - c1 - xh * c2)
    bound = r * (3 * U * g.abs() + d1 + 4 * U * c1.abs() + xh.abs() * d2 + 6 * U * (xh * c2).abs()) * 1.01 + 2 * U * want.abs()
    inside(dx, want, bound + (want.abs() + bound) * STORE[dtype] + TINY, "dx")
    inside(dw, (G * xh).sum(0), 7 * U * (G * xh).abs().sum(0), "dweight")         # xhat's two, two multiply-adds, the join's
    inside(db, G.sum(0), 4 * U * G.abs().sum(0), "dbias")


def test_layer_norm_gradients_against_differences():
    """dx, dweight and dbias of sum(c * y) against central differences of the forward formula in 64 bits; and of the kernel's own
    forward along random directions."""
    ops = _ops()
    rows, cols, eps = 4, 24, 1e-5
    x, w, b, c = randn(rows, cols, seed=1), 1 + 0.2 * randn(cols, seed=2), 0.3 * randn(cols, seed=3), randn(rows, cols, seed=4)

    def value(xx, ww, bb):
        m = xx.mean(1, keepdim=True)
        d = xx - m
        return (((d * d).mean(1, keepdim=True) + eps).rsqrt() * d * ww + bb).clamp(min=0).mul(c.double()).sum()

    act, mean, rstd = ops.layer_norm_fwd(x, w, b, eps=eps, relu=True)
    got = ops.layer_norm_bwd(x, w, mean, rstd, c, act=act)
    args = [x.double(), w.double(), b.double()]
    for k, grad in enumerate(got):
        flat = args[k].reshape(-1)
        for i in range(0, flat.numel(), 5):
            h = 1e-6
            old = flat[i].item()
            flat[i] = old + h
            up = value(*args)
            flat[i] = old - h
            down = value(*args)
            flat[i] = old
            # (h^2 times a third derivative of order 10, and 2^-53 of a value of order 30 over 2 h: both under 1e-8; fp32 roundings)
            assert abs(float(grad.reshape(-1)[i]) - float(up - down) / (2 * h)) < 2e-5, (k, i)
    # along a direction through the kernel's forward: outputs good to 1e-6, divided by 2 h = 2e-2, over 96 terms of order 1; curvature h^2
    for seed in range(3):
        v, h = randn(rows, cols, seed=50 + seed), 1e-2
        f = [float((ops.layer_norm_fwd(x + s * h * v, w, b, eps=eps)[0].double() * c.double()).sum()) for s in (1, -1)]
        lin = float((ops.layer_norm_bwd(x, w, mean, rstd, c)[0].double() * v.double()).sum())
        assert abs((f[0] - f[1]) / (2 * h) - lin) < 1e-2 * (1 + abs(lin)), seed


def test_layer_norm_is_reproducible_and_adds_to_what_is_there():
    ops = _ops()
    x, w, dout = randn(5003, 770, seed=1), 1 + 0.2 * randn(770, seed=2), randn(5003, 770, seed=3)
    _, mean, rstd = ops.layer_norm_fwd(x, w, None)
    first = ops.layer_norm_bwd(x, w, mean, rstd, dout)
    for _ in range(3):
        again = ops.layer_norm_bwd(x, w, mean, rstd, dout)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    dw, db = randn(770, seed=4), randn(770, seed=5)
    w0, b0 = dw.clone(), db.clone()
    r = ops.layer_norm_bwd(x, w, mean, rstd, dout, dweight=dw, dbias=db)
    assert r[1] is dw and r[2] is db and torch.equal(dw, w0 + first[1]) and torch.equal(db, b0 + first[2])


def test_layer_norm_refusals():
    ops = _ops()
    x, w = randn(4, 8), randn(8)
    out, mean, rstd = ops.layer_norm_fwd(x, w, w)
    for call, kind in [(lambda: ops.layer_norm_fwd(x.half()), TypeError), (lambda: ops.layer_norm_fwd(x.t()), RuntimeError),
                       (lambda: ops.layer_norm_fwd(x, w[:4].contiguous()), ValueError), (lambda: ops.layer_norm_fwd(x, w.bfloat16()), ValueError),
                       (lambda: ops.layer_norm_fwd(x, None, w), ValueError), (lambda: ops.layer_norm_fwd(x, w, eps=-1.0), ValueError),
                       (lambda: ops.layer_norm_fwd(x[:, :0].contiguous()), ValueError), (lambda: ops.layer_norm_fwd(x, w.cpu()), RuntimeError),
                       (lambda: ops.layer_norm_fwd(x[0, 0]), ValueError),
                       (lambda: ops.layer_norm_bwd(x, w, mean, rstd, x.bfloat16()), ValueError),
                       (lambda: ops.layer_norm_bwd(x, w, mean, rstd, x[:2].contiguous()), ValueError),
                       (lambda: ops.layer_norm_bwd(x, w, mean[:2].contiguous(), rstd, x), ValueError),
                       (lambda: ops.layer_norm_bwd(x, w, mean, rstd.double(), x), ValueError),
                       (lambda: ops.layer_norm_bwd(x, w, mean, rstd, x, act=x[:1].contiguous()), ValueError),
                       (lambda: ops.layer_norm_bwd(x, w, mean, rstd, x, dweight=w), ValueError),
                       (lambda: ops.layer_norm_bwd(x, None, mean, rstd, x, dweight=w, dbias=w), ValueError),
                       (lambda: ops.layer_norm_bwd(x, w, mean, rstd, x.cpu()), RuntimeError)]:
        with pytest.raises(kind):
            call()


# ------------------------------------------------------------------------------------------------ gradient norm and clipping
def flats(tensors):
    return torch.cat([t.double().reshape(-1) for t in tensors]) if tensors else torch.zeros(0, device=DEV, dtype=torch.float64)


def check_clip(tensors, max_norm, scales=None):
    """norm and coefficient against fp64 (both rounded to fp32 once), the gradients in place: the coefficient's rounding and the product's."""
    ops = _ops()
    before = [t.clone() for t in tensors]
    s = torch.cat([torch.full((t.numel(),), float(v), device=DEV, dtype=torch.float64) for t, v in zip(tensors, scales or [1.0] * len(tensors))])
    norm = float((flats(before) * s).norm())
    c = min(1.0, max_norm / (norm + 1e-6))
    table = ops.GradTable(tensors, scales)
    clip = ops.grad_norm(table, max_norm)
    assert clip.shape == (2,) and clip.dtype == torch.float32
    assert all(torch.equal(a, b) for a, b in zip(before, tensors))              # the norm alone changes nothing
    for got in (clip, ops.grad_clip(table, max_norm)):
        assert abs(float(got[0]) - norm) <= (U + 1e-12) * norm, (float(got[0]), norm)
        # (|c| is between norms: U of its own, and the fp64 norm's 1e-12)
        assert abs(float(got[1]) - c) <= (U + 1e-11) * c, (float(got[1]), c)
    for t, old in zip(tensors, before):
        want = old.double() * c
        inside(t, want, want.abs() * ((1 + STORE[t.dtype]) * (1 + 1.01 * U) - 1) + 2.0 ** -133, "gradient")
        if c == 1.0:
            assert torch.equal(t, old)
    return clip


@pytest.mark.parametrize("limit", [0.25, 1e9, 0.0, float("inf")])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 5, 255, 256, 1023, 4097, 16383, 16384, 16385, 32769, 65536, 100003, 3000001])
def test_grad_clip_one_tensor(n, dtype, limit):
    check_clip([randn(n, seed=n, dtype=dtype)], limit)


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("count", [2, 17, 160, 1500])
def test_grad_clip_many_tensors(count, offset):
    """Tensors of both types and very different sizes, empty ones among them, at odd addresses inside two buffers whose gaps stay."""
    rng = np.random.RandomState(count)
    sizes = (np.exp(rng.uniform(0, np.log(30000), count)).astype(int) * (rng.uniform(size=count) > 0.1)).tolist()
    sizes[0] = 70001
    place = {torch.float32: 0, torch.bfloat16: 0}
    spots = []
    for i, n in enumerate(sizes):
        t = DTYPES[i % 2]
        spots.append((t, place[t] + offset, n))
        place[t] += offset + n + 5
    store = {t: torch.full((m + 16,), 3.0, device=DEV, dtype=t) for t, m in place.items()}
    tensors = [store[t][a:a + n] for t, a, n in spots]
    used = {t: torch.zeros(m + 16, device=DEV, dtype=torch.bool) for t, m in place.items()}
    for (t, a, n), v in zip(spots, tensors):
        v.copy_(randn(n, seed=7 + a))
        used[t][a:a + n] = True
    check_clip(tensors, 2.0, scales=[0.5 + (i % 5) for i in range(count)])
    for t in DTYPES:
        assert bool((store[t][~used[t]] == 3.0).all())


def test_grad_norm_scales_of_any_size():
    """fp32 squares of these would overflow or vanish; the norm does neither."""
    ops = _ops()
    for scale in (1e-30, 1e-22, 1e-38, 1e20, 3e30, 1e36):
        g = randn(5000, seed=1) * scale
        n = float(g.double().norm())
        clip = ops.grad_norm([g], 1.0)
        assert abs(float(clip[0]) - n) <= 2 * U * n, scale
    big = [torch.full((9,), 3e38, device=DEV)]                                  # the norm itself is past fp32: shown as infinity, still clipped
    clip = ops.grad_clip(big, 1e38)
    assert float(clip[0]) == float("inf") and abs(float(clip[1]) - 1 / 9) < 1e-7 and abs(float(big[0][0]) / 3e38 - 1 / 9) < 1e-7


def test_grad_norm_of_values_that_are_not_finite():
    """As the formula has it: an infinite norm gives the coefficient 0 (0 * inf = NaN at its place, 0 elsewhere), a NaN a NaN."""
    ops = _ops()
    for bad, norm in ((float("nan"), float("nan")), (float("inf"), float("inf")), (-float("inf"), float("inf"))):
        for n in (5, 40000):
            g = randn(n, seed=2)
            g[n // 2] = bad
            clip = ops.grad_clip([g], 1.0).cpu()
            assert np.isnan(float(clip[0])) if np.isnan(norm) else float(clip[0]) == norm
            if np.isnan(norm):
                assert np.isnan(float(clip[1])) and bool(g.isnan().all())
            else:
                assert float(clip[1]) == 0.0 and bool(g[n // 2].isnan()) and int(g.isnan().sum()) == 1 and float(g[0].abs()) == 0.0
    assert ops.grad_norm([torch.full((3,), float("inf"), device=DEV)]).tolist() == [float("inf"), 1.0]      # no limit, no clipping


def test_grad_clip_layouts_and_refusals():
    ops = _ops()
    conv = randn(8, 4, 3, 3, seed=1).to(memory_format=torch.channels_last)
    check_clip([conv, randn(6, 10, seed=2).t(), randn(1, seed=3).view(()), torch.empty(0, 5, device=DEV)], 0.5)
    zeros = [torch.zeros(100, device=DEV)]
    assert ops.grad_clip(zeros, 1.0).tolist() == [0.0, 1.0]
    assert ops.grad_norm([torch.empty(0, device=DEV)], 1.0).tolist() == [0.0, 1.0]
    assert ops.grad_clip([torch.empty(0, device=DEV)], 1.0).tolist() == [0.0, 1.0]
    g = randn(100)
    for call, kind in [(lambda: ops.GradTable([g, g]), ValueError), (lambda: ops.GradTable([g[:60], g[59:]]), ValueError),
                       (lambda: ops.GradTable([g[::2]]), ValueError), (lambda: ops.GradTable([g.half()]), TypeError),
                       (lambda: ops.GradTable([g, g.cpu()]), RuntimeError), (lambda: ops.GradTable([g], [1.0, 2.0]), ValueError),
                       (lambda: ops.GradTable([g], [float("nan")]), RuntimeError), (lambda: ops.grad_norm([g], -1.0), ValueError),
                       (lambda: ops.grad_clip([g], float("nan")), ValueError), (lambda: ops.grad_scale([g], g), ValueError),
                       (lambda: ops.grad_scale([g], torch.ones(2)), RuntimeError),
                       (lambda: ops.sgd_flat(g, g[:50], g, 0.1, clip=torch.ones(2, device=DEV)), ValueError),
                       (lambda: ops.sgd_flat(g, g, g, 0.1, clip=torch.ones(3, device=DEV)), TypeError),
                       (lambda: ops.sgd_flat(g[1:], g[1:], g[1:], 0.1, clip=torch.ones(2, device=DEV)), RuntimeError)]:
        with pytest.raises(kind):
            call()


def test_grad_norm_past_32_bit_offsets():
    """One bfloat16 tensor of 2^31 + 11 elements."""
    ops = _ops()
    n = (1 << 31) + 11
    g = torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    g[-11:] = 2.0
    g[5] = 1.0
    clip = ops.grad_clip([g], 0.5)
    assert abs(float(clip[0]) - 45 ** 0.5) <= 2 * U * 7
    want = torch.tensor(2.0 * float(clip[1])).bfloat16()
    assert bool((g[-11:] == want.to(DEV)).all()) and float(g[-12]) == 0.0


def test_grad_table_from_two_streams_at_once():
    """Two norms of one table in flight: each call has scratch of its own."""
    ops = _ops()
    grads = [randn(n, seed=n) for n in (3000001, 17, 70000)]
    table = ops.GradTable(grads)
    want = ops.grad_norm(table, 1.0).clone()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.grad_norm(table, 1.0))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("n", [1, 3, 4, 1027, 296512, 5000003])
@pytest.mark.parametrize("limit", [0.1, 1e9])
def test_sgd_flat_with_a_clip(n, limit):
    """Against fp64; with nothing to clip the bits of the step without a clip."""
    ops = _ops()
    p, g, b = randn(n, seed=1), randn(n, seed=2), randn(n, seed=3)
    p0, b0 = p.clone(), b.clone()
    lr, mom, wd, gs = 0.03, 0.9, 1e-4, 0.5
    clip = ops.grad_norm(ops.GradTable([g], [gs]), limit)
    ops.sgd_flat(p, g, b, lr, mom, wd, grad_scale=gs, clip=clip)
    G, P, B = g.double(), p0.double(), b0.double()
    c = min(1.0, limit / (float((gs * G).norm()) + 1e-6))
    d = gs * c * G + wd * P
    wb = mom * B + d
    wp = P - lr * wb
    # constants enter as fp32 values: U each; d: scale (2), product, sum; buf: product and sum; p: product and sum
    db = (5 * U * (gs * c * G).abs() + 3 * U * (wd * P).abs() + 2 * U * (mom * B).abs() + 2 * U * wb.abs()) * 1.01
    inside(b, wb, db + TINY, "buf")
    inside(p, wp, lr * db + 2 * U * (lr * wb).abs() + U * wp.abs() + TINY, "param")
    if c == 1.0:
        p1, b1 = p0.clone(), b0.clone()
        ops.sgd_flat(p1, g, b1, lr, mom, wd, grad_scale=gs)
        assert torch.equal(p, p1) and torch.equal(b, b1)


# ------------------------------------------------------------------------------------------------ together
class _Step:
    """A projection head's training step as a program writes it: Linear, layer norm with ReLU, Linear, and back, into one flat buffer,
    then the clipped SGD step over it."""

    def __init__(self, seed, rows=96, width=256, out=64):
        torch.manual_seed(seed)
        self.shapes = [(width, width), (width,), (width,), (width,), (out, width), (out,)]
        sizes = [int(np.prod(s)) for s in self.shapes]
        self.flat = torch.randn(sum(sizes), device=DEV) * 0.05
        self.grad, self.buf = torch.zeros_like(self.flat), torch.zeros_like(self.flat)
        at = np.cumsum([0] + sizes)
        self.p = [self.flat[a:a + n].view(s) for a, n, s in zip(at, sizes, self.shapes)]
        self.g = [self.grad[a:a + n].view(s) for a, n, s in zip(at, sizes, self.shapes)]
        self.x, self.target = torch.randn(rows, width, device=DEV), torch.randn(rows, out, device=DEV)
        self.table = _ops().GradTable(self.g)

    def run(self):
        ops = _ops()
        w0, b0, nw, nb, w1, b1 = self.p
        h = ops.linear_fwd(self.x, w0, b0)
        a, mean, rstd = ops.layer_norm_fwd(h, nw, nb, relu=True)
        y = ops.linear_fwd(a, w1, b1)
        dy = (y - self.target) / y.shape[0]
        self.grad.zero_()
        da = ops.linear_bwd(a, ops.transpose_f32(w1), dy, self.g[4], self.g[5])
        dh = ops.layer_norm_bwd(h, nw, mean, rstd, da, act=a, dweight=self.g[2], dbias=self.g[3])[0]
        dx = ops.linear_bwd(self.x, ops.transpose_f32(w0), dh, self.g[0], self.g[1])
        clip = ops.grad_norm(self.table, 0.05)
        ops.sgd_flat(self.flat, self.grad, self.buf, 0.1, clip=clip)
        return dx, clip


def test_head_step_against_autograd():
    """The run of them together: gradients, norm and updated parameters of two steps against torch autograd in 64 bits with
    clip_grad_norm_ and torch.optim.SGD.  (relative to the largest entry: the Linears' fp32 sums of 256 products, 256 u = 1.5e-5, through
    three more layers)"""
    s = _Step(0)
    ref = [p.detach().double().clone().requires_grad_() for p in s.p]
    opt = torch.optim.SGD(ref, lr=0.1, momentum=0.9, weight_decay=1e-4)
    x = s.x.double().requires_grad_()
    for _ in range(2):
        dx, clip = s.run()
        opt.zero_grad()
        x.grad = None
        h = torch.nn.functional.layer_norm(x @ ref[0].t() + ref[1], (256,), ref[2], ref[3], 1e-5).relu()
        (0.5 * ((h @ ref[4].t() + ref[5] - s.target.double()) ** 2).sum() / 96).backward()
        norm = torch.nn.utils.clip_grad_norm_(ref, 0.05)
        assert float(norm) > 0.05 and abs(float(clip[0]) - float(norm)) < 1e-4 * float(norm)
        opt.step()
        assert float((dx.double() - x.grad).abs().max()) < 1e-4 * float(x.grad.abs().max())
        for mine, g, want in zip(s.p, s.g, ref):
            assert float((g.double() * clip[1].double() - want.grad).abs().max()) < 2e-4 * float(want.grad.abs().max()) + 1e-9
            assert float((mine.double() - want.detach()).abs().max()) < 2e-5 * float(want.detach().abs().max()) + 1e-7


def test_capture_and_replay():
    """Forward, backward, norm, clipping and step captured into a graph, replayed between eager calls of the same operators: every replay
    has the eager result's bits.  Two graphs over one table."""
    ops = _ops()
    x, w, b, dout = randn(777, 515, seed=1), 1 + 0.2 * randn(515, seed=2), randn(515, seed=3), randn(777, 515, seed=4)
    grads = [randn(n, seed=n) for n in (40001, 7, 300000)]
    fresh = [t.clone() for t in grads]
    table = ops.GradTable(grads)
    param, buf = randn(40000, seed=8), randn(40000, seed=9)
    p0, b0 = param.clone(), buf.clone()

    def work():
        for t, f in zip(grads, fresh):
            t.copy_(f)
        out, mean, rstd = ops.layer_norm_fwd(x, w, b, relu=True)
        dx, dw, db = ops.layer_norm_bwd(x, w, mean, rstd, dout, act=out)
        norm = ops.grad_norm(table, 0.3)
        clip = ops.grad_clip(table, 1.0)
        param.copy_(p0)
        buf.copy_(b0)
        ops.sgd_flat(param, grads[2][:40000], buf, 0.1, clip=norm)
        return [out, mean, rstd, dx, dw, db, norm, clip] + grads + [param, buf]

    want = [t.clone() for t in work()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = work()
            with pytest.raises(RuntimeError, match="before the capture"):
                ops.GradTable(grads)
        graphs.append((g, outs))
    for k in range(4):
        for g, outs in graphs:
            for t in outs:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            for i, (a, e) in enumerate(zip(outs, want)):
                assert torch.equal(a, e), (k, i)
        eager = work()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(eager, want))


def test_operators_on_a_side_stream():
    """Called under another stream, the work is ordered on that stream (inputs made there just before)."""
    ops = _ops()
    s = torch.cuda.Stream()
    x0, w = randn(2000, 2048, seed=1), 1 + 0.2 * randn(2048, seed=2)
    want = ops.layer_norm_fwd(x0 * 3 + 1, w, None)[0]
    norm = ops.grad_norm([x0 * 3 + 1])
    table = None
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s):
            x = x0 * 3
            x += 1
            got = ops.layer_norm_fwd(x, w, None)[0]
            table = ops.GradTable([x])
            n = ops.grad_norm(table)
        s.synchronize()
        assert torch.equal(got, want) and torch.equal(n, norm)


# ------------------------------------------------------------------------------------------------ the model and the solver
def _model(**kw):
    from vince_amd.config import make_args
    from vince_amd.models.vince_model import VinceModel
    torch.manual_seed(3)
    model = VinceModel(make_args(backbone="ResNet18", input_size=(64, 64), batch_size=16, vince_queue_size=64, **kw))
    for n, p in model.named_parameters():
        if "embedding_norm" in n:
            p.data.add_(0.2 * torch.randn(p.shape))
    model.to(DEV)
    model.train()
    return model


@pytest.mark.parametrize("jigsaw", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_model_head_norm_against_autograd(dtype, jigsaw):
    """VinceModel(head_norm="layer"): embeddings and head gradients against torch in 64 bits on the trunk's own features.  (bf16: the
    head's Linears multiply bfloat16 hi + lo halves, 2^-16 a product)"""
    import torch.nn.functional as F
    model = _model(compute_dtype=dtype, head_norm="layer", jigsaw=jigsaw)
    from oracle import vince_oracle as vo
    data = vo.structured_frames(8, 66 if jigsaw else 64, 66 if jigsaw else 64, seed=4).to(DEV)
    orders = torch.rand(8, 9, generator=torch.Generator().manual_seed(1)).argsort(1).to(DEV)
    model.zero_grad()
    spatial, pooled, pre, emb = model._run_encoder(data, jigsaw, orders if jigsaw else None)
    c = randn(*emb.shape, seed=5)
    (emb * c).sum().backward()
    torch.cuda.synchronize()
    if jigsaw:
        names = ["jigsaw_linear", "jigsaw_embedding.0", "jigsaw_embedding_norm", "jigsaw_embedding.2"]
    else:
        names = ["embedding.0", "embedding_norm", "embedding.2"]
    mods = dict(model.named_modules())
    ref = {n: [p.detach().double().contiguous().requires_grad_() for p in mods[n].parameters()] for n in names}
    f = pooled.detach().double()
    if jigsaw:
        f = F.linear(f, *ref["jigsaw_linear"]).view(8, 9, -1)
        f = torch.gather(f, 1, orders[:, :, None].expand_as(f)).reshape(8, -1)
    k = 1 if jigsaw else 0
    h = F.layer_norm(F.linear(f, *ref[names[k]]), (ref[names[k + 1]][0].numel(),), *ref[names[k + 1]], 1e-5).relu()
    want = F.normalize(F.linear(h, *ref[names[k + 2]]), dim=1)
    (want * c.double()).sum().backward()
    tol = 2e-4 if dtype == "fp32" else 3e-3
    assert float((emb.double() - want).abs().max()) < tol * float(want.abs().max())
    for n in names:
        for p, r in zip(mods[n].parameters(), ref[n]):
            assert float((p.grad.double() - r.grad).norm()) < 5 * tol * float(r.grad.norm()), n


@pytest.mark.parametrize("world", [1, 4])
def test_flat_sgd_with_max_grad_norm_is_clip_and_sgd(world):
    """FlatSGD(max_grad_norm) against torch's clip_grad_norm_ + SGD on copies of the same gradients, with a head that has never run.
    world 4: the buffer holds sums over ranks, of which the step and the norm take the mean (grad_scale)."""
    from oracle import vince_oracle as vo
    from vince_amd.optim import FlatSGD
    model = _model(compute_dtype="fp32", head_norm="layer", jigsaw=True)
    opt = FlatSGD(model, lr=0.1, max_grad_norm=0.5)
    opt.grad_scale = 1.0 / world
    named = [(n, p) for n, p in model.named_parameters() if p.grad is not None and not n.startswith("jigsaw")]
    ref = {n: p.detach().double().clone().requires_grad_() for n, p in named}
    idle = {n: p.detach().clone() for n, p in model.named_parameters() if n.startswith("jigsaw")}
    ropt = torch.optim.SGD(list(ref.values()), lr=0.1, momentum=0.9, weight_decay=1e-4)
    for it in range(3):
        data = vo.structured_frames(8, 64, 64, seed=it).to(DEV)
        model.zero_grad()
        emb = model._run_encoder(data)[3]
        (emb * randn(*emb.shape, seed=it)).sum().mul(5.0 if it < 2 else 1e-3).backward()
        before = {n: p.grad.clone() for n, p in named}
        for n, _ in named:
            ref[n].grad = before[n].double() / world
        norm = float(torch.nn.utils.clip_grad_norm_(list(ref.values()), 0.5))
        opt.step()
        ropt.step()
        assert abs(float(opt.last_clip[0]) - norm) < 1e-6 * norm and (float(opt.last_clip[1]) < 1) == (norm > 0.5)
        for n, p in named:
            assert torch.equal(p.grad, before[n])                              # the buffer's gradients are not rewritten
            assert float((p.detach().double() - ref[n].detach()).abs().max()) < 1e-5 * float(ref[n].abs().max()) + 1e-7, n
    assert all(torch.equal(dict(model.named_parameters())[n], v) for n, v in idle.items())


@pytest.mark.parametrize("limit", [0.05, 0.005])
def test_clipping_under_the_data_parallel_reducer(limit):
    """The single-rank form of a data-parallel step with clipping: the last gradient bucket arrives late, the norm waits for it, nothing
    stays pending, and the step is the plain solver's (bounds of two such fp32 steps: the atomics' order)."""
    import os
    import torch.distributed as dist
    from vince_amd.config import make_args
    from vince_amd.data_source import SyntheticFrames
    from vince_amd.solvers.vince_solver import VinceSolver

    def run(force):
        torch.manual_seed(0)
        os.environ.pop("VINCE_FORCE_DP", None)
        if force:
            os.environ["VINCE_FORCE_DP"] = "1"
        args = make_args(backbone="ResNet18", batch_size=16, vince_queue_size=64, input_size=(64, 64), compute_dtype="fp32", head_norm="layer",
                         max_grad_norm=limit, batch_source=SyntheticFrames(16, 64, 64, 1, device=DEV, seed=5))
        solver = VinceSolver(args)
        torch.manual_seed(1)
        solver.vince_queue.vector_queue.copy_(torch.nn.functional.normalize(torch.randn(64, 64), dim=1))
        solver.reset_epoch()
        p0 = solver.model._flat.clone()
        solver.run_train_iteration()
        torch.cuda.synchronize()
        m = solver.model
        assert (solver.reducer is not None) == force and m._late is None and m._deferred_step is None and not m._stem_pending
        norm, c = (float(v) for v in solver.optimizer.last_clip)
        want = min(1.0, limit / (norm + 1e-6))         # (this step's norm is 0.026: one limit above it, one below)
        assert abs(norm - float(m._flat_grad.double().norm())) < 1e-5 * norm and abs(c - want) < 1e-6 * want
        return norm, p0, m._flat.clone()

    os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
    os.environ.setdefault("MASTER_PORT", "29537")
    dist.init_process_group("nccl", rank=0, world_size=1)
    try:
        n0, a0, b0 = run(False)
        n1, a1, b1 = run(True)
    finally:
        os.environ.pop("VINCE_FORCE_DP", None)
        dist.destroy_process_group()
        from vince_amd._lib import lib
        lib().vince_set_side_streams(2)
    assert torch.equal(a0, a1) and abs(n0 - n1) < 2e-2 * n0
    assert float((b0 - b1).norm()) < 5e-2 * float((b0 - a0).norm())


def test_solver_with_head_norm_and_clipping():
    """VinceSolver with both options, side decoders included, deferred stem join on: every step's norm is finite and is the norm of the
    gradients it leaves (the side decoders' unscaled), the parameters move by the clipped amount, nothing stays pending."""
    from vince_amd.config import make_args
    from vince_amd.data_source import SyntheticFrames
    from vince_amd.solvers.vince_solver import VinceSolver

    class Labelled(SyntheticFrames):
        def __call__(self, loader_id=0):
            b = super().__call__(loader_id)
            b["data_source"] = "IN"
            b["imagenet_labels"] = (torch.arange(self.batch_size, device=self.device) * 37) % 1000
            return b

    torch.manual_seed(0)
    args = make_args(backbone="ResNet18", batch_size=16, vince_queue_size=64, input_size=(64, 64), compute_dtype="bf16", use_imagenet=True,
                     batch_source=Labelled(16, 64, 64, 1, device=DEV, seed=5), head_norm="layer", max_grad_norm=0.01)
    solver = VinceSolver(args)
    solver.reset_epoch()
    opt, model = solver.optimizer, solver.model
    assert solver.defer_stem and opt.max_grad_norm == 0.01
    for it in range(3):
        p0, b0 = model._flat[:model._n_train].clone(), opt.momentum_buffer.clone()
        loss = solver.run_train_iteration()[0]["nce_loss"]
        torch.cuda.synchronize()
        assert model._deferred_step is None and not model._stem_pending and model._late is None
        norm, c = (float(v) for v in opt.last_clip)
        extra = [p.grad.double() / c for p in model.imagenet_decoders.parameters()]
        want = float(torch.cat([model._flat_grad.double()] + [e.reshape(-1) for e in extra]).norm())
        assert np.isfinite(float(loss)) and norm > 0.01 and abs(norm - want) < 1e-5 * want and abs(c - 0.01 / norm) < 1e-3 * c
        d = model._flat_grad.double() * c + 1e-4 * p0.double()
        buf = 0.9 * b0.double() + d
        lr = opt.param_groups[0]["lr"]
        moved = p0.double() - lr * buf
        assert float((model._flat[:model._n_train].double() - moved).abs().max()) < 1e-6
    key = solver.queue_model.queue_network
    assert key.head_norm and torch.isfinite(key.embedding_norm.weight).all()
