"""layernorm_fwd / layernorm_bwd against 64 bits: types, widths, alignments and
strides, rows of one value, of equal values and far from zero, infinities and
NaN, the gradient against the formula and against differences, refusals."""
import threading

import pytest
import torch

from kernelproblems_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
EPS = 1e-5
# A row's sums: up to 130 terms one after the other and a tree of ten levels, in
# 32 bits: 140 * 2^-24, and a handful of single roundings behind them.
REL = 1e-5
U = 2.0 ** -24  # half a step of 32 bits


def rand(*shape, seed=0, std=1.0, mean=0.0, dtype=BF):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)


def weight(N, dtype=BF, seed=99):
    return (1 + 0.1 * rand(N, seed=seed, dtype=F32)).to(dtype)


def half_step(t64, dtype):
    """Half a step of the type at a value (2^-126 and below: of the smallest normal)."""
    return t64.abs().clamp_min(2.0 ** -126) * (torch.finfo(dtype).eps / 2)


def within(got, want, bound, what):
    d = (got.double() - want).abs()
    bad = d > bound
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {d.numel()}, worst over by {(d - bound).max().item():.3g}"


def check_fwd(x, w, b, res, out):
    y, h, mean, rstd = out
    N = x.shape[-1]
    h64 = x.double() if res is None else (res.double() + x.double()).to(x.dtype).double()
    if res is None:
        assert h is None
    elif h is not None:
        assert h.dtype == x.dtype and torch.equal(h.double(), h64)
    m64 = h64.mean(-1)
    far = h64 - m64[..., None]
    var = far.square().mean(-1)
    r64 = (var + EPS).rsqrt()
    w64 = torch.ones(N, dtype=torch.float64, device=DEV) if w is None else w.double()
    b64 = torch.zeros(N, dtype=torch.float64, device=DEV) if b is None else b.double()
    off = REL * h64.abs().mean(-1)  # of the mean
    # the deviations are all off by as much, their squares' sum by N times its square
    rel = REL + (off.square() / (var + EPS))
    if mean is not None:
        assert mean.dtype == F32 and rstd.dtype == F32 and mean.shape == x.shape[:-1]
        within(mean, m64, off, "mean")
        within(rstd, r64, rel * r64, "rstd")
    y64 = far * r64[..., None] * w64 + b64
    slack = ((off * r64)[..., None] + far.abs() * (r64 * (rel + REL))[..., None]) * w64.abs() + REL * b64.abs()
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    within(y, y64, half_step(y64, y.dtype) * 1.001 + slack, "y")


def check_bwd(dy, x, mean, rstd, w, dres, out, want_dw=True, want_db=True):
    dx, dw, db = out
    N = x.shape[-1]
    rows = lambda t: t.reshape(-1, N).double()  # noqa: E731
    d, r = rows(dy), rstd.reshape(-1, 1).double()
    xhat = (rows(x) - mean.reshape(-1, 1).double()) * r
    g = d * (1.0 if w is None else w.double())
    a, c = g.mean(-1, keepdim=True), (xhat * g).mean(-1, keepdim=True)
    want = (g - a - xhat * c) * r
    parts = (g.abs() + g.abs().mean(-1, keepdim=True) + xhat.abs() * (xhat * g).abs().mean(-1, keepdim=True)) * r
    if dres is not None:
        want = want + rows(dres)
    assert dx.dtype == x.dtype and dx.shape == x.shape and dx.is_contiguous()
    within(dx.reshape(-1, N), want, half_step(want, dx.dtype) * 1.001 + REL * parts, "dx")
    for name, got, wanted, terms in (("dw", dw, want_dw and w is not None, d * xhat), ("db", db, want_db, d)):
        if not wanted:
            assert got is None
            continue
        assert got.dtype == F32 and got.shape == (N,)
        within(got, terms.sum(0), REL * terms.abs().sum(0) + 1e-30, name)


SHAPES = [(1, 1), (3, 2), (3, 7), (40, 8), (37, 24), (1000, 64), (333, 80), (129, 128), (65, 129), (50, 250), (33, 256),
          (21, 264), (19, 512), (20, 511), (11, 1000), (10, 1001), (9, 1024), (9, 1025), (8, 1032), (17, 2568),
          (13, 2567), (1, 4096), (5, 4096), (7, 5120), (5, 5123), (6, 8192), (3, 8200), (3, 12288), (2, 12291),
          (2, 16384), (2, 16385), (3, 20000), (2, 30001)]


@pytest.mark.parametrize("M,N", SHAPES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_forward(M, N, dtype):
    x, w, b, res = (rand(M, N, seed=1, mean=0.5, dtype=dtype), weight(N, dtype), rand(N, seed=5, dtype=dtype),
                    rand(M, N, seed=2, dtype=dtype))
    check_fwd(x, w, b, res, ops.layernorm_fwd(x, w, b, EPS, residual=res))
    check_fwd(x, w, b, None, ops.layernorm_fwd(x, w, b, EPS))
    check_fwd(x, None, None, None, ops.layernorm_fwd(x, eps=EPS))
    other = F32 if dtype == BF else BF
    w2 = weight(N, other)
    y, h, mean, rstd = ops.layernorm_fwd(x, w2, None, EPS, residual=res, write_h=False, save_stats=False)
    assert h is None and mean is None and rstd is None
    check_fwd(x, w2, None, res, (y, h, mean, rstd))


def stats(x):
    far = x.double() - x.double().mean(-1, keepdim=True)
    return x.double().mean(-1).float(), (far.square().mean(-1) + EPS).rsqrt().float()


@pytest.mark.parametrize("M,N", SHAPES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradient(M, N, dtype):
    x, w = rand(M, N, seed=1, mean=0.5, dtype=dtype), weight(N, dtype)
    dy, dres = rand(M, N, seed=3, std=1e-2, dtype=dtype), rand(M, N, seed=4, std=1e-2, dtype=dtype)
    mean, rstd = stats(x)
    check_bwd(dy, x, mean, rstd, w, dres, ops.layernorm_bwd(dy, x, mean, rstd, w, dres=dres))
    check_bwd(dy, x, mean, rstd, w, None, ops.layernorm_bwd(dy, x, mean, rstd, w))
    check_bwd(dy, x, mean, rstd, None, None, ops.layernorm_bwd(dy, x, mean, rstd))
    check_bwd(dy, x, mean, rstd, w, dres, ops.layernorm_bwd(dy, x, mean, rstd, w, dres=dres, compute_db=False),
              want_db=False)
    w2 = weight(N, F32 if dtype == BF else BF)
    check_bwd(dy, x, mean, rstd, w2, None, ops.layernorm_bwd(dy, x, mean, rstd, w2, compute_dw=False), want_dw=False)
    out = ops.layernorm_bwd(dy, x, mean, rstd, w, compute_dw=False, compute_db=False)
    check_bwd(dy, x, mean, rstd, w, None, out, want_dw=False, want_db=False)


@pytest.mark.parametrize("M,N", [(5000, 64), (3001, 100), (2500, 768), (1500, 1001), (900, 4096), (700, 4099)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_rows(M, N, dtype):
    """Several rows for each block, the same bits in every run."""
    x, w, b = rand(M, N, seed=1, mean=2.0, dtype=dtype), weight(N, dtype), rand(N, seed=5, dtype=dtype)
    dy, dres = rand(M, N, seed=3, dtype=dtype), rand(M, N, seed=4, dtype=dtype)
    out = ops.layernorm_fwd(x, w, b, EPS)
    check_fwd(x, w, b, None, out)
    grads = ops.layernorm_bwd(dy, x, out[2], out[3], w, dres=dres)
    check_bwd(dy, x, out[2], out[3], w, dres, grads)
    again = ops.layernorm_bwd(dy, x, out[2], out[3], w, dres=dres)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    grads = ops.layernorm_bwd(dy, x, out[2], out[3], w)
    check_bwd(dy, x, out[2], out[3], w, None, grads)


def shifted(t, by):
    """A copy of t that starts `by` values behind a 16-byte boundary."""
    buf = torch.zeros(t.numel() + by + 8, dtype=t.dtype, device=DEV)
    out = buf[by:by + t.numel()].view(t.shape)
    out.copy_(t)
    return out


@pytest.mark.parametrize("N", [64, 100, 129, 1000, 1001, 1003, 4096, 4098, 9001])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("by", [(1, 1, 1), (3, 3, 3), (4, 4, 4), (0, 1, 2), (2, 0, 0)])
def test_any_alignment(N, dtype, by):
    M = 13
    x, w, b, res = (rand(M, N, seed=1, dtype=dtype), weight(N, dtype), rand(N, seed=5, dtype=dtype),
                    rand(M, N, seed=2, dtype=dtype))
    dy = rand(M, N, seed=3, dtype=dtype)
    mean, rstd = stats(x)
    x1, r1, d1 = shifted(x, by[0]), shifted(res, by[1]), shifted(dy, by[2])
    check_fwd(x, w, b, res, ops.layernorm_fwd(x1, shifted(w, 1), shifted(b, 3), EPS, residual=r1))
    check_bwd(dy, x, mean, rstd, w, res, ops.layernorm_bwd(d1, x1, mean, rstd, shifted(w, 1), dres=r1))


@pytest.mark.parametrize("N,wide", [(64, 192), (128, 129), (1000, 1008), (1001, 1009), (4096, 12288), (96, 97), (257, 1024)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_row_strides(N, wide, dtype):
    """Rows inside wider ones, as slices of a packed projection are."""
    M = 50
    packed = [rand(M, wide, seed=s, dtype=dtype) for s in (1, 2, 3, 4)]
    x, res, dy, dres = (t[:, wide - N:] for t in packed)
    w, b = weight(N, dtype), rand(N, seed=5, dtype=dtype)
    check_fwd(x, w, b, res, ops.layernorm_fwd(x, w, b, EPS, residual=res))
    mean, rstd = stats(x)
    check_bwd(dy, x, mean, rstd, w, dres, ops.layernorm_bwd(dy, x, mean, rstd, w, dres=dres))
    one = x[:1].expand(M, N)  # every row the same memory
    check_fwd(one, w, b, None, ops.layernorm_fwd(one, w, b, EPS))


def test_shapes_and_empty():
    w = weight(64)
    y, h, mean, rstd = ops.layernorm_fwd(rand(2, 3, 64), w, w, residual=rand(2, 3, 64, seed=1))
    assert y.shape == h.shape == (2, 3, 64) and mean.shape == rstd.shape == (2, 3)
    y, h, mean, rstd = ops.layernorm_fwd(rand(64), w)
    assert y.shape == (64,) and mean.shape == ()
    dx, dw, db = ops.layernorm_bwd(rand(64), rand(64), mean, rstd, w)
    assert dx.shape == (64,) and dw.shape == db.shape == (64,)
    y, h, mean, rstd = ops.layernorm_fwd(rand(0, 64), w)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dw, db = ops.layernorm_bwd(rand(0, 64), rand(0, 64), mean, rstd, w)
    assert dx.shape == (0, 64) and bool((dw == 0).all()) and bool((db == 0).all())
    y, _, mean, _ = ops.layernorm_fwd(rand(0, 0))
    assert y.shape == (0, 0) and mean.shape == (0,)


@pytest.mark.parametrize("N", [1, 8, 64, 129, 1000, 1001, 4096, 20000])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_without_spread(N, dtype):
    """Equal values: no deviation, rstd 1 / sqrt(eps), y the bias.  (Whole numbers: their sums are exact.)"""
    x = torch.tensor([0.0, 3.0, -7.0], device=DEV)[:, None].expand(3, N).to(dtype).contiguous()
    w, b = weight(N, dtype), rand(N, seed=5, dtype=dtype)
    y, _, mean, rstd = ops.layernorm_fwd(x, w, b, EPS)
    # the mean is one division of an exact sum, and each row's deviations at most its rounding
    assert bool((mean - x[:, 0].float()).abs().max() <= 7 * 2.0 ** -23)
    assert torch.allclose(rstd, torch.full_like(rstd, EPS ** -0.5), rtol=1e-5)
    within(y, b.double().expand(3, N), half_step(b.double(), dtype) + 7 * 2.0 ** -23 * EPS ** -0.5 * w.double().abs(), "y")


@pytest.mark.parametrize("N", [64, 1000, 1001, 4096, 20000])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_values_that_are_not_finite_stay_in_their_row(N, dtype):
    x, w, dy = rand(6, N, seed=1, dtype=dtype), weight(N, dtype), rand(6, N, seed=2, dtype=dtype)
    clean = ops.layernorm_fwd(x, w, None, EPS)
    bad = x.clone()
    bad[1, N // 2], bad[3, 0], bad[4, N - 1] = float("inf"), float("nan"), float("-inf")
    got = ops.layernorm_fwd(bad, w, None, EPS)
    for i in (0, 2, 5):
        assert torch.equal(got[0][i], clean[0][i]) and got[2][i] == clean[2][i] and got[3][i] == clean[3][i]
    for i in (1, 3, 4):
        assert bool(torch.isnan(got[0][i]).all()) and bool(torch.isnan(got[3][i]))
    a = ops.layernorm_bwd(dy, x, clean[2], clean[3], w)
    b = ops.layernorm_bwd(dy, bad, got[2], got[3], w)
    for i in (0, 2, 5):
        assert torch.equal(a[0][i], b[0][i])
    for i in (1, 3, 4):
        assert bool(torch.isnan(b[0][i]).all())
    assert bool(torch.isnan(b[1]).all()) and torch.equal(a[2], b[2])


@pytest.mark.parametrize("N", [64, 1000, 1001, 4096, 20000])
def test_a_mean_far_from_zero(N):
    """A thousand deviations from zero: the deviations keep the digits that 32 bits leave them."""
    x = rand(40, N, seed=1, mean=1000.0, dtype=F32)
    check_fwd(x, weight(N, F32), None, None, ops.layernorm_fwd(x, weight(N, F32), None, EPS))


FAR = [1, 3, 7, 64, 100, 129, 500, 1000, 1001, 4096, 4099, 8192, 12288, 16384, 20000]


@pytest.mark.parametrize("N", FAR)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("residual", [False, True])
def test_rows_of_one_value(N, dtype, residual):
    """Any value, not whole numbers alone: the mean is that value, y the bias, to the last bit."""
    values = torch.tensor([1000.3, -0.1, 3e-3, 12345.678, 0.0, -7e4], device=DEV)
    x = values[:, None].expand(6, N).to(dtype).contiguous()
    w, b = weight(N, dtype), rand(N, seed=5, dtype=dtype)
    y, h, mean, rstd = ops.layernorm_fwd(x, w, b, EPS, residual=0.5 * x if residual else None)
    h = h if residual else x
    assert torch.equal(mean, h[:, 0].float())
    assert torch.equal(y, b.expand(6, N))
    # distances from a mean of some roundings, of the row and of parts of it
    var = (4 * U * h[:, 0].double()).square() + 8 * U * (REL * h[:, 0].double()).square()
    within(rstd, torch.full_like(var, EPS ** -0.5), EPS ** -0.5 * (var / EPS + 8 * U), "rstd")


@pytest.mark.parametrize("N", [16392, 100001, 3_000_001])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_long_rows_of_one_value(N, dtype):
    x = torch.tensor([1000.3, -0.1, 12345.678], device=DEV)[:, None].expand(3, N).to(dtype).contiguous()
    b = rand(N, seed=5, dtype=dtype)
    y, _, mean, _ = ops.layernorm_fwd(x, weight(N, dtype), b, EPS)
    assert torch.equal(mean, x[:, 0].float()) and torch.equal(y, b.expand(3, N))


@pytest.mark.parametrize("N", FAR[3:])
@pytest.mark.parametrize("far", [1e3, -1e4])
def test_a_mean_far_from_zero_is_off_by_its_last_place(N, far):
    x, w = rand(40, N, seed=1, mean=far, dtype=F32), weight(N, F32)
    y, _, mean, rstd = ops.layernorm_fwd(x, w, None, EPS)
    m64 = x.double().mean(-1)
    d = x.double() - m64[:, None]
    var = d.square().mean(-1)
    r64 = (var + EPS).rsqrt()
    # its own rounding; the distances' sums, of the deviations and of what the first mean is off by
    off = U * m64.abs() * 1.001 + REL * (d.abs().mean(-1) + REL * m64.abs())
    rel = REL + 8 * U * (REL * m64).square() / (var + EPS)
    within(mean, m64, off, "mean")
    within(rstd, r64, rel * r64, "rstd")
    y64 = d * r64[:, None] * w.double()
    slack = (off[:, None] + d.abs() * (rel + 4 * U)[:, None]) * r64[:, None] * w.double().abs()
    within(y, y64, slack, "y")


@pytest.mark.parametrize("N", FAR)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_the_mean_of_a_row_with_infinities(N, dtype):
    """Is infinite, or not a number where two of them have two signs; the rows beside it are as they were."""
    x = rand(4, N, seed=1, dtype=dtype)
    clean = ops.layernorm_fwd(x, None, None, EPS)
    x[1, N // 2], x[2, N - 1], x[2, 0] = float("inf"), float("-inf"), float("inf") if N > 1 else float("-inf")
    y, _, mean, rstd = ops.layernorm_fwd(x, None, None, EPS)
    assert mean[1] == float("inf") and (bool(torch.isnan(mean[2])) if N > 1 else mean[2] == float("-inf"))
    assert bool(torch.isnan(y[1:3]).all()) and bool(torch.isnan(rstd[1:3]).all())
    for i in (0, 3):
        assert torch.equal(y[i], clean[0][i]) and mean[i] == clean[2][i] and rstd[i] == clean[3][i]


@pytest.mark.parametrize("N", [48, 129, 1024, 2567])
def test_gradient_against_differences(N):
    M, step = 6, 1e-2
    x, w, b, dy = (rand(M, N, seed=1, dtype=F32), weight(N, F32), rand(N, seed=5, dtype=F32), rand(M, N, seed=2, dtype=F32))
    _, _, mean, rstd = ops.layernorm_fwd(x, w, b, EPS)
    dx, dw, db = ops.layernorm_bwd(dy, x, mean, rstd, w)
    loss = lambda x, w, b: (ops.layernorm_fwd(x, w, b, EPS)[0].double() * dy.double()).sum()  # noqa: E731
    for name, grad, args in (("x", dx, (0,)), ("w", dw, (1,)), ("b", db, (2,))):
        d = rand(*grad.shape, seed=7, dtype=F32)
        plus, minus = ([t + s * d if i in args else t for i, t in enumerate((x, w, b))] for s in (step, -step))
        diff = (loss(*plus) - loss(*minus)) / (2 * step)
        want = (grad.double() * d.double()).sum()
        # the third derivative's term (step^2 times values of order one), and y's roundings over the step
        bound = (step ** 2 + 2.0 ** -22 / step) * (dy.double().norm() * d.double().norm() * (1 if name == "x" else M ** 0.5))
        assert abs(diff - want) <= bound, f"{name}: {diff.item()} {want.item()} {bound.item()}"


def test_values_past_2_31():
    """The last rows lie beyond what 32 bits count."""
    M, N = (1 << 18) + 5, 8192
    x = torch.zeros(M, N, dtype=BF, device=DEV)
    dy = torch.zeros(M, N, dtype=BF, device=DEV)
    at = torch.tensor([0, 1, 262143, 262144, M - 1], device=DEV)
    x[at], dy[at] = rand(5, N, seed=1, mean=0.5), rand(5, N, seed=2)
    w = weight(N)
    y, _, mean, rstd = ops.layernorm_fwd(x, w, None, EPS)
    check_fwd(x[at], w, None, None, (y[at], None, mean[at], rstd[at]))
    assert bool((y[2:1000] == 0).all()) and bool((y[-1000:-10] == 0).all())
    del y
    dx, dw, db = ops.layernorm_bwd(dy, x, mean, rstd, w)
    check_bwd(dy[at], x[at], mean[at], rstd[at], w, None, (dx[at], dw, db))


@pytest.mark.parametrize("M,N,dtype,by", [(262144, 8192, F32, 0), (1 << 24, 64, F32, 0), (1 << 23, 96, BF, 0), (1 << 20, 64, F32, 1),
                                          (1 << 20, 1000, BF, 0), (70000, 16000, BF, 0), (300000, 1001, F32, 0)])
def test_long_sums_of_rows_that_are_alike(M, N, dtype, by):
    """Every row the same, so that the roundings of a column's sum all go one way; over
    hundreds and thousands of rows for a thread.  by: dy lies unlike x."""
    x, w = rand(1, N, seed=1, mean=0.5, dtype=dtype), weight(N, dtype)
    dy = rand(1, N, seed=3, dtype=dtype)
    dy[0, 0], dy[0, 1] = 0.3, 0.1
    one = lambda t: t.expand(M, N)  # noqa: E731
    mean, rstd = stats(x)
    dx, dw, db = ops.layernorm_bwd(one(shifted(dy, by) if by else dy), one(x), mean.expand(M).contiguous(),
                                   rstd.expand(M).contiguous(), w)
    assert all(torch.equal(dx[i], dx[0]) for i in (1, M // 2, M - 1))
    del dx
    term = dy[0].double()
    within(db, M * term, REL * M * term.abs(), "db")
    term = term * (x[0].double() - mean.double()) * rstd.double()
    # (and each term's own two roundings)
    within(dw, M * term, (REL + 2.0 ** -23) * M * term.abs(), "dw")


@pytest.mark.parametrize("N", [40, 129, 600, 1001, 2570, 4099, 8192, 16001])
@pytest.mark.parametrize("by", [1, 3, 4])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_all_tensors_alike_off_a_boundary(N, by, dtype):
    """The C ABI with outputs, too, `by` values behind a boundary.  The first row's begin and
    the last one's end are then not copied but written into their place in the ring, which
    the rows behind go over: the same, right results in several runs, and nothing beside them."""
    M = 6000 if N < 2000 else 2500
    code = _lib.FRAG_DT_BF16 if dtype == BF else _lib.FRAG_DT_F32
    ptr = lambda t: t.data_ptr()  # noqa: E731
    x, dy, w, b = rand(M, N, seed=1, mean=0.5, dtype=dtype), rand(M, N, seed=3, dtype=dtype), weight(N, dtype), rand(N, dtype=dtype)
    xs, ds = shifted(x, by), shifted(dy, by)
    mean, rstd = torch.empty(M, device=DEV), torch.empty(M, device=DEV)
    dw, db = torch.empty(N, device=DEV), torch.empty(N, device=DEV)
    need = _lib.load().frag_layernorm_bwd_workspace_bytes(M, N)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    held = []
    for _ in range(10):
        y, h, dx = (shifted(torch.zeros_like(x), by) for _ in range(3))
        _lib.call("frag_layernorm_fwd", ptr(xs), N, ptr(ds), N, ptr(w), ptr(b), ptr(y), ptr(h), ptr(mean), ptr(rstd),
                  M, N, EPS, code, code, torch.cuda.current_stream().cuda_stream)
        _lib.call("frag_layernorm_bwd", ptr(ds), N, ptr(h), N, ptr(mean), ptr(rstd), ptr(w), ptr(xs), N, ptr(dx),
                  ptr(dw), ptr(db), M, N, code, code, ptr(ws), need, torch.cuda.current_stream().cuda_stream)
        for t in (y, h, dx):
            around = t.view(-1).as_strided((t.numel() + by + 8,), (1,), 0)
            assert not bool(around[:by].any()) and not bool(around[by + t.numel():].any())
        held.append([t.clone() for t in (y, h, mean, rstd, dx, dw, db)])
    y, h, mean, rstd, dx, dw, db = held[0]
    check_fwd(x, w, b, dy, (y, h, mean, rstd))
    check_bwd(dy, h, mean, rstd, w, x, (dx, dw, db))
    assert all(torch.equal(a, c) for again in held[1:] for a, c in zip(held[0], again))


@pytest.mark.parametrize("N", [16385, 1 << 20, 3_000_001])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_long_rows_of_values_that_are_alike(N, dtype):
    """Thousands of terms for a thread, whose roundings all go one way: the squares of
    values of one magnitude, and gradients that are equal."""
    x = torch.full((3, N), 0.3, device=DEV)
    x[:, ::2] *= -1
    x[1] += 0.7  # (and a mean that is not zero)
    x, w = x.to(dtype), weight(N, dtype)
    dy = torch.full((3, N), 0.1, device=DEV).to(dtype)
    dy[2] += rand(N, seed=1, dtype=dtype)
    out = ops.layernorm_fwd(x, w, None, EPS)
    check_fwd(x, w, None, None, out)
    check_fwd(x, None, None, 2 * x, ops.layernorm_fwd(x, None, None, EPS, residual=2 * x))
    check_bwd(dy, x, out[2], out[3], w, None, ops.layernorm_bwd(dy, x, out[2], out[3], w))
    check_bwd(dy, x, out[2], out[3], None, None, ops.layernorm_bwd(dy, x, out[2], out[3], None))


def test_streams_and_graphs():
    x, w, b, dy = rand(64, 4096, seed=1), weight(4096), rand(4096, seed=5), rand(64, 4096, seed=2)
    want = ops.layernorm_fwd(x, w, b)
    grads = ops.layernorm_bwd(dy, x, want[2], want[3], w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.layernorm_fwd(x, w, b)
        og = ops.layernorm_bwd(dy, x, other[2], other[3], w)
    side.synchronize()
    assert torch.equal(other[0], want[0]) and all(torch.equal(a, c) for a, c in zip(og, grads))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.layernorm_fwd(x, w, b)
        hg = ops.layernorm_bwd(dy, x, held[2], held[3], w)
    x.copy_(rand(64, 4096, seed=8))
    dy.copy_(rand(64, 4096, seed=9))
    graph.replay()
    torch.cuda.synchronize()
    want = ops.layernorm_fwd(x, w, b)
    grads = ops.layernorm_bwd(dy, x, want[2], want[3], w)
    assert torch.equal(held[0], want[0]) and all(torch.equal(a, c) for a, c in zip(hg, grads))


@pytest.mark.parametrize("M,N", [(1, 64), (9, 513), (1000, 129), (1 << 20, 64), (1 << 20, 121), (200001, 505), (300000, 520),
                                 (100003, 1001), (60000, 8192), (40001, 16001), (4000, 20000)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_the_workspace_is_enough(M, N, dtype):
    """Nothing is written behind the bytes that the gradient asks for."""
    x, w = rand(1, N, seed=1, mean=0.5, dtype=dtype), weight(N, dtype)
    mean, rstd = (t.expand(M).contiguous() for t in stats(x))
    dy = rand(1, N, seed=2, dtype=dtype)
    need = _lib.load().frag_layernorm_bwd_workspace_bytes(M, N)
    ws = torch.full((need + (8 << 20),), 77, dtype=torch.uint8, device=DEV)
    dx, dw, db = torch.empty(M, N, dtype=dtype, device=DEV), torch.empty(N, device=DEV), torch.empty(N, device=DEV)
    code = _lib.FRAG_DT_BF16 if dtype == BF else _lib.FRAG_DT_F32
    for dres in (None, x.data_ptr()):
        _lib.call("frag_layernorm_bwd", dy.data_ptr(), 0, x.data_ptr(), 0, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(),
                  dres, 0, dx.data_ptr(), dw.data_ptr(), db.data_ptr(), M, N, code, code, ws.data_ptr(), need,
                  torch.cuda.current_stream().cuda_stream)
        assert bool((ws[need:] == 77).all())
        within(db, M * dy[0].double(), REL * M * dy[0].double().abs(), "db")


def test_more_blocks_than_an_sm_holds_in_a_graph():
    """The pass that adds the partials starts beside the last of the gradient's blocks, and
    waits for all of them: captured, and replayed on other values."""
    M, N = 310000, 520
    x, dy, w = rand(M, N, seed=1, mean=0.5), rand(M, N, seed=2), weight(N)
    mean, rstd = stats(x)
    ops.layernorm_bwd(dy, x, mean, rstd, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [ops.layernorm_bwd(dy, x, mean, rstd, w) for _ in range(2)]
    for seed in (3, 4):
        dy.copy_(rand(M, N, seed=seed))
        graph.replay()
        want = ops.layernorm_bwd(dy, x, mean, rstd, w)
        assert all(torch.equal(a, b) for out in held for a, b in zip(out, want))
    check_bwd(dy, x, mean, rstd, w, None, want)


def test_two_threads_behind_every_variant():
    """A kernel's largest shared memory is remembered for each of more than a hundred
    kernels: where one found no place, two threads' calls of it with different widths
    would lower it under each other's launches."""
    for dtype in (BF, F32):
        for N in (48, 120, 248, 504, 1000, 1024, 49, 121, 249, 499, 1001, 2049):
            x = rand(5, N, seed=N, dtype=dtype)
            mean, rstd = stats(x)
            for w in (weight(N, BF), weight(N, F32)):
                for res in (None, x):
                    check_fwd(x, w, None, res, ops.layernorm_fwd(x, w, None, EPS, residual=res))
                    check_bwd(x, x, mean, rstd, w, res, ops.layernorm_bwd(x, x, mean, rstd, w, dres=res))
    for N in (64, 512, 1000, 1024, 2048, 4096, 5120, 8192, 12288, 16384):
        x, w = rand(64, N, seed=N), weight(N)
        ops.rmsnorm_fwd(x, w)
        ops.add_rmsnorm_fwd(x, x, w)
    errors = []

    def run(N, M, stream):
        with torch.cuda.stream(stream):
            x, w = rand(M, N, seed=N), weight(N)
            want = ops.layernorm_fwd(x, w, None, EPS)
            grads = ops.layernorm_bwd(x, x, want[2], want[3], w)
            try:
                for _ in range(300):
                    out = ops.layernorm_fwd(x, w, None, EPS)
                    assert torch.equal(out[0], want[0])
                    assert all(torch.equal(a, b) for a, b in zip(ops.layernorm_bwd(x, x, want[2], want[3], w), grads))
            except Exception as e:  # noqa: BLE001
                errors.append(e)
    threads = [threading.Thread(target=run, args=(N, M, torch.cuda.Stream())) for N, M in ((1032, 4), (16376, 2000), (8200, 300))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]


def test_workspace():
    M, N = 200, 1000
    x, dy, w = rand(M, N, seed=1), rand(M, N, seed=2), weight(N)
    mean, rstd = stats(x)
    want = ops.layernorm_bwd(dy, x, mean, rstd, w)
    for size in (16, 64 << 20):
        ws = torch.empty(size, dtype=torch.uint8, device=DEV)
        got = ops.layernorm_bwd(dy, x, mean, rstd, w, workspace=ws)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("N", [64, 4096])
def test_tensors_that_hold_no_values_are_refused(N):
    """What torch.func's transforms hand on has no memory of its own: an error, and the next call is as ever."""
    x, w = rand(4, N, seed=1), weight(N)
    want = ops.layernorm_fwd(x, w)
    for call in (lambda: torch.func.grad(lambda t: ops.layernorm_fwd(t, w)[0].float().sum())(x),
                 lambda: torch.func.vmap(lambda t: ops.layernorm_fwd(t, w)[0])(x[None]),
                 lambda: torch.func.grad(lambda t: ops.layernorm_fwd(x, t)[0].float().sum())(w),
                 lambda: torch.func.grad(lambda t: ops.layernorm_fwd(x, w, residual=t)[0].float().sum())(x),
                 lambda: torch.func.vmap(lambda t: ops.layernorm_bwd(t, x, want[2], want[3], w)[0])(x[None]),
                 lambda: torch.func.grad(lambda t: ops.grad_norm([x, t])[0])(x)):
        with pytest.raises(RuntimeError):
            call()
        assert torch.equal(ops.layernorm_fwd(x, w)[0], want[0])


def test_refusals():
    x, w = rand(4, 64), weight(64)
    mean, rstd = stats(x)
    bad = [(TypeError, lambda: ops.layernorm_fwd(x.half(), w)), (TypeError, lambda: ops.layernorm_fwd(x, w.half())),
           (TypeError, lambda: ops.layernorm_fwd(x, w, w.float())), (ValueError, lambda: ops.layernorm_fwd(x, w[:32])),
           (ValueError, lambda: ops.layernorm_fwd(x.cpu(), w)), (ValueError, lambda: ops.layernorm_fwd(x, w.cpu())),
           (ValueError, lambda: ops.layernorm_fwd(x, w, residual=x[:2])),
           (TypeError, lambda: ops.layernorm_fwd(x, w, residual=x.float())),
           (ValueError, lambda: ops.layernorm_fwd(x.t())), (ValueError, lambda: ops.layernorm_fwd(torch.tensor(1.0, device=DEV))),
           (ValueError, lambda: ops.layernorm_fwd(rand(3, 0))),
           (ValueError, lambda: ops.layernorm_fwd(rand(4, 6, 64)[:, :4])),  # no single row stride
           (ValueError, lambda: ops.layernorm_bwd(x[:2], x, mean, rstd, w)),
           (TypeError, lambda: ops.layernorm_bwd(x.float(), x, mean, rstd, w)),
           (TypeError, lambda: ops.layernorm_bwd(x, x, mean.double(), rstd, w)),
           (ValueError, lambda: ops.layernorm_bwd(x, x, mean[:2], rstd, w)),
           (ValueError, lambda: ops.layernorm_bwd(x, x, mean, rstd, w, dres=x[:2])),
           (ValueError, lambda: ops.layernorm_bwd(x, x, mean, rstd, w, workspace=torch.empty(4)))]
    for error, call in bad:
        with pytest.raises(error):
            call()
    torch.cuda.synchronize()
