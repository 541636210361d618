"""rmsnorm_quant_fwd / rmsnorm_quant_bwd against 64 bits: widths, groups that
are cut, both formats and scale types, rows of zeros, infinities and NaN,
strides, the gradient against the formula and against differences, refusals."""
import pytest
import torch

from kernelproblems_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
F32, E8 = torch.float32, torch.float8_e8m0fnu
EPS = 1e-5
# rstd and all that follows: sums of up to 64 terms by one thread and then a
# tree, in 32 bits, and a handful of single roundings
REL = 5e-6


def rand(*shape, seed=0, std=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(torch.bfloat16)


def weight(N, seed=99):
    return (1 + 0.1 * rand(N, seed=seed).float()).to(torch.bfloat16)


def check_quant(q, scale, y, group, slack):
    """q and scale of the 64-bit rows y; `slack` bounds the 32-bit error of y."""
    M, N = y.shape
    top = torch.finfo(q.dtype).max
    size = group or N
    at = torch.arange(N, device=DEV) // size
    most = torch.stack([b.abs().amax(1) for b in y.split(size, 1)], 1)
    err = torch.stack([b.amax(1) for b in slack.split(size, 1)], 1)
    s = scale.double().view(M, -1)
    assert s.shape == most.shape
    want = torch.where(most > 0, (most / top).clamp_min(2.0 ** -126), 1.0)
    off = err / top + REL * want
    if scale.dtype == E8:
        lo, hi = torch.exp2(torch.ceil(torch.log2(want - off))), torch.exp2(torch.ceil(torch.log2(want + off)))
        assert bool(((s >= lo) & (s <= hi)).all())
    else:
        assert bool(((s - want).abs() <= off).all())
    t = y / s[:, at]
    # half a step: 2^-4 (E4M3) or 2^-3 (E5M2) of the value, or of the smallest normal
    half, tiny = (2.0 ** -4, 2.0 ** -10) if q.dtype == E4 else (2.0 ** -3, 2.0 ** -17)
    bound = torch.clamp_min(half * t.abs(), tiny) * 1.0001 + slack / s[:, at] + REL * t.abs()
    d = (q.view(M, N).double() - t).abs()
    assert bool((d <= bound).all()), f"{(d - bound).max().item():.3g}"
    # and what is further than that from a tie is the correctly rounded one
    off = slack / s[:, at] + REL * t.abs()
    lo, hi = ((t + e).clamp(-top, top).float().to(q.dtype).double() for e in (-off, off))
    assert bool(((q.view(M, N).double() >= lo) & (q.view(M, N).double() <= hi)).all())


def forward64(x, w, res):
    h = x.double() if res is None else (res.double() + x.double()).to(torch.bfloat16).double()
    rstd = (h.square().mean(-1) + EPS).rsqrt()
    return h, rstd, h * rstd[:, None] * w.double()


def check_fwd(x, w, res, out, group):
    q, scale, h, rstd = out
    M, N = x.reshape(-1, x.shape[-1]).shape
    x2, r2 = x.reshape(M, N), None if res is None else res.reshape(M, N)
    h64, r64, y64 = forward64(x2, w, r2)
    if res is None:
        assert h is None
    elif h is not None:
        assert torch.equal(h.view(M, N).double(), h64)
    if rstd is not None:
        assert bool(((rstd.view(M).double() - r64).abs() <= REL * r64).all())
    check_quant(q, scale, y64, group, REL * y64.abs())


SHAPES = [(1, 1), (3, 7), (1, 4096), (5, 64), (33, 1000), (4, 1001), (17, 2568), (9, 8192), (2, 16384),
          (3, 20000), (2, 30001), (300, 128), (64, 96)]


@pytest.mark.parametrize("M,N", SHAPES)
@pytest.mark.parametrize("group", [0, 32, 64, 128])
def test_forward(M, N, group):
    x, w, res = rand(M, N, seed=1), weight(N), rand(M, N, seed=2)
    for dtype in (E4, E5):
        for sd in (F32, E8):
            check_fwd(x, w, res, ops.rmsnorm_quant_fwd(x, w, EPS, residual=res, dtype=dtype, group=group,
                                                       scale_dtype=sd), group)
    check_fwd(x, w, None, ops.rmsnorm_quant_fwd(x, w, EPS, group=group), group)
    q, scale, h, rstd = ops.rmsnorm_quant_fwd(x, w, EPS, residual=res, group=group, write_h=False, save_rstd=False)
    assert h is None and rstd is None
    check_fwd(x, w, res, (q, scale, h, rstd), group)


def test_shapes_and_empty():
    w = weight(64)
    q, s, h, r = ops.rmsnorm_quant_fwd(rand(2, 3, 64), w, residual=rand(2, 3, 64, seed=1), group=32)
    assert q.shape == (2, 3, 64) and s.shape == (2, 3, 2) and h.shape == (2, 3, 64) and r.shape == (2, 3)
    q, s, _, _ = ops.rmsnorm_quant_fwd(rand(64), w)
    assert q.shape == (64,) and s.shape == ()
    q, s, _, r = ops.rmsnorm_quant_fwd(rand(0, 64), w, group=64)
    assert q.shape == (0, 64) and s.shape == (0, 1) and r.shape == (0,)
    dx, q, s, dw = ops.rmsnorm_quant_bwd(rand(0, 64), rand(0, 64), torch.empty(0, device=DEV), w)
    assert dx.shape == (0, 64) and bool((dw == 0).all())


@pytest.mark.parametrize("N", [64, 1000, 1001, 4096])
@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("sd", [F32, E8])
def test_zero_rows_and_values_that_are_not_finite(N, group, sd):
    x, w = rand(6, N, seed=3), weight(N)
    x[0] = 0
    x[1, N // 2] = float("inf")
    x[2, N // 3] = float("nan")
    x[4] = 1e-30  # far below eps: y is tiny but not zero
    q, scale, _, rstd = ops.rmsnorm_quant_fwd(x, w, EPS, group=group, scale_dtype=sd)
    q, s = q.float(), scale.float().view(6, -1)
    assert bool((q[0] == 0).all()) and bool((s[0] == 1).all())
    assert rstd[1] == 0 and torch.isnan(rstd[2])
    assert torch.isnan(q[1, N // 2]) and not bool(torch.isfinite(s[1, (N // 2) // (group or N)]))
    others = torch.ones(N, dtype=torch.bool, device=DEV)
    if group:  # the other groups of that row are zeros
        others[(N // 2) // group * group:(N // 2) // group * group + group] = False
        assert bool((q[1, others] == 0).all())
    assert bool(torch.isnan(q[2]).all()) and not bool(torch.isfinite(s[2]).any())
    for row in (3, 5):
        check_fwd(x[row:row + 1], w, None, (ops.rmsnorm_quant_fwd(x, w, EPS, group=group, scale_dtype=sd)[0][row:row + 1],
                                            scale[row:row + 1], None, rstd[row:row + 1]), group)
    y = 1e-30 / EPS ** 0.5 * w.double()
    want = torch.stack([b.abs().amax() for b in y.split(group or N)]) / 448
    assert bool((s[4].double() >= want * 0.99).all()) and bool((s[4].double() <= want * 2.01).all())


@pytest.mark.parametrize("N", [64, 1000, 4096])
def test_strided_rows(N):
    w = weight(N)
    x = rand(5, N + 24, seed=4)[:, 8:8 + N]
    res = rand(10, N, seed=5)[::2]
    check_fwd(x, w, res, ops.rmsnorm_quant_fwd(x, w, EPS, residual=res, group=32), 32)
    odd = rand(5, N + 3, seed=6)[:, 1:1 + N]  # rows at odd addresses
    check_fwd(odd, w, res, ops.rmsnorm_quant_fwd(odd, w, EPS, residual=res), 0)
    one = rand(1, N, seed=7).expand(5, N)  # one row for all
    check_fwd(one, w, None, ops.rmsnorm_quant_fwd(one, w, EPS), 0)
    dy, r = rand(5, 2 * N, seed=8)[:, :N], torch.rand(5, device=DEV) + 0.5
    check_bwd(dy, x, r, w, res, ops.rmsnorm_quant_bwd(dy, x, r, w, dres=res, group=64), 64)


def backward64(dy, x, rstd, w, dres):
    dy, xhat, r = dy.double(), x.double() * rstd.double()[:, None], rstd.double()[:, None]
    g = dy * w.double()
    mean = (xhat * g).mean(-1, keepdim=True)
    dx = (g - xhat * mean) * r
    # what the 32-bit error is relative to
    size = (g.abs() + xhat.abs() * (xhat * g).abs().mean(-1, keepdim=True)) * r
    if dres is not None:
        dx, size = dx + dres.double(), size + dres.double().abs()
    return dx, size, (dy * xhat).sum(0), (dy * xhat).abs().sum(0)


def check_bwd(dy, x, rstd, w, dres, out, group):
    dx, q, scale, dw = out
    want, size, dw64, dwsize = backward64(dy, x, rstd, w, dres)
    if dx is not None:
        err = (dx.double() - want).abs()
        assert bool((err <= 2.0 ** -8 * want.abs() * 1.001 + REL * size + 1e-38).all())
    check_quant(q, scale, want, group, REL * size)
    if dw is not None:
        assert bool(((dw.double() - dw64).abs() <= 5e-6 * dwsize + 1e-38).all())


@pytest.mark.parametrize("M,N", SHAPES + [(777, 136), (2000, 256)])
@pytest.mark.parametrize("group", [0, 32, 128])
def test_backward(M, N, group):
    x, dy, w, dres = rand(M, N, seed=1), rand(M, N, seed=2, std=1e-3), weight(N), rand(M, N, seed=3, std=1e-3)
    rstd = (x.float().square().mean(-1) + EPS).rsqrt()
    for dtype in (E4, E5):
        for sd in (F32, E8):
            for dr in (None, dres):
                check_bwd(dy, x, rstd, w, dr, ops.rmsnorm_quant_bwd(dy, x, rstd, w, dres=dr, dtype=dtype, group=group,
                                                                    scale_dtype=sd), group)
    dx, q, s, dw = ops.rmsnorm_quant_bwd(dy, x, rstd, w, group=group, write_dx=False, compute_dw=False)
    assert dx is None and dw is None
    check_bwd(dy, x, rstd, w, None, (dx, q, s, dw), group)


def test_backward_is_reproducible():
    x, dy, w = rand(1537, 1032, seed=1), rand(1537, 1032, seed=2), weight(1032)
    rstd = (x.float().square().mean(-1) + EPS).rsqrt()
    a, b = (ops.rmsnorm_quant_bwd(dy, x, rstd, w, dres=dy) for _ in range(2))
    for u, v in zip(a, b):
        assert torch.equal(u.float(), v.float())


@pytest.mark.parametrize("N", [64, 1001])
def test_gradient_matches_differences(N):
    """Difference quotients of sum(dy * norm(h) * w) + sum(dres * h), in 64
    bits, along random directions of x and of w; the forward's saved h and
    rstd are what the gradient reads."""
    x, res, w = rand(6, N, seed=1), rand(6, N, seed=2), weight(N)
    dy, dres = rand(6, N, seed=3), rand(6, N, seed=4)
    _, _, h, rstd = ops.rmsnorm_quant_fwd(x, w, EPS, residual=res)
    dx, q, scale, dw = ops.rmsnorm_quant_bwd(dy, h, rstd, w, dres=dres)

    def loss(h64, w64):
        r = (h64.square().mean(-1, keepdim=True) + EPS).rsqrt()
        return (dy.double() * h64 * r * w64).sum() + (dres.double() * h64).sum()
    for seed in (5, 6):
        v, u = rand(6, N, seed=seed).double(), rand(N, seed=seed + 2).double()
        e = 1e-4
        H, W = h.double(), w.double()
        along = (loss(H + e * v, W) - loss(H - e * v, W)) / (2 * e)
        # 8 standard deviations of the bf16 roundings, the quotient's e^2 term
        assert (along - (dx.double() * v).sum()).abs() <= 8 * 2.0 ** -9 * (dx.double() * v).norm() + 1e-5
        along8 = (q.double() * scale.double()[:, None] * v).sum()
        assert (along - along8).abs() <= 8 * 2.0 ** -3 * (dx.double() * v).norm()
        along = (loss(H, W + e * u) - loss(H, W - e * u)) / (2 * e)
        assert (along - (dw.double() * u).sum()).abs() <= 1e-5 * (dw.double() * u).abs().sum()


def test_agrees_with_the_unquantised_pair():
    """The same h and rstd as add_rmsnorm_fwd; 8 bits of its y to one step."""
    x, res, w = rand(64, 4096, seed=1), rand(64, 4096, seed=2), weight(4096)
    h0, y, r0 = ops.add_rmsnorm_fwd(res, x, w, EPS)
    q, s, h, r = ops.rmsnorm_quant_fwd(x, w, EPS, residual=res, group=128)
    assert torch.equal(h, h0) and torch.allclose(r, r0, rtol=1e-6)
    back = q.float() * s.repeat_interleave(128, -1)
    # (the smallest magnitudes: half the format's smallest step, in scales)
    assert bool(((back - y.float()).abs() <= 2.0 ** -3.9 * y.float().abs() + s.max() * 2.0 ** -10).all())


def test_refusals():
    x, w, r = rand(4, 64), weight(64), torch.ones(4, device=DEV)
    with pytest.raises(TypeError):
        ops.rmsnorm_quant_fwd(x.float(), w)
    with pytest.raises(TypeError):
        ops.rmsnorm_quant_fwd(x, w, dtype=torch.int8)
    with pytest.raises(TypeError):
        ops.rmsnorm_quant_fwd(x, w, scale_dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.rmsnorm_quant_fwd(x, w, group=48)
    with pytest.raises(ValueError):
        ops.rmsnorm_quant_fwd(x, weight(32))
    with pytest.raises(ValueError):
        ops.rmsnorm_quant_fwd(x, w, residual=rand(5, 64))
    with pytest.raises(ValueError):
        ops.rmsnorm_quant_fwd(x.cpu(), w.cpu())
    with pytest.raises(ValueError):
        ops.rmsnorm_quant_fwd(rand(64, 64).t(), w)
    with pytest.raises(ValueError):
        ops.rmsnorm_quant_fwd(rand(4, 6, 64)[:, :5], w)  # no single row stride
    with pytest.raises(ValueError):
        ops.rmsnorm_quant_bwd(x, x, r[:3], w)
    with pytest.raises(TypeError):
        ops.rmsnorm_quant_bwd(x, x, r.double(), w)
    with pytest.raises(ValueError):
        ops.rmsnorm_quant_bwd(x, x, r, w, dres=rand(4, 32))
    with pytest.raises(ValueError):
        ops.rmsnorm_quant_bwd(x, x, r, w, workspace=torch.empty(1 << 20, dtype=torch.uint8))


GRIDS = """
import sys
import torch
from cuda.bindings import driver
from kernelproblems_b200 import ops
order = [(20000, 256, False), (20000, 1024, False), (20000, 4096, True), (20000, 4096, False), (20000, 1000, False)]
w = {N: torch.ones(N, dtype=torch.bfloat16, device="cuda") for _, N, _ in order}
grids = []
for M, N, res in order[::int(sys.argv[1])]:
    x = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    call = lambda: ops.rmsnorm_quant_fwd(x, w[N], residual=x if res else None)
    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    h = driver.CUgraph(graph.raw_cuda_graph())
    _, _, n = driver.cuGraphGetNodes(h)
    _, nodes, n = driver.cuGraphGetNodes(h, n)
    assert n == 1
    err, p = driver.cuGraphKernelNodeGetParams(nodes[0])
    assert int(err) == 0
    grids.append(f"{M}x{N}{res} {p.gridDimX} of {p.blockDimX}")
print(sorted(grids))
"""


def test_grid_does_not_depend_on_earlier_calls():
    """Each kernel's resident blocks are its own: the same calls in the other
    order, in a process of their own, get the same grids."""
    import subprocess
    import sys
    from pathlib import Path
    runs = [subprocess.run([sys.executable, "-c", GRIDS, step], cwd=Path(__file__).resolve().parent.parent, timeout=300,
                           capture_output=True, text=True) for step in ("1", "-1")]
    assert all(r.returncode == 0 for r in runs), runs[0].stderr + runs[1].stderr
    assert runs[0].stdout == runs[1].stdout


# Rows enough that blocks and warps take several (the next row's loads ahead,
# alternating slots, a last block that is cut; the gradient's ring reused, with
# both parities of its barriers), each width's own kernel.
LONG = [(40013, 256), (40013, 504), (40013, 1000), (9001, 4096), (3001, 8200), (1501, 16384), (20011, 300), (5003, 1001)]


@pytest.mark.parametrize("M,N", LONG)
@pytest.mark.parametrize("group", [0, 32, 128])
def test_forward_of_many_rows(M, N, group):
    x, w, res = rand(M, N, seed=31), weight(N), rand(M, N, seed=32)
    x[5::7] *= 30  # neighbouring rows of one block differ
    x[3::64] = 0
    for r in (None, res):
        check_fwd(x, w, r, ops.rmsnorm_quant_fwd(x, w, EPS, residual=r, group=group), group)


@pytest.mark.parametrize("M,N", [(20011, 136), (20011, 512), (12007, 1032), (9001, 4096), (6007, 4104), (3001, 5120),
                                 (3001, 6144), (3001, 6152), (3001, 8192), (1501, 8200), (1501, 16384), (20011, 300),
                                 (5003, 1001), (1501, 9001)])
@pytest.mark.parametrize("group", [0, 128])
def test_backward_of_many_rows(M, N, group):
    x, dy, w, dres = rand(M, N, seed=33), rand(M, N, seed=34, std=1e-3), weight(N), rand(M, N, seed=35, std=1e-3)
    dy[5::7] *= 30
    x[3::64] = 0
    rstd = (x.float().square().mean(-1) + EPS).rsqrt()
    for dr in (None, dres):
        check_bwd(dy, x, rstd, w, dr, ops.rmsnorm_quant_bwd(dy, x, rstd, w, dres=dr, group=group), group)
    ops.check_status()


@pytest.mark.parametrize("N", [264, 300, 504, 513, 520, 1016, 1032, 4100, 4104, 5120, 6144, 6152, 8191, 8200, 9001, 16383])
def test_widths_at_the_variants_borders(N):
    x, dy, w, res = rand(37, N, seed=36), rand(37, N, seed=37), weight(N), rand(37, N, seed=38)
    rstd = (x.float().square().mean(-1) + EPS).rsqrt()
    for group in (0, 64):
        for r in (None, res):
            check_fwd(x, w, r, ops.rmsnorm_quant_fwd(x, w, EPS, residual=r, group=group, scale_dtype=E8), group)
            check_bwd(dy, x, rstd, w, r, ops.rmsnorm_quant_bwd(dy, x, rstd, w, dres=r, group=group), group)


def test_rows_of_no_values_are_refused():
    x, w, r = rand(5, 0), rand(0), torch.ones(5, device=DEV)
    with pytest.raises(ValueError, match="at least one"):
        ops.rmsnorm_quant_fwd(x, w)
    with pytest.raises(ValueError, match="at least one"):
        ops.rmsnorm_quant_fwd(x, w, residual=x, group=32)
    with pytest.raises(ValueError, match="at least one"):
        ops.rmsnorm_quant_bwd(x, x, r, w)
    q, s, _, rstd = ops.rmsnorm_quant_fwd(rand(0, 0), w)  # no rows either
    assert q.shape == (0, 0) and s.shape == rstd.shape == (0,)
