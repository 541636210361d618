"""orthogonalize and muon_update against the same steps in 64 bits: sizes from
one element on, tall and wide, strides, spectra, schedules, zeros and NaN, the
update in place, and refusals."""
import math

import pytest
import torch

from kernelproblems_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
# Relative Frobenius error of the result.  The products' fp16 rounding, worked
# through the five steps in a 64-bit emulation of the scheme: up to 1.5e-3 at
# sizes of 24, 1.3e-3 at 64, 0.9e-3 at 512 (spectra: flat, 1/k, 16 strong
# directions over a rest of 2%); the bf16 result's own: 1.7e-3.
TOL = 3e-3
SMALL_TOL = 2.0 ** -8 + 2e-3  # a few elements: one rounding's worst


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def exact(g, steps=5, co=ops.NEWTON_SCHULZ, eps=1e-7):
    x = g.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    co = [co] * steps if isinstance(co[0], float) else co
    for a, b, c in co:
        A = x @ x.mT
        x = a * x + (b * A + c * A @ A) @ x
    return x.mT if tall else x


def off(got, want):
    return (torch.linalg.matrix_norm(got.double() - want) / torch.linalg.matrix_norm(want)).max().item()


def tol(g):
    return TOL if min(g.shape[-2:]) >= 16 else SMALL_TOL


SIZES = [(1, 1), (1, 7), (5, 1), (3, 200), (16, 16), (96, 160), (127, 129), (128, 128), (160, 96), (129, 1000),
         (257, 64), (64, 1031), (500, 500), (333, 1025), (1024, 256), (700, 1300), (100, 2050), (4096, 128), (16, 4097),
         (129, 5000), (2049, 1793), (2000, 2312), (1100, 4000)]


@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sizes(m, n, dtype):
    g = normal(m, n, seed=m + n, dtype=dtype)
    o = ops.orthogonalize(g)
    assert o.dtype == torch.bfloat16 and o.shape == g.shape and o.is_contiguous()
    assert off(o, exact(g)) <= tol(g)
    ops.check_status()


@pytest.mark.parametrize("m,n", [(64, 100), (512, 512), (300, 1000), (1000, 300)])
@pytest.mark.parametrize("spectrum", ["one over k", "strong and weak", "rank one", "scaled"])
def test_spectra(m, n, spectrum):
    g = normal(m, n, seed=1)
    if spectrum == "one over k":
        u, s, v = torch.linalg.svd(g.double(), full_matrices=False)
        g = (u / torch.arange(1, len(s) + 1, device=DEV)) @ v
    elif spectrum == "strong and weak":
        g = normal(m, 16, seed=2) @ normal(16, n, seed=3) + 0.02 * g
    elif spectrum == "rank one":
        g = normal(m, 1, seed=2) @ normal(1, n, seed=3)
    else:
        g = g * 1e12
    g = g.float()
    o = ops.orthogonalize(g)
    if spectrum == "rank one":  # the rest is rounding noise: only the one direction is compared
        u, s, v = torch.linalg.svd(g.double(), full_matrices=False)
        got, want = (u[:, 0] @ x.double() @ v[0] for x in (o, exact(g)))
        assert abs(got - want) <= TOL * abs(want)
    else:
        assert off(o, exact(g)) <= TOL
    small = ops.orthogonalize(g * 1e-3 / g.abs().max())  # the norm does not matter
    assert off(small, o.double()) <= 2 * TOL or spectrum == "rank one"


@pytest.mark.parametrize("shape", [(3, 100, 60), (2, 2, 33, 140), (5, 128, 256), (3, 130, 515)])
def test_batches(shape):
    g = normal(*shape, seed=4)
    o = ops.orthogonalize(g)
    assert off(o, exact(g)) <= TOL
    for i in range(shape[0]):  # every matrix by itself, to the bit
        assert torch.equal(ops.orthogonalize(g[i]), o[i])


def test_batch_of_large_matrices():
    g = normal(2, 1800, 1810, seed=4)  # (the batch's count may choose another tile: not bit for bit)
    assert off(ops.orthogonalize(g), exact(g)) <= TOL


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(dtype):
    base = normal(4, 130, 222, seed=5, dtype=dtype)
    for g in (base[0].t(), base[:, 3:100, 7:201], base[::2, ::2, ::3], base[1:2].expand(3, 130, 222),
              base.transpose(1, 2), base[:1, None].expand(1, 3, 130, 222), normal(60, 1, seed=6, dtype=dtype).expand(60, 70)[:, :1]):
        o = ops.orthogonalize(g)
        assert torch.equal(o, ops.orthogonalize(g.contiguous()))
        assert off(o, exact(g)) <= tol(g)


def test_schedules():
    g = normal(200, 300, seed=7)
    for steps, co in ((1, ops.NEWTON_SCHULZ), (2, (1.5, -0.5, 0.0)), (8, (1.875, -1.25, 0.375)),
                      (3, [(8.0, -22.0, 16.0), (4.0, -6.0, 2.8), (1.875, -1.25, 0.375)])):
        o = ops.orthogonalize(g, steps=steps, coefficients=co)
        assert off(o, exact(g, steps, co)) <= TOL
    g = normal(64, 64, seed=8) * 1e-4  # eps as large as the norm
    assert off(ops.orthogonalize(g, eps=0.01), exact(g, eps=0.01)) <= TOL


def test_zero_and_not_finite():
    g = normal(4, 70, 90, seed=9)
    want = ops.orthogonalize(g)
    g[1] = 0
    g[2, 3, 4] = float("nan")
    o = ops.orthogonalize(g)
    assert bool((o[1] == 0).all()) and bool(torch.isnan(o[2]).all())
    assert torch.equal(o[0], want[0]) and torch.equal(o[3], want[3])
    g[2, 3, 4] = float("inf")
    assert bool(torch.isnan(ops.orthogonalize(g)[2]).all())


@pytest.mark.parametrize("shape", [(0, 8, 8), (2, 0, 8), (2, 8, 0), (0, 0)])
def test_empty(shape):
    assert ops.orthogonalize(torch.empty(shape, device=DEV)).shape == shape


def test_reproducible_with_buffers_and_on_another_stream():
    g = normal(300, 700, seed=10)
    want = ops.orthogonalize(g)
    out = torch.empty(300, 700, dtype=torch.bfloat16, device=DEV)
    ws = torch.full((ops.orthogonalize_workspace_bytes(1, 300, 700),), 255, dtype=torch.uint8, device=DEV)
    assert ops.orthogonalize(g, out=out, workspace=ws) is out and torch.equal(out, want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.orthogonalize(g)
    s.synchronize()
    assert torch.equal(other, want)


@pytest.mark.parametrize("m,n", [(200, 100), (300, 700), (2304, 2304)])  # a cluster, blocks, pairs of blocks
def test_in_a_graph(m, n):
    g = normal(m, n, seed=11)
    out = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
    ws = torch.empty(ops.orthogonalize_workspace_bytes(1, m, n), dtype=torch.uint8, device=DEV)
    want = ops.orthogonalize(g, out=out, workspace=ws).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.orthogonalize(g, out=out, workspace=ws)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)


UNIT = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -22}  # fp32: a few roundings


@pytest.mark.parametrize("shape", [(96, 160), (2, 200, 77), (1, 5), (512, 1024), (700, 301), (1900, 2100), (120, 2600)])
@pytest.mark.parametrize("pd,gd,md", [(torch.float32, torch.float32, torch.float32),
                                      (torch.bfloat16, torch.bfloat16, torch.bfloat16),
                                      (torch.float32, torch.bfloat16, torch.float32),
                                      (torch.bfloat16, torch.float32, torch.float32)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_update(shape, pd, gd, md, nesterov):
    p, g, m = (normal(*shape, seed=s, dtype=d) for s, d in ((12, pd), (13, gd), (14, md)))
    lr, mu, wd, scale = 0.02, 0.9, 0.1, 0.7
    m64 = mu * m.double() + (1 - mu) * g.double()
    o = exact(mu * m64 + (1 - mu) * g.double() if nesterov else m64)
    p64 = (1 - lr * wd) * p.double() - lr * scale * o
    kw = dict(lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd, scale=scale)
    before = [t.clone() for t in (p, g, m)]
    p1, m1 = ops.muon_update(p, g, m, **kw)
    assert all(torch.equal(a, b) for a, b in zip(before, (p, g, m)))
    assert p1.dtype == pd and m1.dtype == md
    assert bool(((m1.double() - m64).abs() <= UNIT[md] * (m.abs() + g.abs()).double()).all())
    err = torch.linalg.vector_norm(p1.double() - p64)
    assert err <= tol(p) * lr * scale * torch.linalg.vector_norm(o) + UNIT[pd] * torch.linalg.vector_norm(p64)
    # in place: the same bits
    q, n = p.clone(), m.clone()
    assert ops.muon_update(q, g, n, param_out=q, momentum_out=n, **kw) == (q, n)
    assert torch.equal(q, p1) and torch.equal(n, m1)


@pytest.mark.parametrize("m,n", [(24, 100), (96, 160), (128, 700), (1500, 100), (3, 200)])
def test_short_sided_updates_in_32_bits(m, n):
    """With a side of at most 128 and weights in 32 bits the products take three
    terms: 5e-7 in a 64-bit emulation at 24 x 100, accumulators in 32 bits
    beside it; the step is as large as the weights, so that it shows."""
    p, g, mom = (normal(m, n, seed=s) for s in (22, 23, 24))
    p1, _ = ops.muon_update(p, g, mom, lr=1.0, momentum=0.5, nesterov=False, scale=math.sqrt(max(m, n)))
    o = exact(0.5 * mom.double() + 0.5 * g.double())
    p64 = p.double() - math.sqrt(max(m, n)) * o
    err = torch.linalg.vector_norm(p1.double() - p64)
    assert err <= 1e-5 * math.sqrt(max(m, n)) * torch.linalg.vector_norm(o) + 2.0 ** -22 * torch.linalg.vector_norm(p64)


def test_update_of_strided_tensors():
    p, g, m = (normal(130, 90, seed=s).t() for s in (15, 16, 17))
    p1, m1 = ops.muon_update(p, g, m, lr=0.1)
    p2, m2 = ops.muon_update(p.contiguous(), g.contiguous(), m.contiguous(), lr=0.1)
    assert torch.equal(p1, p2) and torch.equal(m1, m2)


def test_calls_on_two_streams_at_once():
    gs = [normal(700, 900, seed=s) for s in (20, 21)]
    want = [ops.orthogonalize(g) for g in gs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in gs]
    got = []
    for _ in range(3):
        for g, s in zip(gs, streams):
            with torch.cuda.stream(s):
                got.append(ops.orthogonalize(g))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])
    ops.check_status()


def test_refusals():
    g = normal(8, 8)
    with pytest.raises(ValueError):
        ops.orthogonalize(g, steps=33)
    with pytest.raises(TypeError):
        ops.orthogonalize(g.half())
    with pytest.raises(ValueError):
        ops.orthogonalize(g[0])
    with pytest.raises(ValueError):
        ops.orthogonalize(g.cpu())
    with pytest.raises(ValueError):
        ops.orthogonalize(g, steps=0)
    with pytest.raises(ValueError):
        ops.orthogonalize(g, coefficients=[(1.0, 2.0, 3.0)] * 4)
    with pytest.raises(ValueError):
        ops.orthogonalize(g, coefficients=(math.nan, 1.0, 1.0))
    with pytest.raises(ValueError):
        ops.orthogonalize(g, out=torch.empty(8, 9, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError):
        ops.orthogonalize(normal(4, 6, 8, 8)[:, :5])
    with pytest.raises(ValueError):  # a repeated dimension inside another
        ops.orthogonalize(normal(4, 1, 8, 8).expand(4, 3, 8, 8))
    with pytest.raises(ValueError):
        ops.muon_update(g, normal(8, 9), g.clone(), lr=0.1)
    with pytest.raises(ValueError):
        ops.muon_update(g, g.clone(), g.clone(), lr=math.inf)
    with pytest.raises(ValueError):
        ops.muon_update(g, g.clone(), g.clone(), lr=0.1, momentum=1.5)
    with pytest.raises(ValueError):  # the gradient would be overwritten while it is read
        h = g.clone()
        ops.muon_update(g, h, g.clone(), lr=0.1, param_out=h)
    with pytest.raises(ValueError):
        o = torch.empty_like(g)
        ops.muon_update(g, g.clone(), g.clone(), lr=0.1, param_out=o, momentum_out=o)
    with pytest.raises(ValueError):
        ops.muon_update(g, g.clone(), g.clone(), lr=0.1, workspace=torch.empty(9, dtype=torch.uint8))


@pytest.mark.parametrize("shape", [(5, 64, 100), (2, 300, 700), (130, 60)])
def test_in_place(shape):
    g = normal(*shape, seed=25, dtype=torch.bfloat16)
    want = ops.orthogonalize(g)
    assert ops.orthogonalize(g, out=g) is g and torch.equal(g, want)


def test_outputs_over_other_matrices_are_refused():
    buf = normal(5, 64, 100, seed=26, dtype=torch.bfloat16)
    before = buf.clone()
    with pytest.raises(ValueError, match="overlaps"):
        ops.orthogonalize(buf[:4], out=buf[1:])
    with pytest.raises(ValueError, match="overlaps"):
        ops.orthogonalize(buf[0, :64, :64].t(), out=buf[0].flatten()[:4096].view(64, 64))
    assert torch.equal(buf, before)


def test_one_cluster_a_matrix_takes_no_workspace():
    assert all(ops.orthogonalize_workspace_bytes(4000, m, n) == 0 for m, n in ((128, 1024), (4096, 128), (1, 1), (64, 100)))
    assert ops.orthogonalize_workspace_bytes(1, 128, 4097) > 0 and ops.orthogonalize_workspace_bytes(1, 129, 129) > 0
    g = normal(600, 128, 1024, seed=27, dtype=torch.bfloat16)  # 157 MB; the other form's workspace is 500
    out = torch.empty_like(g)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.orthogonalize(g, out=out)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20
    assert off(out[::97], exact(g[::97])) <= TOL
    # the caller's is left alone
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device=DEV)
    assert torch.equal(ops.orthogonalize(g[:2], workspace=ws), out[:2]) and not bool(ws.any())


@pytest.mark.parametrize("m,n", [(100, 128), (128, 2048), (300, 700), (700, 301), (2304, 2304)])
@pytest.mark.parametrize("norm", [1e-3, 1e-6, 1e-8])
def test_norm_far_below_eps(m, n, norm):
    """|G| = norm * eps: X stays small through all steps, which then only
    multiply it.  hi is off by up to 2^-25 and hi + lo by 2^-36 (of 256 times
    an element), uniformly: 0.6 * 2^-44 * sqrt(mn) / norm of X, 8e-3 for the
    largest at 1e-8, and the same again from the steps after (each a third as
    much); under 1e-3 with the rest of TOL elsewhere."""
    g = normal(m, n, seed=28)
    g = g / torch.linalg.matrix_norm(g) * (norm * 1e-2)
    want = exact(g, eps=1e-2)
    noise = 0.6 * 2.0 ** -44 * math.sqrt(m * n) / norm * 1.5
    assert off(ops.orthogonalize(g, eps=1e-2), want) <= TOL + noise


@pytest.mark.parametrize("m,n", [(64, 100), (96, 160), (128, 700)])
@pytest.mark.parametrize("norm", [1e-3, 1e-6])
def test_short_sided_update_with_a_norm_far_below_eps(m, n, norm):
    """Weights in 32 bits with a side of at most 128: X is off by up to 2^-33 an
    element in each step, multiplied by the steps after (3.4445^5 = 485)."""
    g = normal(m, n, seed=29)
    g = g / torch.linalg.matrix_norm(g) * (norm * 1e-2)
    p, mom = torch.zeros_like(g), torch.zeros_like(g)
    p1, _ = ops.muon_update(p, g, mom, lr=1.0, momentum=0.0, nesterov=False, eps=1e-2)
    assert bool(((p1.double() + exact(g, eps=1e-2)).abs() <= 485 * 1.5 * 2.0 ** -33 + 1e-5 / math.sqrt(max(m, n)) * norm * 485).all())
