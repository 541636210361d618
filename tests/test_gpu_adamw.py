"""adamw_update and grad_norm against 64 bits: types, sizes, alignments, many
tensors, states in 32 and 8 bits, steps and rates on the device, graphs,
gradients that are not finite, and refusals."""
import math
import warnings

import pytest
import torch

from kernelproblems_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
U = 2.0 ** -24  # half a step of 32 bits


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def make(sizes, dtype, seed=0, std=1.0, shift=0, gap=0):
    """Tensors of the sizes (ints or shapes) inside one buffer: `shift` values
    before the first, `gap` between them."""
    shapes = [(s,) if isinstance(s, int) else s for s in sizes]
    numels = [math.prod(s) for s in shapes]
    buf = torch.full((shift + sum(numels) + gap * len(sizes) + 8,), 7.0, dtype=dtype, device=DEV)
    out, at, g = [], shift, gen(seed)
    for shape, n in zip(shapes, numels):
        buf[at:at + n] = (torch.randn(n, generator=g, device=DEV) * std).to(dtype)
        out.append(buf[at:at + n].view(shape))
        at += n + gap
    return out, buf


def fill(states, seed=3, std=1e-2, zeros=True):
    """Random moments, through what the states hold: as a run of steps would leave them."""
    g = gen(seed)
    for i, p in enumerate(states.params):
        a, n = states.offsets[i], p.numel()
        m, r = (torch.randn(n, generator=g, device=DEV) * std for _ in range(2))
        if zeros and n > 300:
            m[130:260] = 0
            r[130:260] = 0
        put(states, a, n, m, r.abs())


def put(states, a, n, m, r):
    held = -(-n // 128) * 128
    m, r = (torch.cat([t, torch.zeros(held - n, device=DEV)]) for t in (m, r))
    if states.dtype == F32:
        states.exp_avg[a:a + held], states.exp_avg_sq[a:a + held] = m, r.square()
        return
    for t, to, scale in ((m, states.exp_avg, states.exp_avg_scale), (r, states.exp_avg_sq, states.exp_avg_sq_scale)):
        t = t.view(-1, 128)
        s = t.abs().amax(1) / 448
        s = torch.where(s > 0, s, torch.ones_like(s))
        to[a:a + held] = (t / s[:, None]).to(E4).view(-1)
        scale[a // 128:(a + held) // 128] = s


def moments64(states):
    """(m, v) of every value held, in 64 bits."""
    m, v = states.exp_avg.double(), states.exp_avg_sq.double()
    if states.dtype != F32:
        m = (m.view(-1, 128) * states.exp_avg_scale.double()[:, None]).view(-1)
        v = (v.view(-1, 128) * states.exp_avg_sq_scale.double()[:, None]).view(-1).square()
    return m, v


def expected(states, grads, lr, step, betas, eps, scale, decay, lr_scale):
    """What the step should leave, in 64 bits: parameters by tensor, moments flat;
    and a part of the parameters' error."""
    m, v = moments64(states)
    p, off = [], []
    for i, g in enumerate(grads):
        a, n = states.offsets[i], states.params[i].numel()
        if g is None:
            p.append(states.params[i].double())
            off.append(None)
            continue
        g = g.double().view(-1) * scale
        m[a:a + n] = betas[0] * m[a:a + n] + (1 - betas[0]) * g
        v[a:a + n] = betas[1] * v[a:a + n] + (1 - betas[1]) * g * g
        hat = m[a:a + n] / (1 - betas[0] ** step)
        root = (v[a:a + n] / (1 - betas[1] ** step)).sqrt() + eps
        u, rate = hat / root, lr * lr_scale[i]
        # what m's own roundings move the step by where its two terms cancel
        off.append((5 * U * rate * 2 * (1 - betas[0]) / (1 - betas[0] ** step) * g.abs() / root).view(states.params[i].shape))
        w = states.params[i].double()
        p.append(w - rate * (decay[i] * w + u.view(w.shape)))
    return p, m, v, off


def check_eight(q, scale, y, off, root):
    """q and scale of the 64-bit values y, known to within `off` of themselves."""
    y, q, scale = y.view(-1, 128), q.double().view(-1, 128), scale.double()
    most = y.abs().amax(1)
    want = torch.where(most > 0, (most / 448).clamp_min(2.0 ** -126), 1.0)
    # the largest value's own error, the product with 1 / 448 and that constant's rounding
    assert bool(((scale - want).abs() <= (off + 3 * U) * want).all())
    t = y / scale[:, None]
    # the reciprocal and the product that q is rounded from
    e = t.abs() * (off + 3 * U)
    lo, hi = ((t + s * e).clamp(-448, 448).float().to(E4).double() for s in (-1, 1))
    if root:
        lo, hi = (torch.where(y > 0, b.clamp_min(2.0 ** -9), b) for b in (lo, hi))
    assert bool(((q >= lo) & (q <= hi)).all())
    near = (q - t).abs() <= torch.clamp_min(2.0 ** -4 * t.abs(), 2.0 ** -10) * 1.001
    assert bool((near | (root & (q == 2.0 ** -9))).all())


def run_and_check(sizes, dtype, gdtype, state, *, copies=False, shift=0, gap=0, gshift=None, step=7, lr=1e-2,
                  betas=(0.9, 0.95), eps=1e-8, scale=None, decay=0.1, lr_scale=1.0, skip=(), seed=0):
    params, buf = make(sizes, dtype, seed, shift=shift, gap=gap)
    grads, _ = make(sizes, gdtype, seed + 1, std=1e-2, shift=shift if gshift is None else gshift, gap=gap)
    for g in grads:
        if g.numel() > 600:
            g.view(-1)[128:512] = 0  # whole groups without a gradient
    grads = [None if i in skip else g for i, g in enumerate(grads)]
    cp = make(sizes, BF, seed + 2, shift=shift, gap=gap)[0] if copies else None
    states = ops.AdamWStates(params, dtype=state, weight_decay=decay, lr_scale=lr_scale, copies=cp)
    fill(states)
    each = lambda v: [v] * len(sizes) if isinstance(v, (int, float)) else v  # noqa: E731
    s64 = 1.0 if scale is None else scale.double().item()
    before, outside = [p.clone() for p in params], buf.clone()
    held = [t.clone() for t in (states.exp_avg.view(torch.uint8), states.exp_avg_sq.view(torch.uint8))]
    p64, m64, v64, off = expected(states, grads, lr, step, betas, eps, s64, each(decay), each(lr_scale))
    kept = [None if c is None else c.clone() for c in (cp or [])]
    ops.adamw_update(states, grads, lr=lr, step=step, betas=betas, eps=eps, grad_scale=scale)
    for i, (p, w) in enumerate(zip(params, p64)):
        if grads[i] is None:
            assert torch.equal(p, before[i]) and (not copies or torch.equal(cp[i], kept[i]))
            continue
        u = (w - before[i].double()).abs() + lr * each(lr_scale)[i] * each(decay)[i] * before[i].double().abs()
        # the product with keep and its own rounding; the step: three roundings each of m and of the root's
        # square, the root, rate, quotient (2^-22) and the denominator
        slack = 2 * U * before[i].double().abs() + 24 * U * u + off[i]
        half = w.abs().clamp_min(2.0 ** -126) * torch.finfo(dtype).eps / 2
        assert bool(((p.double() - w).abs() <= half * 1.001 + slack).all()), (i, sizes[i])
        if copies:
            assert bool(((cp[i].double() - w).abs() <= w.abs().clamp_min(2.0 ** -126) * 2.0 ** -8 * 1.001 + slack + half).all())
    # three roundings of each of the two terms, each smaller than the sum of their magnitudes
    g64 = torch.zeros_like(m64)
    for i, g in enumerate(grads):
        if g is not None:
            g64[states.offsets[i]:states.offsets[i] + g.numel()] = g.double().view(-1).abs() * s64
    used = torch.zeros_like(m64, dtype=torch.bool)
    for i, g in enumerate(grads):
        if g is not None:
            used[states.offsets[i]:states.offsets[i] + -(-g.numel() // 128) * 128] = True
    if state == F32:
        mag = m64.abs() + 2 * (1 - betas[0]) * g64
        assert bool(((states.exp_avg.double() - m64).abs() <= 5 * U * mag + 2.0 ** -140)[used].all())
        assert bool(((states.exp_avg_sq.double() - v64).abs() <= 6 * U * v64 + 2.0 ** -140)[used].all())
    else:
        m_off = (5 * U * (m64.abs() + 2 * (1 - betas[0]) * g64)).view(-1, 128)
        at = used.view(-1, 128)[:, 0]
        m = m64.view(-1, 128)
        check_cancelling(states.exp_avg.view(-1, 128)[at], states.exp_avg_scale[at], m[at], m_off[at])
        check_eight(states.exp_avg_sq.view(-1, 128)[at].view(-1), states.exp_avg_sq_scale[at],
                    v64.sqrt().view(-1, 128)[at].reshape(-1), 5 * U, True)  # half of v's 6, and the root's 2^-23
    # what no tensor of the step holds is as it was: states without a gradient, and memory around the parameters
    wide = 4 if state == F32 else 1
    now = [states.exp_avg.view(torch.uint8), states.exp_avg_sq.view(torch.uint8)]
    untouched = ~used.repeat_interleave(wide)
    assert all(torch.equal(a[untouched], b[untouched]) for a, b in zip(now, held))
    behind = torch.ones_like(used)
    for i, p in enumerate(params):
        behind[states.offsets[i]:states.offsets[i] + p.numel()] = False
    assert bool((states.exp_avg.float()[behind] == 0).all()) and bool((states.exp_avg_sq.float()[behind] == 0).all())
    inside = torch.zeros_like(buf, dtype=torch.bool)
    for p in params:
        a = (p.data_ptr() - buf.data_ptr()) // buf.element_size()
        inside[a:a + p.numel()] = True
    assert torch.equal(buf[~inside], outside[~inside])
    return states, params, grads


def check_cancelling(q, scale, y, off):
    """As check_eight, where each value is known to within its own `off`."""
    q, scale = q.double(), scale.double()
    most = y.abs().amax(1)
    want = torch.where(most > 0, (most / 448).clamp_min(2.0 ** -126), 1.0)
    assert bool(((scale - want).abs() <= off.amax(1) / 448 + 3 * U * want).all())
    t = y / scale[:, None]
    e = t.abs() * 3 * U + off / scale[:, None]
    lo, hi = ((t + s * e).clamp(-448, 448).float().to(E4).double() for s in (-1, 1))
    assert bool(((q >= lo) & (q <= hi)).all())


SIZES = [[1], [7], [8], [127], [128], [129], [1000], [4096], [4097], [2048], [2049], [70001], [(33, 65)], [(3, 5, 7)],
         [0, 5, 0], [1] * 40, [300, 1, 4096, 128, 0, 9000], list(range(1, 60)), [5000] * 33, [100] * 600]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("state", [F32, E4])
def test_sizes(sizes, state):
    run_and_check(sizes, F32, F32, state)
    run_and_check(sizes, BF, BF, state)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("gdtype", [BF, F32])
@pytest.mark.parametrize("state", [F32, E4])
@pytest.mark.parametrize("shift,gap,gshift", [(0, 0, 0), (0, 8, 0), (1, 0, 1), (3, 1, 5), (4, 4, 4), (0, 0, 1), (1, 0, 0)])
def test_types_and_alignments(dtype, gdtype, state, shift, gap, gshift):
    sizes = [5000, 64, 4096, 1, 777, 12345]
    run_and_check(sizes, dtype, gdtype, state, shift=shift, gap=gap, gshift=gshift)
    run_and_check(sizes, dtype, gdtype, state, shift=shift, gap=gap, gshift=gshift, copies=True,
                  scale=torch.tensor(0.37, device=DEV), decay=[0.1, 0.0, 0.2, 0.0, 0.0, 0.1],
                  lr_scale=[1.0, 2.0, 0.5, 1.0, 0.0, 1.0])


@pytest.mark.parametrize("state", [F32, E4])
@pytest.mark.parametrize("kw", [dict(step=1), dict(step=100000), dict(betas=(0.0, 0.0)), dict(betas=(0.0, 0.999)),
                                dict(betas=(0.99, 0.5)), dict(lr=0.0), dict(lr=1.0, decay=0.5), dict(eps=1e-3), dict(eps=2.0 ** -126),
                                dict(skip=(0,)), dict(skip=(1, 2)), dict(skip=(0, 1, 2))])
def test_constants_and_missing_gradients(state, kw):
    run_and_check([1000, 4096, 300], F32, BF, state, **kw)


@pytest.mark.parametrize("state", [F32, E4])
@pytest.mark.parametrize("shift", [1, 2, 3, 4, 5, 6, 7])
def test_every_place_between_boundaries(shift, state):
    """Ends of tensors, of a warp's 256 values and of a block's 1024 at every place
    between two 16-byte boundaries, of parameters and gradients apart."""
    sizes = [1, 7, 9, 255, 256, 257, 264, 511, 1023, 1024, 1025, 1288, 2048, 2055]
    run_and_check(sizes, BF, BF, state, shift=shift, gap=16 - shift, gshift=8 - shift)
    run_and_check(sizes, F32, BF, state, shift=shift, gap=shift, gshift=shift, copies=True)
    run_and_check(sizes, BF, F32, state, shift=0, gap=8, gshift=shift)


@pytest.mark.parametrize("shift", [0, 3])
def test_states_in_8_bits_are_the_formulas_in_32(shift):
    """Codes as elementary 32-bit operations give them, each rounded, over several
    steps; their scales to one last place (the roots' step of Newton's iteration is
    rounded to nearest but where 2^-21 of all arguments lie by a midpoint)."""
    n, (b1, b2) = 300000, (0.9, 0.95)
    (p,), _ = make([n], F32, 0, shift=shift)
    s = ops.AdamWStates([p], dtype=E4)
    pad = s.exp_avg.numel() - n
    m = torch.zeros(n + pad, device=DEV).view(-1, 128)
    r = torch.zeros_like(m)
    for step in range(1, 5):
        (g,), _ = make([n], BF, step, std=1e-3, shift=shift)
        g = g * torch.exp(2 * torch.randn(n, device=DEV, generator=gen(step + 10))).bfloat16()
        g[1000:3000] = 0
        ops.adamw_update(s, [g], lr=1e-4, step=step, betas=(b1, b2))
        g32 = torch.nn.functional.pad(g.float(), (0, pad)).view(-1, 128)
        m = b1 * m + (1 - b1) * g32
        r = torch.sqrt(b2 * (r * r) + (1 - b2) * g32 * g32)
        held = []
        for y, codes, scale in ((m, s.exp_avg, s.exp_avg_scale), (r, s.exp_avg_sq, s.exp_avg_sq_scale)):
            most = y.abs().amax(-1)
            want = torch.where(most > 0, (most * (1.0 / 448)).clamp_min(2.0 ** -126), 1.0)
            q = y * (1.0 / want)[:, None]
            q = torch.where(y > 0, q.clamp_min(2.0 ** -9), q) if y is r else q
            q = q.clamp(-448, 448).to(E4)
            assert torch.equal(q.view(-1).float(), codes.float())
            assert ((scale - want).abs() <= 2.0 ** -23 * want).all()
            held.append(codes.float().view(-1, 128) * scale[:, None])
        m, r = held


def first_scales(g, r, betas):
    """The scales of the roots that one step leaves of groups whose values are all
    alike: gradient g, root r before.  A group's scale is its root times 1 / 448."""
    grad = g[:, None].expand(-1, 128).reshape(-1).contiguous()
    s = ops.AdamWStates([torch.zeros(grad.numel(), device=DEV)], dtype=E4)
    s.exp_avg_sq.copy_(torch.full_like(s.exp_avg_sq, 256.0, dtype=F32))
    s.exp_avg_sq_scale.copy_(r / 256)
    ops.adamw_update(s, [grad], lr=1e-4, step=1, betas=betas)
    return s.exp_avg_sq_scale


def scales_of(v):
    """sqrt(v) rounded to 32 bits once (a 64-bit root holds twice the digits and two
    more, so rounding it again is rounding the root), times 1 / 448."""
    s = v.double().sqrt().float() * (1.0 / 448)
    return torch.where(v > 0, s.clamp_min(2.0 ** -126), 1.0)


def test_roots_of_every_mantissa_are_rounded_to_nearest():
    """All 2^24 numbers of two binades, the second moments v = a + 0.75 g^2 of a = r^2 / 4."""
    b2 = 0.25
    for lo in range(0, 1 << 24, 1 << 18):
        at = torch.arange(lo, lo + (1 << 18), device=DEV)
        v = ((at % (1 << 23)).float() * 2.0 ** -23 + 1) * (1.0 if lo < 1 << 23 else 2.0)
        k = (16 * v.sqrt()).floor() - 1  # a = (k / 16)^2 is exact, and v - a at least 1 / 16
        a, r = (k / 16).square(), k / 8
        g = ((v.double() - a.double()) / (1 - b2)).sqrt().float()
        for step in (1, -1, 2, -2, 3, -3):  # the gradient near it with which the rounded operations meet v
            near = (g.view(torch.int32) + step).view(F32)
            g = torch.where(a + (g * (1 - b2)) * g == v, g, torch.where(a + (near * (1 - b2)) * near == v, near, g))
        assert bool((a + (g * (1 - b2)) * g == v).all())
        assert torch.equal(first_scales(g, r, (0.9, b2)), scales_of(v))


def test_roots_of_all_sizes_are_rounded_to_nearest():
    """From what underflows to what overflows nearly; and of nothing."""
    e = torch.rand(1 << 15, generator=gen(1), device=DEV) * 144 - 80
    g = (1 + torch.rand(1 << 15, generator=gen(2), device=DEV)) * e.floor().exp2()
    g[:100] = 0
    want = scales_of((g * 0.5) * g)
    assert torch.equal(first_scales(g, torch.zeros_like(g), (0.9, 0.5)), want) and bool((want == 1).any())


@pytest.mark.parametrize("shift", [1, 3])
def test_states_in_8_bits_of_shifted_gradients_are_the_aligned_ones(shift):
    """Gradients, parameters and copies off 16-byte boundaries leave the same bits."""
    sizes, held = [70001, 130, 4096], []
    for by in (0, shift):
        params, _ = make(sizes, F32, 0, shift=by, gap=by)
        grads, _ = make(sizes, BF, 1, std=1e-3, shift=by, gap=by)
        assert by == 0 or all(g.data_ptr() % 16 for g in grads)
        copies, _ = make(sizes, BF, 2, shift=by, gap=by)
        s = ops.AdamWStates(params, dtype=E4, copies=copies)
        for step in range(1, 5):
            for i, g in enumerate(grads):
                g.mul_(torch.exp(torch.randn(g.shape, generator=gen(10 * step + i), device=DEV)).bfloat16())
            ops.adamw_update(s, grads, lr=1e-3, step=step)
        held.append([*params, *copies, s.exp_avg.float(), s.exp_avg_sq.float(), s.exp_avg_scale, s.exp_avg_sq_scale])
    assert all(torch.equal(a, b) for a, b in zip(*held))


@pytest.mark.parametrize("b2", [0.95, 0.98])
def test_states_in_8_bits_over_hundreds_of_steps(b2):
    """Gradients that fall tenfold but for one value of each group: the codes are the
    formula's in 32 bits all the way, and the roots follow what fell (documented as 1.0 and
    1.04 times the true ones after 20 / (1 - beta2) steps, by a simulation on the CPU; a
    median of 8128 values, each of some half step of E4M3, moves by less than 0.01)."""
    b1, groups = 0.9, 64
    s = ops.AdamWStates([torch.zeros(groups * 128, device=DEV)], dtype=E4)
    m, r, v64 = (torch.zeros(groups, 128, device=DEV) for _ in range(3))
    v64 = v64.double()

    def eight(y, least):
        most = y.abs().amax(-1)
        scale = torch.where(most > 0, (most * (1.0 / 448)).clamp_min(2.0 ** -126), 1.0)
        q = y * (1.0 / scale)[:, None]
        q = torch.where(y > 0, q.clamp_min(2.0 ** -9), q) if least else q
        return q.clamp(-448, 448).to(E4).float(), scale

    g, warm = gen(1), round(5 / (1 - b2))
    for step in range(1, warm + round(20 / (1 - b2)) + 1):
        grad = torch.randn(groups, 128, generator=g, device=DEV)
        if step > warm:
            grad[:, 1:] *= 0.1
        ops.adamw_update(s, [grad.view(-1)], lr=1e-4, step=step, betas=(b1, b2))
        m, r = b1 * m + (1 - b1) * grad, torch.sqrt(b2 * (r * r) + (1 - b2) * grad * grad)
        v64 = b2 * v64 + (1 - b2) * grad.double() ** 2
        (mq, ms), (rq, rs) = eight(m, False), eight(r, True)
        m, r = mq * ms[:, None], rq * rs[:, None]
    for codes, scale, q, want in ((s.exp_avg, s.exp_avg_scale, mq, ms), (s.exp_avg_sq, s.exp_avg_sq_scale, rq, rs)):
        assert torch.equal(codes.float().view(-1, 128), q) and torch.equal(scale, want)
    ratio = (r.double() / v64.sqrt())[:, 1:].median().item()
    assert abs(ratio - {0.95: 1.0, 0.98: 1.04}[b2]) < 0.02


def test_betas_that_8_bits_do_not_follow_warn():
    def step(betas, dtype):
        ops.adamw_update(ops.AdamWStates([torch.zeros(128, device=DEV)], dtype=dtype), [torch.ones(128, device=DEV)],
                         lr=1e-3, step=1, betas=betas)
    for betas in ((0.9, 0.99), (0.96, 0.95)):
        with pytest.warns(RuntimeWarning, match="8 bits"):
            step(betas, E4)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        step((0.95, 0.98), E4)
        step((0.99, 0.999), F32)


def test_a_large_tensor():
    """Values past 2^31, and a tensor behind them."""
    n = (1 << 31) + 1000
    p = torch.zeros(n, dtype=BF, device=DEV)
    q = torch.ones(300, dtype=BF, device=DEV)
    g = torch.zeros(n, dtype=BF, device=DEV)
    g[-1000:], g[:1000] = 1.0, -1.0
    states = ops.AdamWStates([p, q], dtype=E4)
    ops.adamw_update(states, [g, torch.ones(300, dtype=BF, device=DEV)], lr=0.5, step=1)
    assert bool((p[-1000:] == -0.5).all()) and bool((p[:1000] == 0.5).all()) and bool((p[1000:-1000] == 0).all())
    assert bool((q == 0.5).all())
    norm, _ = ops.grad_norm([g])
    assert norm.item() == pytest.approx(math.sqrt(2000), rel=1e-6)


@pytest.mark.parametrize("state", [F32, E4])
def test_step_and_rate_on_the_device(state):
    sizes = [1000, 300]
    one, _, grads = run_and_check(sizes, F32, F32, state, step=5, lr=3e-3)
    params, _ = make(sizes, F32, 0)
    two = ops.AdamWStates(params, dtype=state, weight_decay=0.1)
    fill(two)
    lr = torch.tensor(3e-3, device=DEV)
    ops.adamw_update(two, grads, lr=lr, step=torch.tensor([5], device=DEV))
    for a, b in zip(one.params, two.params):  # the rate is 3e-3 rounded to 32 bits
        assert bool(((a - b).abs() <= 2 * U * a.abs() + 2 * U * 3e-3 * 3).all())
    for k, t in two.state_dict().items():
        if k != "numel":
            assert torch.equal(t.view(torch.uint8), getattr(one, k).view(torch.uint8))


@pytest.mark.parametrize("state", [F32, E4])
def test_captured_and_replayed(state):
    """A step with its clip factor in a graph: the count of steps, gradients and rate are read anew."""
    sizes = [5000, 64, 777]

    def begin():
        params, _ = make(sizes, F32, 0)
        return ops.AdamWStates(params, dtype=state, weight_decay=0.1), torch.tensor(1e-2, device=DEV)
    eager, lr = begin()
    held, lr2 = begin()
    grads, buf = make(sizes, F32, 1)
    step = torch.zeros((), dtype=torch.int64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up on states of its own
        ops.adamw_update(begin()[0], grads, lr=lr2, step=1, grad_scale=ops.grad_norm(grads, max_norm=1.0)[1])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.add_(1)
        norm, scale = ops.grad_norm(grads, max_norm=1.0)
        ops.adamw_update(held, grads, lr=lr2, step=step, grad_scale=scale)
    for i in range(1, 4):
        buf.copy_(torch.randn(buf.shape, generator=gen(50 + i), device=DEV))
        lr.fill_(1e-2 / i)
        lr2.fill_(1e-2 / i)
        graph.replay()
        n, s = ops.grad_norm(grads, max_norm=1.0)
        ops.adamw_update(eager, grads, lr=lr, step=i, grad_scale=s)
        assert torch.equal(n, norm) and torch.equal(s, scale)
        for a, b in zip(eager.params, held.params):
            assert bool(((a - b).abs() <= 2 * U * a.abs() + 1e-2 * 8 * U * i).all())


@pytest.mark.parametrize("state", [F32, E4])
@pytest.mark.parametrize("how", ["nan scale", "inf scale", "norm of inf", "nan rate", "step 0"])
def test_nothing_changes(state, how):
    params, _ = make([500, 5000], F32, 0)
    grads, _ = make([500, 5000], F32, 1)
    copies, _ = make([500, 5000], BF, 2)
    states = ops.AdamWStates(params, dtype=state, weight_decay=0.1, copies=copies)
    fill(states)
    before = [t.clone() for t in (*params, *copies, *(t for k, t in states.state_dict().items() if k != "numel"))]
    kw = dict(lr=1e-2, step=3)
    if how == "norm of inf":
        grads[1][77] = float("inf")
        norm, kw["grad_scale"] = ops.grad_norm(grads, max_norm=1.0)
        assert torch.isinf(norm) and torch.isnan(kw["grad_scale"])
    elif how == "nan rate":
        kw["lr"] = torch.tensor(float("nan"), device=DEV)
    elif how == "step 0":
        kw["step"] = torch.zeros((), dtype=torch.int64, device=DEV)
    else:
        kw["grad_scale"] = torch.tensor(float(how[:3]), device=DEV)
    ops.adamw_update(states, grads, **kw)
    after = (*params, *copies, *(t for k, t in states.state_dict().items() if k != "numel"))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, after))


@pytest.mark.parametrize("shift", [0, 1])
def test_values_that_are_not_finite(shift):
    """32 bits: one value; 8 bits: its group."""
    for state in (F32, E4):
        params, _ = make([1000], F32, 0, shift=shift)
        grads, _ = make([1000], F32, 1, shift=shift)
        clean = [t.clone() for t in params]
        a, b = ops.AdamWStates(clean, dtype=state), ops.AdamWStates(params, dtype=state)
        ops.adamw_update(a, grads, lr=1e-2, step=1)
        grads[0][300] = float("nan")
        ops.adamw_update(b, grads, lr=1e-2, step=1)
        nan = torch.zeros(1000, dtype=torch.bool, device=DEV)
        nan[300] = True
        assert bool(torch.isnan(params[0])[nan].all()) and torch.equal(params[0][~nan], clean[0][~nan])
        m, v = b.moments(0)
        if state == E4:
            nan[256:384] = True
        assert bool(torch.isnan(m)[nan].all()) and bool(torch.isnan(v)[nan].all())
        assert torch.equal(m[~nan], a.moments(0)[0][~nan]) and torch.equal(v[~nan], a.moments(0)[1][~nan])


@pytest.mark.parametrize("shift", [0, 1])
def test_a_small_root_beside_a_large_one_does_not_become_zero(shift):
    """2^-20 of the group's largest: below E4M3's range, held at its smallest number."""
    params, _ = make([256], F32, 0, shift=shift)
    grads, _ = make([256], F32, 1, shift=shift)
    grads[0].fill_(2.0 ** -20)
    grads[0][5], grads[0][7] = 1.0, 0.0
    states = ops.AdamWStates(params, dtype=E4)
    ops.adamw_update(states, grads, lr=1e-3, step=1, betas=(0.9, 0.95))
    r = states.exp_avg_sq.float()
    assert r[5] == 448 and r[7] == 0 and bool((r[[0, 1, 6, 127]] == 2.0 ** -9).all()) and bool((r[128:] == 448).all())


def test_a_parameter_whose_data_was_replaced():
    params, _ = make([300, 500], F32, 0)
    grads, _ = make([300, 500], F32, 1)
    states = ops.AdamWStates(params, dtype=F32)
    ref = [p.clone() for p in params]
    other = ops.AdamWStates(ref, dtype=F32)
    ops.adamw_update(states, grads, lr=1e-2, step=1)
    ops.adamw_update(other, grads, lr=1e-2, step=1)
    params[1].data = params[1].clone()
    ops.adamw_update(states, grads, lr=1e-2, step=2)
    ops.adamw_update(other, grads, lr=1e-2, step=2)
    assert all(torch.equal(a, b) for a, b in zip(params, ref))
    for data in (params[1].to(BF), params[1][:400].clone(), params[0][:250].clone()):
        keep, params[1].data = params[1].data, data
        with pytest.raises((TypeError, ValueError)):
            ops.adamw_update(states, grads, lr=1e-2, step=3)
        params[1].data = keep


def test_states_saved_and_loaded():
    for state in (F32, E4):
        a, params, grads = run_and_check([1000, 129], F32, F32, state)
        saved = {k: v if k == "numel" else v.clone() for k, v in a.state_dict().items()}
        again = [p.clone() for p in params]
        b = ops.AdamWStates(again, dtype=state, weight_decay=0.1)
        b.load_state_dict(saved)
        for s in (a, b):
            ops.adamw_update(s, grads, lr=1e-2, step=8)
        assert all(torch.equal(x, y) for x, y in zip(params, again))
        with pytest.raises(ValueError):
            ops.AdamWStates([params[0].clone()], dtype=state).load_state_dict(saved)
        with pytest.raises(ValueError):
            ops.AdamWStates(again, dtype=E4 if state == F32 else F32).load_state_dict(saved)
        m, v = a.moments(1)
        assert m.shape == params[1].shape and bool((v >= 0).all())


# ------------------------------------------------------------------ the norm

@pytest.mark.parametrize("sizes", SIZES + [[40000, 16384, 16385, 100003], [3_000_001, 17]], ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("shift,gap", [(0, 0), (1, 0), (3, 1), (0, 5)])
def test_norm(sizes, shift, gap):
    a, _ = make(sizes, F32, 1, shift=shift, gap=gap)
    b, _ = make(sizes, BF, 2, shift=shift, gap=gap)
    for grads in (a, b, [x for pair in zip(a, b) for x in pair]):
        want = math.sqrt(sum(g.double().square().sum().item() for g in grads))
        for max_norm in (0.5 * want, 2 * want):
            norm, scale = ops.grad_norm(grads, max_norm=max_norm)
            # at most 32 terms in 32 bits (40 roundings with their join), halved by the root, and the result's own
            assert abs(norm.item() - want) <= 22 * U * want
            assert abs(scale.item() - min(1.0, max_norm / want)) <= 26 * U
        again, none = ops.grad_norm([None, *grads])
        assert none is None and torch.equal(again, norm)


def test_norm_of_nothing_and_of_what_is_not_finite():
    g = [torch.zeros(1000, device=DEV), torch.zeros(0, device=DEV)]
    norm, scale = ops.grad_norm(g, max_norm=1.0)
    assert norm == 0 and scale == 1 and norm.shape == scale.shape == ()
    norm, scale = ops.grad_norm(g[1:], max_norm=1.0)
    assert norm == 0 and scale == 1
    for bad in (float("inf"), float("nan"), float("-inf")):
        g[0][999] = bad
        norm, scale = ops.grad_norm(g, max_norm=1.0)
        assert not torch.isfinite(norm) and torch.isnan(scale)
    # a long run of equal values, whose roundings all go one way
    g = [torch.full((60_000_000,), 0.1, device=DEV)]
    want = math.sqrt(60_000_000) * g[0][0].double().item()
    assert abs(ops.grad_norm(g)[0].item() - want) <= 22 * U * want


def test_norm_on_other_streams():
    g, _ = make([100000, 77], F32, 1)
    ws = torch.empty(1 << 16, dtype=torch.uint8, device=DEV)
    want = ops.grad_norm(g, max_norm=1.0, workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.grad_norm(g, max_norm=1.0)
    side.synchronize()
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_rates_beyond_32_bits_are_refused():
    p, _ = make([300, 500], F32, 0)
    g, _ = make([300, 500], F32, 1)
    before = [t.clone() for t in p]
    for lr, scale in ((1e39, 1.0), (-1e39, 1.0), (1e30, [1.0, 1e30]), (float("nan"), 1.0), (1e39, [0.5, 0.5])):
        with pytest.raises(ValueError):
            ops.adamw_update(ops.AdamWStates(p, lr_scale=scale), g, lr=lr, step=1)
    with pytest.raises(ValueError):
        ops.AdamWStates(p, lr_scale=1e39)
    with pytest.raises(ValueError):
        ops.AdamWStates(p, weight_decay=[0.0, -1e39])
    assert all(torch.equal(a, b) for a, b in zip(before, p))
    ops.adamw_update(ops.AdamWStates(p, lr_scale=[1e-30, 1e-30]), g, lr=1e30, step=1)
    assert not any(torch.equal(a, b) for a, b in zip(before, p))


def test_refusals():
    p, _ = make([300, 500], F32, 0)
    g, _ = make([300, 500], F32, 1)
    states = ops.AdamWStates(p)
    up = lambda grads=g, **kw: ops.adamw_update(states, grads, **{"lr": 1e-3, "step": 1, **kw})  # noqa: E731
    bad = [(ValueError, lambda: ops.AdamWStates([])), (TypeError, lambda: ops.AdamWStates([p[0].half()])),
           (ValueError, lambda: ops.AdamWStates([p[0].cpu()])), (ValueError, lambda: ops.AdamWStates([p[0].view(10, 30).t()])),
           (ValueError, lambda: ops.AdamWStates([p[0], p[0]])), (ValueError, lambda: ops.AdamWStates([p[0], p[0][200:]])),
           (ValueError, lambda: ops.AdamWStates(p, copies=[None])), (TypeError, lambda: ops.AdamWStates(p, dtype=BF)),
           (ValueError, lambda: ops.AdamWStates(p, copies=[p[0], None])), (ValueError, lambda: ops.AdamWStates(p, weight_decay=[0.1])),
           (ValueError, lambda: ops.AdamWStates(p, lr_scale=float("nan"))), (TypeError, lambda: ops.AdamWStates([1.0])),
           (ValueError, lambda: ops.AdamWStates(p, copies=[None, p[0].view(BF)[:500]])),  # shares memory with p[0]
           (TypeError, lambda: ops.adamw_update(p, g, lr=1e-3, step=1)), (ValueError, lambda: up(g[:1])),
           (ValueError, lambda: up([g[0], g[1][:300]])), (ValueError, lambda: up([g[0], g[1].view(50, 10)])),
           (TypeError, lambda: up([g[0], g[1].half()])), (ValueError, lambda: up([g[0], g[1].cpu()])),
           (ValueError, lambda: up([g[0], torch.empty(1000, device=DEV)[::2]])), (ValueError, lambda: up(step=0)),
           (ValueError, lambda: up(step=1.0)), (ValueError, lambda: up(lr=float("inf"))), (ValueError, lambda: up(betas=(1.0, 0.9))),
           (ValueError, lambda: up(betas=(0.9, -0.1))), (ValueError, lambda: up(eps=-1.0)), (ValueError, lambda: up(eps=0.0)), (ValueError, lambda: up(eps=1e-40)),
           (TypeError, lambda: up(grad_scale=torch.ones((), dtype=torch.float64, device=DEV))),
           (ValueError, lambda: up(grad_scale=torch.ones(()))), (ValueError, lambda: up(grad_scale=torch.ones(2, device=DEV))),
           (TypeError, lambda: up(step=torch.ones((), device=DEV))),
           (ValueError, lambda: ops.grad_norm([])), (ValueError, lambda: ops.grad_norm([None])),
           (TypeError, lambda: ops.grad_norm([g[0].half()])), (ValueError, lambda: ops.grad_norm([g[0].cpu()])),
           (ValueError, lambda: ops.grad_norm([g[0], g[1].cpu()])), (ValueError, lambda: ops.grad_norm(g, max_norm=0.0)),
           (ValueError, lambda: ops.grad_norm(g, max_norm=float("inf"))), (TypeError, lambda: ops.grad_norm([3])),
           (ValueError, lambda: ops.grad_norm([g[0].view(10, 30).t()]))]
    before = [t.clone() for t in p]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail(f"refusal {i} did not come")
    keep, states.exp_avg = states.exp_avg, states.exp_avg[:128]
    with pytest.raises(ValueError):
        up()
    states.exp_avg = keep
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, p))
