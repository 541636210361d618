"""rope_scaled against a 64-bit rotation: layouts, part of the head, scaled
frequencies, positions deep in a long context, strides, in-place use, the
gradient, and its refusals."""
import math

import pytest
import torch

from kernelproblems_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(x, pos, plan, layout, backward=False):
    """(rotated values in 64 bits, m(|a| + |b|) of each element's pair)."""
    x = x.double()
    half, m = plan.rotary_dim // 2, plan.attention_factor
    angle = 2 * math.pi * torch.remainder(pos.double()[..., None] * plan.turns.to(x.device), 1.0)
    cos, sin = (m * angle.cos())[:, :, None], (m * angle.sin())[:, :, None] * (-1 if backward else 1)
    out, size = x.clone(), torch.zeros_like(x)
    ia = torch.arange(half, device=x.device) * (1 if layout == "neox" else 2)
    ib = ia + (half if layout == "neox" else 1)
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * cos - b * sin, b * cos + a * sin
    size[..., ia] = size[..., ib] = m * (a.abs() + b.abs())
    return out, size


def check(got, x, pos, plan, layout, backward=False):
    """One rounding to bf16 (at most 2^-8 of the value) and the 32-bit errors of a sine
    or cosine (under 2^-21), its product with m and the rotation's two products."""
    want, size = reference(x, pos, plan, layout, backward)
    err = (got.double() - want).abs()
    bound = 2.0 ** -8 * want.abs() * 1.001 + 4e-6 * size
    assert bool((err <= bound).all()), f"worst excess {(err - bound).max().item():.3g}"
    assert torch.equal(got[..., plan.rotary_dim:], x[..., plan.rotary_dim:])


def rand(*shape, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)


PLANS = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
         dict(scaling="smooth", factor=8.0), dict(scaling="parts", factor=4.0),
         dict(scaling="parts", factor=16.0, attention_factor=0.7)]


@pytest.mark.parametrize("layout", ["neox", "interleaved"])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (96, 48), (80, 20), (80, 80), (64, 2), (256, 256),
                                   (160, 160), (96, 24), (512, 512), (36, 12), (34, 34), (1000, 512), (7, 2)])
def test_heads(D, rot, layout):
    plan = ops.RopeFrequencies(D, rotary_dim=rot)
    q, k = rand(2, 5, 6, D, seed=1), rand(2, 5, 1, D, seed=2)
    pos = torch.tensor([[0, 1, 7, 100, 8191], [131071, 3, 2, 1, 0]], device=DEV)
    for backward in (False, True):
        oq, ok = ops.rope_scaled(q, k, pos, freqs=plan, layout=layout, backward=backward)
        check(oq, q, pos, plan, layout, backward)
        check(ok, k, pos, plan, layout, backward)


@pytest.mark.parametrize("kw", PLANS)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_scalings_and_long_positions(kw, dtype):
    plan = ops.RopeFrequencies(128, rotary_dim=96, **kw)
    q = rand(1, 9, 4, 128, seed=3)
    pos = torch.tensor([0, 1, 4095, 65536, 1 << 20, (1 << 24) + 1, (1 << 30) + 7, 2 ** 31 - 1, -5], device=DEV,
                       dtype=dtype)
    oq, none = ops.rope_scaled(q, None, pos, freqs=plan)
    assert none is None
    check(oq, q, pos[None].expand(1, 9), plan, "neox")


@pytest.mark.parametrize("B,S,Hq,Hk", [(1, 1, 32, 8), (7, 1, 5, 1), (1, 513, 16, 16), (3, 129, 40, 8), (2, 2049, 3, 0)])
def test_tokens(B, S, Hq, Hk):
    plan = ops.RopeFrequencies(128, scaling="smooth", factor=8.0)
    q, k = rand(B, S, Hq, 128, seed=4), rand(B, S, Hk, 128, seed=5) if Hk else None
    oq, ok = ops.rope_scaled(q, k, None, freqs=plan)
    pos = torch.arange(S, device=DEV).expand(B, S)
    check(oq, q, pos, plan, "neox")
    if Hk:
        check(ok, k, pos, plan, "neox")


@pytest.mark.parametrize("B,S,H", [(0, 4, 2), (2, 0, 2), (2, 3, 0)])
def test_empty(B, S, H):
    plan = ops.RopeFrequencies(64)
    oq, _ = ops.rope_scaled(rand(B, S, H, 64), None, None, freqs=plan)
    assert oq.shape == (B, S, H, 64)


@pytest.mark.parametrize("layout", ["neox", "interleaved"])
@pytest.mark.parametrize("D,rot", [(128, 128), (96, 32), (80, 20)])
def test_strides(D, rot, layout):
    plan = ops.RopeFrequencies(D, rotary_dim=rot, scaling="parts", factor=4.0)
    pos = torch.arange(33, device=DEV, dtype=torch.int32)
    packed = rand(2, 33, 6, D, seed=6)
    bhsd = rand(2, 5, 33, D, seed=7).transpose(1, 2)
    odd = rand(2, 33, 5 * D + 3, seed=8)[..., 1:1 + 5 * D].unflatten(-1, (5, D))  # rows at odd addresses
    shared = rand(2, 33, 1, D, seed=9).expand(2, 33, 5, D)
    for q in (packed[:, :, :4], packed[:, :, 4:], bhsd, odd, shared):
        for backward in (False, True):
            oq, _ = ops.rope_scaled(q, None, pos, freqs=plan, layout=layout, backward=backward)
            check(oq, q, pos[None].expand(2, 33), plan, layout, backward)
    oq, ok = ops.rope_scaled(bhsd, packed, pos, freqs=plan, layout=layout, out_layout="bhsd")
    assert oq.transpose(1, 2).is_contiguous()
    check(oq, bhsd, pos[None].expand(2, 33), plan, layout)
    check(ok, packed, pos[None].expand(2, 33), plan, layout)


@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (80, 20)])
def test_in_place_leaves_the_rest(D, rot):
    plan = ops.RopeFrequencies(D, rotary_dim=rot)
    packed = rand(2, 17, 8, D, seed=10)
    before = packed.clone()
    q, k = packed[:, :, :4], packed[:, :, 4:6]
    ops.rope_scaled(q, k, None, freqs=plan, out_q=q, out_k=k)
    pos = torch.arange(17, device=DEV).expand(2, 17)
    check(packed[:, :, :6], before[:, :, :6], pos, plan, "neox")
    assert torch.equal(packed[:, :, 6:], before[:, :, 6:])


@pytest.mark.parametrize("layout", ["neox", "interleaved"])
def test_gradient_is_the_transpose_and_matches_differences(layout):
    """<g, R x> = <R'g, x>; and the difference quotient of <g, R(x + e v)>
    along v is <R'g, v>.  Both sides carry one bf16 rounding of each value."""
    plan = ops.RopeFrequencies(96, rotary_dim=48, scaling="parts", factor=8.0)
    x, g, v = (rand(2, 50, 4, 96, seed=s) for s in (11, 12, 13))
    pos = torch.arange(100, device=DEV).view(2, 50) * 977
    rx = ops.rope_scaled(x, None, pos, freqs=plan, layout=layout)[0].double()
    rg = ops.rope_scaled(g, None, pos, freqs=plan, layout=layout, backward=True)[0].double()
    g64, x64, v64 = g.double(), x.double(), v.double()
    n = 2.0 ** -9 * 8  # 8 standard deviations of independent roundings
    slack = n * ((g64 * rx).norm() + (rg * x64).norm())
    assert (g64 * rx).sum().sub((rg * x64).sum()).abs() <= slack
    e = 0.25
    up = reference(x64 + e * v64, pos, plan, layout)[0]
    down = reference(x64 - e * v64, pos, plan, layout)[0]
    quotient = (g64 * (up - down)).sum() / (2 * e)
    assert (quotient - (rg * v64).sum()).abs() <= n * (rg * v64).norm()


def test_another_stream():
    plan = ops.RopeFrequencies(128)
    q = rand(2, 64, 8, 128, seed=14)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        oq, _ = ops.rope_scaled(q, None, None, freqs=plan)
    s.synchronize()
    check(oq, q, torch.arange(64, device=DEV).expand(2, 64), plan, "neox")


def test_refusals():
    plan = ops.RopeFrequencies(64, rotary_dim=32)
    q = rand(2, 4, 3, 64)
    with pytest.raises(TypeError):
        ops.rope_scaled(q.float(), freqs=plan)
    with pytest.raises(TypeError):
        ops.rope_scaled(q, freqs=None)
    with pytest.raises(ValueError):
        ops.rope_scaled(q.cpu(), freqs=plan)
    with pytest.raises(ValueError):
        ops.rope_scaled(rand(2, 4, 3, 128), freqs=plan)
    with pytest.raises(ValueError):
        ops.rope_scaled(q[0], freqs=plan)
    with pytest.raises(ValueError):
        ops.rope_scaled(q, freqs=plan, layout="other")
    with pytest.raises(ValueError):
        ops.rope_scaled(q, rand(2, 5, 3, 64), freqs=plan)
    with pytest.raises(ValueError):
        ops.rope_scaled(q, None, torch.arange(5, device=DEV), freqs=plan)
    with pytest.raises(ValueError):
        ops.rope_scaled(q, None, torch.arange(4), freqs=plan)
    with pytest.raises(TypeError):
        ops.rope_scaled(q, None, torch.arange(4, device=DEV).float(), freqs=plan)
    with pytest.raises(ValueError):  # overlaps q, shifted
        wide = rand(2, 5, 3, 64)
        ops.rope_scaled(wide[:, :4], freqs=plan, out_q=wide[:, 1:])
    with pytest.raises(ValueError):  # an expanded output
        ops.rope_scaled(q, freqs=plan, out_q=torch.empty(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV).expand(2, 4, 3, 64))
    with pytest.raises(ValueError):  # the two outputs are one buffer
        o = torch.empty_like(q)
        ops.rope_scaled(q, q.clone(), freqs=plan, out_q=o, out_k=o)
    with pytest.raises(TypeError):
        ops.rope_scaled(q, freqs=plan, out_q=torch.empty(2, 4, 3, 64, device=DEV))
    with pytest.raises(ValueError):
        ops.rope_scaled(rand(2, 4, 64, 3).transpose(2, 3), freqs=plan)


@pytest.mark.parametrize("D,rot", [(128, 128), (96, 32), (80, 20)])
def test_in_place_on_head_major_slices(D, rot):
    """q and k of one packed [B, H, S, D] tensor."""
    plan = ops.RopeFrequencies(D, rotary_dim=rot)
    packed = rand(3, 8, 17, D, seed=15)
    before = packed.clone().transpose(1, 2)
    q, k = packed[:, :4].transpose(1, 2), packed[:, 4:6].transpose(1, 2)
    ops.rope_scaled(q, k, None, freqs=plan, out_q=q, out_k=k)
    pos = torch.arange(17, device=DEV).expand(3, 17)
    after = packed.transpose(1, 2)
    check(after[:, :, :6], before[:, :, :6], pos, plan, "neox")
    assert torch.equal(after[:, :, 6:], before[:, :, 6:])


def test_outputs_that_meet_across_sequences_are_refused():
    plan = ops.RopeFrequencies(64)
    y = torch.empty(4, 3, 5, 64, dtype=torch.bfloat16, device=DEV)
    q, k = rand(2, 4, 5, 64), rand(2, 4, 5, 64, seed=1)
    with pytest.raises(ValueError, match="overlap"):
        ops.rope_scaled(q, k, None, freqs=plan, out_q=y[:, 0:2].transpose(0, 1), out_k=y[:, 1:3].transpose(0, 1))


def test_outputs_over_the_other_input_are_refused():
    plan = ops.RopeFrequencies(64)
    q, k = rand(1, 3, 4, 64), rand(1, 3, 4, 64, seed=1)
    before = q.clone(), k.clone()
    for kw in (dict(out_q=k), dict(out_k=q), dict(out_q=k, out_k=q)):
        with pytest.raises(ValueError, match="overlap"):
            ops.rope_scaled(q, k, None, freqs=plan, **kw)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    out = torch.empty_like(q)  # one output given, the other input in place
    ops.rope_scaled(q, k, None, freqs=plan, out_q=out, out_k=k)
    check(out, before[0], torch.arange(3, device=DEV)[None], plan, "neox")
    check(k, before[1], torch.arange(3, device=DEV)[None], plan, "neox")


def test_in_place_with_other_strides_of_single_dimensions():
    """One token a sequence, one sequence or one head: that dimension's stride
    says nothing, and views of the same elements may differ in it."""
    plan = ops.RopeFrequencies(64)
    for x, view in ((rand(3, 1, 4, 64), lambda t: t.view(3, 4, 1, 64).transpose(1, 2)),
                    (rand(1, 5, 4, 64), lambda t: t.as_strided(t.shape, (64, 256, 64, 1))),
                    (rand(2, 5, 1, 64), lambda t: t.as_strided(t.shape, (320, 64, 8, 1)))):
        before, out = x.clone(), view(x)
        assert out.data_ptr() == x.data_ptr() and out.stride() != x.stride()
        got, _ = ops.rope_scaled(x, None, None, freqs=plan, out_q=out)
        assert got is out
        check(x, before, torch.arange(x.shape[1], device=DEV).expand(x.shape[:2]), plan, "neox")
