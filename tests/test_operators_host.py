"""RopeFrequencies on the CPU: the scaling rules at their ends, and refusals."""
import ctypes as C
import math

import pytest
import torch

from kernelproblems_b200 import _lib, ops


def freq(plan):
    return plan.turns * 2 * math.pi


def plain(rot, theta=500000.0):
    return theta ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)


def test_unscaled_and_linear():
    assert torch.allclose(freq(ops.RopeFrequencies(128)), plain(128), rtol=1e-14)
    p = ops.RopeFrequencies(128, rotary_dim=64, scaling="linear", factor=4.0)
    assert p.rotary_dim == 64 and torch.allclose(freq(p), plain(64) / 4, rtol=1e-14)
    assert p.attention_factor == 1.0


def test_base_slows_the_last_pair_by_the_factor():
    f, g = plain(128), freq(ops.RopeFrequencies(128, scaling="base", factor=8.0))
    assert g[0] == pytest.approx(1.0) and (f[-1] / g[-1]).item() == pytest.approx(8.0, rel=1e-12)


def test_smooth_keeps_short_waves_and_slows_long_ones():
    f = plain(128)
    g = freq(ops.RopeFrequencies(128, scaling="smooth", factor=8.0, original_context=8192))
    turns = 8192 * f / (2 * math.pi)
    assert torch.allclose(g[turns >= 4], f[turns >= 4], rtol=1e-14)
    assert torch.allclose(g[turns <= 1], f[turns <= 1] / 8, rtol=1e-14)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and bool(((g < f) & (g > f / 8))[mid].all())


def test_parts_keeps_the_first_pairs_and_slows_the_last():
    f, p = plain(128), ops.RopeFrequencies(128, scaling="parts", factor=4.0, original_context=4096)
    g = freq(p)
    turns = 4096 * f / (2 * math.pi)
    assert torch.allclose(g[turns > 34], f[turns > 34], rtol=1e-14)
    assert torch.allclose(g[turns < 0.7], f[turns < 0.7] / 4, rtol=1e-14)
    assert p.attention_factor == pytest.approx(0.1 * math.log(4) + 1)
    assert ops.RopeFrequencies(128, scaling="parts", factor=4.0, attention_factor=0.5).attention_factor == 0.5


@pytest.mark.parametrize("kw", [dict(rotary_dim=130), dict(rotary_dim=63), dict(rotary_dim=0), dict(theta=0.0),
                                dict(theta=float("nan")), dict(scaling="other"), dict(factor=0.5),
                                dict(factor=float("inf")), dict(original_context=0), dict(high_turns=1.0),
                                dict(slow_turns=40.0), dict(low_turns=-1.0),
                                dict(scaling="base", rotary_dim=2)])
def test_plan_refusals(kw):
    with pytest.raises(ValueError):
        ops.RopeFrequencies(128, **kw)


def test_rot_limit():
    with pytest.raises(ValueError):
        ops.RopeFrequencies(1024)
    assert ops.RopeFrequencies(1024, rotary_dim=512).turns.numel() == 256


def test_entry_points_reject_bad_arguments_on_the_host():
    lib = _lib.load()
    turns = (C.c_double * 64)()
    t = (_lib.RopeTensor * 1)(_lib.RopeTensor(None, None, 2, 0, 0, 0, 0, 0, 0, 0, 0))
    rope = lambda t, n, B, S, D, rot, lay=0, tu=turns: lib.frag_rope_scaled(  # noqa: E731
        t, n, B, S, D, rot, None, 0, 0, 0, tu, 1.0, lay, 0, None)
    assert rope(None, 1, 1, 1, 128, 128) == 1
    assert rope(t, 3, 1, 1, 128, 128) == 1
    assert rope(t, 1, -1, 1, 128, 128) == 1
    assert rope(t, 1, 1, 1, 128, 128, lay=2) == 1
    assert rope(t, 1, 1, 1, 128, 128, tu=None) == 1
    assert rope(t, 1, 1, 1, 128, 130) == 2
    assert rope(t, 1, 1, 1, 128, 127) == 2
    assert rope(t, 1, 1, 1, 128, 128) == 1   # null tensors
    assert rope(t, 1, 0, 1, 128, 128) == 0   # nothing to do
    fwd = lambda M, N, fmt=0, group=0: lib.frag_rmsnorm_quant_fwd(  # noqa: E731
        None, N, None, 0, None, None, None, None, None, M, N, 1e-5, fmt, group, 0, None)
    assert fwd(4, 64) == 1 and fwd(-1, 64) == 1 and fwd(4, 64, fmt=2) == 1
    assert fwd(4, 64, group=48) == 2 and fwd(4, 0) == 2 and fwd(0, 64) == 0
    bwd = lambda M, N, fmt=1, group=0: lib.frag_rmsnorm_quant_bwd(  # noqa: E731
        None, N, None, N, None, None, None, 0, None, None, None, None, M, N, fmt, group, 0, None, 0, None)
    assert bwd(4, 64) == 1 and bwd(-1, 64) == 1 and bwd(4, 64, fmt=7) == 1
    assert bwd(4, 64, group=1) == 2 and bwd(0, 64) == 0


def test_orthogonalize_rejects_bad_arguments_on_the_host():
    lib = _lib.load()
    co = (C.c_float * 15)(*([3.4, -4.8, 2.0] * 5))
    none = _lib.Matrix(None, 0, 8, 1, 0)
    orth = lambda E, m, n, steps=5, c=co, g=none: lib.frag_orthogonalize(  # noqa: E731
        C.byref(g), None, E, m, n, steps, c, 1e-7, None, 0, None)
    assert orth(1, 8, 8) == 1 and orth(-1, 8, 8) == 1 and orth(1, 8, 8, steps=0) == 1 and orth(1, 8, 8, c=None) == 1
    assert orth(1, 8, 8, steps=33) == 2 and orth(1 << 20, 8, 8) == 2 and orth(1, 1 << 25, 8) == 2
    assert orth(1, 1 << 16, 1 << 16) == 2  # 2^32 elements
    assert orth(0, 8, 8) == 0 and orth(1, 0, 8) == 0
    assert lib.frag_muon_update(C.byref(none), C.byref(none), C.byref(none), None, None, 1, 8, 8, 0.1, 0.9, 1, 0.0, 1.0,
                                5, co, 1e-7, None, 0, None) == 1
    assert lib.frag_orthogonalize_workspace_bytes(0, 8, 8) == 0


def addresses(t):
    """Every byte of a tensor."""
    at = torch.zeros(1, dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n) * s).reshape(-1)
    return set((at[:, None] * t.element_size() + t.data_ptr() + torch.arange(t.element_size())).reshape(-1).tolist())


def test_overlap_of_packed_slices():
    packed = torch.empty(2, 5, 8, 16, dtype=torch.bfloat16)  # [B, S, H, D]
    assert not ops._overlaps(packed[:, :, :4], packed[:, :, 4:6])
    assert ops._overlaps(packed[:, :, :5], packed[:, :, 4:6])
    major = torch.empty(2, 8, 5, 16, dtype=torch.bfloat16).transpose(1, 2)  # [B, H, S, D] storage
    assert not ops._overlaps(major[:, :, :4], major[:, :, 4:6])
    assert ops._overlaps(major[:, :, :4], major[:, :, 3:6])
    # sequences that are disjoint row by row, although row 1 of one is row 0 of the other
    y = torch.empty(4, 3, 5, 8)
    assert ops._overlaps(y[:, 0:2].transpose(0, 1), y[:, 1:3].transpose(0, 1))
    assert not ops._overlaps(y[:, 0:1], y[:, 1:3]) and not ops._overlaps(y[:0], y)
    flat = torch.empty(64)
    assert not ops._overlaps(flat[::2], flat[1::2]) and ops._overlaps(flat[::2], flat[1::3])
    assert ops._overlaps(flat[:4], flat.view(torch.bfloat16)[7:]) and not ops._overlaps(flat[:4], flat.view(torch.bfloat16)[8:])


@pytest.mark.parametrize("seed", range(4))
def test_overlap_against_every_address(seed):
    import random
    r = random.Random(seed)
    buf = torch.empty(4000, dtype=r.choice([torch.bfloat16, torch.float32]))
    other = buf.view(torch.bfloat16)
    for _ in range(300):
        shape = [r.randint(1, 4) for _ in range(r.randint(1, 4))]
        a = buf.as_strided(shape, [r.choice([0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 40, 64]) for _ in shape], r.randint(0, 60))
        if r.random() < 0.5:  # the same strides, as of slices
            b = buf.as_strided([max(1, n + r.choice([-1, 0, 1])) for n in shape], a.stride(), r.randint(0, 60))
        else:
            shape = [r.randint(1, 4) for _ in range(r.randint(1, 4))]
            b = r.choice([buf, other]).as_strided(shape, [r.choice([0, 1, 2, 4, 5, 8, 16, 20, 64]) for _ in shape],
                                                  r.randint(0, 60))
        assert ops._overlaps(a, b) == bool(addresses(a) & addresses(b)), (a.shape, a.stride(), b.shape, b.stride())


def test_rope_outputs_and_the_other_input():
    """Strides only: the check runs before anything is launched."""
    q, k = (torch.empty(2, 3, 4, 16, dtype=torch.bfloat16) for _ in range(2))
    new = torch.empty_like
    ops._check_rope_outs(q, k, q, k)
    ops._check_rope_outs(q, k, q, new(k))
    ops._check_rope_outs(q, k, new(q), k)
    packed = torch.empty(2, 3, 6, 16, dtype=torch.bfloat16)
    ops._check_rope_outs(packed[:, :, :4], packed[:, :, 4:], packed[:, :, :4], packed[:, :, 4:])
    for oq, ok in ((k, new(k)), (new(q), q), (k, q), (q, q), (k, k)):
        with pytest.raises(ValueError, match="overlap"):
            ops._check_rope_outs(q, k, oq, ok)
    with pytest.raises(ValueError, match="overlap"):  # two heads of k
        ops._check_rope_outs(packed[:, :, :4], packed[:, :, 4:], packed[:, :, 2:], new(packed[:, :, 4:]))


def test_matrix_outputs_and_what_they_replace():
    buf = torch.empty(5, 8, 8, dtype=torch.bfloat16)
    g, other = buf[:4], torch.empty(4, 8, 8, dtype=torch.bfloat16)
    ops._check_replaces(torch.empty_like(g), "out", g, (g,))
    ops._check_replaces(g, "out", g, (g,))
    ops._check_replaces(buf[:4], "out", g, (g, other))
    halves = torch.empty(4, 8, 16)[:, :, :8]  # fp32, every second run of 8
    ops._check_replaces(torch.empty_like(halves, memory_format=torch.contiguous_format), "out", halves, (halves,))
    wide = torch.empty(4, 8, 8)
    for out, like, inputs in ((buf[1:], g, (g,)), (g, other, (g, other)),
                              (wide.view(torch.bfloat16).flatten()[:256].view(4, 8, 8), wide, (wide,)),
                              (g, buf.as_strided((4, 8, 8), (64, 1, 8)), (buf.as_strided((4, 8, 8), (64, 1, 8)),))):
        with pytest.raises(ValueError, match="overlaps"):
            ops._check_replaces(out, "out", like, inputs)


def test_smoke_has_no_matrix_for_pairs_of_blocks():
    """Pairs of blocks take over from 56 tiles of 256 x 256 (three quarters of 74 pairs)."""
    import __graft_entry__ as entry
    import inspect
    assert "SMOKE_MATRICES" in inspect.getsource(entry.smoke)
    for m, n in entry.SMOKE_MATRICES:
        assert 4 * -(-m // 256) * -(-n // 256) < 3 * 74
