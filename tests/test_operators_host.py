"""RopeFrequencies on the CPU: the scaling rules at their ends, and refusals."""
import ctypes as C
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from kernelproblems_b200 import _build, _lib, ops


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


def test_layernorm_rejects_bad_arguments_on_the_host():
    lib = _lib.load()
    fwd = lambda M, N, dt=0, wdt=0, x=None, y=None, h=None: lib.frag_layernorm_fwd(  # noqa: E731
        x, N, None, 0, None, None, y, h, None, None, M, N, 1e-5, dt, wdt, None)
    assert fwd(4, 64) == 1 and fwd(-1, 64) == 1 and fwd(4, 64, dt=2) == 1 and fwd(4, 64, wdt=3) == 1
    assert fwd(4, 0) == 2 and fwd(1 << 31, 8) == 2 and fwd(0, 64) == 0
    assert fwd(4, 64, x=16, y=64, h=128) == 1  # h without a residual
    assert fwd(4, 64, x=17, y=64) == 3 and fwd(4, 64, dt=1, x=16, y=66) == 3
    bwd = lambda M, N, dt=0, dw=None, p=None, x=None: lib.frag_layernorm_bwd(  # noqa: E731
        p, N, x or p, N, p, p, None, None, 0, p, dw, None, M, N, dt, 0, None, 0, None)
    assert bwd(4, 64) == 1 and bwd(-1, 64) == 1 and bwd(4, 64, dt=2) == 1
    assert bwd(4, 0) == 2 and bwd(0, 64) == 0 and bwd(4, 64, dw=64, p=64) == 4 and bwd(4, 64, p=64, x=65) == 3
    assert lib.frag_layernorm_bwd_workspace_bytes(0, 64) == 0
    assert lib.frag_layernorm_bwd_workspace_bytes(4, 64) >= 2 * 4 * 64


def test_lists_of_tensors_are_checked_on_the_host():
    lib = _lib.load()
    one = lambda kind, v: (kind * 1)(v)  # noqa: E731
    ptr, num, code = one(C.c_void_p, 64), one(C.c_int64, 10), one(C.c_int32, 1)
    norm = lambda p=ptr, n=num, c=code, count=1, top=1.0, out=64, scale=None, ws=None, size=0: lib.frag_grad_norm(  # noqa: E731
        p, n, c, count, top, out, scale, ws, size, None)
    assert norm() == 4 and norm(ws=8, size=1 << 20) == 3  # workspace missing, not aligned
    assert norm(count=-1) == 1 and norm(p=None) == 1 and norm(out=None) == 1 and norm(scale=64, top=0.0) == 1
    assert norm(scale=64, top=float("nan")) == 1 and norm(n=one(C.c_int64, -1)) == 1 and norm(c=one(C.c_int32, 5)) == 1
    assert norm(p=one(C.c_void_p, 66)) == 3 and norm(p=one(C.c_void_p, None)) == 1
    assert lib.frag_grad_norm_workspace_bytes(1) > 0

    def adamw(t=None, grads=ptr, codes=code, count=1, m=64, v=64, ms=None, vs=None, lr=1e-3, b1=0.9, b2=0.9, eps=1e-8, step=1):
        table = (_lib.AdamWTensor * 1)(t or _lib.AdamWTensor(64, None, 10, 0, 1.0, 0.0, 1))
        return lib.frag_adamw_update(table, grads, codes, count, m, v, ms, vs, lr, None, b1, b2, eps, step, None, None, None)
    T = _lib.AdamWTensor
    assert adamw(count=-1) == 1 and adamw(grads=None) == 1 and adamw(b1=1.0) == 1 and adamw(b2=-0.1) == 1
    assert adamw(eps=-1.0) == 1 and adamw(eps=0.0) == 1 and adamw(eps=1e-39) == 1 and adamw(lr=float("nan")) == 1 and adamw(step=0) == 1 and adamw(ms=64) == 1
    assert adamw(m=None) == 1 and adamw(m=68) == 3 and adamw(codes=one(C.c_int32, 2)) == 1
    assert adamw(T(None, None, 10, 0, 1.0, 0.0, 1)) == 1 and adamw(T(64, None, -1, 0, 1.0, 0.0, 1)) == 1
    assert adamw(T(64, None, 10, 64, 1.0, 0.0, 1)) == 3 and adamw(T(66, None, 10, 0, 1.0, 0.0, 1)) == 3
    assert adamw(T(64, 65, 10, 0, 1.0, 0.0, 1)) == 3 and adamw(T(64, None, 10, 0, float("inf"), 0.0, 1)) == 1
    assert adamw(T(64, None, 10, 0, 1.0, 0.0, 7)) == 1 and adamw(T(64, None, 0, 0, 1.0, 0.0, 1)) == 0 and adamw(count=0) == 0


def test_rates_that_are_not_finite_in_32_bits_are_refused():
    """The kernel leaves everything as it is for such a rate: from the host it is an error."""
    lib, code = _lib.load(), (C.c_int32 * 1)(1)
    ptr = (C.c_void_p * 1)(64)

    def adamw(lr, lr_scale=1.0):
        table = (_lib.AdamWTensor * 1)(_lib.AdamWTensor(64, None, 10, 0, lr_scale, 0.0, 1))
        return lib.frag_adamw_update(table, ptr, code, 1, 68, 64, None, None, lr, None, 0.9, 0.9, 1e-8, 1, None, None, None)
    # (states that are not aligned are the next refusal)
    assert adamw(1e-3) == 3 and adamw(3e38) == 3 and adamw(1e30, 1e-30) == 3
    assert adamw(1e39) == 1 and adamw(1e30, 1e30) == 1 and adamw(-1e39) == 1
    for values in (1e39, [1e39], float("nan")):
        with pytest.raises(ValueError, match="32 bits"):
            ops._each(values, 1, "lr_scale")
    assert ops._each([3e38], 1, "lr_scale") == [3e38]
    end = 2.0 ** 128 - 2.0 ** 103
    for v in (end, -end, math.nextafter(end, 0), -math.nextafter(end, 0), float("inf"), float("nan"), 0.0, 2.0 ** -200):
        assert ops._finite(v) == math.isfinite(C.c_float(v).value)


def test_states_need_cuda_tensors():
    for bad in ([], [torch.zeros(8)], [torch.zeros(8).half()], [1.0]):
        with pytest.raises((ValueError, TypeError)):
            ops.AdamWStates(bad)
    with pytest.raises(ValueError):
        ops.grad_norm([torch.zeros(8)])
    with pytest.raises(ValueError):
        ops.layernorm_fwd(torch.zeros(2, 8))


def test_the_binding_leaves_what_it_does_not_take():
    """CPU tensors, lists of other things, wrong counts: None, and the Python path's errors."""
    b = _lib.binding()
    x = torch.zeros(2, 8)
    assert b.layernorm_fwd(x, None, None, 1e-5, None, True, True) is None
    assert b.layernorm_fwd("x", None, None, 1e-5, None, True, True) is None and b.layernorm_fwd(x) is None
    assert b.layernorm_bwd(x, x, x, x, None, None, True, True) is None
    assert b.grad_norm([x], 1.0) is None and b.grad_norm([], None) is None and b.grad_norm(x, None) is None
    assert b.grad_norm([None, x], float("nan")) is None and b.grad_norm([x, 3], 1.0) is None
    assert b.adamw(*[None] * 19) is None and b.adamw() is None
    assert b.adamw([x], 0, 0, 0, [x], 0, x, x, None, None, 0, 0.0, None, 0.9, 0.9, 1e-8, 1, None, None) is None
    with pytest.raises(TypeError):
        b.bind(1)


def test_a_missing_binding_fails_loudly(tmp_path, monkeypatch):
    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.setattr(_lib, "LIB_PATH", tmp_path / "libfrag.so")
    with pytest.raises(FileNotFoundError):
        _lib.binding()


def test_the_binding_is_of_this_torch_and_python():
    path = _lib.LIB_PATH.with_name(_build.binding_name())
    assert path.exists() and torch.__version__ in path.name and f"{sys.version_info.major}{sys.version_info.minor}" in path.name
    assert _lib.binding().__file__ == str(path)


@pytest.fixture
def build_in(tmp_path, monkeypatch):
    """_build with its files under tmp_path and a compiler that only makes them."""
    made = []

    def run(cmd, **kw):
        out = Path(cmd[cmd.index("-o") + 1])
        out.write_text("")
        made.append(out.name)
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(_build, "BUILD_DIR", tmp_path / "objects")
    monkeypatch.setattr(_build, "LIB_PATH", tmp_path / "libfrag.so")
    monkeypatch.setattr(_build, "nvcc", lambda: "nvcc")
    monkeypatch.setattr(_build.subprocess, "run", run)
    return made


def test_the_library_is_linked_where_the_binding_does_not_build(build_in, monkeypatch):
    def fails(*a):
        raise RuntimeError("no host compiler that fits")
    monkeypatch.setattr(_build, "build_binding", fails)
    with pytest.raises(RuntimeError, match="that fits"):
        _build.build()
    assert _build.LIB_PATH.exists() and "adamw.o" in build_in


def test_the_library_is_built_without_torch(build_in, monkeypatch):
    monkeypatch.setattr(_build.importlib.util, "find_spec", lambda name: None)
    monkeypatch.setattr(_build, "build_binding", lambda *a: pytest.fail("torch is not there"))
    assert _build.build() == _build.LIB_PATH and _build.LIB_PATH.exists()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are no memory")
@pytest.mark.parametrize("N", [64, 4096, 4097, 20000])
def test_no_device_is_a_status(N):
    lib = _lib.load()
    assert lib.frag_layernorm_fwd(64, N, None, 0, None, None, 64, None, None, None, 8, N, 1e-5, 0, 0, None) == 6
    assert lib.frag_layernorm_bwd(64, N, 64, N, 64, 64, None, None, 0, 64, None, None, 8, N, 0, 0, None, 0, None) == 6
