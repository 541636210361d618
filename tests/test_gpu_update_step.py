"""Layer norm, the gradients' norm and AdamW together, as a training step uses
them: the example runs, its gradients are those of its formulas in 64 bits, and a
whole step replays from a graph."""
import importlib.util
from pathlib import Path

import pytest
import torch

from kernelproblems_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parent.parent / "examples" / "norm_and_update_step.py"
    spec = importlib.util.spec_from_file_location("norm_and_update_step", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_example_runs(example):
    losses = example.train(4, report=lambda line: None)
    assert len(losses) == 4 and all(torch.isfinite(torch.tensor(losses)))


def norm64(x, w, b):
    far = x - x.mean(-1, keepdim=True)
    return far * (far.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w + b


def test_gradients(example):
    tower = example.Tower(300, 256, 128, DEV, seed=3)
    for name in ("w1", "w2"):
        tower.weights[name].add_(0.1 * torch.randn(256, device=DEV))
    ids = torch.randint(0, 300, (700,), device=DEV)
    out, saved = tower.forward(ids)
    dout = (torch.randn(out.shape, device=DEV) / out.numel()).to(BF)
    got = tower.backward(dout, saved)
    p = {k: v.double().requires_grad_() for k, v in tower.weights.items()}
    e = p["table"][ids]
    z = norm64(e, p["w1"], p["b1"]) @ p["proj1"].t()
    want = torch.autograd.grad((norm64(e + z, p["w2"], p["b2"]) @ p["proj2"].t() * dout.double()).sum(), list(p.values()))
    for name, a, b in zip(tower.NAMES, got, want):
        # between the formulas and a gradient lie at most ten tensors rounded to bf16, each off by 2^-8 at
        # most: ten times that of the whole, in the 2-norm
        assert (a.double() - b).norm() <= 10 * 2.0 ** -8 * b.norm(), name


def test_a_whole_step_in_a_graph(example):
    """The step's count, its rate and its clip factor are on the device."""
    steps, tokens = 3, 512
    eager, held = (example.Tower(200, 128, 64, DEV, seed=5, states=torch.float8_e4m3fn) for _ in range(2))
    ids = torch.zeros(tokens, dtype=torch.int64, device=DEV)
    target = torch.zeros(tokens, 64, device=DEV)
    step, lr = torch.zeros((), dtype=torch.int64, device=DEV), torch.tensor(0.01, device=DEV)

    def one(tower, count, rate):
        out, saved = tower.forward(ids)
        grads = tower.backward(((out.float() - target) / out.numel()).to(BF), saved)
        return tower.update(grads, rate, count, max_norm=0.01)

    warm = example.Tower(200, 128, 64, DEV, seed=5, states=torch.float8_e4m3fn)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(warm, torch.ones((), dtype=torch.int64, device=DEV), lr)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.add_(1)
        norm = one(held, step, lr)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    for i in range(1, steps + 1):
        ids.copy_(torch.randint(0, 200, (tokens,), generator=g, device=DEV))
        target.copy_(torch.randn(target.shape, generator=g, device=DEV))
        graph.replay()
        want = one(eager, i, lr)
        assert torch.equal(norm, want)
        for a, b in zip(eager.masters, held.masters):
            # the two correction factors may round differently on the host and on the device: 2^-24 of a step of 0.01
            assert bool(((a - b).abs() <= 0.01 * 2.0 ** -22 * i + 2.0 ** -23 * a.abs()).all())
        for a, b in zip(held.masters, eager.masters):
            a.copy_(b)
    assert step.item() == steps
    ops.check_status()
