"""A training step of a small tower with this library's operators:

  token embedding and its gradient     ops.embedding_fwd, ops.embedding_bwd
  layer norm, with and without the     ops.layernorm_fwd, ops.layernorm_bwd
  residual's addition, and gradients
  the norm of all gradients            ops.grad_norm
  the update of all parameters         ops.AdamWStates, ops.adamw_update

The projections are library products.  Parameters are fp32 masters; the step
writes the bf16 weights that the model reads.  Nothing in a step waits for the
host, so that it can be captured into a graph.

    python examples/norm_and_update_step.py [--steps 30]
"""
import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
from kernelproblems_b200 import ops  # noqa: E402

BF = torch.bfloat16


class Tower:
    """out = norm2(e + norm1(e) W1') W2' of the tokens' embeddings e."""

    NAMES = ("table", "w1", "b1", "proj1", "w2", "b2", "proj2")

    def __init__(self, vocab, dim, width, device, seed=0, states=torch.float32):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=g, device=device)  # noqa: E731
        ones, zeros = torch.ones(dim, device=device), torch.zeros(dim, device=device)
        self.masters = [rand(vocab, dim), ones, zeros, rand(dim, dim) / math.sqrt(dim), ones.clone(), zeros.clone(),
                        rand(width, dim) / math.sqrt(dim)]
        self.weights = dict(zip(self.NAMES, (p.to(BF) for p in self.masters)))
        decay = [0.1 if p.dim() == 2 else 0.0 for p in self.masters]
        self.states = ops.AdamWStates(self.masters, dtype=states, weight_decay=decay, copies=list(self.weights.values()))

    def forward(self, ids):
        p = self.weights
        e = ops.embedding_fwd(ids, p["table"]).view(-1, p["table"].shape[1])
        y1, _, mean1, rstd1 = ops.layernorm_fwd(e, p["w1"], p["b1"])
        z = y1 @ p["proj1"].t()
        y2, h, mean2, rstd2 = ops.layernorm_fwd(z, p["w2"], p["b2"], residual=e)
        return y2 @ p["proj2"].t(), (ids, e, y1, mean1, rstd1, h, y2, mean2, rstd2)

    def backward(self, dout, saved):
        """The gradients in NAMES' order, fp32 but for the projections'."""
        p = self.weights
        ids, e, y1, mean1, rstd1, h, y2, mean2, rstd2 = saved
        dproj2 = dout.t() @ y2
        dh, dw2, db2 = ops.layernorm_bwd(dout @ p["proj2"], h, mean2, rstd2, p["w2"])
        dproj1 = dh.t() @ y1
        de, dw1, db1 = ops.layernorm_bwd(dh @ p["proj1"], e, mean1, rstd1, p["w1"], dres=dh)
        dtable = ops.embedding_bwd(de, ids, p["table"].shape[0])
        return [dtable, dw1, db1, dproj1, dw2, db2, dproj2]

    def update(self, grads, lr, step, max_norm=1.0):
        norm, scale = ops.grad_norm(grads, max_norm=max_norm)
        ops.adamw_update(self.states, grads, lr=lr, step=step, grad_scale=scale)
        return norm


def train(steps=30, tokens=2048, vocab=1000, dim=512, width=384, lr=0.01, device="cuda", report=print):
    student, teacher = (Tower(vocab, dim, width, device, seed=s, states=t)
                        for s, t in ((0, torch.float8_e4m3fn), (1, torch.float32)))
    g = torch.Generator(device=device)
    g.manual_seed(2)
    losses, norms = [], []
    for step in range(1, steps + 1):
        ids = torch.randint(0, vocab, (tokens,), generator=g, device=device)
        out, saved = student.forward(ids)
        diff = out.float() - teacher.forward(ids)[0].float()
        losses.append(0.5 * diff.square().mean())
        grads = student.backward((diff / diff.numel()).to(BF), saved)
        norms.append(student.update(grads, lr, step))
    losses, norms = torch.stack(losses).tolist(), torch.stack(norms).tolist()
    ops.check_status()
    for i in range(0, steps, max(1, steps // 6)):
        report(f"step {i:3d}  loss {losses[i]:.4f}  gradients' norm {norms[i]:.4f}")
    report(f"last      loss {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    train(ap.parse_args().steps)
