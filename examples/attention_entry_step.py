"""A training step of an attention layer's entry with this library's operators:

  residual add + RMSNorm into 8 bits   ops.rmsnorm_quant_fwd
  q, k projection of the 8-bit values  torch._scaled_mm (a library product)
  rotary positions, scaled             ops.rope_scaled
  their gradients                      ops.rope_scaled(backward=True), ops.rmsnorm_quant_bwd
  the projection's weight update       ops.muon_update

The student's q and k learn to match a teacher projection's.

    python examples/attention_entry_step.py [--steps 30]
"""
import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
from kernelproblems_b200 import ops  # noqa: E402


def quantised_rows(w):
    """8-bit rows of a weight and their scales."""
    scale = w.float().abs().amax(1, keepdim=True) / 448
    return (w.float() / scale).to(torch.float8_e4m3fn), scale


class Entry:
    """Norm weight and q, k projection of a layer of `heads` + `kv_heads` heads."""

    def __init__(self, dim, heads, kv_heads, head_dim, device, seed=0):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.norm = torch.ones(dim, dtype=torch.bfloat16, device=device)
        self.proj = torch.randn((heads + kv_heads) * head_dim, dim, generator=g, device=device) / math.sqrt(dim)
        self.momentum = torch.zeros_like(self.proj)
        # half of every head is rotated; the context is eight times the original one
        self.freqs = ops.RopeFrequencies(head_dim, rotary_dim=head_dim // 2, scaling="smooth", factor=8.0)

    def forward(self, residual, x, positions):
        B, S, dim = x.shape
        q8, scale, h, rstd = ops.rmsnorm_quant_fwd(x, self.norm, residual=residual)
        w8, wscale = quantised_rows(self.proj)
        qk = torch._scaled_mm(q8.view(-1, dim), w8.t(), scale_a=scale.view(-1, 1), scale_b=wscale.t(),
                              out_dtype=torch.bfloat16).view(B, S, -1, self.head_dim)
        q, k = qk[:, :, :self.heads], qk[:, :, self.heads:]
        out = ops.rope_scaled(q, k, positions, freqs=self.freqs, out_q=q, out_k=k)  # in place
        return out, (q8, scale, h, rstd)

    def backward(self, dq, dk, saved, positions, dres=None):
        """Gradients of the projection, the norm weight and the residual
        stream (in bf16, and in 8 bits for the projection below)."""
        q8, scale, h, rstd = saved
        B, S, dim = h.shape
        d = torch.empty(B, S, self.heads + self.kv_heads, self.head_dim, dtype=torch.bfloat16, device=h.device)
        ops.rope_scaled(dq, dk, positions, freqs=self.freqs, backward=True, out_q=d[:, :, :self.heads],
                        out_k=d[:, :, self.heads:])
        d = d.view(B * S, -1)
        y = (q8.float() * scale[..., None]).view(B * S, dim)
        dproj = d.float().t() @ y
        dy = (d @ self.proj.to(torch.bfloat16)).view(B, S, dim)
        dx, dx8, dscale, dnorm = ops.rmsnorm_quant_bwd(dy, h, rstd, self.norm, dres=dres)
        return dproj, dnorm, dx, (dx8, dscale)

    def update(self, dproj, lr):
        ops.muon_update(self.proj, dproj, self.momentum, lr=lr, weight_decay=0.01,
                        scale=0.2 * math.sqrt(max(self.proj.shape)), param_out=self.proj, momentum_out=self.momentum)


def train(steps=30, B=2, S=512, dim=512, heads=8, kv_heads=2, head_dim=64, lr=0.02, device="cuda", report=print):
    student, teacher = (Entry(dim, heads, kv_heads, head_dim, device, seed=s) for s in (0, 1))
    g = torch.Generator(device=device)
    g.manual_seed(2)
    losses = []
    for step in range(steps):
        residual, x = (torch.randn(B, S, dim, generator=g, device=device).to(torch.bfloat16) for _ in range(2))
        positions = torch.randint(0, 65536 - S, (B, 1), generator=g, device=device) + torch.arange(S, device=device)
        (q, k), saved = student.forward(residual, x, positions)
        (tq, tk), _ = teacher.forward(residual, x, positions)
        dq, dk = (a.float() - b.float() for a, b in ((q, tq), (k, tk)))
        losses.append(0.5 * (dq.square().mean() + dk.square().mean()))
        n = dq.numel() + dk.numel()
        dproj, dnorm, dx, _ = student.backward((dq / n).to(torch.bfloat16), (dk / n).to(torch.bfloat16), saved, positions)
        student.update(dproj, lr)
    losses = torch.stack(losses).tolist()
    ops.check_status()
    for i in range(0, steps, max(1, steps // 6)):
        report(f"step {i:3d}  loss {losses[i]:.4f}")
    report(f"last      loss {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    train(ap.parse_args().steps)
