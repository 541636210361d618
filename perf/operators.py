"""The operators around a decoder layer's library products, as measured cases:

  rope       rotary positions of q and k, both pair layouts, part of the head,
             frequencies scaled for long contexts, forward and gradient
  norm8      (residual add +) RMSNorm with its output in 8 bits and scales
  norm8_bwd  the gradient of (residual add +) RMSNorm, also in 8 bits and scales
  ortho      a gradient's Newton-Schulz orthogonalisation
  muon       a whole weight update by it: momentum, orthogonalisation, step

``run`` computes each in its plain form (elementary torch operations in 32
bits, rounded once) where ``own`` is false, and calls the framework's operators
where it is true.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
SCALE = {"f32": torch.float32, "e8m0": torch.float8_e8m0fnu}
DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
NS = (3.4445, -4.7750, 2.0315)  # coefficients of the quintic step
NS_EPS = 1e-7
LR, MOMENTUM, DECAY = 1e-4, 0.95, 0.1


def listed():
    return [
        # one new token for each of 32 sequences deep in a long context
        dict(name="rope decode", op="rope", B=32, S=1, Hq=32, Hk=8, D=128, rot=128, layout="neox",
             scaling="smooth", factor=8.0, context=131072, backward=False, packed=False),
        # a training batch, every head dimension rotated
        dict(name="rope train", op="rope", B=8, S=4096, Hq=32, Hk=8, D=128, rot=128, layout="neox",
             scaling="smooth", factor=8.0, context=131072, backward=False, packed=False),
        # the gradient, half of an odd-sized head, pairs side by side, q and k
        # inside one packed projection, an odd sequence length
        dict(name="rope gradient part", op="rope", B=3, S=1537, Hq=20, Hk=4, D=96, rot=48,
             layout="interleaved", scaling="parts", factor=4.0, context=65536, backward=True, packed=True),
        # eight decoded tokens on their way into an 8-bit projection
        dict(name="norm8 decode", op="norm8", M=8, N=4096, residual=True, group=0, scale="f32", fmt="e4m3"),
        # a training batch of a wide model, scales for 128 values each
        dict(name="norm8 train", op="norm8", M=32768, N=8192, residual=True, group=128, scale="f32",
             fmt="e4m3"),
        # an odd count of tokens, a last group that is cut, power-of-two scales
        dict(name="norm8 ragged", op="norm8", M=1537, N=1000, residual=False, group=32, scale="e8m0",
             fmt="e4m3"),
        # the training batch's gradient for the projection below the residual
        dict(name="norm8 gradient", op="norm8_bwd", M=8192, N=4096, residual=True, group=0, scale="f32",
             fmt="e5m2"),
        # the same of an odd token count and width
        dict(name="norm8 gradient odd", op="norm8_bwd", M=777, N=2568, residual=True, group=128, scale="f32",
             fmt="e5m2"),
        # the smallest matrix: an adapter's or a router's
        dict(name="ortho small", op="ortho", E=1, m=96, n=160, dtype="bf16"),
        # the key and value projection of a 4096-wide model
        dict(name="ortho kv", op="ortho", E=1, m=1024, n=4096, dtype="bf16"),
        # a stack of tall odd matrices in 32 bits
        dict(name="ortho tall odd", op="ortho", E=3, m=1111, n=517, dtype="f32"),
        # the largest projection of a 4096-wide model, 32-bit weights and momentum
        dict(name="muon mlp", op="muon", E=1, m=4096, n=14336, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "rope", "norm8", "norm8", "norm8_bwd", "ortho", "ortho", "muon"])
    if op == "rope":
        D = rng.choice([64, 80, 96, 128, 160, 256])
        rot = rng.choice([D, D, D // 2, D // 2, 32, 24 if rng.random() < 0.5 else 20])
        Hk = rng.choice([1, 2, 4, 8, 8])
        Hq = Hk * rng.choice([1, 3, 4, 5, 8])
        B = rng.choice([1, 1, 2, 3, 8])
        most = 8 * 4096 * 40 * 128 // (B * (Hq + Hk) * D)
        S = min(most, _log(rng, 1, 8192))
        return dict(op=op, B=B, S=S, Hq=Hq, Hk=Hk, D=D, rot=rot, layout=rng.choice(["neox", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "base", "smooth", "parts"]),
                    factor=rng.choice([2.0, 4.0, 8.0]), context=rng.choice([8192, 32768, 131072]),
                    backward=rng.random() < 0.4, packed=rng.random() < 0.4)
    if op in ("norm8", "norm8_bwd"):
        # widths: sixteen times an odd number, or any odd number
        N = 2 * _log(rng, 32, 7000) + 1
        if rng.random() < 0.75:
            N = 16 * (2 * _log(rng, 2, 256) + 1) if rng.random() < 0.7 else rng.choice([1024, 2048, 4096, 8192])
        M = min(32768 * 8192 // N, _log(rng, 1, 32768))
        return dict(op=op, M=M, N=N, residual=rng.random() < 0.6, group=rng.choice([0, 0, 32, 64, 128]),
                    scale=rng.choice(["f32", "f32", "e8m0"]), fmt="e4m3" if op == "norm8" else "e5m2")
    E = rng.choice([1, 1, 1, 2, 4])
    m, n = _log(rng, 16, 6000), _log(rng, 16, 6000)
    if rng.random() < 0.4:
        m, n = 16 * (2 * (m // 32) + 1), 16 * (2 * (n // 32) + 1)
    return dict(op=op, E=E, m=m, n=n, dtype=rng.choice(["bf16", "f32"]))


# ---------------------------------------------------------------- frequencies

def _inverse_frequencies(c):
    """theta^(-2j/rot), scaled for a longer context, in 64 bits, and the
    factor on the rotated values."""
    rot, theta, f, orig = c["rot"], 500000.0, c["factor"], 8192
    j = torch.arange(rot // 2, dtype=torch.float64)
    if c["scaling"] == "base":  # a larger base: the last pair is slowed by the whole factor
        theta = theta * f ** (rot / (rot - 2.0))
    inv = theta ** (-2.0 * j / rot)
    if c["scaling"] == "linear":
        return inv / f, 1.0
    if c["scaling"] == "smooth":  # by wavelength: short ones stay, long ones are slowed, a ramp between
        low, high = 1.0, 4.0
        turns = orig * inv / (2 * math.pi)  # turns within the original context
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return keep * inv + (1 - keep) * inv / f, 1.0
    if c["scaling"] == "parts":  # by pair index, a ramp between two turn counts
        fast, slow = 32.0, 1.0
        at = lambda r: rot * math.log(orig / (2 * math.pi * r)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
        slowed = ((j - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return slowed * inv / f + (1 - slowed) * inv, 0.1 * math.log(f) + 1.0
    return inv, 1.0


# -------------------------------------------------------------------- prepare

def _normal(g, *shape, dtype=torch.bfloat16, std=1.0):
    t = torch.randn(shape, generator=g, device=DEV)
    return (t.mul_(std) if std != 1.0 else t).to(dtype)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op = c["op"]
    if op == "rope":
        B, S, Hq, Hk, D = c["B"], c["S"], c["Hq"], c["Hk"], c["D"]
        if c["packed"]:  # q, k and v of one projection's output
            qkv = _normal(g, B, S, Hq + 2 * Hk, D)
            c["q"], c["k"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
        else:
            c["q"], c["k"] = _normal(g, B, S, Hq, D), _normal(g, B, S, Hk, D)
        first = torch.randint(0, c["context"] - S + 1, (B, 1), generator=g, device=DEV)
        c["pos"] = first + torch.arange(S, device=DEV)
        if own:
            c["plan"] = _plan(c)
        else:
            inv, m = _inverse_frequencies(c)
            c["plan"] = (inv.to(DEV, torch.float32), m)
        return c
    if op in ("norm8", "norm8_bwd"):
        M, N = c["M"], c["N"]
        channel = torch.ones(N, device=DEV)  # a few channels are far larger than the rest
        channel[torch.randint(0, N, (max(1, N // 256),), generator=g, device=DEV)] = 20.0
        x = torch.randn(M, N, generator=g, device=DEV).mul_(channel)
        x[63::64] = 0  # padding tokens
        c["x"] = x.to(torch.bfloat16)
        c["w"] = (1 + 0.1 * torch.randn(N, generator=g, device=DEV)).to(torch.bfloat16)
        if op == "norm8":
            c["res"] = _normal(g, M, N) if c["residual"] else None
        else:
            c["dy"] = _normal(g, M, N, std=1e-3)
            c["dres"] = _normal(g, M, N, std=1e-3) if c["residual"] else None
            c["rstd"] = (c["x"].float().square().mean(-1) + EPS).rsqrt()
        return c
    E, m, n = c["E"], c["m"], c["n"]
    r = max(1, min(m, n) // 8)  # a gradient: a few strong directions over a weak rest
    G = torch.randn(E, m, r, generator=g, device=DEV) @ torch.randn(E, r, n, generator=g, device=DEV)
    G = G.div_(math.sqrt(r)).add_(torch.randn(E, m, n, generator=g, device=DEV), alpha=0.3).mul_(1e-3)
    G = G if E > 1 else G[0]
    c["grad"] = G.to(DTYPE[c["dtype"]])
    if op == "muon":
        c["param"] = _normal(g, *G.shape, dtype=DTYPE[c["dtype"]], std=0.02)
        c["mom"] = _normal(g, *G.shape, dtype=DTYPE[c["dtype"]], std=5e-4)
    return c


def _plan(c):
    from kernelproblems_b200 import ops
    return ops.RopeFrequencies(c["D"], rotary_dim=c["rot"], theta=500000.0, scaling=c["scaling"],
                               factor=c["factor"], original_context=8192)


# ------------------------------------------------------------------------ run

def run(state):
    return _own(state) if own else _plain(state)


def _own(c):
    from kernelproblems_b200 import ops
    op = c["op"]
    if op == "rope":
        return ops.rope_scaled(c["q"], c["k"], c["pos"], freqs=c["plan"], layout=c["layout"],
                               backward=c["backward"])
    if op == "norm8":
        q, scale, h, rstd = ops.rmsnorm_quant_fwd(c["x"], c["w"], EPS, residual=c["res"], dtype=FP8[c["fmt"]],
                                                  group=c["group"], scale_dtype=SCALE[c["scale"]])
        return (q, scale, rstd) if h is None else (q, scale, rstd, h)
    if op == "norm8_bwd":
        dx, q, scale, dw = ops.rmsnorm_quant_bwd(c["dy"], c["x"], c["rstd"], c["w"], dres=c["dres"],
                                                 dtype=FP8[c["fmt"]], group=c["group"],
                                                 scale_dtype=SCALE[c["scale"]])
        return q, scale, dx, dw
    if op == "ortho":
        return ops.orthogonalize(c["grad"], steps=5, coefficients=NS, eps=NS_EPS)
    return ops.muon_update(c["param"], c["grad"], c["mom"], lr=LR, momentum=MOMENTUM, nesterov=True,
                           weight_decay=DECAY, scale=0.2 * math.sqrt(max(c["m"], c["n"])), steps=5,
                           coefficients=NS, eps=NS_EPS)


def _plain(c):
    op = c["op"]
    if op == "rope":
        inv, m = c["plan"]
        angle = c["pos"].float()[..., None, None] * inv
        cos, sin = torch.cos(angle) * m, torch.sin(angle) * (-m if c["backward"] else m)
        turn = _halves if c["layout"] == "neox" else _pairs
        return turn(c["q"], cos, sin, c["rot"]), turn(c["k"], cos, sin, c["rot"])
    if op == "norm8":
        h = c["x"] if c["res"] is None else (c["res"].float() + c["x"].float()).to(torch.bfloat16)
        hf = h.float()
        rstd = 1.0 / torch.sqrt((hf * hf).mean(-1, keepdim=True) + EPS)
        q, scale = _quantised(hf * rstd * c["w"].float(), c)
        return (q, scale, rstd[:, 0]) if c["res"] is None else (q, scale, rstd[:, 0], h)
    if op == "norm8_bwd":
        dy, xhat = c["dy"].float(), c["x"].float() * c["rstd"][:, None]
        gw = dy * c["w"].float()
        dx = (gw - xhat * (xhat * gw).mean(-1, keepdim=True)) * c["rstd"][:, None]
        dx = dx if c["dres"] is None else c["dres"].float() + dx
        q, scale = _quantised(dx, c)
        return q, scale, dx.to(torch.bfloat16), (dy * xhat).sum(0)
    if op == "ortho":
        return _orthogonal(c["grad"].float()).to(torch.bfloat16)
    g = c["grad"].float()
    mom = MOMENTUM * c["mom"].float() + (1 - MOMENTUM) * g
    o = _orthogonal(MOMENTUM * mom + (1 - MOMENTUM) * g)
    step = LR * 0.2 * math.sqrt(max(c["m"], c["n"]))
    param = (1 - LR * DECAY) * c["param"].float() - step * o
    return param.to(c["param"].dtype), mom.to(c["mom"].dtype)


def _halves(x, cos, sin, rot):
    x = x.float()
    a, b, rest = x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(torch.bfloat16)


def _pairs(x, cos, sin, rot):
    x = x.float()
    a, b, rest = x[..., 0:rot:2], x[..., 1:rot:2], x[..., rot:]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest],
                     -1).to(torch.bfloat16)


def _quantised(y, c):
    """One scale for each row, or for each `group` values of it (the last group may be cut): the largest
    magnitude becomes the format's largest value; 1 where all are zero."""
    M, N = y.shape
    top = torch.finfo(FP8[c["fmt"]]).max
    group = c["group"] or N
    blocks = torch.nn.functional.pad(y, (0, -N % group)).view(M, -1, group)
    most = blocks.abs().amax(-1)
    scale = torch.where(most > 0, (most * (1.0 / top)).clamp_min(2.0 ** -126), 1.0)
    if c["scale"] == "e8m0":  # the power of two above
        mantissa, exponent = torch.frexp(scale)
        scale = torch.ldexp(torch.ones_like(scale), exponent - (mantissa == 0.5).to(exponent.dtype))
    q = (blocks / scale[..., None]).clamp(-top, top).view(M, -1)[:, :N].to(FP8[c["fmt"]])
    scale = scale if c["group"] else scale[:, 0]
    return q, scale.to(SCALE[c["scale"]])


def _orthogonal(g):
    x = g / (torch.sqrt((g * g).sum((-2, -1), keepdim=True)) + NS_EPS)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = _step(_step(_step(_step(_step(x)))))
    return x.mT if tall else x


def _step(x):
    a, b, c = NS
    gram = x @ x.mT
    return a * x + (b * gram + c * (gram @ gram)) @ x


# ----------------------------------------------------------------------- work

def work(case):
    c = case
    op = c["op"]
    if op == "rope":
        values = c["B"] * c["S"] * (c["Hq"] + c["Hk"]) * c["D"]
        return {"bytes": 4 * values + 8 * c["B"] * c["S"],
                "flops": 3 * c["B"] * c["S"] * (c["Hq"] + c["Hk"]) * c["rot"]}
    if op in ("norm8", "norm8_bwd"):
        M, N = c["M"], c["N"]
        scales = M * (-(-N // c["group"]) if c["group"] else 1) * (1 if c["scale"] == "e8m0" else 4)
        if op == "norm8":  # x (and the residual) read, 8 bits (and the sum) written
            return {"bytes": M * N * (2 + 1 + (4 if c["residual"] else 0)) + scales + 4 * M + 2 * N,
                    "flops": 6 * M * N}
        return {"bytes": M * N * (2 + 2 + (2 if c["residual"] else 0) + 2 + 1) + scales + 4 * M + 6 * N,
                "flops": 12 * M * N}
    size = c["E"] * c["m"] * c["n"]
    s, l = min(c["m"], c["n"]), max(c["m"], c["n"])
    # five steps of a symmetric product, a symmetric square and a full product
    flops = 5 * c["E"] * (s * s * l + s * s * s + 2 * s * s * l)
    b = 2 if c["dtype"] == "bf16" else 4
    return {"bytes": size * (b + 2) if op == "ortho" else size * 5 * b, "flops": flops}


# ---------------------------------------------------------------------- exact

def exact(case, seed):
    c = prepare(case, seed)
    op = c["op"]
    if op == "rope":
        inv, m = _inverse_frequencies(c)
        angle = c["pos"].double()[:, :, None, None] * inv.to(DEV)
        turn = torch.polar(torch.full_like(angle, m), -angle if c["backward"] else angle)
        return tuple(_turned(c[t].double(), turn, c) for t in ("q", "k"))
    if op == "norm8":
        h = c["x"].double()
        if c["res"] is not None:
            h = (h + c["res"].double()).to(torch.bfloat16).double()
        rstd = (h.pow(2).sum(-1) / c["N"] + EPS).pow(-0.5)
        q, scale = _scaled(torch.einsum("mn,m,n->mn", h, rstd, c["w"].double()), c)
        return (q, scale, rstd) if c["res"] is None else (q, scale, rstd, h)
    if op == "norm8_bwd":
        x, r, dy, w = c["x"].double(), c["rstd"].double(), c["dy"].double(), c["w"].double()
        along = torch.einsum("mn,mn,n->m", x, dy, w)  # the gradient along the row itself
        dx = torch.einsum("mn,n,m->mn", dy, w, r) - x * (along * r ** 3 / c["N"])[:, None]
        if c["dres"] is not None:
            dx = dx + c["dres"].double()
        q, scale = _scaled(dx, c)
        return q, scale, dx, torch.einsum("mn,mn,m->n", dy, x, r)
    g = c["grad"].double()
    if op == "ortho":
        return _definition(g)
    mom = c["mom"].double().lerp(g, 1 - MOMENTUM)
    param = c["param"].double() * (1 - LR * DECAY)
    return param - LR * 0.2 * math.sqrt(max(c["m"], c["n"])) * _definition(g.lerp(mom, MOMENTUM)), mom


def _turned(x, turn, c):
    """The rotation as a product of complex numbers."""
    rot = c["rot"]
    part = x[..., :rot]
    pairs = part.unflatten(-1, (2, rot // 2)).mT if c["layout"] == "neox" else part.unflatten(-1, (rot // 2, 2))
    done = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    x[..., :rot] = (done.mT if c["layout"] == "neox" else done).flatten(-2)
    return x


def _scaled(y, c):
    """The values that the 8 bits stand for before they are rounded, and the scales."""
    M, N = y.shape
    top = torch.finfo(FP8[c["fmt"]]).max
    group = c["group"] or N
    at = torch.arange(N, device=DEV) // group
    most = torch.stack([block.abs().amax(1) for block in y.split(group, 1)], 1)
    scale = torch.where(most > 0, most / top, 1.0)
    if c["scale"] == "e8m0":
        scale = torch.exp2(torch.ceil(torch.log2(scale)))
    return y / scale[:, at], scale if c["group"] else scale[:, 0]


def _definition(g):
    """x p(x' x) for each step, on the side with the smaller Gram matrix."""
    a, b, c = NS
    wide = g.shape[-1] > g.shape[-2]
    x = (g.mT if wide else g) / (torch.linalg.vector_norm(g, dim=(-2, -1), keepdim=True) + NS_EPS)
    eye = torch.eye(x.shape[-1], dtype=torch.float64, device=DEV)
    for _ in range(5):
        gram = x.mT @ x
        x = x @ (a * eye + gram @ (b * eye + c * gram))
    return x.mT if wide else x
