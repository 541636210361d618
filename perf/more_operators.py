"""Layer norm and the update of what the orthogonalised step leaves over, as measured cases:

  layernorm      (residual add +) layer norm, with its saved mean and rstd
  layernorm_bwd  its gradient, with the sums over rows for weight and bias
  grad_norm      the norm of all gradients of a model and the factor that clips it
  adamw          one AdamW step over many tensors at once, states in 32 bits or
                 in 8 bits with a scale for 128 values

``run`` computes each in its plain form (elementary torch operations in 32
bits, rounded once) where ``own`` is false, and calls the framework's operators
where it is true.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
GROUP = 128  # values of a tensor that share a scale; each tensor starts a new group
LR, BETAS, ADAM_EPS, DECAY, STEP = 1e-4, (0.9, 0.95), 1e-8, 0.1, 37
MAX_NORM = 1.0


def listed():
    return [
        # eight decoded tokens between two layers
        dict(name="layernorm decode", op="layernorm", M=8, N=4096, dtype="bf16", residual=True, bias=True),
        # a training batch of a wide model
        dict(name="layernorm train", op="layernorm", M=32768, N=8192, dtype="bf16", residual=True, bias=True),
        # odd counts, no bias, a network in 32 bits
        dict(name="layernorm ragged", op="layernorm", M=1537, N=1001, dtype="f32", residual=False, bias=False),
        # a training batch's gradient, with the residual stream's own
        dict(name="layernorm gradient", op="layernorm_bwd", M=8192, N=4096, dtype="bf16", residual=True, bias=True),
        # the norm of each key head: many short rows, few columns to sum into
        dict(name="layernorm gradient heads", op="layernorm_bwd", M=262144, N=128, dtype="bf16", residual=False,
             bias=True),
        # odd counts of rows and columns
        dict(name="layernorm gradient odd", op="layernorm_bwd", M=777, N=2567, dtype="bf16", residual=True, bias=True),
        # the gradients of all norms of a model: many small tensors
        dict(name="grad norm vectors", op="grad_norm", kind="many", n=130, lo=4096, hi=4096, g="f32", shift=0),
        # the gradients of a decoder layer
        dict(name="grad norm layer", op="grad_norm", kind="layer", n=9, lo=4096, hi=14336, g="bf16", shift=0),
        # the weights of all norms of a model
        dict(name="adamw vectors", op="adamw", kind="many", n=130, lo=4096, hi=4096, p="f32", g="f32", state="f32",
             copy=False, clip=True, shift=0),
        # the embedding table: its gradient comes in 32 bits, the model reads it in bf16
        dict(name="adamw table", op="adamw", kind="many", n=1, lo=128256 * 4096, hi=128256 * 4096, p="f32", g="f32",
             state="f32", copy=True, clip=True, shift=0),
        # a decoder layer in bf16 with states in 8 bits
        dict(name="adamw layer 8 bits", op="adamw", kind="layer", n=9, lo=4096, hi=14336, p="bf16", g="bf16",
             state="e4m3", copy=False, clip=True, shift=0),
        # tensors of odd sizes in a flat buffer that starts off any alignment
        dict(name="adamw ragged 8 bits", op="adamw", kind="many", n=37, lo=65, hi=500001, p="f32", g="bf16",
             state="e4m3", copy=True, clip=False, shift=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layernorm", "layernorm", "layernorm_bwd", "layernorm_bwd", "grad_norm", "adamw", "adamw", "adamw"])
    if op in ("layernorm", "layernorm_bwd"):
        N = 2 * _log(rng, 16, 8000) + 1
        if rng.random() < 0.7:
            N = 16 * (2 * _log(rng, 2, 500) + 1) if rng.random() < 0.5 else rng.choice([64, 128, 256, 768, 1024, 2048,
                                                                                       4096, 5120, 8192, 12288])
        M = min(32768 * 8192 // N // 2, _log(rng, 1, 262144))
        return dict(op=op, M=M, N=N, dtype=rng.choice(["bf16", "bf16", "f32"]), residual=rng.random() < 0.5,
                    bias=rng.random() < 0.7)
    n = _log(rng, 1, 300)
    lo = _log(rng, 1, 100000)
    hi = max(lo, min(_log(rng, 64, 200000000), 400000000 // n))
    case = dict(op=op, kind="many", n=n, lo=min(lo, hi), hi=hi, g=rng.choice(["bf16", "f32"]),
                shift=rng.choice([0, 0, 0, 1, 3]))
    if op == "adamw":
        case["p"] = rng.choice(["bf16", "f32", "f32"])
        case.update(state=rng.choice(["f32", "e4m3"]), copy=case["p"] == "f32" and rng.random() < 0.5,
                    clip=rng.random() < 0.6)
    return case


def _sizes(c):
    """Values of each tensor: a decoder layer's, or `n` from `lo` to `hi` in equal ratios."""
    if c["kind"] == "layer":
        d, f = c["lo"], c["hi"]
        return [d, d * d, d * d // 4, d * d // 4, d * d, d, d * f, d * f, d * f]
    ratio = math.log(c["hi"] / c["lo"]) / max(c["n"] - 1, 1)
    return [int(round(c["lo"] * math.exp(ratio * i))) for i in range(c["n"])]


def _groups(c):
    return [-(-s // GROUP) for s in _sizes(c)]


# -------------------------------------------------------------------- prepare

def _normal(g, *shape, dtype=torch.bfloat16, std=1.0):
    t = torch.randn(shape, generator=g, device=DEV)
    return (t.mul_(std) if std != 1.0 else t).to(dtype)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return _rows(c, g) if c["op"] in ("layernorm", "layernorm_bwd") else _tensors(c, g)


def _rows(c, g):
    M, N, dt = c["M"], c["N"], DTYPE[c["dtype"]]
    channel = torch.ones(N, device=DEV)  # a few channels are far larger than the rest
    channel[torch.randint(0, N, (max(1, N // 256),), generator=g, device=DEV)] = 20.0
    x = torch.randn(M, N, generator=g, device=DEV).mul_(channel).add_(torch.randn(M, 1, generator=g, device=DEV))
    x[63::64] = 0  # padding tokens
    c["x"] = x.to(dt)
    del x
    c["w"] = (1 + 0.1 * torch.randn(N, generator=g, device=DEV)).to(dt)
    c["b"] = _normal(g, N, dtype=dt, std=0.1) if c["bias"] else None
    if c["op"] == "layernorm":
        c["res"] = _normal(g, M, N, dtype=dt) if c["residual"] else None
        return c
    c["dy"] = _normal(g, M, N, dtype=dt, std=1e-3)
    c["dres"] = _normal(g, M, N, dtype=dt, std=1e-3) if c["residual"] else None
    xf = c["x"].float()
    c["mean"] = xf.mean(-1)
    c["rstd"] = (xf.sub_(c["mean"][:, None]).square_().mean(-1) + EPS).rsqrt()
    return c


def _tensors(c, g):
    """Every tensor starts at a multiple of GROUP values in a flat buffer that
    starts `shift` values into its memory; the values between two are zero."""
    sizes, groups = _sizes(c), _groups(c)
    total = GROUP * sum(groups)
    starts = [GROUP * sum(groups[:i]) for i in range(len(sizes))]
    count = torch.tensor(groups, device=DEV)
    held = torch.tensor(sizes, device=DEV).repeat_interleave(count)
    at = GROUP * (torch.arange(total // GROUP, device=DEV) - (count.cumsum(0) - count).repeat_interleave(count))
    pad = torch.arange(GROUP, device=DEV) >= (held - at)[:, None]  # values behind a tensor's end
    strength = torch.exp(torch.randn(total // GROUP, 1, generator=g, device=DEV)).mul_(1e-3)
    untouched = torch.rand(total // GROUP, 1, generator=g, device=DEV) < 0.2  # rows that no token came by
    untouched[0] = False
    strength.masked_fill_(untouched, 0)

    def flat(t, dtype):
        out = torch.zeros(total + c["shift"], dtype=dtype, device=DEV)[c["shift"]:]
        out.copy_(t.masked_fill_(pad, 0).view(-1))
        return out

    def normal(scale):
        return torch.randn(total // GROUP, GROUP, generator=g, device=DEV).mul_(scale)

    c["g"] = flat(normal(strength), DTYPE[c["g"]])
    c["grads"] = [c["g"][a:a + s] for a, s in zip(starts, sizes)]
    if c["op"] == "grad_norm":
        return c
    c["clip"] = torch.tensor(0.7, device=DEV) if c["clip"] else None
    decay = [DECAY if i % 2 or c["n"] == 1 else 0.0 for i in range(len(sizes))]
    c["decay"], c["count"] = torch.tensor(decay, device=DEV), count
    c["p"] = flat(normal(0.02), DTYPE[c["p"]])
    m, v = normal(0.3 * strength), normal(0.5 * strength).square_()
    m.masked_fill_(pad, 0)
    v.masked_fill_(pad, 0)
    c["copy"] = torch.zeros(total, dtype=torch.bfloat16, device=DEV) if c["copy"] else None
    if c["state"] == "f32":
        state = (m.view(-1), v.view(-1))
    else:
        state = (*_eight(m), *_eight(v.sqrt_(), floor=True))
    del m, v
    if own:
        from kernelproblems_b200 import ops
        cut = lambda t: [t[a:a + s] for a, s in zip(starts, sizes)]  # noqa: E731
        plan = ops.AdamWStates(cut(c["p"]), dtype=torch.float32 if c["state"] == "f32" else torch.float8_e4m3fn,
                               weight_decay=decay, copies=None if c["copy"] is None else cut(c["copy"]))
        held = ((plan.exp_avg, plan.exp_avg_sq) if c["state"] == "f32" else
                (plan.exp_avg, plan.exp_avg_scale, plan.exp_avg_sq, plan.exp_avg_sq_scale))
        for to, t in zip(held, state):
            to.copy_(t)
        c["plan"], state = plan, held
    c["states"] = state
    return c


# ------------------------------------------------------------------------ run

def run(state):
    return _own(state) if own else _plain(state)


def _own(c):
    from kernelproblems_b200 import ops
    op = c["op"]
    if op == "layernorm":
        y, h, mean, rstd = ops.layernorm_fwd(c["x"], c["w"], c["b"], EPS, residual=c["res"])
        return (y, mean, rstd) if h is None else (y, mean, rstd, h)
    if op == "layernorm_bwd":
        return ops.layernorm_bwd(c["dy"], c["x"], c["mean"], c["rstd"], c["w"], dres=c["dres"],
                                 compute_db=c["bias"])
    if op == "grad_norm":
        return ops.grad_norm(c["grads"], max_norm=MAX_NORM)
    ops.adamw_update(c["plan"], c["grads"], lr=LR, step=STEP, betas=BETAS, eps=ADAM_EPS, grad_scale=c["clip"])
    return c["p"], c["copy"], c["states"]


def _plain(c):
    op = c["op"]
    if op == "layernorm":
        h = c["x"] if c["res"] is None else (c["res"].float() + c["x"].float()).to(c["x"].dtype)
        hf = h.float()
        mean = hf.mean(-1, keepdim=True)
        t = hf - mean
        rstd = 1.0 / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)
        y = t * rstd * c["w"].float()
        y = (y if c["b"] is None else y + c["b"].float()).to(h.dtype)
        return (y, mean[:, 0], rstd[:, 0]) if c["res"] is None else (y, mean[:, 0], rstd[:, 0], h)
    if op == "layernorm_bwd":
        dy, xhat = c["dy"].float(), (c["x"].float() - c["mean"][:, None]) * c["rstd"][:, None]
        gw = dy * c["w"].float()
        dx = (gw - gw.mean(-1, keepdim=True) - xhat * (xhat * gw).mean(-1, keepdim=True)) * c["rstd"][:, None]
        dx = dx if c["dres"] is None else c["dres"].float() + dx
        return dx.to(c["x"].dtype), (dy * xhat).sum(0), dy.sum(0) if c["bias"] else None
    if op == "grad_norm":
        g = c["g"].float()
        norm = torch.sqrt((g * g).sum())
        return norm, torch.where(torch.isfinite(norm), MAX_NORM / norm.clamp_min(MAX_NORM), math.nan)
    return _adamw(c)


def _adamw(c):
    (b1, b2), t = BETAS, STEP
    eight = c["state"] == "e4m3"
    g = c["g"].float().view(-1, GROUP)
    g = g if c["clip"] is None else g * c["clip"]
    if eight:
        mq, ms, rq, rs = c["states"]
        m = mq.float().view(-1, GROUP) * ms[:, None]
        v = (rq.float().view(-1, GROUP) * rs[:, None]).square()
    else:
        m, v = (s.view(-1, GROUP) for s in c["states"])
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    root = torch.sqrt(v)
    step = (LR / (1 - b1 ** t)) * m / (root * (1 / math.sqrt(1 - b2 ** t)) + ADAM_EPS)
    keep = (1 - LR * c["decay"]).repeat_interleave(c["count"])[:, None]
    p = (c["p"].float().view(-1, GROUP) * keep - step).view(-1)
    c["p"] = p.to(c["p"].dtype)
    c["copy"] = None if c["copy"] is None else p.to(torch.bfloat16)
    c["states"] = (*_eight(m), *_eight(root, floor=True)) if eight else (m.view(-1), v.view(-1))
    return c["p"], c["copy"], c["states"]


def _eight(y, floor=False):
    """e4m3 and a scale for each group: the largest magnitude becomes 448.
    `floor`: what is not zero stays so (the smallest e4m3 is 2^-9)."""
    most = y.abs().amax(-1)
    scale = torch.where(most > 0, (most * (1.0 / 448)).clamp_min(2.0 ** -126), 1.0)
    q = y * (1.0 / scale)[:, None]
    q = torch.where(y > 0, q.clamp_min(2.0 ** -9), q) if floor else q
    return q.clamp(-448, 448).to(torch.float8_e4m3fn).view(-1), scale


# ----------------------------------------------------------------------- work

def work(case):
    c = case
    op = c["op"]
    if op in ("layernorm", "layernorm_bwd"):
        M, N, b = c["M"], c["N"], DTYPE[c["dtype"]].itemsize
        vectors = 2 if c["bias"] else 1
        if op == "layernorm":  # x (and the residual) read, y (and the sum) written
            return {"bytes": M * N * b * (4 if c["residual"] else 2) + 8 * M + vectors * b * N, "flops": 8 * M * N}
        return {"bytes": M * N * b * (4 if c["residual"] else 3) + 8 * M + (b + 4 * vectors) * N,
                "flops": 14 * M * N}
    values = sum(_sizes(c))
    g = DTYPE[c["g"]].itemsize
    if op == "grad_norm":
        return {"bytes": values * g, "flops": 2 * values}
    state = 16 * values if c["state"] == "f32" else 4 * values + 16 * sum(_groups(c))
    return {"bytes": values * (g + 2 * DTYPE[c["p"]].itemsize + (2 if c["copy"] else 0)) + state,
            "flops": 16 * values}


# ---------------------------------------------------------------------- exact

def exact(case, seed):
    c = prepare(case, seed)
    op = c["op"]
    if op == "layernorm":
        h = c["x"].double()
        if c["res"] is not None:
            h = (h + c["res"].double()).to(c["x"].dtype).double()
        var, mean = torch.var_mean(h, -1, correction=0)
        rstd = (var + EPS).pow(-0.5)
        y = torch.einsum("mn,m,n->mn", h - mean[:, None], rstd, c["w"].double())
        y = y if c["b"] is None else y + c["b"].double()
        return (y, mean, rstd) if c["res"] is None else (y, mean, rstd, h)
    if op == "layernorm_bwd":
        dy, w, r = c["dy"].double(), c["w"].double(), c["rstd"].double()
        far = c["x"].double() - c["mean"].double()[:, None]
        gw = dy * w
        # the gradient less its parts along the constant row and along x - mean
        dx = gw - (torch.mv(gw, torch.ones_like(w)) / c["N"])[:, None]
        dx -= far * (torch.einsum("mn,mn->m", far, gw) * r * r / c["N"])[:, None]
        dx *= r[:, None]
        dx = dx if c["dres"] is None else dx + c["dres"].double()
        return dx, torch.einsum("mn,mn,m->n", dy, far, r), dy.sum(0) if c["bias"] else None
    if op == "grad_norm":
        norm = torch.linalg.vector_norm(c["g"].double())
        return norm, (MAX_NORM / norm).clamp_max(1.0)
    g = c["g"].double() * (1.0 if c["clip"] is None else c["clip"].double())
    wide = lambda q, s: (q.double().view(-1, GROUP) * s.double()[:, None]).view(-1)  # noqa: E731
    if c["state"] == "e4m3":
        mq, ms, rq, rs = c["states"]
        m, v = wide(mq, ms), wide(rq, rs).pow(2)
    else:
        m, v = (s.double() for s in c["states"])
    m = m.lerp(g, 1 - BETAS[0])
    v = v.lerp(g * g, 1 - BETAS[1])
    hat = m / (1 - BETAS[0] ** STEP)
    turn = hat / ((v / (1 - BETAS[1] ** STEP)).sqrt() + ADAM_EPS)
    decay = c["decay"].double().repeat_interleave(c["count"] * GROUP)
    p = c["p"].double()
    p = p - LR * (turn + decay * p)
    copy = None if c["copy"] is None else p
    if c["state"] == "f32":
        return p, copy, (m, v)
    return p, copy, (*_values(m), *_values(v.sqrt()))


def _values(y):
    """What the 8 bits stand for before they are rounded, and the scales."""
    y = y.view(-1, GROUP)
    scale = y.abs().max(-1).values / 448
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    return (y / scale[:, None]).view(-1), scale
