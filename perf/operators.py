"""The operators around the layer in a training step, as cases that can be timed and compared.

Three operators of a language model's training step that stand beside the Mixture-of-Experts layer:

  head loss       softmax cross entropy of the vocabulary product x W^T, its logits never kept, with the gradients of x and W
  residual norm   y = alpha x + gate * rmsnorm(h) * post,  u = rmsnorm(y) * pre: the norm after a block, its gate, the skip
                  connection with its scale and the norm before the next block, with all gradients
  AdamW           one step over many tensors at once, moments in 8 or in 32 bits

``run`` computes a case in plain torch operations (``own`` false) or through this package's calls (``own`` true).
``exact`` is the same from the definition, in 64 bits.
"""
import math

import torch

own = False

IGNORED = -100
BLOCK = 256            # elements that share a scale of the 8-bit moments
T0 = 100               # optimiser steps behind the first one taken here
LR, B1, B2, EPS, DECAY = 3e-4, 0.9, 0.999, 1e-8, 0.01
NORM_EPS = 1e-5


def listed():
    return [
        # scoring a handful of continuations: latency
        dict(name="loss of 16 tokens", op="loss", n=16, c=512, v=32000, ignored=0.0, train=False),
        # evaluation of a prompt set whose padding is ignored, a vocabulary that divides by nothing
        dict(name="loss, odd sizes", op="loss", n=777, c=1024, v=50021, ignored=0.25, train=False),
        # one micro-batch of the medium configuration
        dict(name="loss and gradients", op="loss", n=8192, c=512, v=32000, ignored=0.0, train=True),
        # fine-tuning on answers only: half of the tokens carry no loss
        dict(name="half of the tokens ignored", op="loss", n=3001, c=1024, v=50021, ignored=0.5, train=True),
        # one micro-batch of a wide model over a large vocabulary
        dict(name="large vocabulary", op="loss", n=8192, c=2048, v=131072, ignored=0.0, train=True),
        # a decode step of eight sequences
        dict(name="norms of 8 tokens", op="norm", n=8, c=1024, dtype="bf16", per_gate=0, train=False),
        # a prompt of the decode configuration's width, one gate per sequence
        dict(name="norms of a prompt", op="norm", n=16384, c=1024, dtype="bf16", per_gate=2048, train=False),
        # FP32 tokens, a width that is no power of two, gates whose sequences end inside the last one
        dict(name="norms, FP32, odd sizes", op="norm", n=1021, c=320, dtype="fp32", per_gate=256, train=True),
        # a micro-batch of the 64-expert configuration
        dict(name="norms and gradients", op="norm", n=32768, c=2048, dtype="bf16", per_gate=0, train=True),
        # the small repository configuration: 50 small tensors, latency
        dict(name="adamw, small layer, 32 bits", op="adamw", e=8, c=128, h=512, extra=0, bits=32, grad="fp32"),
        # a layer of 64 experts: 386 tensors from 64 to half a million elements
        dict(name="adamw, 64 experts, 8 bits", op="adamw", e=64, c=1024, h=512, extra=0, bits=8, grad="fp32"),
        # the vocabulary matrix of the largest loss beside a small layer, gradients in BF16
        dict(name="adamw, vocabulary, 8 bits", op="adamw", e=8, c=128, h=512, extra=131072 * 2048, bits=8, grad="bf16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("loss", "loss", "norm", "adamw"))
    if op == "loss":
        c, v = 8 * _spread(rng, 16, 256), _spread(rng, 1000, 131072)
        train = rng.random() < 0.6
        return dict(op=op, n=_spread(rng, 1, 8192), c=c, v=v, ignored=rng.choice((0.0, 0.0, 0.25, 0.5, 0.9)), train=train)
    if op == "norm":
        n = _spread(rng, 1, 32768)
        return dict(op=op, n=n, c=8 * _spread(rng, 16, 256), dtype=rng.choice(("bf16", "bf16", "fp32")),
                    per_gate=rng.choice((0, 0, max(1, n // rng.randint(1, 9)))), train=rng.random() < 0.6)
    return dict(op=op, e=_spread(rng, 2, 64), c=8 * _spread(rng, 8, 128), h=_spread(rng, 64, 1408),
                extra=rng.choice((0, _spread(rng, 1000, 50000000))), bits=rng.choice((8, 8, 32)), grad=rng.choice(("fp32", "bf16")))


def _valid(case):
    return case["n"] - int(case["n"] * case["ignored"])


def _sizes(case):
    """Elements of each tensor: the layer's parameters (router, then per expert gate, up and down with their biases), then one more."""
    e, c, h = case["e"], case["c"], case["h"]
    return [c * e, e] + [c * h, h, c * h, h, h * c, c] * e + ([case["extra"]] if case["extra"] else [])


def _gates(case):
    return -(-case["n"] // case["per_gate"]) if case["per_gate"] else 1


def work(case):
    if case["op"] == "loss":
        n, c, v, valid = case["n"], case["c"], case["v"], _valid(case)
        moved, flops = 2 * valid * c + 2 * v * c + 4 * n + 8 * n, 2 * valid * c * v
        if case["train"]:
            moved, flops = moved + 2 * n * c + 2 * v * c + 4 * n, 3 * flops
        return {"bytes": moved, "flops": flops}
    if case["op"] == "norm":
        nc, size, small = case["n"] * case["c"], 2 if case["dtype"] == "bf16" else 4, 4 * case["c"] * (_gates(case) + 2)
        moved = 4 * nc * size + small
        if case["train"]:                        # x, h, dy, du once, y, u, dx, dh once
            moved = 8 * nc * size + 3 * small
        return {"bytes": moved, "flops": nc * (9 if not case["train"] else 34)}
    k = sum(_sizes(case))
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": k * (8 + (2 if case["grad"] == "bf16" else 4) + 2 + state), "flops": k * 16}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    if case["op"] == "loss":
        n, c, v = case["n"], case["c"], case["v"]
        w = normal(v, c, std=1.5 / math.sqrt(c), dtype=torch.bfloat16)
        targets = torch.randint(0, v, (n,), generator=gen, device="cuda", dtype=torch.int32)
        # hidden states that know something of their targets: a few of the tokens are nearly certain
        sure = torch.rand(n, 1, generator=gen, device="cuda") * 5.0
        x = (normal(n, c) + sure * w[targets.long()].float()).to(torch.bfloat16)
        order = torch.randperm(n, generator=gen, device="cuda")
        targets[order[_valid(case):]] = IGNORED
        d_loss = torch.full((n,), 1.0 / max(1, _valid(case)), device="cuda")
        return dict(case=case, x=x, w=w, targets=targets, d_loss=d_loss)
    if case["op"] == "norm":
        n, c = case["n"], case["c"]
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        s = dict(case=case, x=normal(n, c, std=2.0, dtype=dtype), h=normal(n, c, std=0.7, dtype=dtype), alpha=0.9)
        s["post"], s["pre"] = normal(c, std=0.1) + 1.0, normal(c, std=0.1) + 1.0
        s["gate"] = normal(_gates(case), c, std=0.3)
        if case["train"]:
            s["dy"], s["du"] = normal(n, c, dtype=dtype), normal(n, c, dtype=dtype)
            s["d_post"], s["d_pre"], s["d_gate"] = torch.zeros_like(s["post"]), torch.zeros_like(s["pre"]), torch.zeros_like(s["gate"])
        return s
    sizes = _sizes(case)
    total = sum(-(-k // BLOCK) for k in sizes) * BLOCK          # every tensor starts on a block of its own
    starts, real, at = [], torch.zeros(total, dtype=torch.bool, device="cuda"), 0
    for k in sizes:
        starts.append(at)
        real[at:at + k] = True
        at += -(-k // BLOCK) * BLOCK
    w = torch.where(real, normal(total, std=0.02), 0.0)
    # gradients of very different size from block to block, as from tensor to tensor
    size = torch.exp(torch.rand(total // BLOCK, 1, generator=gen, device="cuda") * 8.0 - 12.0)
    g = torch.where(real, (normal(total // BLOCK, BLOCK) * size).reshape(-1), 0.0)
    m = torch.where(real, (normal(total // BLOCK, BLOCK, std=0.3) * size).reshape(-1), 0.0)
    v = torch.where(real, ((normal(total // BLOCK, BLOCK, std=0.5) * size).square() + (0.2 * size).square()).reshape(-1), 0.0)
    s = dict(case=case, w=w, g=g.to(torch.bfloat16) if case["grad"] == "bf16" else g, copy=w.to(torch.bfloat16), starts=starts, sizes=sizes, t=T0, seed=seed & 0x7FFFFFFF)
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        half = torch.full((total,), 1 << 15, dtype=torch.int32, device="cuda")
        s["m"], s["m_scale"] = _to8(m, _exponent(m.abs(), 1), half)
        s["v"], s["v_scale"] = _to8(v.sqrt(), _exponent(v, 2), half)
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------
def _plain_loss(s):
    x, w, targets = s["x"], s["w"].float(), s["targets"].long()
    valid = (targets >= 0) & (targets < w.shape[0])
    x = torch.where(valid[:, None], x.float(), 0.0)
    label = torch.where(valid, targets, 0)
    z = x @ w.T
    top = z.amax(1)
    e = (z - top[:, None]).exp_()
    total = e.sum(1)
    lse = top + total.log()
    loss = torch.where(valid, lse - z.gather(1, label[:, None])[:, 0], 0.0)
    lse = torch.where(valid, lse, 0.0)
    if not s["case"]["train"]:
        return loss, lse
    del z
    up = torch.where(valid, s["d_loss"], 0.0)
    e *= (up / total)[:, None]
    e.scatter_add_(1, label[:, None], -up[:, None])
    return loss, lse, (e @ w).to(torch.bfloat16), (e.T @ x).to(torch.bfloat16)


def _plain_norm(s):
    case, x, h = s["case"], s["x"].float(), s["h"].float()
    gate = s["gate"].repeat_interleave(case["per_gate"], 0)[:x.shape[0]] if case["per_gate"] else s["gate"]
    r1 = 1.0 / (h.square().mean(1, keepdim=True) + NORM_EPS).sqrt()
    normed = h * r1 * s["post"]
    y = s["alpha"] * x + gate * normed
    r2 = 1.0 / (y.square().mean(1, keepdim=True) + NORM_EPS).sqrt()
    u = y * r2 * s["pre"]
    dtype = s["x"].dtype
    if not case["train"]:
        return y.to(dtype), u.to(dtype)
    du = s["du"].float()
    y_hat, d_hat = y * r2, du * s["pre"]
    dy = s["dy"].float() + r2 * (d_hat - y_hat * (d_hat * y_hat).mean(1, keepdim=True))
    h_hat, g_hat = h * r1, dy * gate * s["post"]
    dh = r1 * (g_hat - h_hat * (g_hat * h_hat).mean(1, keepdim=True))
    s["d_pre"] += (du * y_hat).sum(0)
    s["d_post"] += (dy * gate * h_hat).sum(0)
    d_gate = dy * normed
    if case["per_gate"]:
        rows = torch.nn.functional.pad(d_gate, (0, 0, 0, _gates(case) * case["per_gate"] - x.shape[0]))
        s["d_gate"] += rows.view(_gates(case), case["per_gate"], -1).sum(1)
    else:
        s["d_gate"] += d_gate.sum(0)
    return y.to(dtype), u.to(dtype), (s["alpha"] * dy).to(dtype), dh.to(dtype), s["d_post"], s["d_pre"], s["d_gate"]


def _mixed(h):
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & 0xFFFFFFFF
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _random(count, seed, t, device):
    """32 random bits per element: the finaliser of MurmurHash3 over the element's place, the seed and the step."""
    i = torch.arange(count, dtype=torch.int64, device=device)
    return _mixed((i & 0xFFFFFFFF) ^ _mixed((seed * 0x9E3779B1 + t) & 0xFFFFFFFF) ^ ((i >> 32) * 0x9E3779B1 & 0xFFFFFFFF))


def _power(e):
    """2^e for whole numbers -126 to 127."""
    return ((e + 127) << 23).view(torch.float32)


def _exponent(a, root):
    """Per block: the power of two below its largest value (root 2: below the square root of that)."""
    e = (a.view(-1, BLOCK).amax(1).view(torch.int32) >> 23) - 127
    return e.clamp(min=-100) if root == 1 else e >> 1


def _to8(x, exponent, random16):
    """Stochastic rounding to a sign, 4 bits of exponent and 3 of mantissa, a block's largest value between 128 and 256 units:
    the 16 random bits are added below the last kept bit."""
    x = x.view(-1, BLOCK)
    a = x.abs() * _power(7 - exponent)[:, None]
    low = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)                # fixed steps of 2^-9 below
    bits = (a + low).view(torch.int32) + (random16.view(-1, BLOCK) << 4)
    q = (bits & ~0xFFFFF).view(torch.float32) - low
    return torch.copysign(q, x).to(torch.float8_e4m3fn).view(-1), _power(exponent - 7)


def _plain_adamw(s):
    case = s["case"]
    s["t"] += 1
    w, g, t = s["w"], s["g"].float(), s["t"]
    if case["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1).square()
    m, v = B1 * m + (1.0 - B1) * g, B2 * v + (1.0 - B2) * g * g
    w = w - (LR * DECAY) * w - LR * (m / (1.0 - B1 ** t)) / ((v / (1.0 - B2 ** t)).sqrt() + EPS)
    s["w"].copy_(w)
    s["copy"].copy_(w)
    if case["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return s["w"], s["copy"], s["m"], s["v"]
    random = _random(m.numel(), s["seed"], t, m.device)
    s["m"], s["m_scale"] = _to8(m, _exponent(m.abs(), 1), (random & 0xFFFF).to(torch.int32))
    s["v"], s["v_scale"] = _to8(v.sqrt(), _exponent(v, 2), (random >> 16).to(torch.int32))
    return s["w"], s["copy"], s["m"], s["m_scale"], s["v"], s["v_scale"]


# ---- this package's calls -------------------------------------------------------------------------------------------
def _own_loss(s):
    import mgpt_b200
    loss, lse = mgpt_b200.head_loss(s["x"], s["w"], s["targets"])
    if not s["case"]["train"]:
        return loss, lse
    dx, dw = mgpt_b200.head_loss_backward(s["x"], s["w"], s["targets"], lse, s["d_loss"])
    return loss, lse, dx, dw


def _own_norm(s):
    import mgpt_b200
    args = dict(post_scale=s["post"], gate=s["gate"], pre_scale=s["pre"], alpha=s["alpha"], eps=NORM_EPS, tokens_per_gate=s["case"]["per_gate"])
    y, u, stats = mgpt_b200.residual_norm(s["x"], s["h"], **args)
    if not s["case"]["train"]:
        return y, u
    dx, dh = mgpt_b200.residual_norm_backward(s["x"], s["h"], stats, s["dy"], s["du"], d_post_scale=s["d_post"], d_gate=s["d_gate"], d_pre_scale=s["d_pre"], **args)
    return y, u, dx, dh, s["d_post"], s["d_pre"], s["d_gate"]


def _own_adamw(s):
    import mgpt_b200
    if "optimiser" not in s:                     # a program makes it once, when its tensors exist
        def parts(flat):
            return [flat[a:a + k] for a, k in zip(s["starts"], s["sizes"])]

        state = (s["m"], s["v"]) if s["case"]["bits"] == 32 else (s["m"], s["v"], s["m_scale"], s["v_scale"])
        s["optimiser"] = mgpt_b200.AdamW(parts(s["w"]), parts(s["g"]), copies=parts(s["copy"]), state_bits=s["case"]["bits"], state=state, weight_decay=DECAY, seed=s["seed"])
    s["t"] += 1
    s["optimiser"].step(s["t"], lr=LR, beta1=B1, beta2=B2, eps=EPS)
    if s["case"]["bits"] == 32:
        return s["w"], s["copy"], s["m"], s["v"]
    return s["w"], s["copy"], s["m"], s["m_scale"], s["v"], s["v_scale"]


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_loss(state) if op == "loss" else _own_norm(state) if op == "norm" else _own_adamw(state)
    return _plain_loss(state) if op == "loss" else _plain_norm(state) if op == "norm" else _plain_adamw(state)


# ---- the definition, in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "loss":
        n, v = case["n"], case["v"]
        wd = s["w"].double()
        loss, lse = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
        dx = torch.zeros(n, case["c"], dtype=torch.float64, device="cuda")
        dw = torch.zeros_like(wd) if case["train"] else None
        kept = torch.nonzero(s["targets"] >= 0)[:, 0]
        for rows in torch.split(kept, 1024):
            x, label = s["x"][rows].double(), s["targets"][rows].long()
            z = x @ wd.T
            total = torch.logsumexp(z, 1)
            lse[rows], loss[rows] = total, total - z[torch.arange(len(rows), device="cuda"), label]
            if case["train"]:
                p = torch.exp(z - total[:, None])
                p[torch.arange(len(rows), device="cuda"), label] -= 1.0
                p *= s["d_loss"][rows].double()[:, None]
                dx[rows] = p @ wd
                dw += p.T @ x
        return (loss, lse, dx, dw) if case["train"] else (loss, lse)
    if case["op"] == "norm":
        leaves = {k: s[k].double().requires_grad_(case["train"]) for k in ("x", "h", "post", "pre", "gate")}
        row = torch.arange(case["n"], device="cuda") // case["per_gate"] if case["per_gate"] else torch.zeros(case["n"], dtype=torch.int64, device="cuda")
        h, c = leaves["h"], case["c"]
        normed = h / torch.sqrt((h * h).sum(1, keepdim=True) / c + NORM_EPS) * leaves["post"]
        y = s["alpha"] * leaves["x"] + leaves["gate"][row] * normed
        u = y / torch.sqrt((y * y).sum(1, keepdim=True) / c + NORM_EPS) * leaves["pre"]
        if not case["train"]:
            return y, u
        d = torch.autograd.grad((y, u), [leaves[k] for k in ("x", "h", "post", "pre", "gate")], (s["dy"].double(), s["du"].double()))
        return y.detach(), u.detach(), *d
    t = T0 + 1
    outs = [[] for _ in range(4 if case["bits"] == 32 else 6)]
    total = s["w"].numel()
    random = _random(total, s["seed"], t, "cuda") if case["bits"] == 8 else None
    step = BLOCK << 17
    for a in range(0, total, step):
        part = slice(a, min(total, a + step))
        blocks = slice(a // BLOCK, -(-part.stop // BLOCK))
        w, g = s["w"][part].double(), s["g"][part].double()
        m, v = s["m"][part].double(), s["v"][part].double()
        if case["bits"] == 8:
            m = m * s["m_scale"][blocks].double().repeat_interleave(BLOCK)
            v = (v * s["v_scale"][blocks].double().repeat_interleave(BLOCK)) ** 2
        m, v = B1 * m + (1.0 - B1) * g, B2 * v + (1.0 - B2) * g * g
        w = w * (1.0 - LR * DECAY) - LR * (m / (1.0 - B1 ** t)) / (torch.sqrt(v / (1.0 - B2 ** t)) + EPS)
        got = [w, w]
        if case["bits"] == 32:
            got += [m, v]
        else:
            for x, bits, least in ((m, random[part] & 0xFFFF, -100.0), (torch.sqrt(v), random[part] >> 16, -64.0)):
                x = x.view(-1, BLOCK)
                unit = torch.pow(2.0, torch.floor(torch.log2(x.abs().amax(1))).clamp(min=least) - 7.0)
                y = x.abs() / unit[:, None]
                grid = torch.pow(2.0, torch.floor(torch.log2(y)).clamp(min=-6.0) - 3.0)
                y = torch.floor(y / grid + bits.view(-1, BLOCK).double() / 65536.0) * grid
                got += [torch.where(x < 0, -y, y).view(-1), unit]
        for o, x in zip(outs, got):
            o.append(x)
    return tuple(torch.cat(o) for o in outs)
