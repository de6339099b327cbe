"""Routing to experts and activations kept in 8 bits, as cases that can be timed and compared.

Two operators of a Mixture-of-Experts block in training and in generation:

  routing   softmax or sigmoid scores of the experts, a bias that balances their load, groups of experts, the k largest,
            renormalised weights; with the gradient of the logits
  kept      activations kept for the backward pass in 8 bits, 32 channels to a power of two: kept and restored alone, and as
            the x and h of the norms around a block, whose gradients are formed from them

``run`` computes a case in plain torch operations (``own`` false) or through this package's calls (``own`` true).
``exact`` is the same from the definition, in 64 bits.
"""
import math

import torch

own = False

TINY = 1e-20           # beside the sum that the weights are divided by
NORM_EPS = 1e-5
GROUP = 32             # channels that share an exponent


def listed():
    return [
        # a decode step of eight sequences, many small experts in groups
        dict(name="routing of 8 tokens, 256 experts", op="route", n=8, e=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4, renorm=True, dtype="fp32", train=False),
        # a prompt through the 64-expert configuration's router: softmax, four of 64
        dict(name="routing, 64 experts, softmax", op="route", n=32768, e=64, k=4, score="softmax", bias=False, groups=1, top_groups=1, renorm=True, dtype="fp32", train=False),
        # one micro-batch, balanced by a bias, with the gradient
        dict(name="routing, 256 experts in groups", op="route", n=32768, e=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4, renorm=True, dtype="fp32", train=True),
        # BF16 logits, sizes that divide by nothing, weights as they are
        dict(name="routing, odd sizes", op="route", n=1021, e=155, k=6, score="softmax", bias=True, groups=5, top_groups=3, renorm=False, dtype="bf16", train=True),
        # several micro-batches at once, softmax over many experts
        dict(name="routing, many tokens", op="route", n=131072, e=128, k=8, score="softmax", bias=False, groups=1, top_groups=1, renorm=True, dtype="fp32", train=True),
        # the residual stream of a few tokens: latency
        dict(name="kept, 64 tokens", op="keep", n=64, c=1024, dtype="bf16"),
        # FP32 tokens, a last group that is not whole
        dict(name="kept, FP32, odd sizes", op="keep", n=3001, c=1000, dtype="fp32"),
        # the residual stream of a micro-batch of the 64-expert configuration
        dict(name="kept, micro-batch", op="keep", n=32768, c=2048, dtype="bf16"),
        # norms of a few tokens, all gradients: latency
        dict(name="norms from kept, 64 tokens", op="norm", n=64, c=1024, dtype="bf16", per_gate=0),
        # FP32 tokens, a width that is no power of two, gates whose sequences end inside the last one
        dict(name="norms from kept, FP32, odd sizes", op="norm", n=2047, c=1032, dtype="fp32", per_gate=512),
        # a micro-batch of the 64-expert configuration
        dict(name="norms from kept, micro-batch", op="norm", n=32768, c=2048, dtype="bf16", per_gate=0),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("route", "route", "keep", "norm"))
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 5, 8, 16))
        size = max(2, _spread(rng, 8, 384) // groups)
        e, top_groups = groups * size, rng.randint(1, groups)
        n = min(_spread(rng, 1, 131072), (131072 * 128) // e)
        return dict(op=op, n=n, e=e, k=rng.randint(1, min(12, top_groups * size)), score=rng.choice(("softmax", "sigmoid")), bias=rng.random() < 0.5,
                    groups=groups, top_groups=top_groups, renorm=rng.random() < 0.6, dtype=rng.choice(("fp32", "fp32", "bf16")), train=rng.random() < 0.6)
    n, c, dtype = _spread(rng, 1, 32768), 8 * _spread(rng, 8, 256), rng.choice(("bf16", "bf16", "fp32"))
    if dtype == "fp32":
        n = min(n, (16384 * 2048) // c)
    if op == "keep":
        return dict(op=op, n=n, c=c, dtype=dtype)
    return dict(op=op, n=n, c=c, dtype=dtype, per_gate=rng.choice((0, 0, max(1, n // rng.randint(1, 9)))))


def _gates(case):
    return -(-case["n"] // case["per_gate"]) if case["per_gate"] else 1


def _size(case):
    return 2 if case["dtype"] == "bf16" else 4


def work(case):
    size = _size(case)
    if case["op"] == "route":
        n, e, k = case["n"], case["e"], case["k"]
        moved = n * e * size + 8 * n * k + 4 * e * (1 + case["bias"])
        flops = n * e * 12 + n * e * k
        if case["train"]:
            moved, flops = moved + n * e * size + 4 * n * k, flops + n * e * 8
        return {"bytes": moved, "flops": flops}
    nc, kept = case["n"] * case["c"], case["n"] * (case["c"] + -(-case["c"] // GROUP))
    if case["op"] == "keep":                     # x read, its kept form written and, later, read, the restored x written
        return {"bytes": 2 * nc * size + 2 * kept, "flops": nc * 6}
    # x, h, dy, du once, y, u, dx, dh once; the kept x and h written by the forward pass and read by the backward one
    return {"bytes": 8 * nc * size + 4 * kept + 12 * case["c"] * (_gates(case) + 2), "flops": nc * 44}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    n = case["n"]
    if case["op"] == "route":
        e = case["e"]
        # some experts are liked by most tokens; the bias has learnt part of it
        liked = normal(e, std=0.7)
        s = dict(case=case, logits=(normal(n, e, std=1.2) + liked).to(dtype), bias=None)
        if case["bias"]:
            s["bias"] = (normal(e, std=0.02) - 0.08 * liked) / (1.0 if case["score"] == "sigmoid" else e / 8)
        s["counts"] = torch.zeros(e, dtype=torch.int32, device="cuda")
        if case["train"]:
            s["d_weights"] = normal(n, case["k"])
        return s
    c = case["c"]
    # a few channels of a residual stream are much larger than the others
    sizes = torch.exp(normal(c, std=0.8))
    s = dict(case=case, x=(normal(n, c, std=2.0) * sizes).to(dtype))
    if case["op"] == "keep":
        return s
    s["h"], s["alpha"] = (normal(n, c, std=0.7) * sizes.flip(0)).to(dtype), 0.9
    s["post"], s["pre"] = normal(c, std=0.1) + 1.0, normal(c, std=0.1) + 1.0
    s["gate"] = normal(_gates(case), c, std=0.3)
    s["dy"], s["du"] = normal(n, c, dtype=dtype), normal(n, c, dtype=dtype)
    s["d_post"], s["d_pre"], s["d_gate"] = torch.zeros_like(s["post"]), torch.zeros_like(s["pre"]), torch.zeros_like(s["gate"])
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------
def _scores(z, score):
    if score == "sigmoid":
        return 1.0 / (1.0 + (-z).exp())
    p = (z - z.amax(1, keepdim=True)).exp()
    return p / p.sum(1, keepdim=True)


def _plain_route(s):
    case, z = s["case"], s["logits"].double()          # (which of two experts is ahead may hang on the last bits)
    n, e, k, groups = case["n"], case["e"], case["k"], case["groups"]
    p = _scores(z, case["score"])
    c = p if s["bias"] is None else p + s["bias"].double()
    order = z if s["bias"] is None else c
    if case["top_groups"] < groups:
        best = c.view(n, groups, e // groups).sort(dim=2, descending=True).values[:, :, :2].sum(2)
        kept = torch.zeros(n, groups, dtype=torch.bool, device=z.device)
        kept.scatter_(1, best.sort(stable=True, dim=1, descending=True).indices[:, :case["top_groups"]], True)
        order = torch.where(kept.repeat_interleave(e // groups, 1), order, -math.inf)
    top = order.sort(stable=True, dim=1, descending=True).indices[:, :k]
    g = p.gather(1, top)
    total = g.sum(1, keepdim=True) + TINY
    scale = _scale(case)
    w = g / total * scale if case["renorm"] else g * scale
    s["counts"].scatter_add_(0, top.reshape(-1), torch.ones(n * k, dtype=torch.int32, device=z.device))
    out = top.int(), w.float(), s["counts"]
    if not case["train"]:
        return out
    dw = s["d_weights"].double()
    dg = (dw - (dw * g).sum(1, keepdim=True) / total) / total * scale if case["renorm"] else dw * scale
    dz = torch.zeros_like(z)
    if case["score"] == "sigmoid":
        dz.scatter_(1, top, dg * g * (1.0 - g))
    else:
        dz.scatter_(1, top, dg)
        dz = p * (dz - (dg * g).sum(1, keepdim=True))
    return *out, dz.to(s["logits"].dtype)


def _scale(case):
    return 2.5 if case["renorm"] and case["score"] == "sigmoid" else 1.0


def _power(e):
    """2^e for whole numbers -126 to 127."""
    return ((e + 127) << 23).view(torch.float32)


def _kept(x):
    """x in 8 bits, as the values they stand for: per 32 channels of a row the least power of two in whose units the largest rounds to 127 at most."""
    n, c = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -c % GROUP)).view(n, -1, GROUP)
    largest = x.abs().amax(2, keepdim=True).view(torch.int32)
    e = (((largest + 0x10000) >> 23) - 133).clamp(min=-126)           # (127.5 units and more round to 128: the next power)
    return ((x * _power(-e)).round() * _power(e)).view(n, -1)[:, :c]


def _plain_norm(s):
    case, x, h = s["case"], s["x"].float(), s["h"].float()
    gate = s["gate"].repeat_interleave(case["per_gate"], 0)[:x.shape[0]] if case["per_gate"] else s["gate"]
    r1 = 1.0 / (h.square().mean(1, keepdim=True) + NORM_EPS).sqrt()
    y = s["alpha"] * x + gate * (h * r1 * s["post"])
    r2 = 1.0 / (y.square().mean(1, keepdim=True) + NORM_EPS).sqrt()
    u = y * r2 * s["pre"]
    dtype = s["x"].dtype
    out = y.to(dtype), u.to(dtype)
    # backward: from what was kept
    h_hat = _kept(s["h"]) * r1
    normed = h_hat * s["post"]
    y_hat = (s["alpha"] * _kept(s["x"]) + gate * normed) * r2
    du = s["du"].float()
    d_hat = du * s["pre"]
    dy = s["dy"].float() + r2 * (d_hat - y_hat * (d_hat * y_hat).mean(1, keepdim=True))
    g_hat = dy * gate * s["post"]
    dh = r1 * (g_hat - h_hat * (g_hat * h_hat).mean(1, keepdim=True))
    s["d_pre"] += (du * y_hat).sum(0)
    s["d_post"] += (dy * gate * h_hat).sum(0)
    d_gate = dy * normed
    if case["per_gate"]:
        rows = torch.nn.functional.pad(d_gate, (0, 0, 0, _gates(case) * case["per_gate"] - x.shape[0]))
        s["d_gate"] += rows.view(_gates(case), case["per_gate"], -1).sum(1)
    else:
        s["d_gate"] += d_gate.sum(0)
    return *out, (s["alpha"] * dy).to(dtype), dh.to(dtype), s["d_post"], s["d_pre"], s["d_gate"]


# ---- this package's calls -------------------------------------------------------------------------------------------
def _own_route(s):
    import mgpt_b200
    case = s["case"]
    how = dict(score=case["score"], renormalise=case["renorm"], scale=_scale(case))
    top, w = mgpt_b200.route(s["logits"], case["k"], bias=s["bias"], groups=case["groups"], top_groups=case["top_groups"], counts=s["counts"], **how)
    if not case["train"]:
        return top, w, s["counts"]
    return top, w, s["counts"], mgpt_b200.route_backward(s["logits"], top, s["d_weights"], **how)


def _own_keep(s):
    import mgpt_b200
    return mgpt_b200.restore8(mgpt_b200.keep8(s["x"]))


def _own_norm(s):
    import mgpt_b200
    args = dict(post_scale=s["post"], gate=s["gate"], pre_scale=s["pre"], alpha=s["alpha"], eps=NORM_EPS, tokens_per_gate=s["case"]["per_gate"])
    y, u, stats, (x8, h8) = mgpt_b200.residual_norm(s["x"], s["h"], keep=True, **args)
    dx, dh = mgpt_b200.residual_norm_backward(x8, h8, stats, s["dy"], s["du"], d_post_scale=s["d_post"], d_gate=s["d_gate"], d_pre_scale=s["d_pre"], **args)
    return y, u, dx, dh, s["d_post"], s["d_pre"], s["d_gate"]


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_route(state) if op == "route" else _own_keep(state) if op == "keep" else _own_norm(state)
    return _plain_route(state) if op == "route" else _kept(state["x"]).to(state["x"].dtype) if op == "keep" else _plain_norm(state)


# ---- the definition, in 64 bits -------------------------------------------------------------------------------------
def _exact_route(s):
    case, z = s["case"], s["logits"].double().requires_grad_(s["case"]["train"])
    n, e, k, groups = case["n"], case["e"], case["k"], case["groups"]
    p = torch.sigmoid(z) if case["score"] == "sigmoid" else torch.softmax(z, 1)
    with torch.no_grad():
        c = (p.detach() + s["bias"].double()) if s["bias"] is not None else p.detach().clone()
        left = c.clone() if s["bias"] is not None else z.detach().clone()
        rows = torch.arange(n, device="cuda")
        if case["top_groups"] < groups:
            in_groups = c.view(n, groups, -1)
            first = in_groups.argmax(2, keepdim=True)
            score = in_groups.gather(2, first)[:, :, 0] + in_groups.scatter(2, first, -math.inf).amax(2)
            out = torch.ones(n, groups, dtype=torch.bool, device="cuda")
            for _ in range(case["top_groups"]):                          # (argmax: the first of equals)
                best = score.argmax(1)
                out[rows, best], score[rows, best] = False, -math.inf
            left[out.repeat_interleave(e // groups, 1)] = -math.inf
        chosen = []
        for _ in range(k):
            best = left.argmax(1)
            left[rows, best] = -math.inf
            chosen.append(best)
        top = torch.stack(chosen, 1)
    g = p.gather(1, top)
    w = _scale(case) * (g / (g.sum(1, keepdim=True) + TINY) if case["renorm"] else g)
    if not case["train"]:
        return top.int(), w, None
    return top.int(), w.detach(), None, torch.autograd.grad(w, z, s["d_weights"].double())[0]


def _exact_kept(x):
    x = x.double()
    out = torch.empty_like(x)
    for a in range(0, x.shape[1], GROUP):
        part = x[:, a:a + GROUP]
        largest = part.abs().amax(1, keepdim=True)
        e = (torch.floor(torch.log2(largest.clamp(min=2.0 ** -200))) - 7.0).clamp(min=-126.0)
        unit = ((e.long() + 1023) << 52).view(torch.float64)             # 2^e without a last bit that is off (ties to even)
        for _ in range(3):                                               # the least power that will do
            unit = torch.where(torch.round(largest / unit) > 127.0, 2.0 * unit, unit)
        out[:, a:a + GROUP] = torch.round(part / unit) * unit
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s)
    if case["op"] == "keep":
        return _exact_kept(s["x"])
    parts = []
    sums = [torch.zeros(s[k].shape, dtype=torch.float64, device="cuda") for k in ("post", "pre", "gate")]
    c, alpha, post, pre = case["c"], s["alpha"], s["post"].double(), s["pre"].double()
    for a in range(0, case["n"], 4096):
        rows = slice(a, min(case["n"], a + 4096))
        which = torch.arange(rows.start, rows.stop, device="cuda") // case["per_gate"] if case["per_gate"] else torch.zeros(rows.stop - a, dtype=torch.int64, device="cuda")
        gate = s["gate"].double()[which]
        x, h, up, du = (s[k][rows].double() for k in ("x", "h", "dy", "du"))
        n1 = torch.sqrt((h * h).sum(1, keepdim=True) / c + NORM_EPS)
        y = alpha * x + gate * post * h / n1
        n2 = torch.sqrt((y * y).sum(1, keepdim=True) / c + NORM_EPS)
        u = pre * y / n2
        # the norms' gradients with the kept tokens over the forward pass's sizes
        h, x = _exact_kept(s["h"][rows]) / n1, _exact_kept(s["x"][rows])
        yn = (alpha * x + gate * post * h) / n2
        inner = ((du * pre) * yn).sum(1, keepdim=True) / c
        d = up + (du * pre - yn * inner) / n2
        dn = d * gate * post
        dh = (dn - h * ((dn * h).sum(1, keepdim=True) / c)) / n1
        sums[0] += (d * gate * h).sum(0)
        sums[1] += (du * yn).sum(0)
        sums[2].index_add_(0, which, d * post * h)
        parts.append((y, u, alpha * d, dh))
    return (*(torch.cat(p) for p in zip(*parts)), *sums)
