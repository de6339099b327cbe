"""A small language model trained with the layer and the operators beside it: a whole training step without attention.

    python examples/train_lm.py [--steps 60] [--routing sigmoid] [--kept-bits 8]

Each block is the Mixture-of-Experts layer between two norms, with a gate per channel on the residual stream:

    u = rmsnorm(x)*pre,   x' = alpha*x + gate * rmsnorm(moe(u))*post

The embedding is the head as well.  What a step consists of:

    embedding rows -> [MoELayer.forward, residual_norm] x blocks -> head_loss
    head_loss_backward -> [residual_norm_backward, MoELayer.backward] x blocks -> embedding rows' gradients
    AdamW over every tensor at once, moments in 8 bits

With ``--routing`` the layers choose their experts by softmax or sigmoid scores with renormalised weights, under a bias that is moved towards
equal loads after every step; with ``--kept-bits 8`` what the norms keep for their backward pass is in 8 bits.

The data are sequences in which a token fixes the next one nine times out of ten; the first tokens of each sequence carry no loss.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from mgpt_b200 import AdamW, MoELayer, check_status, head_loss, head_loss_backward, residual_norm, residual_norm_backward  # noqa: E402


class Model:
    def __init__(self, vocab=1000, dim=128, hidden=256, experts=8, top_k=2, blocks=2, alpha=1.0, seed=0, state_bits=8, routing=None, kept_bits=16):
        g = torch.Generator().manual_seed(seed)
        self.alpha, self.dim, self.keep = alpha, dim, kept_bits == 8
        self.embed = (torch.randn(vocab, dim, generator=g) * 0.1).cuda()             # the masters are FP32
        self.head = self.embed.bfloat16()                                            # the copy that the products read
        self.d_embed = torch.zeros_like(self.embed)
        self.moe, self.bias, self.small, self.d_small = [], [], [], []
        for _ in range(blocks):
            layer = MoELayer(dim, hidden, experts, top_k)
            layer.load_parameters([torch.randn(p.shape, generator=g).numpy() * (p.shape[0] ** -0.5 if p.shape[0] > 1 else 0.0) for p in layer.get_parameters()])
            self.moe.append(layer)
            self.bias.append(torch.zeros(experts).cuda() if routing else None)
            if routing:
                layer.set_routing(routing, bias=self.bias[-1], renormalise=True)
            self.small.append(dict(pre=torch.ones(dim).cuda(), post=torch.ones(dim).cuda(), gate=torch.full((1, dim), 0.5).cuda()))
        self.final = torch.ones(dim).cuda()                                          # scale of the norm in front of the head
        self.d_small = [{k: torch.zeros_like(v) for k, v in s.items()} for s in self.small]
        self.d_final = torch.zeros_like(self.final)
        weights = [self.embed, self.final] + [p for m in self.moe for p in m.get_parameters()] + [v for s in self.small for v in s.values()]
        self.grads = [self.d_embed, self.d_final] + [p.grad for m in self.moe for p in m.get_parameters()] + [v for s in self.d_small for v in s.values()]
        # decay for the matrices, none for scales, gates and biases
        self.optimiser = AdamW(weights, self.grads, copies=[self.head] + [None] * (len(weights) - 1), state_bits=state_bits, seed=seed,
                               weight_decay=[0.01 if min(w.shape) > 1 and w.dim() == 2 else 0.0 for w in weights])
        self.t = 0

    def norm_args(self, i):
        """Arguments of the call between block i and what follows it: the next block's norm, or the head's."""
        s = self.small[i]
        return dict(post_scale=s["post"], gate=s["gate"], pre_scale=self.small[i + 1]["pre"] if i + 1 < len(self.small) else self.final, alpha=self.alpha)

    def step(self, tokens, targets, lr=3e-3):
        """One training step; returns the mean loss (on the device)."""
        for g in self.grads:
            g.zero_()
        rows = tokens.reshape(-1)
        x = self.head[rows.long()]
        first = dict(pre_scale=self.small[0]["pre"], alpha=0.0)                      # the norm in front of the first block: y = x
        x0 = x
        x, u, stats0 = residual_norm(x0, x0, **first)
        kept = []
        for i, moe in enumerate(self.moe):
            h = moe.forward(u)
            y, v, stats, *kept8 = residual_norm(x, h, keep=self.keep, **self.norm_args(i))
            kept.append((*(kept8[0] if self.keep else (x, h)), stats))
            x, u = y, v
        targets = targets.reshape(-1)
        loss, lse = head_loss(u, self.head, targets)
        share = (targets >= 0).float()
        share /= share.sum()
        du, _ = head_loss_backward(u, self.head, targets, lse, share, self.d_embed)   # (FP32: added to)
        dy = torch.zeros_like(du)
        for i in reversed(range(len(self.moe))):
            x, h, stats = kept[i]
            d = self.d_small[i]
            d_pre = self.d_small[i + 1]["pre"] if i + 1 < len(self.small) else self.d_final
            dy, dh = residual_norm_backward(x, h, stats, dy, du, d_post_scale=d["post"], d_gate=d["gate"], d_pre_scale=d_pre, **self.norm_args(i))
            du = self.moe[i].backward(dh)
        _, dx0 = residual_norm_backward(x0, x0, stats0, dy, du, d_pre_scale=self.d_small[0]["pre"], **first)
        self.d_embed.index_add_(0, rows.long(), dx0.float())
        self.t += 1
        self.optimiser.step(self.t, lr=lr)
        for m, bias in zip(self.moe, self.bias):
            m.sync_weights()                                                         # the layer's own BF16 copies
            if bias is not None and lr:                                              # experts with more tokens than the mean are asked less
                counts = m.workspace_view("counts", torch.int32, (m.E,)).float()
                bias += 1e-3 * torch.sign(counts.mean() - counts)
        return (loss * share).sum()


def batch(n, length, vocab, seed):
    """Sequences whose next token is a fixed function of the token, nine times out of ten; targets of the first eight are ignored."""
    g = torch.Generator().manual_seed(seed)
    follow = torch.randperm(vocab, generator=torch.Generator().manual_seed(1))
    t = torch.randint(0, vocab, (n, length + 1), generator=g)
    keep = torch.rand(n, length, generator=g) < 0.9
    for i in range(length):
        t[:, i + 1] = torch.where(keep[:, i], follow[t[:, i]], t[:, i + 1])
    targets = t[:, 1:].clone()
    targets[:, :8] = -1
    return t[:, :-1].int().cuda(), targets.int().cuda()


def train(steps=60, vocab=1000, seed=0, state_bits=8, report=None, **how):
    model = Model(vocab=vocab, seed=seed, state_bits=state_bits, **how)
    losses = []
    for i in range(steps):
        losses.append(model.step(*batch(32, 64, vocab, 100 + i)))
        if report and (i % report == 0 or i + 1 == steps):
            print(f"step {i:4d}  loss {float(losses[-1]):.4f}")
    check_status()
    for m in model.moe:
        m.check_status()
    return [float(v) for v in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    ap.add_argument("--routing", choices=("softmax", "sigmoid"))
    ap.add_argument("--kept-bits", type=int, default=16, choices=(8, 16))
    args = ap.parse_args()
    train(args.steps, state_bits=args.state_bits, report=10, routing=args.routing, kept_bits=args.kept_bits)
