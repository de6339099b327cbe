"""AdamW where every warp takes many blocks, from many tensors: rings that are filled again, tensors that change on the way, both lengths of runs.

Bounds as in the tests of small tensors: with u = 2^-24, m and v go through three and four roundings a step, w through two of its own size and
about 16 of the update's.  Codes of m, the units and the copies are exact; a code of the root of v may be its neighbour where the root's last
bits decide (2^-16 of them), and is the smallest one where the rounding's bits would make it zero.
"""
import pytest
import torch

from mgpt_b200 import AdamW

pytestmark = pytest.mark.gpu
U, BLOCK = 2.0 ** -24, 256
LR, B1, B2, EPS = 1e-2, 0.9, 0.999, 1e-8


def _mixed(h):
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & 0xFFFFFFFF
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _exponent(a):
    return (a.contiguous().view(torch.int32) >> 23) - 127


def _codes(a, unit, random16):
    a = torch.ldexp(a, -unit[:, None])
    low = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)
    return (((a + low).view(torch.int32) + (random16 << 4)) & ~0xFFFFF).view(torch.float32) - low


def _make(sizes, offsets, dtypes, std, seed):
    """Tensors of these sizes, each some elements behind a boundary of 16 bytes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    starts, at = [], 0
    for k, o in zip(sizes, offsets):
        starts.append(at + o)
        at += -(-(k + o) // 8) * 8
    flat = torch.randn(at, device="cuda", generator=g) * std
    both = {d: flat.to(d) for d in set(dtypes)}
    return [both[d][a:a + k] for a, k, d in zip(starts, sizes, dtypes)]


def _cases():
    some = [1, 255, 70001, 257, 4096, 30000, 7, 0, 65536, 512, 12345, 2048]
    f, b = torch.float32, torch.bfloat16
    yield "one tensor", [10_000_001], [0], [f]
    yield "one tensor off its boundary", [10_000_001], [1], [b]
    yield "few large ones", [6_000_000, 255, 6_000_001, 1, 3_000_000], [0, 0, 0, 3, 2], [b, f, b, f, f]
    yield "many", [some[(i * 5 + i // 12) % 12] for i in range(600)], [(i // 3) % 4 if i % 3 == 0 else 0 for i in range(600)], [f if i % 4 else b for i in range(600)]


@pytest.mark.parametrize("name,sizes,offsets,dtypes", [pytest.param(*c, id=c[0]) for c in _cases()])
@pytest.mark.parametrize("bits", [8, 32])
def test_many_blocks_per_warp(bits, name, sizes, offsets, dtypes):
    w, g = _make(sizes, offsets, [torch.float32] * len(sizes), 0.05, 1), _make(sizes, offsets[::-1] if len(sizes) > 9 else offsets, dtypes, 1e-3, 2)
    c = [a.bfloat16() if i % 5 != 4 else None for i, a in enumerate(w)]
    decay = [0.1 * (i % 3) for i in range(len(sizes))]
    opt = AdamW(w, g, copies=c, state_bits=bits, weight_decay=decay, seed=77)
    blocks = [-(-k // BLOCK) for k in sizes]
    total = sum(blocks) * BLOCK
    assert opt.blocks * BLOCK == total and opt.blocks > 10 * 2 * 148 * 8          # ten blocks for each warp of two thread blocks per SM
    place = torch.cat([torch.arange(k, device="cuda") + BLOCK * sum(blocks[:i]) for i, k in enumerate(sizes)])
    size = torch.tensor(sizes, device="cuda")
    D = torch.repeat_interleave(torch.tensor(decay, device="cuda", dtype=torch.float64), size)
    W = torch.cat(w).double()
    rough = torch.zeros_like(W)
    m, v = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    for t in (1, 2, 3):
        G = torch.zeros(total, device="cuda")
        G[place] = torch.cat([a.float() for a in g])
        opt.step(t, lr=LR, beta1=B1, beta2=B2, eps=EPS)
        if bits == 8:
            m, v = B1 * m + (1.0 - B1) * G, B2 * v + ((1.0 - B2) * G) * G
            m2, v2 = m.view(-1, BLOCK), v.view(-1, BLOCK)
            em, ev = _exponent(m2.abs().amax(1)).clamp(min=-100) - 7, (_exponent(v2.amax(1)) >> 1) - 7
            key = _mixed((77 * 0x9E3779B1 + t) & 0xFFFFFFFF)
            r = _mixed(torch.arange(total, device="cuda") ^ key).view(-1, BLOCK)
            cm = torch.copysign(_codes(m2.abs(), em, (r & 0xFFFF).int()), m2)
            cv = _codes(v2.sqrt(), ev, (r >> 16).int())
            cv = torch.where((v2 > 0) & (cv == 0), 2.0 ** -9, cv)
            one = torch.ones_like(m2[:, 0])
            assert torch.equal(opt.m_scale, torch.ldexp(one, em)) and torch.equal(opt.v_scale, torch.ldexp(one, ev))
            got_m, got_v = opt.m.float().view(-1, BLOCK), opt.v.float().view(-1, BLOCK)
            assert torch.equal(got_m, cm)
            off = got_v != cv
            step = torch.exp2(torch.floor(torch.log2(cv.clamp(min=2.0 ** -9))) - 3).clamp(min=2.0 ** -9)
            assert int(off.sum()) <= 2 + total * 2.0 ** -16 and ((got_v - cv).abs() <= 1.001 * step).all()
            del off, step, cm, cv, r
        else:
            m, v = B1 * m.double() + (1.0 - B1) * G.double(), B2 * v.double() + (1.0 - B2) * G.double().square()
        up = LR * (m[place].double() / (1 - B1 ** t)) / ((v[place].double() / (1 - B2 ** t)).sqrt() + EPS)
        W = W * (1 - LR * D) - up
        now = torch.cat(w)
        rough = rough + 3 * U * W.abs() + 20 * U * up.abs()
        assert ((now.double() - W).abs() <= rough).all()
        for a, b in zip(w, c):
            assert b is None or torch.equal(b, a.bfloat16())
        if bits == 32:
            # the terms of m are at most the largest gradient so far, which is this one's size
            assert ((opt.m.double() - m).abs() <= 12 * U * G.double().abs()).all() and ((opt.v.double() - v).abs() <= 12 * U * v).all()
        else:
            m, v = (got_m * opt.m_scale[:, None]).view(-1), (got_v * opt.v_scale[:, None]).view(-1).square()
            W, rough = now.double(), torch.zeros_like(rough)
        for a in g:
            a.neg_()
    assert not int(opt.found_nonfinite)
