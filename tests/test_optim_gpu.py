"""AdamW over many tensors against its formulas: in 64 bits for the weights and the 32-bit moments, and against a model of the
8-bit moments in numpy, whose FP32 operations are the kernel's one by one.

Bounds, with u = 2^-24: m and v go through three and four roundings; w through two of its own size and about 16 of the update's
(root and quotient of the 8-bit form are good to 2 ulp each).  The model's codes of m and all scales are the kernel's, bit for bit; a
code of the root of v may be the next one where the root's last bits decide, which is 2^-18 of them.
"""
import numpy as np
import pytest
import torch

from mgpt_b200 import AdamW, MoeError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8)
f32 = np.float32


def _mixed(h):
    h = h ^ (h >> np.uint64(16))
    h = (h * np.uint64(0x85EBCA6B)) & np.uint64(0xFFFFFFFF)
    h = h ^ (h >> np.uint64(13))
    h = (h * np.uint64(0xC2B2AE35)) & np.uint64(0xFFFFFFFF)
    return h ^ (h >> np.uint64(16))


def _codes(a, unit_exp, random16):
    """Values over 2^unit_exp to three bits of mantissa, stochastically: the values the codes stand for, in units."""
    a = np.ldexp(a, -unit_exp[:, None]).astype(f32)
    low = np.where(a < f32(2.0 ** -6), f32(2.0 ** -6), f32(0))
    bits = (a + low).astype(f32).view(np.uint32) + (random16.astype(np.uint32) << np.uint32(4))
    return (bits & np.uint32(0xFFF00000)).view(f32) - low


def _exponent(a):
    return (np.ascontiguousarray(a).view(np.int32) >> 23) - 127


def _model8(m, ms, s, vs, g, t, seed, beta1=0.9, beta2=0.999, **_):
    """One step of the 8-bit moments: codes (as values), units, and the FP32 moments before rounding; arrays [blocks, 256]."""
    m, v = m * ms[:, None], np.square(s * vs[:, None])
    m1 = f32(beta1) * m + f32(1.0 - beta1) * g
    v1 = f32(beta2) * v + (f32(1.0 - beta2) * g) * g
    bad = ~(np.isfinite(m1) & np.isfinite(v1))
    m1, v1 = np.where(bad, m, m1).astype(f32), np.where(bad, v, v1).astype(f32)
    em, ev = np.maximum(_exponent(np.abs(m1).max(1)), -100) - 7, (_exponent(v1.max(1)) >> 1) - 7
    key = _mixed(np.uint64((seed * 0x9E3779B1 + t) & 0xFFFFFFFF))
    r = _mixed(np.arange(m.size, dtype=np.uint64).reshape(m.shape) ^ key)
    cm = np.copysign(_codes(np.abs(m1), em, r & np.uint64(0xFFFF)), m1)
    cs = _codes(np.sqrt(v1), ev, r >> np.uint64(16))
    return cm, np.ldexp(f32(1), em), cs, np.ldexp(f32(1), ev), m1, v1, bad


def _tensors(sizes, grad=torch.float32, seed=0, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def make(dtype, std):
        flat = (torch.randn(sum(sizes) + offset + 8 * len(sizes), device="cuda", generator=g) * std).to(dtype)
        out, at = [], offset
        for k in sizes:
            out.append(flat[at:at + k])
            at += k if offset else -(-k // 8) * 8                    # offset: whatever boundary comes
        return out

    return make(torch.float32, 0.05), make(grad, 1e-3), make(torch.bfloat16, 1.0)


def _update(w, m1, v1, t, decay, lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8):
    up = lr * (m1 / (1 - beta1 ** t)) / (np.sqrt(v1 / (1 - beta2 ** t)) + eps)
    return w * (1 - lr * decay) - up, 3 * U * np.abs(w) + 20 * U * np.abs(up)


SIZES = [[1], [255, 256, 257], [7, 0, 2048, 1, 513], [64 * 64, 64, 64 * 100, 100] * 5, [70001]]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
def test_32_bit_moments(sizes, offset, grad):
    w, g, c = _tensors(sizes, grad, seed=len(sizes), offset=offset)
    decay = [0.1 * (i % 3) for i in range(len(sizes))]
    opt = AdamW(w, g, copies=c, state_bits=32, weight_decay=decay)
    want = [(a.double().cpu().numpy(), np.zeros(a.numel()), np.zeros(a.numel())) for a in w]
    rough = [np.zeros(a.numel()) for a in w]
    for t in (1, 2, 3):
        opt.step(t, **HYPER)
        for i, a in enumerate(g):
            x = a.double().cpu().numpy()
            m1, v1 = 0.9 * want[i][1] + (1.0 - 0.9) * x, 0.999 * want[i][2] + (1.0 - 0.999) * x * x
            new, tol = _update(want[i][0], m1, v1, t, decay[i])
            want[i], rough[i] = (new, m1, v1), rough[i] + tol
            a.neg_()                                                # (another gradient of the same sizes)
    at = 0
    for i, a in enumerate(w):
        k = a.numel()
        assert (np.abs(a.double().cpu().numpy() - want[i][0]) <= rough[i]).all()
        m, v = opt.m[at:at + k].double().cpu().numpy(), opt.v[at:at + k].double().cpu().numpy()
        assert (np.abs(m - want[i][1]) <= 12 * U * np.abs(g[i].double().cpu().numpy())).all()
        assert (np.abs(v - want[i][2]) <= 12 * U * want[i][2]).all()
        assert torch.equal(c[i], a.bfloat16())
        at += -(-k // 256) * 256
    assert at == opt.m.numel() and not int(opt.found_nonfinite)


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16])
def test_8_bit_moments_follow_their_model(sizes, offset, grad):
    w, g, c = _tensors(sizes, grad, seed=7 + len(sizes), offset=offset)
    opt = AdamW(w, g, copies=c, state_bits=8, weight_decay=0.1, seed=12345)
    blocks = opt.blocks
    state = [np.zeros((blocks, 256), f32), np.ones(blocks, f32), np.zeros((blocks, 256), f32), np.ones(blocks, f32)]
    real = np.zeros((blocks, 256), bool)
    for t in (1, 2, 3):
        before = [a.double().cpu().numpy() for a in w]
        G, at = np.zeros((blocks, 256), f32), 0
        for a in g:
            k = a.numel()
            G.reshape(-1)[at:at + k] = a.float().cpu().numpy()
            real.reshape(-1)[at:at + k] = True
            at += -(-k // 256) * 256
        opt.step(t, **HYPER)
        cm, ms, cs, vs, m1, v1, _ = _model8(*state, G, t, 12345)
        got = [x.float().cpu().numpy().reshape(blocks, 256) for x in (opt.m, opt.v)]
        assert np.array_equal(opt.m_scale.cpu().numpy(), ms) and np.array_equal(opt.v_scale.cpu().numpy(), vs)
        assert np.array_equal(got[0], cm)
        off = got[1] != cs
        step = np.maximum(np.exp2(np.floor(np.log2(np.maximum(cs, 2.0 ** -9))) - 3), 2.0 ** -9)
        assert off.sum() <= 2 + off.size * 2.0 ** -16 and (np.abs(got[1] - cs) <= 1.001 * step).all()
        assert not got[0][~real].any() and not got[1][~real].any()
        at = 0
        for i, a in enumerate(w):
            k = a.numel()
            new, tol = _update(before[i], m1.reshape(-1)[at:at + k].astype(np.float64), v1.reshape(-1)[at:at + k].astype(np.float64), t, 0.1)
            assert (np.abs(a.double().cpu().numpy() - new) <= tol).all()
            assert torch.equal(c[i], a.bfloat16())
            at += -(-k // 256) * 256
            g[i].mul_(-0.5)
        state = [got[0], ms, got[1], vs]


def test_rounding_is_unbiased():
    """A constant gradient for 400 steps: the mean of v follows its recursion, which rounding to nearest would leave where it is.
    Each step's rounding is off by at most an eighth of the root, independent from element to element: of 65536 elements the mean is
    within 6 standard deviations of 400 such steps."""
    n = 65536
    w, g = torch.zeros(n, device="cuda"), torch.full((n,), 1e-3, device="cuda")
    opt = AdamW([w], [g], state_bits=8, weight_decay=0.0, seed=1)
    opt.step(1, lr=0.0)
    root1 = (opt.v.float() * opt.v_scale.repeat_interleave(256)).double().mean()
    for t in range(2, 401):
        opt.step(t, lr=0.0)
    want = 1e-3 * np.sqrt(1 - 0.999 ** 400)
    got = float((opt.v.float() * opt.v_scale.repeat_interleave(256)).double().mean())
    assert got > 10 * float(root1)                                  # it moved
    # roots are rounded without bias, v is the square of them: each step adds the rounding's variance, at most (root/8)^2/4 of
    # 400 steps' share, to v
    assert want * 0.99 <= got <= want * np.sqrt(1 + 400 / 256) * 1.01


@pytest.mark.parametrize("bits", [8, 32])
def test_gradients_that_are_not_finite(bits):
    w, g, c = _tensors([1000, 300], seed=3)
    opt = AdamW(w, g, copies=c, state_bits=bits, weight_decay=0.1)
    opt.step(1, **HYPER)
    assert not int(opt.found_nonfinite)
    w1 = [a.clone() for a in w]
    unit = opt.m_scale.repeat_interleave(256) if bits == 8 else 1.0
    m1 = opt.m.float() * unit
    bad = [torch.tensor([5, 600]), torch.tensor([299])]
    g[0][5], g[0][600], g[1][299] = float("nan"), float("inf"), 1e30
    opt.step(2, **HYPER)
    assert int(opt.found_nonfinite) == 1
    for a, b, i in zip(w, w1, bad):
        fine = torch.ones(a.numel(), dtype=torch.bool)
        fine[i] = False
        assert torch.equal(a[i], b[i]) and (a[fine] != b[fine]).all() and a.isfinite().all()
    m2 = opt.m.float() * (opt.m_scale.repeat_interleave(256) if bits == 8 else 1.0)
    assert m2.isfinite().all()
    kept = torch.tensor([5, 600, 1024 + 299])
    assert torch.equal(m1[kept], m2[kept]) if bits == 32 else ((m1[kept] - m2[kept]).abs() <= m1[kept].abs() / 4).all()


def test_scaled_gradients_and_same_bits_again():
    for bits in (8, 32):
        runs = []
        for scale in (None, torch.tensor([0.25], device="cuda"), torch.tensor(0.25, device="cuda")):
            w, g, _ = _tensors([5000, 300], seed=4)
            if scale is None:
                for a in g:
                    a.mul_(0.25)
            opt = AdamW(w, g, state_bits=bits, seed=9)
            opt.step(1, grad_scale=scale)
            opt.step(2, grad_scale=scale)
            runs.append([a.clone() for a in w] + [opt.m.clone().float(), opt.v.clone().float()])
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("offset", [1, 2, 4, 8])
@pytest.mark.parametrize("which", ["weights", "grads", "copies"])
def test_boundaries_do_not_matter(bits, offset, which):
    """One of a tensor's three buffers off its boundary by 1, 2, 4 or 8 elements, the others on theirs: the same bits."""
    sizes = [2048, 300, 4096]

    def run(shift):
        t = dict(zip(("weights", "grads", "copies"), _tensors(sizes, torch.bfloat16, seed=11)))
        if shift:
            moved = [torch.empty(a.numel() + shift, dtype=a.dtype, device="cuda")[shift:] for a in t[which]]
            for a, b in zip(moved, t[which]):
                a.copy_(b)
            t[which] = moved
        opt = AdamW(t["weights"], t["grads"], copies=t["copies"], state_bits=bits, seed=3)
        for step in (1, 2):
            opt.step(step, **HYPER)
        return [a.clone() for a in t["weights"] + t["copies"]] + [opt.m.float(), opt.v.float()]

    assert all(torch.equal(a, b) for a, b in zip(run(0), run(offset)))


def test_other_seed_other_rounding_and_continued_state():
    def run(seed, steps, state=None, t0=0):
        w, g, _ = _tensors([4096], seed=5)
        opt = AdamW(w, g, state_bits=8, seed=seed, state=state)
        for t in range(steps):
            opt.step(t0 + t + 1)
        return w[0].clone(), (opt.m.clone(), opt.v.clone(), opt.m_scale.clone(), opt.v_scale.clone())

    _, a = run(1, 3)
    _, b = run(2, 3)
    assert not torch.equal(a[0].float(), b[0].float())
    _, half = run(1, 2)
    _, c = run(1, 1, half, 2)
    assert torch.equal(a[0].float(), c[0].float()) and torch.equal(a[1].float(), c[1].float())


def test_made_on_one_stream_stepped_on_another():
    """The moments are cleared on the stream that the object is made on, which is busy; the first step runs on another."""
    w, g, _ = _tensors([100000], seed=6)
    want = AdamW([w[0].clone()], g, state_bits=32)
    want.step(1)
    side = torch.cuda.Stream()
    dirty = [torch.full((want.m.numel(),), 7.0, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for a in dirty:
            a.record_stream(side)
        del a, dirty
        torch.cuda._sleep(50_000_000)
        opt = AdamW(w, g, state_bits=32)
    opt.step(1)
    torch.cuda.synchronize()
    assert torch.equal(opt.weights[0], want.weights[0]) and torch.equal(opt.m, want.m) and torch.equal(opt.v, want.v)


def test_refusals():
    w, g, c = _tensors([300, 20])
    for bad in (lambda: AdamW([], []), lambda: AdamW(w, g[:1]), lambda: AdamW(w, g, state_bits=4), lambda: AdamW([a.cpu() for a in w], g),
                lambda: AdamW([a.bfloat16() for a in w], g), lambda: AdamW(w, [a.half() for a in g]), lambda: AdamW(w, [g[1], g[0]]),
                lambda: AdamW(w, g, weight_decay=[0.1]), lambda: AdamW(w, g, copies=[a.float() for a in c]),
                lambda: AdamW(w, g, state=(torch.zeros(768, device="cuda"),)), lambda: AdamW(w, g, state_bits=32, state=(torch.zeros(512, device="cuda"), torch.zeros(768, device="cuda")))):
        with pytest.raises(MoeError):
            bad()
    opt = AdamW(w, g)
    for bad in (dict(t=0), dict(t=1, beta1=1.0), dict(t=1, beta2=-0.1), dict(t=1, grad_scale=torch.ones(2, device="cuda")), dict(t=1, grad_scale=torch.ones(1))):
        with pytest.raises(MoeError):
            opt.step(**bad)
    opt.close()
    with pytest.raises(MoeError):
        opt.step(1)
