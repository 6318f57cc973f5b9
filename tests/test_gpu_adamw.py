"""AdamW over many tensors (`AdamW`) against the float64 oracle.

Tolerances.  u = 2^-24.  m and v of one step are sums of two products: off by at most 3 u of the larger (4 u for v); over k steps the
errors add, 4 k u.  The move lr m^ / (sqrt(v^) + eps) adds the roundings of a root, a quotient and three factors: with those of
m and v under 10 (k + 1) u of the move where the terms of m do not cancel, and (1 - beta1) |g| u / sqrt(v) of it where they do, which is
under 40 u of the step size for these gradients.  p is rounded after two more operations: 2 u |p| a step.  16-bit parameters:
half a step of their type each step on top.  The 8-bit codes are decided in 64 bits in the oracle's order of operations, so the
moments are equal to the last bit."""
import numpy as np
import pytest
import torch

import rl_gan_amd as R
from oracle import recurrent_policy as O

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24
LR, BETAS, EPS, DECAY = 2e-3, (0.9, 0.99), 1e-8, 0.1
HYPER = dict(lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY)


def _np(t):
    return t.detach().double().cpu().numpy()


def _make(sizes, kinds, grad_kinds, seed):
    g = torch.Generator(device="cpu").manual_seed(seed)
    params, grads = [], []
    for i, n in enumerate(sizes):
        params.append((torch.randn(n, generator=g) * 0.3).to(TYPES[kinds[i % len(kinds)]]).cuda())
        scale = torch.exp(torch.randn(n, generator=g))
        grads.append((torch.randn(n, generator=g) * scale * 1e-2).to(TYPES[grad_kinds[i % len(grad_kinds)]]).cuda())
    return params, grads


class Host:
    """The oracle's copy: parameters as held (rounded to their types), flat moments."""

    def __init__(self, opt):
        self.opt = opt
        self.p = [_np(p) for p in opt.params]
        m, v = opt.moments()
        self.m, self.v, self.t = _np(m), _np(v), int(opt.steps.item())

    def flat(self, tensors):
        out = np.zeros(self.opt.size)
        for o, t in zip(self.opt.offsets, tensors):
            out[o:o + t.size] = t.reshape(-1)
        return out

    def step(self, grads, lr=LR, scale=1.0):
        self.t += 1
        p, self.m, self.v = O.adamw_step(self.flat(self.p), self.flat([_np(g) for g in grads]), self.m, self.v, self.t, lr, BETAS, EPS,
                                         DECAY, self.opt.state_bits, scale)
        new = [p[o:o + q.size].reshape(q.shape) for o, q in zip(self.opt.offsets, self.p)]
        self.p = [torch.from_numpy(q).to(t.dtype).double().numpy() if t.dtype != torch.float32 else q for q, t in zip(new, self.opt.params)]
        return new

    def check(self, steps, what=""):
        m, v = self.opt.moments()
        if self.opt.state_bits == 8:
            np.testing.assert_array_equal(_np(m), self.m, err_msg=what)
            np.testing.assert_array_equal(_np(v), self.v, err_msg=what)
        else:
            big = np.abs(self.m) + 0.2                           # |(1 - beta1) g| of these gradients stays under 0.2
            assert np.all(np.abs(_np(m) - self.m) <= 4 * steps * U * big), what
            assert np.all(np.abs(_np(v) - self.v) <= 5 * (steps + 1) * U * self.v), what
        assert int(self.opt.steps.item()) == self.t
        for i, (p, q) in enumerate(zip(self.opt.params, self.p)):
            move = 12 * LR                                      # |m^| / sqrt(v^) stays under 12 in these few steps
            tol = steps * (2 * U * (np.abs(q) + move) + 40 * (steps + 1) * U * move)
            if p.dtype != torch.float32:                         # the two may round to neighbours, and go on from there
                tol = tol + steps * torch.finfo(p.dtype).eps * (np.abs(q) + move)
            bad = ~(np.abs(_np(p) - q) <= tol)
            assert not bad.any(), (what, i, int(bad.sum()), _np(p)[bad][:3], q[bad][:3])


SIZES = [1, 3, 4, 63, 64, 65, 200, 255, 257, 2047, 2048, 2049, 4100, 10007]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("kinds,grad_kinds", [(["fp32"], ["fp32"]), (["bf16"], ["bf16"]), (["fp16"], ["fp32"]), (["fp32"], ["bf16", "fp16"]),
                                              (["fp32", "bf16", "fp16"], ["fp16", "fp32", "bf16", "fp32"])])
def test_steps(kinds, grad_kinds, bits):
    params, grads = _make(SIZES, kinds, grad_kinds, 1)
    opt = R.AdamW(params, state_bits=bits, **HYPER)
    host = Host(opt)
    for k in range(3):
        opt.step(grads)
        host.step(grads)
        host.check(k + 1, f"step {k}")
        grads = [(g.float() * -0.7 + 1e-3).to(g.dtype) for g in grads]


@pytest.mark.parametrize("bits", [8, 32])
def test_tensors_at_any_address(bits):
    """Views into one buffer that begin at odd elements, shapes of any rank, and an empty tensor; the rest of the buffer stays."""
    for kind, t in TYPES.items():
        room = (torch.randn(3000, device="cuda") * 0.2).to(t)
        before = room.clone()
        params = [room[1:8], room[9:9 + 64 * 3].view(3, 64), room[203:203], room[301:302].view(()), room[405:405 + 2001]]
        grads = [(torch.randn(p.shape, device="cuda") * 1e-2).to(t) for p in params]
        opt = R.AdamW(params, state_bits=bits, **HYPER)
        host = Host(opt)
        opt.step(grads)
        host.step(grads)
        host.check(1, kind)
        rest = torch.ones(3000, dtype=torch.bool, device="cuda")
        for a, b in ((1, 8), (9, 201), (301, 302), (405, 2406)):
            rest[a:b] = False
        assert torch.equal(room[rest], before[rest])


@pytest.mark.parametrize("bits", [8, 32])
def test_more_tensors_than_a_launch_takes(bits):
    params, grads = _make([17 + i % 90 for i in range(900)], ["fp32", "bf16"], ["fp32"], 2)
    opt = R.AdamW(params, state_bits=bits, **HYPER)
    host = Host(opt)
    for k in range(2):
        opt.step(grads)
        host.step(grads)
        host.check(k + 1)


@pytest.mark.parametrize("bits", [8, 32])
def test_scale_skip_and_rate(bits):
    params, grads = _make([70, 3000], ["fp32"], ["fp16"], 3)
    opt = R.AdamW(params, state_bits=bits, **HYPER)
    host = Host(opt)
    scale = torch.tensor(0.125, device="cuda")
    opt.step(grads, grad_scale=scale)
    host.step(grads, scale=0.125)
    host.check(1)
    held = [p.clone() for p in params] + [t.clone() for t in opt.state_dict().values()]
    opt.step([torch.full_like(g, float("inf")) for g in grads], skip=torch.ones(1, dtype=torch.bool, device="cuda"))
    for a, b in zip(held, params + list(opt.state_dict().values())):
        assert torch.equal(a, b)
    opt.lr = LR / 2                                             # a number goes into the device scalar that the kernels read
    assert torch.is_tensor(opt.lr) and float(opt.lr) == np.float32(LR / 2)
    with pytest.raises(AttributeError):
        opt.steps = 3
    opt.step(grads, skip=torch.zeros((), dtype=torch.uint8, device="cuda"))
    host.step(grads, lr=LR / 2)
    host.check(2)


@pytest.mark.parametrize("bits", [8, 32])
def test_state_goes_out_and_in(bits):
    params, grads = _make([65, 700, 129], ["fp32"], ["fp32"], 4)
    opt = R.AdamW(params, state_bits=bits, **HYPER)
    opt.step(grads)
    other = R.AdamW([p.clone() for p in params], state_bits=bits, **HYPER)
    other.load_state_dict(opt.state_dict())
    third = R.AdamW([p.clone() for p in params], state_bits=bits, **HYPER)
    m, v = opt.moments()
    third.load_moments(m, v, 1)                                 # values that the codes hold come back as the same codes
    for o in (opt, other, third):
        o.step(grads)
    for o in (other, third):
        for a, b in zip(opt.params + list(opt.moments()), o.params + list(o.moments())):
            assert torch.equal(a, b)
    dirty = [t.clone() for t in opt.moments()]                  # what lies between the parameters is not used
    for t in dirty:
        keep = torch.zeros_like(t, dtype=torch.bool)
        for v in opt.views(keep):
            v.fill_(True)
        t[~keep] = float("nan")
    third.load_moments(*dirty, 7)
    assert all(torch.equal(a, b) for a, b in zip(third.moments(), opt.moments())) and int(third.steps) == 7
    parts = opt.views(opt.moments()[0])
    assert [p.shape for p in parts] == [p.shape for p in params] and all((p != 0).any() for p in parts)


def test_values_of_8_bits():
    """load_moments and moments against the oracle's rounding: magnitudes over the whole range of a float, zeros, negative zeros,
    blocks that are all zero and blocks with one number that is not finite."""
    g = torch.Generator(device="cpu").manual_seed(5)
    n = 64 * 400
    m = torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g) * 4)
    v = torch.exp(torch.randn(n, generator=g) * 8)
    m[:64], v[:64] = 0, 0
    m[64:128] = -0.0
    m[200:220], v[210:230] = 0, 0
    m[640:704] *= 1e-30
    v[640:704] *= 1e-30
    m[704:768] *= 1e-38                                          # partly under the normal range
    v[704:768] *= 1e-38
    m[1280:1344] *= 1e30
    v[1280:1344] *= 1e30
    p = torch.zeros(n, device="cuda")
    opt = R.AdamW([p], state_bits=8, **HYPER)
    opt.load_moments(m.cuda(), v.cuda(), 5)
    got_m, got_v = (t.cpu().numpy() for t in opt.moments())
    np.testing.assert_array_equal(got_m, O.round8(m.double().numpy(), True).astype(np.float32))
    root = O.round8(np.sqrt(v.double().numpy()), False).astype(np.float32)
    with np.errstate(under="ignore", over="ignore"):
        np.testing.assert_array_equal(got_v, root * root)
    assert (got_v[(v.numpy() > 1e-30) & (np.arange(n) < 640)] > 0).all()   # a second moment never becomes 0
    m[70], v[140] = float("inf"), float("nan")
    opt.load_moments(m.cuda(), v.cuda(), 5)
    got_m, got_v = opt.moments()
    assert torch.isnan(got_m[64:128]).all() and torch.isfinite(got_m[:64]).all() and torch.isfinite(got_m[128:]).all()
    assert torch.isnan(got_v[128:192]).all() and torch.isfinite(got_v[:128]).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_small_second_moments_do_not_explode(bits):
    """One large gradient among small ones of a block, the same every step: no element moves by more than a few step sizes, where a
    second moment that became 0 would move it by 1e-7 / 1e-12 of them.  The bound: in 32 bits m^ / sqrt(v^) is 1.  In 8 a step's
    rounding is at most 2^-4 of m and 2^-5 of the root; over 20 steps m is at most 1 + 2^-4 sum (b1 (1 + 2^-4))^k < 1.9 of what it
    should be, and v at least (1 - 2^-4)^20 > 0.27 of it: 1.9 / sqrt(0.27) < 4."""
    p = torch.zeros(64, device="cuda")
    g = torch.full((64,), 1e-7, device="cuda")
    g[0] = 1.0
    opt = R.AdamW([p], lr=1e-2, betas=BETAS, eps=1e-12, weight_decay=0.0, state_bits=bits)
    for _ in range(20):
        before = p.clone()
        opt.step([g])
        assert (p - before).abs().max() <= 1e-2 * (4 if bits == 8 else 1.01)


def test_random_rounding_of_one_step():
    """Codes rounded at random against the same rounding of the oracle's moments with the oracle's Philox: a magnitude's 16 bits below
    the code, plus 16 random bits, carry or do not."""
    from oracle import philox
    n, seed, t = 64 * 40, 0x123456789ABCDEF, 6
    g = torch.Generator(device="cpu").manual_seed(9)
    m0, v0 = torch.randn(n, generator=g).cuda(), torch.exp(torch.randn(n, generator=g)).cuda()
    p, grad = torch.zeros(n, device="cuda"), torch.randn(n, generator=g).cuda()
    opt = R.AdamW([p], state_bits=8, rounding="random", seed=seed, **HYPER)
    opt.load_moments(m0, v0, t - 1)
    m0, v0 = (_np(x) for x in opt.moments())
    opt.step([grad])
    m, v = (_np(x) for x in opt.moments())
    em = m0 * BETAS[0] + _np(grad) * (1 - BETAS[0])
    er = np.sqrt(v0 * BETAS[1] + _np(grad) * (1 - BETAS[1]) * _np(grad))
    words = np.array([philox.philox4x32((i, 0, t, 1), (seed & 0xFFFFFFFF, seed >> 32)) for i in range(n // 4)]).reshape(-1)
    for got, want, bits, man in ((np.abs(m), np.abs(em), words >> 16, 3), (np.sqrt(v), er, words & 0xFFFF, 4)):
        high = want.astype(np.float64).view(np.int64) >> 32
        high = (high + (bits << (4 - man))) >> (20 - man) << (20 - man)
        np.testing.assert_array_equal(got, (high << 32).view(np.float64))   # all of these lie within the codes' 16 octaves
    assert np.all(np.sign(m) == np.sign(em))


def test_random_rounding_follows_the_mean():
    """Second moments that decay by 1% a step, half a percent of the root, which is under half a code: to nearest they stay for
    ever; at random their root's mean is the exact one.  A step's rounding has a deviation of at most half a code's 2^-4 of the
    root, independent from step to step: over 300 steps some 2^-5 sqrt(300) = 0.55 of the mean for an element, 0.0034 for the mean
    of 25600; 0.02 is six of those."""
    n = 25600
    for rounding in ("nearest", "random"):
        p = torch.zeros(n, device="cuda")
        opt = R.AdamW([p], state_bits=8, rounding=rounding, seed=3, **HYPER)
        opt.load_moments(torch.zeros(n, device="cuda"), torch.full((n,), 4.0, device="cuda"), 10)
        zero = torch.zeros(n, device="cuda")
        for _ in range(300):
            opt.step([zero])
        root = opt.moments()[1].double().sqrt().mean().item()
        if rounding == "nearest":
            assert root == 2.0
        else:
            want = 2.0 * 0.99 ** 150
            assert abs(root / want - 1) <= 0.02


def test_random_rounding_repeats():
    def run(seed, split):
        params, grads = _make([1000, 77], ["fp32"], ["bf16"], 10)
        opt = R.AdamW(params, state_bits=8, rounding="random", seed=seed, **HYPER)
        for k in range(4):
            opt.step(grads)
            if k == split:                                       # the state handed on to another optimizer
                other = R.AdamW(params, state_bits=8, rounding="random", seed=seed, **HYPER)
                other.load_state_dict(opt.state_dict())
                opt = other
        return params + list(opt.moments())
    a, b, c = run(5, None), run(5, 1), run(6, None)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert not torch.equal(a[2], c[2])


def test_numbers_that_are_not_finite():
    """A NaN gradient spoils its own element (32 bits) or its block (8 bits) and nothing else."""
    for bits in (8, 32):
        params, grads = _make([256, 100], ["fp32"], ["fp32"], 6)
        grads[0][70] = float("nan")
        opt = R.AdamW(params, state_bits=bits, **HYPER)
        opt.step(grads)
        opt.step([torch.zeros_like(g) for g in grads])
        bad = torch.isnan(params[0])
        assert bad[70] and not bad[:64].any() and not bad[128:].any() and torch.isfinite(params[1]).all()
        assert bits == 8 or int(bad.sum()) == 1


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps(bits):
    """Captured steps of two optimizers replayed in turn with eager steps between: counters, rates and gradients are followed."""
    def make(seed):
        params, grads = _make([300, 65, 5000], ["fp32", "bf16"], ["fp32"], seed)
        return R.AdamW(params, state_bits=bits, **HYPER), grads
    pairs = [make(7), make(8)]
    twins = []
    for opt, grads in pairs:
        twins.append(R.AdamW([p.clone() for p in opt.params], state_bits=bits, **HYPER))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    for opt, grads in pairs:
        with torch.cuda.stream(stream):
            opt.step(grads)
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            opt.step(grads)
        graphs.append(g)
    for twin, (_, grads) in zip(twins, pairs):
        twin.step(grads)
    for turn in range(4):
        for (opt, grads), twin, graph in zip(pairs, twins, graphs):
            for x in grads:
                x.mul_(-0.9)
            if turn == 2:
                opt.set_lr(1e-4)
                twin.set_lr(1e-4)
            graph.replay()
            twin.step(grads)
            if turn == 1:
                opt.step(grads)
                twin.step(grads)
        torch.cuda.synchronize()
        for (opt, _), twin in zip(pairs, twins):
            assert int(opt.steps.item()) == int(twin.steps.item())
            for a, b in zip(opt.params + list(opt.moments()), twin.params + list(twin.moments())):
                assert torch.equal(a, b), turn


@pytest.mark.parametrize("bits", [8, 32])
def test_a_tensor_of_more_than_32_bits(bits):
    """The last elements of a tensor of more than 2^31 step as those of a small one do, to the bit."""
    n, tail = (1 << 31) + 64 * 1000 + 37, 64 * 200 + 37
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    rnd = torch.Generator(device="cuda").manual_seed(11)
    p[-tail:] = torch.randn(tail, generator=rnd, device="cuda").bfloat16()
    g[-tail:] = torch.randn(tail, generator=rnd, device="cuda").bfloat16()
    small, small_g = p[-tail:].clone(), g[-tail:].clone()
    big, few = R.AdamW([p], state_bits=bits, **HYPER), R.AdamW([small], state_bits=bits, **HYPER)
    for _ in range(2):
        big.step([g])
        few.step([small_g])
    assert torch.equal(p[-tail:], small) and (p[:1000] == 0).all()
    assert torch.equal(big.first[n - tail:n], few.first[:tail]) and torch.equal(big.second[n - tail:n], few.second[:tail])


def test_refusals():
    p = torch.zeros(10, device="cuda")
    bad = [lambda: R.AdamW([]), lambda: R.AdamW([p], state_bits=16), lambda: R.AdamW([p.cpu()]), lambda: R.AdamW([p.double()]),
           lambda: R.AdamW([p, p]), lambda: R.AdamW([p[:6], p[5:]]), lambda: R.AdamW([torch.zeros(4, 4, device="cuda").t()]),
           lambda: R.AdamW([p], betas=(1.0, 0.9)), lambda: R.AdamW([p], lr=-1.0), lambda: R.AdamW([p], eps=-1.0),
           lambda: R.AdamW([p], weight_decay=float("nan")),
           lambda: R.AdamW([p], rounding="up"), lambda: R.AdamW([p], seed=-1)]
    opt = R.AdamW([p, torch.zeros(3, 4, device="cuda")])
    g = [torch.zeros(10, device="cuda"), torch.zeros(3, 4, device="cuda")]
    one = torch.ones(1, device="cuda")
    bad += [lambda: opt.step(g[:1]), lambda: opt.step([g[0], g[1].t()]), lambda: opt.step([g[0], g[1].double()]),
            lambda: opt.step([g[0].cpu(), g[1]]), lambda: opt.step([g[0], torch.zeros(12, device="cuda")]),
            lambda: opt.step(g, grad_scale=one.double()), lambda: opt.step(g, grad_scale=torch.ones(2, device="cuda")),
            lambda: opt.step(g, skip=one), lambda: opt.step(g, grad_scale=one.cpu()), lambda: opt.set_lr(-1),
            lambda: opt.load_moments(one, one, 1), lambda: opt.load_state_dict({}),
            lambda: opt.load_state_dict(R.AdamW([p]).state_dict())]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was taken")
    q = torch.zeros(10, device="cuda")
    moved = R.AdamW([q])
    q.data = torch.zeros(10, device="cuda")
    with pytest.raises(ValueError):
        moved.step([g[0]])
