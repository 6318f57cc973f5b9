"""The clipped policy loss (`policy_loss`) against the float64 oracle.

Tolerances.  u = 2^-24.  An exponent x log2(e) is rounded twice and 2^x is off by at most 2 u, so e^x of |x| <= 20 (smaller ones
weigh under 1e-8) is off by at most 50 u of itself; a row's sum adds (vocab / 64 + 16) u at most; a probability is therefore off by
P u of itself, P = vocab / 64 + 120, and so are log p and H up to their magnitude (at most log vocab < 12).  The gradient of a row is
k (c (1 - p), c p, eta p (log p + H)): off by at most 4 P u of k (|c| + eta 24).  r = e^(log p - old) and the estimate of the KL follow
log p: their derivative times its error.  Outputs in 16 bits: half a step more."""
import numpy as np
import pytest
import torch

import rl_gan_amd as R
from oracle import recurrent_policy as O

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24
HYPER = dict(clip=(0.2, 0.3), kl_coef=0.05, entropy_coef=0.02, temperature=0.8)


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _inputs(rows, vocab, kind, seed, ref=True, legal=False, weights=True, pad=0, ints=torch.int64):
    g = torch.Generator(device="cpu").manual_seed(seed)
    t = TYPES[kind]
    store = torch.full((rows, vocab + pad), float("nan"), dtype=t)
    z = (torch.randn(rows, vocab, generator=g) * 2).to(t)
    a = torch.randint(0, vocab, (rows,), generator=g)
    z[torch.arange(rows), a] += 3.0
    store[:, :vocab] = z
    mask = None
    if legal:
        mask = torch.rand(rows, vocab, generator=g) > 0.4
        mask[torch.arange(rows), a] = torch.rand(rows, generator=g) > 0.1     # some actions are not legal
        if rows > 2:
            mask[2] = False                                                # and one row has none that is
    zm = z.double() / HYPER["temperature"]
    if legal:
        zm = zm.masked_fill(~mask, -float("inf"))
    lp = torch.log_softmax(zm, 1)[torch.arange(rows), a].float()
    lp = torch.where(torch.isfinite(lp), lp, torch.zeros_like(lp))
    if rows > 3:
        a[1] = -1
    s = dict(logits=store.cuda()[:, :vocab], actions=a.to(ints).cuda(), old_logp=(lp + 0.2 * torch.randn(rows, generator=g)).cuda(),
             advantages=torch.randn(rows, generator=g).cuda(), ref_logp=None, weights=None, legal=None if mask is None else mask.cuda())
    if ref:
        s["ref_logp"] = (lp + 0.3 * torch.randn(rows, generator=g)).cuda()
    if weights:
        w = torch.rand(rows, generator=g)
        if rows > 4:
            w[4] = 0
        s["weights"] = w.cuda()
    return s


def _call(s, grad=True, **more):
    kw = {**HYPER, **more}
    return R.policy_loss(s["logits"], s["actions"], s["old_logp"], s["advantages"], weights=s["weights"], ref_logp=s["ref_logp"],
                         legal=s["legal"], grad=grad, **kw)


def _reference(s, **more):
    kw = {**HYPER, **more}
    if not isinstance(kw["clip"], tuple):
        kw["clip"] = (kw["clip"], kw["clip"])
    return O.policy_loss(_np(s["logits"]), _np(s["actions"]), _np(s["old_logp"]), _np(s["advantages"]), _np(s["weights"]), _np(s["ref_logp"]),
                         None if s["legal"] is None else s["legal"].cpu().numpy(), **kw)


def _check(s, got, ref, grad=True, **more):
    kw = {**HYPER, **more}
    rows, vocab = s["logits"].shape
    P = (vocab / 64 + 120) * U
    loss, logp, entropy, kl, d = ref
    err_lp = P * 12 + 4 * U * np.abs(logp) + 4 * U * np.abs(logp)
    assert np.all(np.abs(_np(got.logp) - logp) <= err_lp), np.abs(_np(got.logp) - logp).max()
    assert np.all(np.abs(_np(got.entropy) - entropy) <= P * 24 + U * entropy)
    dq = np.abs(_np(s["ref_logp"]) - logp) if s["ref_logp"] is not None else np.zeros(rows)
    err_kl = np.expm1(np.minimum(dq, 50)) * err_lp + U * np.abs(kl) + err_lp ** 2 * np.exp(np.minimum(dq, 50))
    a = s["actions"].cpu().numpy()
    used = (a >= 0) & (np.ones(rows) if s["weights"] is None else _np(s["weights"]) != 0).astype(bool)
    if s["legal"] is not None:
        used &= s["legal"].cpu().numpy()[np.arange(rows), np.maximum(a, 0)].astype(bool)
    assert np.all((np.abs(_np(got.kl) - kl) <= err_kl)[used]) and np.all(_np(got.kl)[~used] == 0)
    w = _np(s["weights"]) if s["weights"] is not None else np.full(rows, 1.0 / rows)
    r = np.exp(np.minimum(logp - _np(s["old_logp"]), 50))
    slope = r * np.abs(_np(s["advantages"])) + kw["kl_coef"] * np.expm1(np.minimum(dq, 50))
    per_row = slope * err_lp + kw["entropy_coef"] * (P * 24) + kw["kl_coef"] * err_kl
    bound = float((w * np.where(used, per_row, 0)).sum()) + U * abs(loss)
    assert abs(float(got.loss) - loss) <= bound + 1e-30, (float(got.loss), loss, bound)
    if not grad:
        assert got.dlogits is None
        return
    assert got.dlogits.dtype == s["logits"].dtype and got.dlogits.shape == s["logits"].shape
    g = _np(got.dlogits)
    k = w / kw["temperature"]
    tol = (k * (slope * (4 * P + err_lp) + kw["entropy_coef"] * 24 * 4 * P))[:, None] + U * np.abs(d)
    t = s["logits"].dtype
    if t != torch.float32:
        tol = tol * (1 + torch.finfo(t).eps) + torch.finfo(t).eps / 2 * (np.abs(d) + tol) + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    bad = ~(np.abs(g - d) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], g[bad][:4], d[bad][:4])
    assert np.all(g[~used] == 0)


VOCABS = [1, 2, 3, 4, 7, 13, 16, 17, 18, 29, 31, 32, 57, 63, 64, 65, 121, 128, 129, 200, 255, 256, 257, 500, 512, 513, 1000, 1024, 1025, 2041, 2048, 2049,
          4089, 4096, 4097, 8191, 8192, 8193, 16385, 24577]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("vocab", VOCABS)
def test_widths(vocab, kind):
    rows = 37 if vocab < 600 else 11
    s = _inputs(rows, vocab, kind, 1)
    _check(s, _call(s), _reference(s))
    _check(s, _call(s, grad=False), _reference(s), grad=False)


@pytest.mark.parametrize("kind,vocab", [("fp32", 33000), ("bf16", 49999), ("bf16", 70001), ("fp16", 131072), ("fp32", 140001)])
@pytest.mark.parametrize("rows", [3, 9, 70])
def test_wide_rows(rows, vocab, kind):
    s = _inputs(rows, vocab, kind, 2, legal=rows == 9, pad=3)
    got = _call(s)
    some = slice(0, 9)                                          # (what the oracle has time for)
    part = {k: v if v is None else v[some] for k, v in s.items()}
    ref = _reference(part)
    _check(part, _call(part, grad=False), ref, grad=False)
    if rows > 9:
        got = R.PolicyLoss(_call(part).loss, got.logp[some], got.entropy[some], got.kl[some], got.dlogits[some])
    _check(part, got, ref)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("vocab,rows", [(2, 140001), (9, 140001), (27, 70003), (50, 70003), (64, 70003), (111, 70003), (200, 33001), (256, 33001), (450, 20001),
                                        (900, 9001), (1500, 5001)])
def test_many_rows(rows, vocab, kind):
    """Groups of threads that hold several rows: every row has the bits that it has in a call of few rows; the loss is their sum (in
    64 bits but for the last rounding)."""
    g = torch.Generator(device="cuda").manual_seed(20)
    z = torch.randn(rows, vocab + 1, generator=g, device="cuda").to(TYPES[kind])[:, :vocab]
    a = torch.randint(-1, vocab, (rows,), generator=g, device="cuda")
    s = dict(logits=z, actions=a, old_logp=torch.full((rows,), -float(np.log(vocab)), device="cuda"),
             advantages=torch.randn(rows, generator=g, device="cuda") + 1, weights=torch.rand(rows, generator=g, device="cuda"), ref_logp=None,
             legal=torch.rand(rows, vocab, generator=g, device="cuda") > 0.2 if vocab == 50 else None)
    got = _call(s)
    total = 0.0
    for at in list(range(0, rows, max(1, rows // 7)))[:8]:
        some = slice(at, at + 40)
        part = {k: v if v is None else v[some] for k, v in s.items()}
        few = _call(part)
        for p, q in zip(got[1:], few[1:]):
            assert torch.equal(p[some], q)
    first = {k: v if v is None else v[:20] for k, v in s.items()}
    _check(first, _call(first), _reference(first))
    for at in range(0, rows, 1000):
        total += float(_call({k: v if v is None else v[at:at + 1000] for k, v in s.items()}, grad=False).loss)
    assert abs(total - float(got.loss)) <= 2 * U * abs(total) + (rows / 1000 + 1) * U * abs(total)


@pytest.mark.parametrize("rows", [1, 2, 300, 1500])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_many_wide_rows(rows, kind):
    """The same rows whatever the number of rows: few are shared among workgroups, many are not."""
    s = _inputs(rows, 5003, kind, 3, legal=True)
    got = _call(s)
    some = slice(0, min(rows, 12))
    part = {k: v if v is None else v[some] for k, v in s.items()}
    ref = _reference(part)
    sub = R.PolicyLoss(_call(part).loss, got.logp[some], got.entropy[some], got.kl[some], got.dlogits[some])
    _check(part, sub, ref)


@pytest.mark.parametrize("vocab", [5, 18, 300, 5001, 40000])
@pytest.mark.parametrize("ref,legal,weights,pad,ints", [(False, True, False, 0, torch.int32), (True, True, True, 1, torch.int64),
                                                       (False, False, True, 13, torch.int32)])
def test_options(vocab, ref, legal, weights, pad, ints):
    s = _inputs(14, vocab, "bf16", 4, ref, legal, weights, pad, ints)
    _check(s, _call(s), _reference(s))


@pytest.mark.parametrize("more", [dict(clip=0.0), dict(clip=(1.0, 5.0)), dict(kl_coef=0.0), dict(entropy_coef=0.0), dict(temperature=3.0),
                                  dict(kl_coef=0.0, entropy_coef=0.0, clip=0.1, temperature=1.0)])
@pytest.mark.parametrize("vocab", [18, 6000])
def test_hyperparameters(vocab, more):
    s = _inputs(21, vocab, "fp32", 5)
    _check(s, _call(s, **more), _reference(s, **more), **more)


def test_gradient_against_differences():
    """The gradient against central differences of the call's own loss, row by row (their logits do not meet): a step of 2^-6
    leaves (2^-6)^2 / 6 of the third derivative, which the softmax bounds by some 2 |slope|, and 2 u |loss| / 2^-5 of rounding."""
    s = _inputs(1, 9, "fp32", 6, weights=False)
    s["advantages"].fill_(0.7)
    got = _call(s).dlogits[0]
    h = 2.0 ** -6
    for j in range(9):
        keep = s["logits"][0, j].item()
        s["logits"][0, j] = keep + h
        up = float(_call(s, grad=False).loss)
        s["logits"][0, j] = keep - h
        down = float(_call(s, grad=False).loss)
        s["logits"][0, j] = keep
        assert abs((up - down) / (2 * h) - float(got[j])) <= 4 * h * h + 1e-4


@pytest.mark.parametrize("vocab", [6, 300, 9000, 60000])
@pytest.mark.parametrize("kind", sorted(TYPES))
def test_masked_places_hold_anything(vocab, kind):
    """NaN, infinities and the lowest value where an action is not legal change nothing; -inf as a logit is a probability of 0."""
    s = _inputs(12, vocab, kind, 7, legal=True)
    clean = _call(s)
    low = torch.finfo(TYPES[kind]).min
    for v in (float("nan"), float("inf"), float("-inf"), low):
        t = dict(s, logits=torch.where(s["legal"], s["logits"], torch.full_like(s["logits"], v)))
        got = _call(t)
        for p, q in zip(got, clean):
            assert torch.equal(p, q)
    t = dict(s, logits=torch.where(s["legal"], s["logits"], torch.full_like(s["logits"], float("-inf"))), legal=None)
    got = _call(t)
    for p, q in zip(got, clean):
        assert torch.equal(p, q)


@pytest.mark.parametrize("vocab", [6, 300, 9000, 60000])
def test_one_mask_for_all_rows(vocab):
    s = _inputs(9, vocab, "bf16", 17, legal=True)
    mask = s["legal"][0].clone()
    want = _call(dict(s, legal=mask.repeat(9, 1)))
    got = _call(dict(s, legal=mask.expand(9, -1)))
    for p, q in zip(got, want):
        assert torch.equal(p, q)


@pytest.mark.parametrize("vocab", [5, 3000])
@pytest.mark.parametrize("temperature", [1e-3, 1e4])
def test_far_temperatures(vocab, temperature):
    """Nearly certain and nearly uniform: the oracle's numbers up to an exponent's rounding, which grows with x = dz / temperature."""
    s = _inputs(6, vocab, "fp32", 18, ref=False)
    got, ref = _call(s, temperature=temperature), _reference(s, temperature=temperature)
    reach = float(s["logits"].abs().max()) * 2 / temperature
    assert np.all(np.abs(_np(got.logp) - ref[1]) <= 4 * U * reach + 1e-5)
    assert np.all(np.abs(_np(got.entropy) - ref[2]) <= 1e-4)
    assert torch.isfinite(got.dlogits).all()


@pytest.mark.parametrize("vocab", [6, 300, 9000, 60000])
def test_rows_left_out(vocab):
    """Padding, weight 0, an action that is not allowed, no allowed action at all: zeros, whatever the row's other numbers are."""
    s = _inputs(8, vocab, "fp32", 8, legal=True)
    s["legal"][:] = True
    s["legal"][3] = False
    s["legal"][5, s["actions"][5]] = False
    s["logits"][6, s["actions"][6]] = float("-inf")
    s["logits"][7] = float("-inf")
    nan = float("nan")
    for k in ("old_logp", "advantages", "ref_logp"):
        s[k][[1, 4]] = nan
    s["logits"][1] = nan
    got = _call(s)
    assert torch.isfinite(got.loss)
    for i in (1, 3, 4, 5, 6, 7):
        assert (got.dlogits[i] == 0).all() and got.logp[i] == 0 and got.entropy[i] == 0 and got.kl[i] == 0, i
    for i in (0, 2):
        assert got.logp[i] < 0 and (got.dlogits[i] != 0).any()
    part = {k: v if v is None else v[[0, 2]].contiguous() for k, v in s.items()}
    two = _call(part)
    assert torch.equal(two.dlogits, got.dlogits[[0, 2]]) or (two.dlogits - got.dlogits[[0, 2]]).abs().max() <= 1e-6
    assert abs(float(two.loss) - float(got.loss)) <= 2 * U * abs(float(two.loss)) + 1e-6 * 1e-2


@pytest.mark.parametrize("vocab", [6, 9000])
def test_what_is_wrong_is_seen(vocab):
    """An action beyond the last, a NaN logit, a NaN log-probability: NaN in the loss and that row, no other row touched."""
    for spoil in ("action", "logit", "old"):
        s = _inputs(6, vocab, "fp32", 9)
        clean = _call(s)
        if spoil == "action":
            s["actions"][3] = vocab
        elif spoil == "logit":
            s["logits"][3, 2] = float("nan")
        else:
            s["old_logp"][3] = float("nan")
        got = _call(s)
        assert torch.isnan(got.loss) and torch.isnan(got.dlogits[3]).any()
        keep = [0, 1, 2, 4, 5]
        assert torch.equal(got.dlogits[keep], clean.dlogits[keep]) and torch.equal(got.logp[keep], clean.logp[keep])


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("vocab", [5, 3000])
def test_far_apart_logits(vocab, kind):
    """A certain action (the others at the type's lowest value), all logits equal to the lowest, magnitudes of 1e4: finite."""
    s = _inputs(6, vocab, kind, 10, ref=False)
    low = torch.finfo(TYPES[kind]).min
    s["logits"][0] = low
    s["logits"][0, s["actions"][0]] = 0
    s["logits"][2] = low
    s["logits"][3] = (s["logits"][3].float() * 1e4).clamp(low, -low).to(TYPES[kind])
    got = _call(s)
    ref = _reference(s)
    assert torch.isfinite(got.dlogits[[0, 2]]).all() and float(got.logp[0]) == 0.0 and float(got.entropy[0]) == 0.0
    assert abs(float(got.logp[2]) + np.log(vocab)) <= 1e-5 and abs(float(got.entropy[2]) - np.log(vocab)) <= 1e-5
    np.testing.assert_allclose(_np(got.logp)[3], ref[1][3], rtol=4 * U, atol=1e-5)


@pytest.mark.parametrize("vocab,rows", [(7, 40), (700, 5), (9000, 3), (60000, 2), (9000, 900)])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_gradient_over_the_logits(vocab, rows, kind):
    """out=logits and out=a slice of a wider buffer give the same bits; what lies around the slice stays."""
    s = _inputs(rows, vocab, kind, 11, legal=True, pad=5)
    want = _call(s)
    room = torch.full((rows, vocab + 9), 7.0, dtype=TYPES[kind], device="cuda")
    got = _call(s, out=room[:, 4:4 + vocab])
    assert torch.equal(got.dlogits, want.dlogits) and (room[:, :4] == 7).all() and (room[:, 4 + vocab:] == 7).all()
    got = _call(s, out=s["logits"])
    assert got.dlogits.data_ptr() == s["logits"].data_ptr()
    for p, q in zip(got, want):
        assert torch.equal(p, q)


@pytest.mark.parametrize("vocab", [18, 5000, 90000])
def test_rows_far_apart(vocab):
    """Offsets that pass 32 bits: rows of a buffer of more than 2^32 elements, gradient over the logits.  Which thread holds a column, and
    with it the order of a row's sums, follows from where the row begins within 16 bytes: the same bits are those of near rows that begin
    alike."""
    s = _inputs(3, vocab, "bf16", 21, legal=True)
    room = torch.empty((1 << 32) + (1 << 17), dtype=torch.bfloat16, device="cuda")
    far = room.as_strided((3, vocab), (1 << 31, 1), 5)
    far.copy_(s["logits"])
    ld = (vocab + 7) // 8 * 8
    near = torch.empty(3 * ld + 8, dtype=torch.bfloat16, device="cuda").as_strided((3, vocab), (ld, 1), 5)
    near.copy_(s["logits"])
    want = _call(dict(s, logits=near))
    got = _call(dict(s, logits=far), out=far)
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    _check(s, got, _reference(s))


def test_no_rows():
    s = {k: v if v is None else v[:0] for k, v in _inputs(3, 8, "fp32", 12).items()}
    got = _call(s)
    assert float(got.loss) == 0 and got.dlogits.shape == (0, 8) and got.logp.shape == (0,)


@pytest.mark.parametrize("rows,vocab", [(500, 18), (3, 40000), (3, 90000), (700, 3001)])
def test_captured_graphs_and_streams(rows, vocab):
    """Two captured graphs and eager calls in turn: every replay gives the eager result on the inputs of its time."""
    a, b = _inputs(rows, vocab, "fp32", 13), _inputs(rows, vocab, "bf16", 14, legal=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _call(a), _call(b)
    stream.synchronize()
    graphs, outs = [], []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(_call(s))
        graphs.append(g)
    for turn in range(3):
        for s in (a, b):
            s["advantages"].mul_(-1.5)
            s["logits"].mul_(0.75)
        for g in graphs:
            g.replay()
        want = [_call(s) for s in (a, b)]
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            for p, q in zip(got, ref):
                assert torch.equal(p, q), turn


def test_same_bits_every_time():
    s = _inputs(2000, 900, "bf16", 15)
    first = _call(s)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, _call(s)))


def test_refusals():
    s = _inputs(5, 8, "fp32", 16, legal=True)
    z = s["logits"]
    bad = [
        dict(logits=z.double()), dict(logits=z.cpu()), dict(logits=z[0]), dict(logits=z.t()), dict(logits=z[:1].expand(5, 8)),
        dict(actions=s["actions"].float()), dict(actions=s["actions"][:4]), dict(actions=s["actions"].cpu()),
        dict(old_logp=s["old_logp"].double()), dict(old_logp=None), dict(advantages=s["advantages"][:, None]), dict(advantages=None),
        dict(weights=s["weights"][:2]), dict(ref_logp=s["ref_logp"].half()), dict(legal=s["legal"].float()), dict(legal=s["legal"][:, :4]),
        dict(legal=s["legal"].t().contiguous().t()), dict(legal=s["legal"].cpu()),
    ]
    for change in bad:
        with pytest.raises(ValueError):
            _call({**s, **change})
            raise AssertionError(f"{list(change)} was taken")
    wide = torch.empty(5, 16, device="cuda")
    for more in (dict(clip=-0.1), dict(clip=(1.5, 0.2)), dict(temperature=0.0), dict(temperature=float("nan")), dict(out=z.half()),
                 dict(out=z[:, 1:]), dict(out=torch.empty(1, 8, device="cuda").expand(5, 8)), dict(out=wide.t()[:8].t()[:, :7]),
                 dict(grad=False, out=torch.empty_like(z))):
        with pytest.raises(ValueError):
            _call(s, **more)
            raise AssertionError(f"{more} was taken")
