"""The gated linear recurrence (`gated_scan`, `gated_scan_backward`, `gated_step`, `GatedUnit`) against the float64 oracle.

Tolerances.  With u = 2^-24 a step h = p + take (x - p) rounds three times and takes a gate that is off by at most some 8 u of
itself, so a step adds at most 3 u max(|h|, |x|) + 8 u |x - p| to the error, which later steps multiply by f <= 1; where the
time axis is cut, the factor of a span of T steps is off by at most 10 T u.  Together at most (13 T + 32) u of the largest
magnitude among h, x and the state: loose, but an arithmetic bound.  The same holds for the backward recurrence with the largest
g, and dz has a factor |p - x| / 4 more.  An output in 16 bits is off by half a step of its type on top."""
import numpy as np
import pytest
import torch

import rl_gan_amd as R
from oracle import recurrent_policy as O

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, ref, bound, dtype, what):
    """|got - ref| <= bound + half a step of dtype at ref (and half of its smallest step)"""
    got = _np(got)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    if dtype == torch.float32:
        tol = bound + U * np.abs(ref)
    else:
        tol = bound * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).eps / 2 * (np.abs(ref) + bound) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:3], ref[bad][:3], float(np.max(bound)))


def _inputs(b, n, d, kind, layout, seed, starts=False, lengths=False, reach=2.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    t = TYPES[kind]
    rnd = lambda *s: torch.randn(*s, generator=g)

    def place(v):
        """The values of v [b, n, d] on the GPU in one of the layouts a caller may have."""
        v = v.to(t)
        if layout == "fused":
            both = torch.full((b, n, 2 * d), float("nan"), dtype=t)
            both[..., d:] = v
            return both.cuda()[..., d:]
        if layout == "time":
            return v.transpose(0, 1).contiguous().cuda().transpose(0, 1)
        if layout == "odd":                                     # rows that begin at any element
            wide = torch.full((b, n, d + 3), float("nan"), dtype=t)
            wide[..., 1:d + 1] = v
            return wide.cuda()[..., 1:d + 1]
        return v.cuda()
    s = {"z": place(rnd(b, n, d) * 1.5 + reach), "x": place(rnd(b, n, d)), "state": rnd(b, d).cuda(), "dh": place(rnd(b, n, d)),
         "dstate": rnd(b, d).cuda(), "starts": None, "lengths": None}
    if starts:
        s["starts"] = (torch.rand(b, n, generator=g) < 0.1).cuda()
    if lengths:
        s["lengths"] = torch.randint(-1, n + 2, (b,), generator=g, dtype=torch.int32)   # outside 0 .. n: clamped
        s["lengths"][0], s["lengths"][-1] = (0, n) if b > 1 else (n, n)
        s["lengths"] = s["lengths"].cuda()
    return s


def _host(v):
    return None if v is None else v.cpu().numpy()


def _check(s, kind):
    dtype, n = TYPES[kind], s["z"].shape[1]
    a = (_np(s["z"]), _np(s["x"]))
    st, ln = _host(s["starts"]), _host(s["lengths"])
    h, last = R.gated_scan(s["z"], s["x"], s["state"], starts=s["starts"], lengths=s["lengths"])
    rh, rlast = O.gated_scan(*a, _np(s["state"]), st, ln)
    top = max(1.0, np.abs(_np(s["state"])).max(), np.abs(a[1]).max())
    step = (13 * n + 32) * U
    assert h.dtype == dtype and last.dtype == torch.float32
    _close(h, rh, step * top, dtype, "h")
    _close(last, rlast, step * top, torch.float32, "state")
    dz, dx, ds = R.gated_scan_backward(s["dh"], s["z"], s["x"], h, s["state"], starts=s["starts"], lengths=s["lengths"], dstate=s["dstate"])
    rz, rx, rs = O.gated_scan_backward(_np(s["dh"]), *a, _np(h), _np(s["state"]), st, ln, _np(s["dstate"]))
    # |g| <= |dstate| + sum of f products |dh|: from dx, which is (1 - f) g, and the carry
    take = O.sigmoid(-a[0])
    with np.errstate(invalid="ignore"):                         # 0 / 0 at a gate of exactly 1
        g = np.abs(rx) / take
    big = max(1.0, np.nanmax(g), np.abs(_np(s["dstate"])).max())
    _close(dx, rx, step * big, dtype, "dx")
    _close(dz, rz, step * big * 2 * top, dtype, "dz")
    _close(ds, rs, step * big, torch.float32, "dstate_in")
    return h, last, dz, dx, ds


SHAPES = [(1, 1, 1), (1, 2, 3), (3, 17, 5), (2, 64, 64), (5, 65, 200), (1, 1025, 96), (4, 130, 130), (64, 7, 256), (9, 33, 66)]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("b,n,d", SHAPES)
def test_shapes(b, n, d, kind):
    _check(_inputs(b, n, d, kind, "plain", 1), kind)


@pytest.mark.parametrize("layout", ["plain", "fused", "time", "odd"])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("starts,lengths", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("b,n,d", [(3, 70, 12), (6, 261, 65)])
def test_masks_and_layouts(b, n, d, starts, lengths, kind, layout):
    _check(_inputs(b, n, d, kind, layout, 2, starts, lengths), kind)


@pytest.mark.parametrize("b,n,d,kind", [(1, 6001, 8, "fp32"), (2, 5003, 33, "bf16"), (1, 9000, 130, "fp16"), (3, 2049, 512, "bf16"),
                                        (40, 1100, 64, "fp32")])
@pytest.mark.parametrize("masked", [False, True])
def test_long_sequences(b, n, d, kind, masked):
    """Few units and many steps: the time axis is cut."""
    _check(_inputs(b, n, d, kind, "plain", 3, masked, masked, reach=3.0), kind)


@pytest.mark.parametrize("b,n,d,kind,masked", [(1, 11001, 2048, "fp32", False), (3, 7000, 1111, "fp32", True), (2, 12100, 2000, "bf16", True)])
def test_long_and_large(b, n, d, kind, masked):
    """Few units, many steps and more than the caches hold: workgroups hand maps and states on along the time axis.  (The widths are
    large for the oracle's sake, which walks the steps one by one.)"""
    _check(_inputs(b, n, d, kind, "plain", 16, masked, masked, reach=3.0), kind)


@pytest.mark.parametrize("b,n,d,kind", [(700, 12, 300, "bf16"), (1024, 9, 301, "fp32"), (1500, 31, 256, "fp16"), (1024, 33, 256, "fp32")])
def test_many_units(b, n, d, kind):
    _check(_inputs(b, n, d, kind, "fused", 4, True, True), kind)


def test_extreme_gates():
    """z of +-inf and of the types' largest magnitudes: f is exactly 1 or 0, and nothing is NaN."""
    for kind, t in TYPES.items():
        s = _inputs(2, 40, 8, kind, "plain", 5)
        big = torch.finfo(t).max
        s["z"][:, 3::7], s["z"][:, 5::11], s["z"][0, 8], s["z"][1, 9] = big, -big, float("inf"), float("-inf")
        h = _check(s, kind)[0]
        assert torch.isfinite(h).all()
        # with f = 1 the state stays: both steps hold the same exact value, each within the bound above of it (the second one may
        # begin a span, whose state comes from the maps before it), and for 16 bits they may round to neighbours
        top = max(1.0, float(h.abs().max()))
        assert (h[0, 8].float() - h[0, 7].float()).abs().max() <= (2 * (13 * 40 + 32) * U + torch.finfo(t).eps) * top


@pytest.mark.parametrize("n,d", [(40, 20), (3000, 20), (40000, 200)])
def test_nothing_passes_a_start_or_an_end(n, d):
    """NaN in the state, in an episode before, and behind a sequence's end reaches neither outputs nor gradients."""
    b = 3
    s = _inputs(b, n, d, "fp32", "plain", 6, reach=3.0)
    s["starts"] = torch.zeros(b, n, dtype=torch.bool, device="cuda")
    s["starts"][0, 0] = True
    s["starts"][1, n // 2] = True
    s["lengths"] = torch.tensor([n, n, n // 3], dtype=torch.int32, device="cuda")
    clean = R.gated_scan(s["z"], s["x"], s["state"], starts=s["starts"], lengths=s["lengths"])
    grads = R.gated_scan_backward(s["dh"], s["z"], s["x"], clean[0], s["state"], starts=s["starts"], lengths=s["lengths"], dstate=s["dstate"])
    nan = float("nan")
    s["state"][0] = nan
    s["x"][1, n // 2 - 3] = nan
    for k in ("x", "z", "dh"):
        s[k][2, n // 3:] = nan
    h, last = R.gated_scan(s["z"], s["x"], s["state"], starts=s["starts"], lengths=s["lengths"])
    assert torch.equal(h[0], clean[0][0]) and torch.equal(h[2], clean[0][2]) and torch.equal(last, clean[1])
    assert torch.equal(h[1, n // 2:], clean[0][1, n // 2:]) and torch.isnan(h[1, n // 2 - 3:n // 2]).all()
    assert (h[2, n // 3:] == 0).all()
    dz, dx, ds = R.gated_scan_backward(s["dh"], s["z"], s["x"], h, s["state"], starts=s["starts"], lengths=s["lengths"], dstate=s["dstate"])
    assert torch.equal(dx[0], grads[1][0]) and torch.equal(dz[0], grads[0][0]) and (ds[0] == 0).all()
    assert torch.equal(dx[2], grads[1][2]) and torch.equal(dz[2], grads[0][2]) and torch.equal(ds[2], grads[2][2])
    assert torch.equal(dz[1, n // 2:], grads[0][1, n // 2:]) and torch.equal(dx[1], grads[1][1])
    assert (dz[2, n // 3:] == 0).all() and (dx[2, n // 3:] == 0).all()


@pytest.mark.parametrize("n", [5, 4000, 1000000])
def test_absent_state_and_gradient_are_zeros(n):
    s = _inputs(2, n, 12, "fp32", "plain", 7)
    zero = torch.zeros_like(s["state"])
    a, b = R.gated_scan(s["z"], s["x"]), R.gated_scan(s["z"], s["x"], zero)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ga = R.gated_scan_backward(s["dh"], s["z"], s["x"], a[0])
    gb = R.gated_scan_backward(s["dh"], s["z"], s["x"], a[0], zero, dstate=zero)
    assert all(torch.equal(p, q) for p, q in zip(ga, gb))


def test_a_sequence_in_pieces():
    """The state handed on: two calls give what one gives, up to where their tiles begin."""
    s = _inputs(3, 500, 40, "fp32", "plain", 8)
    h, last = R.gated_scan(s["z"], s["x"], s["state"])
    h1, mid = R.gated_scan(s["z"][:, :201], s["x"][:, :201], s["state"])
    h2, end = R.gated_scan(s["z"][:, 201:], s["x"][:, 201:], mid)
    tol = (13 * 500 + 32) * U * 5
    assert (torch.cat([h1, h2], 1) - h).abs().max() <= tol and (end - last).abs().max() <= tol


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("b,d", [(1, 1), (3, 7), (4096, 256), (5, 1000), (33, 66)])
def test_step(b, d, kind):
    s = _inputs(b, 3, d, kind, "fused", 9, starts=True)
    state = s["state"].clone()
    ref_h, ref_s = O.gated_scan(_np(s["z"]), _np(s["x"]), _np(s["state"]), _host(s["starts"]))
    for t in range(3):
        h = R.gated_step(s["z"][:, t], s["x"][:, t], state, starts=s["starts"][:, t])
        _close(h, ref_h[:, t], 80 * U * 6, TYPES[kind], f"h at step {t}")
    _close(state, ref_s, 80 * U * 6, torch.float32, "state")


@pytest.mark.parametrize("n", [1, 3, 2000])
def test_no_elements(n):
    e = torch.empty(0, n, 5, device="cuda")
    h, s = R.gated_scan(e, e)
    assert h.shape == (0, n, 5) and s.shape == (0, 5)
    z = torch.zeros(2, 0, 5, device="cuda")
    st = torch.randn(2, 5, device="cuda")
    h, s = R.gated_scan(z, z, st)
    assert h.shape == (2, 0, 5) and torch.equal(s, st) and s.data_ptr() != st.data_ptr()
    dz, dx, ds = R.gated_scan_backward(z, z, z, z, st, dstate=st)
    assert dz.shape == (2, 0, 5) and torch.equal(ds, st)


def test_outputs_in_the_callers_buffers():
    """dz and dx as the halves of one buffer, h in a slice: what lies around them stays."""
    for n in (30, 3000):
        s = _inputs(2, n, 24, "bf16", "plain", 10, starts=True)
        room = torch.full((2, n, 40), 7.0, dtype=torch.bfloat16, device="cuda")
        ref = R.gated_scan(s["z"], s["x"], s["state"], starts=s["starts"])
        h, _ = R.gated_scan(s["z"], s["x"], s["state"], starts=s["starts"], out=room[..., 5:29])
        assert torch.equal(h, ref[0]) and (room[..., :5] == 7).all() and (room[..., 29:] == 7).all()
        both = torch.full((2, n, 48), 7.0, dtype=torch.bfloat16, device="cuda")
        a = R.gated_scan_backward(s["dh"], s["z"], s["x"], h, s["state"], starts=s["starts"])
        b = R.gated_scan_backward(s["dh"], s["z"], s["x"], h, s["state"], starts=s["starts"], out=(both[..., :24], both[..., 24:]))
        assert torch.equal(a[0], b[0]) and torch.equal(both[..., :24], a[0]) and torch.equal(both[..., 24:], a[1])


@pytest.mark.parametrize("n", [9, 5000, 360000])
def test_captured_graphs_and_streams(n):
    """Two captured graphs and eager calls in turn, on a stream of their own: every replay gives the eager result."""
    a, b = _inputs(2, n, 32, "fp32", "plain", 11, True, True), _inputs(3, n, 20, "bf16", "plain", 12)

    def both(s):
        h, last = R.gated_scan(s["z"], s["x"], s["state"], starts=s["starts"], lengths=s["lengths"])
        return (h, last) + R.gated_scan_backward(s["dh"], s["z"], s["x"], h, s["state"], starts=s["starts"], lengths=s["lengths"],
                                                 dstate=s["dstate"])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        both(a), both(b)
    stream.synchronize()
    graphs, outs = [], []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(both(s))
        graphs.append(g)
    for turn in range(3):
        for s in (a, b):
            s["x"].add_(0.25)
        for g in graphs:
            g.replay()
        want = [both(s) for s in (a, b)]
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            for p, q in zip(got, ref):
                assert torch.equal(p, q), turn


def test_two_streams_at_once():
    """Long scans on two streams at the same time: workgroups of both wait and go on among each other."""
    a, b = _inputs(2, 250000, 48, "fp32", "plain", 17), _inputs(1, 400000, 64, "fp32", "plain", 18)
    want = [R.gated_scan(s["z"], s["x"], s["state"]) for s in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for turn in range(4):
        for s, stream in zip((a, b), streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append(R.gated_scan(s["z"], s["x"], s["state"]))
    torch.cuda.synchronize()
    for i, (h, last) in enumerate(got):
        assert torch.equal(h, want[i % 2][0]) and torch.equal(last, want[i % 2][1])


def test_rows_far_apart():
    """Offsets that pass 32 bits: rows and steps of a buffer of more than 2^32 elements, forward and backward."""
    b, n, d = 2, 70, 64
    room = torch.empty((1 << 31) + (1 << 21), dtype=torch.bfloat16, device="cuda")
    s = _inputs(b, n, d, "bf16", "plain", 15, starts=True)
    want = R.gated_scan(s["z"], s["x"], s["state"], starts=s["starts"])
    wantb = R.gated_scan_backward(s["dh"], s["z"], s["x"], want[0], s["state"], starts=s["starts"], dstate=s["dstate"])
    for strides in ((1 << 31, 128, 1), (128, 31117312, 1)):       # batch rows, then steps, far apart
        z, x = room.as_strided((b, n, d), strides), room.as_strided((b, n, d), strides, 64)
        z.copy_(s["z"])
        x.copy_(s["x"])
        got = R.gated_scan(z, x, s["state"], starts=s["starts"])
        gotb = R.gated_scan_backward(s["dh"], z, x, want[0], s["state"], starts=s["starts"], dstate=s["dstate"])
        for p, q in zip(got + gotb, want + wantb):
            assert torch.equal(p, q)


@pytest.mark.parametrize("n", [7000, 250000])
def test_same_bits_every_time(n):
    """Whatever order the workgroups of a long sequence come in."""
    s = _inputs(2, n, 48, "fp32", "plain", 13, reach=4.0)
    call = lambda h: R.gated_scan(s["z"], s["x"], s["state"]) + R.gated_scan_backward(s["dh"], s["z"], s["x"], h, s["state"], dstate=s["dstate"])
    first = call(R.gated_scan(s["z"], s["x"], s["state"])[0])
    for _ in range(5):
        assert all(torch.equal(p, q) for p, q in zip(first, call(first[0])))


def test_gated_unit_against_autograd():
    """The layer (dense product, recurrence, both gradients) against torch's float64 autograd of the same formulas."""
    rng = np.random.RandomState(3)
    b, n, k, units = 3, 23, 12, 8
    layer = R.GatedUnit(k, units, rng=rng)
    x = torch.randn(b, n, k, device="cuda")
    state = torch.randn(b, units, device="cuda")
    starts = torch.rand(b, n, device="cuda") < 0.15
    dh, ds = torch.randn(b, n, units, device="cuda"), torch.randn(b, units, device="cuda")
    h, last = layer.forward(x, state, starts)
    dx, dstate = layer.backward(dh, ds)
    w = layer.gates.canon.double().cpu().requires_grad_()
    xr, sr = x.double().cpu().requires_grad_(), state.double().cpu().requires_grad_()
    gates = xr @ w[:k * 2 * units].view(k, 2 * units) + w[k * 2 * units:]
    f, s, hs = torch.sigmoid(gates[..., :units]), sr, []
    for t in range(n):
        s = f[:, t] * torch.where(starts[:, t, None].cpu(), torch.zeros_like(s), s) + (1 - f[:, t]) * gates[:, t, units:]
        hs.append(s)
    hr = torch.stack(hs, 1)
    ((hr * dh.double().cpu()).sum() + (s * ds.double().cpu()).sum()).backward()
    for got, ref in ((h, hr), (last, s), (dx, xr.grad), (dstate, sr.grad), (layer.gates.grad, w.grad)):
        ref = ref.detach().numpy()
        # products of 12 to 69 terms of magnitude up to some 10, then the scan's bound
        assert np.abs(_np(got) - ref).max() <= 1e-5 * max(1.0, np.abs(ref).max())
    step_state = state.clone()
    for t in range(3):
        ht = layer.step(x[:, t], step_state, starts[:, t])
        assert np.abs(_np(ht) - hr[:, t].detach().numpy()).max() <= 1e-5 * 10


def test_refusals():
    s = _inputs(2, 6, 8, "fp32", "plain", 14)
    z, x, st, dh = s["z"], s["x"], s["state"], s["dh"]
    h, _ = R.gated_scan(z, x, st)
    bad = [
        lambda: R.gated_scan(z.double(), x.double()),
        lambda: R.gated_scan(z, x.bfloat16()),
        lambda: R.gated_scan(z, x[:, :5]),
        lambda: R.gated_scan(z[0], x[0]),
        lambda: R.gated_scan(z.cpu(), x),
        lambda: R.gated_scan(z, x.cpu()),
        lambda: R.gated_scan(z.transpose(1, 2), x.transpose(1, 2)),
        lambda: R.gated_scan(z, x, st.bfloat16()),
        lambda: R.gated_scan(z, x, st[:1]),
        lambda: R.gated_scan(z, x, st.t().contiguous().t()),
        lambda: R.gated_scan(z, x, st, starts=torch.zeros(2, 5, dtype=torch.bool, device="cuda")),
        lambda: R.gated_scan(z, x, st, starts=torch.zeros(2, 6, device="cuda")),
        lambda: R.gated_scan(z, x, st, lengths=torch.zeros(2, dtype=torch.int64, device="cuda")),
        lambda: R.gated_scan(z, x, st, lengths=torch.zeros(2, dtype=torch.int32)),
        lambda: R.gated_scan(z, x, st, out=z),
        lambda: R.gated_scan(z, x, st, out=torch.empty(1, 6, 8, device="cuda").expand(2, 6, 8)),
        lambda: R.gated_scan(z, x, st, out=torch.empty(2, 6, 8, device="cuda", dtype=torch.float16)),
        lambda: R.gated_scan_backward(dh, z, x, h[:, :3], st),
        lambda: R.gated_scan_backward(dh, z, x, h, st, dstate=st.double()),
        lambda: R.gated_scan_backward(dh, z, x, h, st, out=(dh, torch.empty_like(z))),
        lambda: R.gated_scan_backward(dh, z, x, h, st, out=(lambda t: (t, t))(torch.empty_like(z))),
        lambda: R.gated_step(z[:, 0], x[:, 0], st.half()),
        lambda: R.gated_step(z[:, 0], x[:, 0], None),
        lambda: R.gated_step(z, x, st),
        lambda: R.gated_step(st, x[:, 0], st),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was taken")
