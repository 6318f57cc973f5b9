"""The recurrent policy's oracle against itself: its gradients against central differences, and the 8-bit floats against a search
of every value that a code can stand for."""
import numpy as np
import pytest

from oracle import recurrent_policy as O


def _differences(f, x, h=1e-6):
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        keep = x[i]
        x[i] = keep + h
        up = f()
        x[i] = keep - h
        g[i] = (up - f()) / (2 * h)
        x[i] = keep
    return g


@pytest.mark.parametrize("masked", [False, True])
def test_scan_gradient_against_differences(masked):
    rng = np.random.RandomState(0)
    b, n, d = 3, 6, 2
    z, x, s, dh, ds = rng.randn(b, n, d), rng.randn(b, n, d), rng.randn(b, d), rng.randn(b, n, d), rng.randn(b, d)
    starts = (rng.rand(b, n) < 0.3) if masked else None
    lengths = np.array([0, 4, 6]) if masked else None

    def value():
        h, last = O.gated_scan(z, x, s, starts, lengths)
        return (h * dh).sum() + (last * ds).sum()
    h, _ = O.gated_scan(z, x, s, starts, lengths)
    got = O.gated_scan_backward(dh, z, x, h, s, starts, lengths, ds)
    for g, v in zip(got, (z, x, s)):
        # central differences: O(h^2) = 1e-12 of the third derivative, 1e-16 / 1e-6 = 1e-10 of rounding
        np.testing.assert_allclose(g, _differences(value, v), rtol=0, atol=1e-8)


@pytest.mark.parametrize("legal", [False, True])
def test_policy_gradient_against_differences(legal):
    rng = np.random.RandomState(1)
    rows, vocab = 7, 5
    z = rng.randn(rows, vocab)
    mask = rng.rand(rows, vocab) > 0.3 if legal else None
    a = rng.randint(0, vocab, rows)
    a[2] = -1
    w = rng.rand(rows)
    w[4] = 0
    adv, old, ref = rng.randn(rows), rng.randn(rows) * 0.3 - 1.5, rng.randn(rows) * 0.3 - 1.5
    call = lambda: O.policy_loss(z, a, old, adv, w, ref, mask, (0.3, 0.4), 0.2, 0.1, 0.8)
    np.testing.assert_allclose(call()[4], _differences(lambda: call()[0], z), rtol=0, atol=1e-8)


@pytest.mark.parametrize("signed", [False, True])
def test_round8_is_the_nearest_code(signed):
    rng = np.random.RandomState(2)
    v = np.exp(rng.randn(20, 64) * 3) * (np.sign(rng.randn(20, 64)) if signed else 1)
    v[3, :60] = 0
    steps, count = (8, 127) if signed else (16, 255)
    for row, got in zip(v, O.round8(v.ravel(), signed).reshape(v.shape)):
        top = np.abs(got).max()
        octave = np.floor(np.log2(top))
        values = np.array([(1 + (k % steps) / steps) * 2.0 ** (octave + k // steps) for k in range(steps - count, steps)])
        for x, y in zip(row, got):
            if x == 0:
                assert y == 0
                continue
            best = values[np.argmin(np.abs(values - abs(x)))]
            if abs(x) < values[0]:
                assert abs(y) in ((0.0, values[0]) if signed else (values[0],))
            else:
                assert abs(abs(y) - abs(x)) <= abs(best - abs(x)) * (1 + 1e-12)
                assert abs(y - x) <= abs(x) / (2 * steps)
