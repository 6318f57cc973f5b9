"""float64 NumPy restatement of the recurrent policy's operators: the gated linear recurrence step by step with its gradient, the
clipped policy loss row by row with its gradient, and AdamW with moments in 64 bits or rounded to the 8-bit floats of its
compact state.  Test infrastructure only."""
import numpy as np


# ---- gated linear recurrence -----------------------------------------------------------------------------
def sigmoid(z):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z))


def gated_scan(z, x, state, starts=None, lengths=None):
    z, x = np.asarray(z, np.float64), np.asarray(x, np.float64)
    b, n, d = z.shape
    s = np.array(state, np.float64) if state is not None else np.zeros((b, d))
    h = np.zeros((b, n, d))
    for i in range(b):
        for t in range(n if lengths is None else min(max(int(lengths[i]), 0), n)):
            p = np.zeros(d) if starts is not None and starts[i, t] else s[i]
            s[i] = sigmoid(z[i, t]) * p + sigmoid(-z[i, t]) * x[i, t]
            h[i, t] = s[i]
    return h, s


def gated_scan_backward(dh, z, x, h, state, starts=None, lengths=None, dstate=None):
    """h: what the forward pass returned (its rounding included)."""
    dh, z, x, h = (np.asarray(v, np.float64) for v in (dh, z, x, h))
    b, n, d = z.shape
    c = np.array(dstate, np.float64) if dstate is not None else np.zeros((b, d))
    dz, dx = np.zeros((b, n, d)), np.zeros((b, n, d))
    for i in range(b):
        for t in reversed(range(n if lengths is None else min(max(int(lengths[i]), 0), n))):
            start = starts is not None and starts[i, t]
            before = h[i, t - 1] if t else (np.asarray(state, np.float64)[i] if state is not None else np.zeros(d))
            p = np.zeros(d) if start else before
            f, take = sigmoid(z[i, t]), sigmoid(-z[i, t])
            g = c[i] + dh[i, t]
            dx[i, t], dz[i, t] = take * g, g * (p - x[i, t]) * f * take
            c[i] = 0.0 if start else f * g
    return dz, dx, c


# ---- clipped policy loss -------------------------------------------------------------------------------------
def policy_loss(logits, actions, old_logp, advantages, weights=None, ref_logp=None, legal=None, clip=(0.2, 0.2), kl_coef=0.0,
                entropy_coef=0.0, temperature=1.0):
    """loss, logp, entropy, kl, dlogits"""
    z = np.array(logits, np.float64)
    rows, vocab = z.shape
    if legal is not None:
        z[~np.asarray(legal, bool)] = -np.inf
    w = np.full(rows, 1.0 / rows) if weights is None else np.asarray(weights, np.float64)
    loss, logp, entropy, kl, d = 0.0, np.zeros(rows), np.zeros(rows), np.zeros(rows), np.zeros((rows, vocab))
    for i in range(rows):
        a = int(actions[i])
        if a < 0 or w[i] == 0:
            continue
        if a >= vocab:
            loss, logp[i], entropy[i], kl[i], d[i] = np.nan, np.nan, np.nan, np.nan, np.nan
            continue
        if z[i, a] == -np.inf:
            continue
        with np.errstate(invalid="ignore", divide="ignore"):
            u = (z[i] - z[i].max()) / temperature
            lp = u - np.log(np.exp(u).sum())
            p = np.exp(lp)
            terms = np.where(p > 0, p * np.where(p > 0, lp, 0.0), p)
        h = -terms.sum()
        r, adv = np.exp(lp[a] - float(old_logp[i])), float(advantages[i])
        low, high = 1 - clip[0], 1 + clip[1]
        held = min(max(r, low), high)
        clipped = r * adv > held * adv
        slope = 0.0 if clipped else -r * adv
        row = -(held if clipped else r) * adv - entropy_coef * h
        if ref_logp is not None:
            q = float(ref_logp[i]) - lp[a]
            kl[i] = np.expm1(q) - q
            row += kl_coef * kl[i]
            slope -= kl_coef * np.expm1(q)
        loss += w[i] * row
        logp[i], entropy[i] = lp[a], h
        d[i] = -slope * p + entropy_coef * (terms + p * h)
        d[i, a] += slope
        d[i] *= w[i] / temperature
    return loss, logp, entropy, kl, d


# ---- AdamW -----------------------------------------------------------------------------------------------------
BLOCK = 64


def round8(v, signed):
    """The values that 8 bits hold of v [blocks * 64]: 3 (signed) or 4 mantissa bits, ties to even; the octave of a block's
    largest rounded magnitude is the top one, 127 or 255 magnitudes count down from its end; under them 0, or for the unsigned
    ones the smallest magnitude.  What a float32 holds as no normal number counts as 0."""
    steps, count = (8, 127) if signed else (16, 255)
    v = np.asarray(v, np.float64).reshape(-1, BLOCK)
    frac, e = np.frexp(np.abs(v))
    near = np.ldexp(np.rint(frac * 2 * steps) / (2 * steps), e)
    near[near < 2.0 ** -126] = 0
    out = np.zeros_like(v)
    for i, row in enumerate(near):
        if not np.all(np.isfinite(row)) or row.max() >= 2.0 ** 128:
            out[i] = np.nan
            continue
        if row.max() == 0:
            continue
        octave = np.frexp(row.max())[1] - 1
        f, ex = np.frexp(row)
        place = (ex - 1 - octave) * steps + np.rint((f * 2 - 1) * steps).astype(int) - (steps - 1) + count
        below = steps - count
        least = np.ldexp(1 + (below % steps) / steps, octave + below // steps)
        kept = np.where(place >= 1, row, 0.0 if signed else least if least >= 2.0 ** -126 else 0.0)
        out[i] = np.where(row > 0, kept, 0.0) * np.sign(v[i])
    return out.reshape(-1)


def adamw_step(p, g, m, v, t, lr, betas, eps, decay, bits, scale=1.0):
    """One step of flat arrays (m and v of 64-element blocks where bits is 8, as values); t counts from 1.  Returns p, m, v."""
    p, g = np.asarray(p, np.float64), np.asarray(g, np.float64) * np.float64(scale)
    m = np.asarray(m, np.float64) * betas[0] + g * (1 - betas[0])
    v = np.asarray(v, np.float64) * betas[1] + g * (1 - betas[1]) * g
    move = (m / (1 - betas[0] ** t)) / (np.sqrt(v / (1 - betas[1] ** t)) + eps)
    p = p * (1 - lr * decay) - lr * move
    if bits == 8:
        m = round8(m, True)
        v = np.square(round8(np.sqrt(v), False).astype(np.float32)).astype(np.float64)
    return p, m, v
