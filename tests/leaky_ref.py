"""Plain 64-bit forms of the token drive and the leaky scan, with bounds on what
32-bit arithmetic may be off by.

A value that is a sum of terms, each a product of some factors, is computed in
32 bits within U = 2^-24 (half a step of f32) per rounding that a term passes.
For the scan a term u_s of h_t is u_s times the decays of t - s steps, so with
    H_t = |a| H_{t-1} + |u_t|             (the sum of the terms' magnitudes)
    J_t = |a| (J_{t-1} + H_{t-1})         (each times its number of steps)
the error of h_t is at most U (K1 H_t + K2 J_t).  K2, the roundings of a step:
the two of the recurrence, the first of them on h + u where the result may be
half as large (3 units), one of the product of decays that joins spans (1), and
the decay itself: exact when given, 8 units for expf (2 ulp) and the division of
the f32 form, 25 for the short exponential and reciprocal of the 16-bit forms
(argument rounded at |z| log2(e) <= 17.4 for |z| <= 12, 2 ulp each for exp and
reciprocal); times s / (1 - s) <= 1.  K1 adds the input's factor and the joins.
Results are then rounded once more to their own type, by at most half a step."""
import numpy as np

U = 2.0 ** -24
K1, K2 = 40.0, {"f32": 16.0, "bf16": 32.0, "f16": 32.0}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
LEAST = {"f32": 2.0 ** -149, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}  # half the smallest subnormal, at most


def close(got, want, bound, kind, what=""):
    """|got - want| <= bound + the rounding to `kind`; NaN and infinities in the same places.  A bound is at
    least U K1 times the magnitudes that pass through a value: where those exceed f32 (3.4e38: gates below -1 or
    above 1 over many steps) an f32 computation overflows on the way, and nothing is compared."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    bound = np.broadcast_to(np.asarray(bound, np.float64), want.shape)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fits = bound < 3.4e38 * U * K1
    got, want, bound = got[fits], want[fits], bound[fits]
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True), what
    if not fine.any():
        return
    off = np.abs(got[fine] - want[fine])
    most = bound[fine] * (1 + 2.0 ** -8) + np.abs(want[fine]) * HALF_STEP[kind] + LEAST[kind]
    if not (off <= most).all():
        k = int(np.nanargmax(np.where(np.isfinite(off), off / most, np.inf)))
        raise AssertionError(f"{what}: off by {off[k]:.3g}, allowed {most[k]:.3g} "
                             f"({(~(off <= most)).sum()} of {off.size} values)")


def decay(z, logit):
    if not logit:
        return z, 1.0 - z
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))


@np.errstate(over="ignore", invalid="ignore")  # gates beyond 1 in magnitude may overflow; see close()
def scan(gate, x, h0, dy=None, dh=None, logit=False, leaky=False, kind="f32"):
    """One sequence batch [b, t, d] in 64 bits: dict of name -> (value, bound).
    gate [b, t, d] or [d]; dy, dh None for zeros."""
    b, t, d = x.shape
    k2 = K2[kind]
    a, k = decay(np.broadcast_to(gate, x.shape), logit)
    u = k * x if leaky else x
    h = np.array(np.broadcast_to(h0, (b, d)), np.float64)
    H, J = np.abs(h), np.zeros_like(h)
    y, past, eh, past_e = (np.zeros((b, t, d)) for _ in range(4))
    for i in range(t):
        past[:, i], past_e[:, i] = h, U * (K1 * H + k2 * J)
        J = np.abs(a[:, i]) * (J + H)
        H = np.abs(a[:, i]) * H + np.abs(u[:, i])
        h = a[:, i] * h + u[:, i]
        y[:, i], eh[:, i] = h, U * (K1 * H + k2 * J)
    out = {"y": (y, eh), "h": (h, U * (K1 * H + k2 * J))}
    if dy is None and dh is None:
        return out
    r = np.zeros((b, d)) if dh is None else np.array(dh, np.float64)
    R, S = np.abs(r), np.zeros_like(r)
    g, eg = np.zeros((b, t, d)), np.zeros((b, t, d))
    for i in reversed(range(t)):
        o = dy[:, i] if dy is not None else 0.0
        g[:, i] = o + r
        G = np.abs(o) + R
        eg[:, i] = U * (K1 * G + k2 * S)
        S = np.abs(a[:, i]) * (S + G)
        R = np.abs(a[:, i]) * G
        r = a[:, i] * g[:, i]
    f = np.abs(k) if leaky else 1.0
    out["dx"] = (g * k if leaky else g, f * (eg + K1 * U * np.abs(g)))
    e = past - x if leaky else past
    da = g * e
    ea = np.abs(e) * eg + np.abs(g) * (past_e + 2 * U * (np.abs(past) + np.abs(x))) + eg * past_e + 4 * U * np.abs(da)
    if gate.ndim == 1:  # the sum over n terms in any order: n U times their magnitudes
        n = b * t
        s = (a * k)[0, 0] if logit and n else 1.0
        out["dgate"] = (da.sum((0, 1)) * s, (ea.sum((0, 1)) + (n + 8) * U * np.abs(da).sum((0, 1))) * np.abs(s) * 1.01
                        + 40 * U * np.abs(da.sum((0, 1)) * s))
    else:
        s = a * k if logit else 1.0
        out["dgate"] = (da * s, (ea + 40 * U * np.abs(da)) * np.abs(s))
    out["dh0"] = (r, U * (K1 * R + k2 * S))
    return out


def embed(tokens, table, scale):
    ok = (tokens >= 0) & (tokens < table.shape[0])
    rows = table[np.where(ok, tokens, 0)]
    return np.where(ok[..., None], rows * np.float64(np.float32(scale)), 0.0)


def embed_grad(tokens, dy, vocab, scale, base=None):
    """(value, bound): a row of m terms is off by at most (m + 3) U times the terms' magnitudes."""
    t = tokens.reshape(-1)
    dy = dy.reshape(t.size, dy.shape[-1])
    ok = (t >= 0) & (t < vocab)
    s = np.float64(np.float32(scale))
    out, mag = np.zeros((vocab, dy.shape[1])), np.zeros((vocab, dy.shape[1]))
    np.add.at(out, t[ok], dy[ok])
    np.add.at(mag, t[ok], np.abs(dy[ok]))
    m = np.bincount(t[ok], minlength=vocab)[:, None]
    want, bound = out * s, (m + 3) * U * mag * abs(s)
    if base is not None:
        want, bound = want + base, bound + 2 * U * (np.abs(base) + mag * abs(s))
    return want, bound
