"""The gated delta rule and its gradients a step at a time in 64 bits, for the tests of snn_delta_scan, and how far
the kernels may be from them."""
import numpy as np

# half a step of a rounding, relative to the value
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def scan(q, k, v, gate, beta, h0, scale=1.0, logit=False, dy=None, dh=None):
    """q, k [t, hk, dk], v [t, h, dv], gate, beta [t, h], h0 [h, dk, dv] of one sequence: a dict of y, h and, with dy
    and dh, the gradients."""
    t, h, dv = v.shape
    hk, dk = q.shape[1:]
    group = h // hk
    with np.errstate(over="ignore"):
        a, b = (1 / (1 + np.exp(-gate)), 1 / (1 + np.exp(-beta))) if logit else (np.exp(gate), beta)
    S, states, y = h0.copy(), [], np.zeros((t, h, dv))
    us, errs = np.zeros((t, h, dv)), np.zeros((t, h, dv))
    for i in range(t):
        states.append(S)
        old = a[i][:, None, None] * S
        kk, qq = np.repeat(k[i], group, 0), np.repeat(q[i], group, 0)
        errs[i] = v[i] - np.einsum("hkv,hk->hv", old, kk)
        us[i] = b[i][:, None] * errs[i]
        S = old + kk[:, :, None] * us[i][:, None, :]
        y[i] = scale * np.einsum("hkv,hk->hv", S, qq)
    out = {"y": y, "h": S}
    if dy is None and dh is None:
        return out
    D = np.zeros_like(S) if dh is None else dh.copy()
    dq, dkk, dvv = np.zeros((t, h, dk)), np.zeros((t, h, dk)), np.zeros((t, h, dv))
    dg, db = np.zeros((t, h)), np.zeros((t, h))
    for i in reversed(range(t)):
        kk, qq = np.repeat(k[i], group, 0), np.repeat(q[i], group, 0)
        old = a[i][:, None, None] * states[i]
        new = old + kk[:, :, None] * us[i][:, None, :]
        if dy is not None:
            D = D + scale * qq[:, :, None] * dy[i][:, None, :]
            dq[i] = scale * np.einsum("hkv,hv->hk", new, dy[i])
        du = np.einsum("hkv,hk->hv", D, kk)
        e = b[i][:, None] * du
        dvv[i] = e
        dkk[i] = np.einsum("hkv,hv->hk", D, us[i]) - np.einsum("hkv,hv->hk", old, e)
        db[i] = (du * errs[i]).sum(-1)
        dold = D - kk[:, :, None] * e[:, None, :]
        da = (dold * states[i]).sum((1, 2))
        dg[i] = a[i] * da
        if logit:
            dg[i] *= 1 - a[i]
            db[i] *= b[i] * (1 - b[i])
        D = a[i][:, None, None] * dold
    out |= {"dq": dq.reshape(t, hk, group, dk).sum(2), "dk": dkk.reshape(t, hk, group, dk).sum(2), "dv": dvv,
            "dgate": dg, "dbeta": db, "dh0": D}
    return out


def rounded(x, kind):
    """x with the 8 bits of bf16 (or untouched)."""
    if kind != "bf16":
        return x
    m, e = np.frexp(x)
    return np.ldexp(np.rint(m * 256), e - 8)


def model(q, k, v, gate, beta, h0, scale=1.0, logit=False, dy=None, dh=None, kind="f32", seed=0):
    """scan() as the kernels take it, by chunks of 64 steps, with the errors that their arithmetic may make drawn at random:
    how far these are from scan() is how far the kernels may be.  A product of matrices in pieces is off by up to 2^-21
    of the sum of its terms' magnitudes: 2^-22 for what two pieces of 11 bits leave of an operand (or for the
    product of the two low pieces), 2^-22 for a sum of up to 128 terms in f32.  One piece of f16 (y of bf16 tensors, p and
    x of their gradients): 2^-11 of an operand.  States, U and R are rounded to bf16 once for the gradients of bf16
    tensors.  A decay between steps is off by 2^-21: two units in the last place of the exponential function, one each of
    its argument's rounding (of magnitudes up to 1; what has decayed further is smaller by more) and of the product."""
    rng = np.random.default_rng(seed)
    t_all, h, dv = v.shape
    hk, dk = q.shape[1:]
    group = h // hk
    one = {"f32": 2.0 ** -21, "f16": 2.0 ** -21, "bf16": 2.0 ** -11}[kind]
    full = 2.0 ** -21

    def mm(a, b, eps=full):
        return a @ b + rng.uniform(-eps, eps, (a.shape[0], b.shape[1])) * (np.abs(a) @ np.abs(b))

    out = {n: np.zeros(s) for n, s in (("y", v.shape), ("h", h0.shape), ("dq", (t_all, hk, dk)), ("dk", (t_all, hk, dk)),
                                       ("dv", v.shape), ("dgate", gate.shape), ("dbeta", beta.shape), ("dh0", h0.shape))}
    with np.errstate(all="ignore"):
        la = -np.log1p(np.exp(-gate)) if logit else gate
        b = 1 / (1 + np.exp(-beta)) if logit else beta
    for j in range(h):
        S, chunks = h0[j].copy(), []
        for c in range(0, t_all, 64):
            e = min(t_all, c + 64)
            K, Q, V, B = k[c:e, j // group], q[c:e, j // group], v[c:e, j], b[c:e, j][:, None]
            n = e - c
            L = la[c:e, j]
            G = np.zeros((n, n))
            for r in range(n):  # G[i, r]: decays of the steps behind r up to i
                G[r:, r] = np.concatenate([[1.0], np.exp(np.cumsum(L[r + 1:]))])
            G = G * (1 + rng.uniform(-full, full, (n, n)) * (1 + np.abs(np.log(np.maximum(G, 1e-30))) / 8))
            since, until = (np.exp(np.cumsum(L)) * (1 + rng.uniform(-full, full, n)))[:, None], G[-1][:, None]
            low = np.tril(np.ones((n, n)), -1)
            A = np.where(low > 0, B * G * mm(K, K.T), 0.0)
            P = np.where(low + np.eye(n) > 0, G * mm(Q, K.T), 0.0)
            T = np.linalg.inv(np.eye(n) + A)
            T = T + rng.uniform(-full, full, T.shape) * (np.abs(T) @ np.abs(np.eye(n) + A) @ np.abs(T)) * low
            U = mm(T, B * (V - since * mm(K, S)))
            out["y"][c:e, j] = scale * (since * mm(Q, S, one) + mm(P, U, one))
            chunks.append((c, e, K, Q, V, B, L, G, since, until, T, P, U, S))
            S = since[-1] * S + mm((until * K).T, U)
        out["h"][j] = S
        if dy is None and dh is None:
            continue
        D = np.zeros_like(S) if dh is None else dh[j].copy()
        for c, e, K, Q, V, B, L, G, since, until, T, P, U, S in reversed(chunks):
            n = e - c
            Z = scale * (dy[c:e, j] if dy is not None else np.zeros_like(V))
            R = mm(T.T, mm(P.T, Z) + until * mm(K, D))
            out["dv"][c:e, j] = B * R
            Sr, Dr, Ur, Rr = (rounded(x, kind) for x in (S, D, U, R))
            low = np.tril(np.ones((n, n)), -1)
            p = (low + np.eye(n)) * G * mm(Z, Ur.T)
            x = -low * G * mm(Rr, Ur.T)
            zq, zk, zm = since * mm(Z, Sr.T), -since * mm(Rr, Sr.T), until * mm(Ur, Dr.T)
            xk, pq = x * mm(K, K.T), p * mm(Q, K.T)
            both = B * xk + pq
            d = (Q * zq).sum(1) + both.sum(1) - both.sum(0) + B[:, 0] * (K * zk).sum(1) - (K * zm).sum(1)
            extra = since[-1, 0] * (Sr * Dr).sum() + (K * zm).sum()
            out["dbeta"][c:e, j] = (Rr * V).sum(1) + (K * zk).sum(1) + xk.sum(1)
            out["dgate"][c:e, j] = np.cumsum(d[::-1])[::-1] + extra
            # the sums that these are of, in f32: 2^-22 of all magnitudes
            size = (np.abs(Q * zq).sum() + 2 * np.abs(both).sum() + np.abs(K * zk).sum() + 2 * np.abs(K * zm).sum()
                    + since[-1, 0] * np.abs(Sr * Dr).sum())
            out["dgate"][c:e, j] += rng.uniform(-1, 1, n) * 2.0 ** -22 * size
            out["dgate"][c:e, j][L == -np.inf] = 0
            out["dq"][c:e, j // group] += zq + mm(p, K, one)
            out["dk"][c:e, j // group] += B * zk + zm + mm(B * x, K, one) + mm((B * x).T, K, one) + mm(p.T, Q, one)
            D = since[-1] * D + mm((since * Q).T, Z) - mm((since * K).T, B * R)
        out["dh0"][j] = D
        if logit:
            with np.errstate(over="ignore"):
                out["dgate"][:, j] *= 1 / (1 + np.exp(gate[:, j]))
            out["dbeta"][:, j] *= b[:, j] * (1 - b[:, j])
    return out


def run(q, k, v, gate, beta, h0, offsets=None, kind="f32", **how):
    """scan() of dense [b, t, ..] or packed [rows, ..] arrays (offsets: a list): a dict of (value, how far off it may be,
    four times the largest error of its head that model() makes: other draws give others)."""
    dy, dh = how.pop("dy", None), how.pop("dh", None)
    n_seq = len(h0)
    dense = offsets is None
    names = ["y", "h"] + (["dq", "dk", "dv", "dgate", "dbeta", "dh0"] if dy is not None or dh is not None else [])
    like = dict(y=v, h=h0, dq=q, dk=k, dv=v, dgate=gate, dbeta=beta, dh0=h0)
    out = {n: [np.zeros(like[n].shape), 0.0] for n in names}
    for i in range(n_seq):
        at = i if dense else slice(offsets[i], offsets[i + 1])
        a = [x[at] for x in (q, k, v, gate, beta)]
        how_i = dict(how, dy=None if dy is None else dy[at], dh=None if dh is None else dh[i])
        want, off = scan(*a, h0[i], **how_i), model(*a, h0[i], kind=kind, seed=i, **how_i)
        for n in names:
            out[n][0][i if n in ("h", "dh0") else at] = want[n]
            if want[n].size:
                out[n][1] = max(out[n][1], 4 * np.abs(off[n] - want[n]).max())
    return out


def close(got, want, kind, name):
    """A value and how far off it may be (run), and one rounding to its type: half a step."""
    got, (want, far) = np.asarray(got, np.float64), want
    assert got.shape == want.shape, (name, got.shape, want.shape)
    if want.size == 0:
        return
    half = HALF["f32"] if name in ("h", "dh0") else HALF[kind]
    # (the rounding is of the computed value, and f16 has no steps below 2^-24)
    far = far * (1 + half) + (2.0 ** -25 if kind == "f16" and name not in ("h", "dh0") else 0.0) + 1e-30
    if kind == "f16" and name not in ("h", "dh0"):  # what is beyond the type's largest value has become infinite
        over = np.abs(want) + far > 65519
        assert (np.sign(got[over]) == np.sign(want[over])).all() and (np.abs(got[over]) > 65000).all()
        got, want = got[~over], want[~over]
    off = np.abs(got - want) - half * np.abs(want)
    assert np.isfinite(got).all() and off.max() <= far, (name, kind, off.max(), far)
