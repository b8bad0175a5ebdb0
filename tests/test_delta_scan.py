"""snn_delta_scan and snn_delta_scan_grad against their 64-bit forms (delta_ref)."""
import ctypes as C

import numpy as np
import pytest

import delta_ref as ref
import snn_b200 as snn

KINDS = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def host(t):
    return t.detach().cpu().double().numpy()


def make(seed, lead, hk, h, dk, dv, kind, logit=False, n_seq=None, strong=False):
    """Inputs of unit keys, as CUDA tensors (kind's type) and h0, dy, dh."""
    import torch
    rng = np.random.default_rng(seed)
    dt = getattr(torch, KINDS[kind])

    def t(x, d=dt):
        return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(d).cuda()

    def unit(x):
        return x / np.sqrt((x ** 2).sum(-1, keepdims=True))

    b = n_seq if n_seq is not None else lead[0]
    q, k = unit(rng.standard_normal((*lead, hk, dk))), unit(rng.standard_normal((*lead, hk, dk)))
    v = rng.standard_normal((*lead, h, dv))
    if logit:
        gate, beta = rng.standard_normal((*lead, h)) * 1.5 + (0.0 if strong else 3.0), rng.standard_normal((*lead, h))
    else:
        gate, beta = -np.exp(rng.standard_normal((*lead, h)) * 1.5 - (0.0 if strong else 3.0)), rng.uniform(0, 1.5, (*lead, h))
    h0, dh = rng.standard_normal((b, h, dk, dv)), rng.standard_normal((b, h, dk, dv)) * 0.3
    dy = rng.standard_normal((*lead, h, dv))
    return [t(x) for x in (q, k, v, gate, beta)], t(h0, torch.float32), t(dy), t(dh, torch.float32)


# ---- the formulas (CPU) ----------------------------------------------------------
@pytest.mark.parametrize("logit", [False, True])
def test_formula_against_differences(logit):
    """The reference's gradients against central differences of its own forward in 64 bits: an error of third order
    in the step, 1e-6 relative for a step of 1e-4, and 2^-52 / 1e-4 of the sum from cancellation."""
    rng = np.random.default_rng(5)
    t, hk, h, dk, dv = 4, 1, 2, 3, 2
    args = [rng.standard_normal(s) for s in ((t, hk, dk), (t, hk, dk), (t, h, dv), (t, h), (t, h), (h, dk, dv))]
    if not logit:
        args[3] = -np.abs(args[3])
    dy, dh = rng.standard_normal((t, h, dv)), rng.standard_normal((h, dk, dv))
    how = dict(logit=logit, scale=0.7)

    def loss(*a):
        r = ref.scan(*a, **how)
        return (r["y"] * dy).sum() + (r["h"] * dh).sum()

    full = ref.scan(*args, dy=dy, dh=dh, **how)
    for i, name in enumerate(("dq", "dk", "dv", "dgate", "dbeta", "dh0")):
        for at in np.ndindex(args[i].shape):
            up, down = [x.copy() for x in args], [x.copy() for x in args]
            up[i][at] += 1e-4
            down[i][at] -= 1e-4
            assert abs((loss(*up) - loss(*down)) / 2e-4 - full[name][at]) < 2e-6 * (1 + abs(full[name][at])), (name, at)


# ---- refusals (CPU) ----------------------------------------------------------------
def call(grad=False, desc=(), **over):
    d = dict(type=0, flags=0, n_seq=2, n_steps=100, hk=2, h=4, dk=8, dv=16, off=None, scale=1.0, res=0)
    d.update(desc)
    heads = {"q": 2 * 8, "k": 2 * 8, "v": 4 * 16, "y": 4 * 16, "dy": 4 * 16, "dq": 2 * 8, "dk": 2 * 8, "dv": 4 * 16}
    width = {n: 8 if n in ("q", "k", "dq", "dk") else 16 for n in heads}
    r = {n: ((i + 1) << 20, 100 * w, w, width[n]) for i, (n, w) in enumerate(heads.items())}
    g = {n: ((i + 1) << 24, 400, 4) for i, n in enumerate(("gate", "beta", "dgate", "dbeta"))}
    a = dict(h0=None, h=None, dh=None, dh0=None, saved=None, sbytes=0, work=1 << 28, bytes=1 << 40)
    if grad:
        a.update(saved=1 << 30, sbytes=1 << 40)
    for k, v in over.items():
        (r if k in r else g if k in g else a)[k] = v
    ro = {k: snn._HEADS.pack(v[0] or 0, *v[1:]) if v else None for k, v in r.items()}
    go = {k: snn._ROWS.pack(v[0] or 0, *v[1:]) if v else None for k, v in g.items()}
    de = snn._DELTA.pack(*(v or 0 for v in d.values()))
    L = snn.lib()
    if grad:
        return L.snn_delta_scan_grad(de, ro["q"], ro["k"], ro["v"], go["gate"], go["beta"], a["saved"], a["sbytes"], ro["dy"],
                                     a["dh"], ro["dq"], ro["dk"], ro["dv"], go["dgate"], go["dbeta"], a["dh0"], a["work"],
                                     a["bytes"], None)
    return L.snn_delta_scan(de, ro["q"], ro["k"], ro["v"], go["gate"], go["beta"], a["h0"], ro["y"], a["h"], a["saved"],
                            a["sbytes"], a["work"], a["bytes"], None)


BAD = [dict(desc=dict(type=3)), dict(desc=dict(flags=2)), dict(desc=dict(n_seq=-1)), dict(desc=dict(n_steps=-1)),
       dict(desc=dict(hk=0)), dict(desc=dict(h=3)), dict(desc=dict(h=1)), dict(desc=dict(h=65536)), dict(desc=dict(dk=0)),
       dict(desc=dict(dk=129)), dict(desc=dict(dv=0)), dict(desc=dict(dv=1025)), dict(desc=dict(off=4100)),
       dict(desc=dict(n_seq=1 << 29, n_steps=1 << 29)), dict(q=None), dict(k=None), dict(v=None), dict(gate=None),
       dict(beta=None), dict(q=(None, 1600, 16, 8)), dict(k=((1 << 20) + 2, 1600, 16, 8)), dict(v=(1 << 20, -1, 64, 16)),
       dict(v=(1 << 20, 6400, -64, 16)), dict(v=(1 << 20, 6400, 64, -16)), dict(gate=((1 << 24) + 2, 400, 4)),
       dict(work=None), dict(work=(1 << 28) + 16), dict(bytes=8)]


@pytest.mark.parametrize("over", BAD + [dict(h0=1026), dict(h=1026), dict(y=None), dict(y=(1 << 20, 6400, 64, 15)),
                                        dict(y=(1 << 20, 6400, 63, 16)), dict(y=(1 << 20, 6399, 64, 16)),
                                        dict(y=(1 << 20, 0, 64, 16)), dict(saved=1 << 30, sbytes=100)])
def test_scan_refuses(over):
    assert call(**over) == 1 and b"delta" in snn.lib().snn_last_error(None)


@pytest.mark.parametrize("over", BAD + [
    dict(dy=None), dict(dh=1026), dict(dh0=1026), dict(saved=None), dict(sbytes=100), dict(dq=None), dict(dk=None),
    dict(dv=None), dict(dgate=None), dict(dbeta=None), dict(dq=(1 << 20, 1600, 15, 8)), dict(dgate=(1 << 24, 400, 3))])
def test_grad_refuses(over):
    assert call(grad=True, **over) == 1 and b"delta" in snn.lib().snn_last_error(None)


def test_null_descriptions_and_sizes():
    n, L = C.c_int64(), snn.lib()
    for fn, how in ((L.snn_delta_scan_saved, ()), (L.snn_delta_scan_workspace, (0,)), (L.snn_delta_scan_grad_workspace, ())):
        assert fn(None, *how, C.byref(n)) == 1
    d = snn._DELTA.pack(1, 0, 3, 100, 2, 4, 128, 100, 0, 1.0, 0)
    assert L.snn_delta_scan_saved(d, None) == 1
    assert L.snn_delta_scan_saved(d, C.byref(n)) == 0 and n.value >= 3 * 2 * 4 * 100 * 128 * 2  # a state a chunk
    d = snn._DELTA.pack(1, 0, 3, 8, 2, 4, 128, 100, 0, 1.0, 0)  # single steps want no workspace
    assert L.snn_delta_scan_workspace(d, 0, C.byref(n)) == 0 and n.value == 0


# ---- GPU ------------------------------------------------------------------------------
def check(kind, b, t, hk, h, dk, dv, logit=False, scale=1.0, seed=0, grads=True, layout=None, strong=False, h0=True, dh=True):
    import torch
    x, s0, dy, d1 = make(seed + t + dk, (b, t), hk, h, dk, dv, kind, logit, strong=strong)

    def lay(v):
        """the same values in other memory: time first, or at an odd element of wider rows"""
        if layout == "tb":
            return v.transpose(0, 1).contiguous().transpose(0, 1)
        if layout == "wide":
            w = torch.empty(*v.shape[:-1], v.shape[-1] + 3, dtype=v.dtype, device="cuda")
            w[..., 1:1 + v.shape[-1]] = v
            return w[..., 1:1 + v.shape[-1]]
        return v

    x, dy = [lay(v) for v in x], lay(dy)
    how = dict(scale=scale, logit=logit)
    zero = np.zeros((b, h, dk, dv))
    want = ref.run(*map(host, x), host(s0) if h0 else zero, dy=host(dy) if grads else None,
                   dh=host(d1) if grads and dh else None, kind=kind, **how)
    y, hh, *saved = snn.delta_scan(*x, s0 if h0 else None, save=grads, **how)
    ref.close(host(y), want["y"], kind, "y")
    ref.close(host(hh), want["h"], kind, "h")
    if grads:
        got = snn.delta_scan_grad(*x, dy, saved[0], dh=d1 if dh else None, **how)
        for name, g in zip(("dq", "dk", "dv", "dgate", "dbeta", "dh0"), got):
            ref.close(host(g), want[name], kind, name)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("t", [1, 2, 8, 9, 63, 64, 65, 130])
def test_lengths(kind, t):
    check(kind, 2, t, 1, 2, 32, 24, seed=t)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dk,dv", [(1, 1), (7, 5), (16, 16), (50, 60), (64, 128), (65, 17), (128, 100), (100, 256), (128, 33), (8, 1000)])
@pytest.mark.parametrize("logit", [False, True])
def test_dims(kind, dk, dv, logit):
    check(kind, 1, 100, 1, 1, dk, dv, logit=logit, scale=dk ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("hk,h", [(1, 3), (2, 4), (3, 3)])
def test_shared_heads(kind, hk, h):
    check(kind, 2, 90, hk, h, 40, 32, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("layout", ["tb", "wide"])
@pytest.mark.parametrize("t", [3, 100])
def test_layouts(kind, layout, t):
    check(kind, 3, t, 2, 4, 24, 40, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("logit", [False, True])
def test_strong_decays_and_missing_states(kind, logit):
    check(kind, 2, 200, 1, 2, 64, 64, logit=logit, strong=True, h0=False, dh=False)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("lengths", [[0], [5, 0, 70, 1], [64, 128, 63, 65, 0, 0, 200], [3, 2, 1], [130] * 9])
@pytest.mark.parametrize("before,behind", [(0, 0), (3, 5)])
def test_packed(kind, lengths, before, behind):
    """Sequences of any lengths, rows of no sequence around them: zero in new results, left alone in given ones."""
    import torch
    off = np.concatenate([[before], before + np.cumsum(lengths)])
    rows, b = int(off[-1]) + behind, len(lengths)
    x, s0, dy, dh = make(11, (rows,), 1, 2, 36, 20, kind, n_seq=b)
    for v in x + [dy]:
        v[:before], v[rows - behind:] = float("nan"), float("nan")
    o = torch.tensor(off, device="cuda")
    want = ref.run(*map(host, x), host(s0), offsets=off.tolist(), dy=host(dy), dh=host(dh), kind=kind)
    y, h, saved = snn.delta_scan(*x, s0, offsets=o, save=True)
    got = dict(zip(("dq", "dk", "dv", "dgate", "dbeta", "dh0"), snn.delta_scan_grad(*x, dy, saved, dh=dh, offsets=o)))
    for name, g in {"y": y, "h": h, **got}.items():
        ref.close(host(g), want[name], kind, name)
    out = torch.full_like(y, 7.0)
    y2, h2 = snn.delta_scan(*x, s0, offsets=o, out=out)
    ref.close(host(y2[before:rows - behind]), (want["y"][0][before:rows - behind], want["y"][1]), kind, "y")
    ref.close(host(h2), want["h"], kind, "h")
    assert (out[:before] == 7).all() and (out[rows - behind:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("logit", [False, True])
def test_segments(kind, logit):
    """Long sequences of few heads are cut into segments that run at once."""
    check(kind, 1, 2500, 1, 2, 40, 24, logit=logit, scale=0.2, grads=kind == "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("lengths", [[4000, 0, 100], [64 * 40, 64 * 25 + 1, 3]])
def test_segments_packed(kind, lengths):
    import torch
    off = np.concatenate([[2], 2 + np.cumsum(lengths)])
    x, s0, _, _ = make(13, (int(off[-1]) + 3,), 1, 1, 20, 36, kind, n_seq=len(lengths))
    want = ref.run(*map(host, x), host(s0), offsets=off.tolist(), kind=kind)
    y, h = snn.delta_scan(*x, s0, offsets=torch.tensor(off, device="cuda"))
    ref.close(host(y), want["y"], kind, "y")
    ref.close(host(h), want["h"], kind, "h")
    y, h, _ = snn.delta_scan(*x, offsets=torch.tensor(off, device="cuda"), save=True)
    want = ref.run(*map(host, x), 0 * host(s0), offsets=off.tolist(), kind=kind)
    ref.close(host(y), want["y"], kind, "y")
    ref.close(host(h), want["h"], kind, "h")


@pytest.mark.gpu
def test_no_sequence_and_no_step():
    import torch
    x, s0, dy, dh = make(1, (2, 0), 1, 1, 8, 8, "bf16")
    y, h, saved = snn.delta_scan(*x, s0, save=True)
    assert y.shape == (2, 0, 1, 8) and torch.equal(h, s0)
    assert torch.equal(snn.delta_scan_grad(*x, dy, saved, dh=dh)[5], dh)
    y, h = snn.delta_scan(*x, s0)
    assert torch.equal(h, s0)
    x, s0, dy, dh = make(1, (5,), 1, 1, 8, 8, "bf16", n_seq=0)
    o = torch.zeros(1, dtype=torch.int64, device="cuda")
    y, h, saved = snn.delta_scan(*x, s0, offsets=o, save=True)
    assert (y == 0).all() and h.shape[0] == 0
    for g in snn.delta_scan_grad(*x, dy, saved, offsets=o):
        assert (g == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("t", [5, 150])
def test_forgetting_all(kind, t):
    """A gate of minus infinity: what was before is gone, whatever it was, and the gate gets no gradient."""
    import torch
    x, s0, dy, dh = make(2, (1, t), 1, 1, 16, 16, kind)
    x[3][:, t // 2] = -float("inf")
    assert snn.delta_scan_grad(*x, dy, snn.delta_scan(*x, s0, logit=True, save=True)[2], dh=dh, logit=True)[3][0, t // 2].item() == 0
    want = ref.run(*map(host, x), host(s0), dy=host(dy), dh=host(dh), kind=kind)
    y, h, saved = snn.delta_scan(*x, s0, save=True)
    ref.close(host(y), want["y"], kind, "y")
    ref.close(host(h), want["h"], kind, "h")
    got = snn.delta_scan_grad(*x, dy, saved, dh=dh)
    for name, g in zip(("dq", "dk", "dv", "dgate", "dbeta", "dh0"), got):
        ref.close(host(g), want[name], kind, name)
    assert got[3][0, t // 2].item() == 0
    y2, h2 = snn.delta_scan(*x, s0)
    ref.close(host(y2), want["y"], kind, "y")
    ref.close(host(h2), want["h"], kind, "h")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 12])
def test_magnitudes(kind, size):
    """Values far from 1: pieces of f16 are taken of scaled values."""
    import torch
    x, s0, dy, dh = make(7, (2, 200), 1, 2, 48, 32, kind)
    x[2] = (x[2] * size).contiguous()
    s0 = s0 * size
    x[0] = x[0] / 8
    want = ref.run(*map(host, x), host(s0), dy=host(dy), dh=host(dh), kind=kind)
    y, h, saved = snn.delta_scan(*x, s0, save=True)
    ref.close(host(y), want["y"], kind, "y")
    ref.close(host(h), want["h"], kind, "h")
    for name, g in zip(("dq", "dk", "dv", "dgate", "dbeta", "dh0"), snn.delta_scan_grad(*x, dy, saved, dh=dh)):
        ref.close(host(g), want[name], kind, name)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
def test_infinities_stay_where_they_belong(kind):
    """An infinity in one column of a value reaches that column alone, one in a query its own answer alone."""
    import torch
    x, s0, dy, dh = make(8, (1, 200), 1, 1, 32, 48, kind)
    want = ref.run(*map(host, x), host(s0), dy=host(dy), dh=host(dh), kind=kind)
    v = x[2].clone()
    v[0, 100, 0, 20] = float("inf")
    y, h = snn.delta_scan(*x[:2], v, *x[3:], s0)
    others = [c for c in range(48) if c != 20]
    ref.close(host(y)[..., others], (want["y"][0][..., others], want["y"][1]), kind, "y")
    ref.close(host(h)[..., others], (want["h"][0][..., others], want["h"][1]), kind, "h")
    ref.close(host(y)[:, :64], (want["y"][0][:, :64], want["y"][1]), kind, "y")
    assert not torch.isfinite(y[0, 100, 0, 20]) and not torch.isfinite(h[..., 20]).all()
    q = x[0].clone()
    q[0, 70, 0, 3] = float("inf")
    y, h = snn.delta_scan(q, *x[1:], s0)
    rows = [t for t in range(200) if t != 70]
    ref.close(host(y)[:, rows], (want["y"][0][:, rows], want["y"][1]), kind, "y")
    ref.close(host(h), want["h"], kind, "h")
    _, _, saved = snn.delta_scan(*x, s0, save=True)
    d = dy.clone()
    d[0, 100, 0, 20] = float("inf")
    dv = snn.delta_scan_grad(*x, d, saved, dh=dh)[2]
    ref.close(host(dv)[..., others], (want["dv"][0][..., others], want["dv"][1]), kind, "dv")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
def test_zero_inputs(kind):
    """No rate, no key, no query: the state only decays, and nothing is divided by."""
    import torch
    x, s0, dy, dh = make(4, (1, 100), 1, 1, 32, 32, kind)
    for zeros in ((4,), (1,), (0, 2), (0, 1, 2, 4)):
        z = [torch.zeros_like(v) if i in zeros else v for i, v in enumerate(x)]
        want = ref.run(*map(host, z), host(s0), dy=host(dy), dh=host(dh), kind=kind)
        y, h, saved = snn.delta_scan(*z, s0, save=True)
        ref.close(host(y), want["y"], kind, "y")
        ref.close(host(h), want["h"], kind, "h")
        for name, g in zip(("dq", "dk", "dv", "dgate", "dbeta", "dh0"), snn.delta_scan_grad(*z, dy, saved, dh=dh)):
            ref.close(host(g), want[name], kind, name)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
def test_steps_in_place_are_the_sequence(kind):
    """Single steps with the state carried in place, and the whole sequence at once."""
    import torch
    x, s0, _, _ = make(9, (3, 70), 2, 4, 64, 96, kind, logit=True)
    want = ref.run(*map(host, x), host(s0), kind=kind, logit=True)
    y, h = snn.delta_scan(*x, s0, logit=True)
    ref.close(host(y), want["y"], kind, "y")
    ref.close(host(h), want["h"], kind, "h")
    state = s0.clone()
    for t in range(70):
        yt, st = snn.delta_scan(*(v[:, t:t + 1] for v in x), state, logit=True, h_out=state)
        assert st is state
        ref.close(host(yt), (want["y"][0][:, t:t + 1], want["y"][1]), kind, "y")
    ref.close(host(state), want["h"], kind, "h")
    h2 = s0.clone()
    snn.delta_scan(*x, h2, logit=True, h_out=h2)
    assert torch.equal(h2, h)


@pytest.mark.gpu
def test_memory_of_long_sequences():
    """Decays next to 1 over 20,000 steps: what decays lose to a rounding would be 2^-25 x 20,000 of the state."""
    import torch
    t = 20000
    q = torch.ones(1, t, 1, 8, device="cuda") / 8 ** 0.5
    k, v = q.clone(), torch.zeros(1, t, 1, 8, device="cuda")
    beta = torch.zeros(1, t, 1, device="cuda")
    h0 = torch.randn(1, 1, 8, 8, device="cuda")
    for g in (-1e-4, -3e-5):
        gate = torch.full((1, t, 1), g, device="cuda")
        want = h0.double() * np.exp(float(gate[0, 0, 0].double()) * t)
        _, h = snn.delta_scan(q, k, v, gate, beta, h0)
        # a rounding of 1 - (the chunk's decay) each of 313 chunks, relative to what it takes off, and one of each product
        assert ((h.double() - want).abs() <= want.abs() * (313 * 2.0 ** -24 + 2.0 ** -23 * abs(g) * t)).all()
        state = h0.clone()
        for _ in range(500):
            snn.delta_scan(q[:, :1], k[:, :1], v[:, :1], gate[:, :1], beta[:, :1], state, h_out=state)
        want = h0.double() * np.exp(float(gate[0, 0, 0].double()) * 500)
        assert ((state.double() - want).abs() <= want.abs() * 500 * 2.0 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_equal_calls_graphs_and_streams(kind):
    """Equal calls give equal bits; a captured step replays on new values; a call on another stream."""
    import torch
    x, s0, dy, dh = make(6, (2, 300), 2, 4, 64, 64, kind)

    def both():
        y, h, saved = snn.delta_scan(*x, s0, save=True)
        return [y, h, *snn.delta_scan_grad(*x, dy, saved, dh=dh)]

    first, again = both(), both()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    y, h = snn.delta_scan(*x, s0, stream=side)
    side.synchronize()
    assert torch.equal(y, first[0]) and torch.equal(h, first[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = both()
    keep = [v.clone() for v in x]
    for v in x[:3]:
        v.copy_(v.flip(1))
    graph.replay()
    want = both()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))
    for v, k in zip(x, keep):
        v.copy_(k)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, first))


@pytest.mark.gpu
def test_binding_refuses():
    import torch
    x, s0, dy, dh = make(3, (2, 20), 1, 2, 16, 16, "bf16")
    q, k, v, gate, beta = x
    y, h, saved = snn.delta_scan(*x, s0, save=True)
    bad = [lambda: snn.delta_scan(q.cpu(), k, v, gate, beta), lambda: snn.delta_scan(q, k, v.float(), gate, beta),
           lambda: snn.delta_scan(q, k[:, :10], v, gate, beta), lambda: snn.delta_scan(q, k, v, gate.float(), beta),
           lambda: snn.delta_scan(q, k, v, gate, beta, s0.bfloat16()), lambda: snn.delta_scan(q, k, v, gate, beta, s0[:1]),
           lambda: snn.delta_scan(q, k, v, gate, beta, offsets=torch.zeros(3, device="cuda")),
           lambda: snn.delta_scan(*x, out=torch.empty_like(v)[:, :3]), lambda: snn.delta_scan(*x, h_out=s0.transpose(2, 3)),
           lambda: snn.delta_scan(q.transpose(2, 3), k, v, gate, beta),
           lambda: snn.delta_scan_grad(*x, None, saved), lambda: snn.delta_scan_grad(*x, dy, saved[:-1]),
           lambda: snn.delta_scan_grad(*x, dy.float(), saved), lambda: snn.delta_scan_grad(*x, dy, saved.float())]
    for f in bad:
        with pytest.raises(snn.SnnError):
            f()
