"""snn_leaky_scan and snn_leaky_scan_grad against their 64-bit forms (leaky_ref)."""
import ctypes as C

import numpy as np
import pytest

import leaky_ref as ref
import snn_b200 as snn

KINDS = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def dt(kind):
    import torch
    return getattr(torch, KINDS[kind])


def host(t):
    return t.detach().cpu().double().numpy()


def same(a, b):
    """Equal values, NaN in the same places."""
    import torch
    return torch.allclose(a, b, rtol=0, atol=0, equal_nan=True)


def make(rng, shape, kind, std=1.0, mean=0.0):
    import torch
    return torch.from_numpy((rng.standard_normal(shape) * std + mean).astype(np.float32)).to(dt(kind)).cuda()


def gate_of(rng, shape, kind, logit):
    import torch
    if logit:
        return make(rng, shape, kind, 2.0, 1.0)
    return torch.from_numpy((1 - np.exp(rng.standard_normal(shape) - 2)).astype(np.float32)).to(dt(kind)).cuda()


# ---- the formulas (CPU) ----------------------------------------------------------
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("leaky", [False, True])
@pytest.mark.parametrize("channel", [False, True])
def test_formula_against_differences(logit, leaky, channel):
    """The reference's gradients against central differences of its own forward in 64 bits: an error of
    third order in the step, 1e-6 relative for a step of 1e-4, and 2^-52 / 1e-4 of the sum from cancellation."""
    rng = np.random.default_rng(5)
    b, t, d = 2, 7, 3
    x, h0, dy, dh = (rng.standard_normal(s) for s in ((b, t, d), (b, d), (b, t, d), (b, d)))
    gate = rng.standard_normal((d,) if channel else (b, t, d)) if logit else \
        rng.uniform(0.2, 0.99, (d,) if channel else (b, t, d))
    how = dict(logit=logit, leaky=leaky)

    def loss(gate, x, h0):
        r = ref.scan(gate, x, h0, **how)
        return (r["y"][0] * dy).sum() + (r["h"][0] * dh).sum()

    full = ref.scan(gate, x, h0, dy, dh, **how)
    for name, i in (("dgate", 0), ("dx", 1), ("dh0", 2)):
        args = [gate, x, h0]
        for at in np.ndindex(args[i].shape):
            e = np.zeros_like(args[i])
            e[at] = 1e-4
            up, down = list(args), list(args)
            up[i], down[i] = args[i] + e, args[i] - e
            assert abs((loss(*up) - loss(*down)) / 2e-4 - full[name][0][at]) < 1e-6 * (1 + abs(full[name][0][at]))


# ---- refusals (CPU) ----------------------------------------------------------------
def call(grad=False, desc=(), **over):
    d = dict(type=0, flags=0, n_seq=2, n_steps=5, n_channels=8, offsets=None)
    d.update(desc)
    r = {k: (8192 + 4096 * i, 40, 8) for i, k in enumerate(("gate", "x", "y", "dgate", "dx"))}
    a = dict(h0=None, h=None, saved=1 << 20, dh=None, dh0=None, work=None, bytes=0)
    for k, v in over.items():
        (r if k in r else a)[k] = v
    ro = {k: snn._ROWS.pack(v[0] or 0, *v[1:]) if v else None for k, v in r.items()}
    de = snn._SCAN.pack(*(v or 0 for v in d.values()))
    L = snn.lib()
    if grad:
        return L.snn_leaky_scan_grad(de, ro["gate"], ro["x"], a["saved"], ro["y"], a["dh"], ro["dgate"], ro["dx"],
                                     a["dh0"], a["work"], a["bytes"], None)
    return L.snn_leaky_scan(de, ro["gate"], ro["x"], a["h0"], ro["y"], a["h"], a["saved"], a["work"], a["bytes"], None)


BAD = [dict(desc=dict(type=3)), dict(desc=dict(flags=16)), dict(desc=dict(n_seq=-1)), dict(desc=dict(n_steps=-1)),
       dict(desc=dict(n_channels=0)), dict(desc=dict(n_channels=1 << 30)),
       dict(desc=dict(n_seq=1 << 20, n_steps=1 << 20, n_channels=1 << 10)), dict(gate=None), dict(x=None),
       dict(gate=(None, 40, 8)), dict(x=(8193, 40, 8)), dict(x=(8192, -40, 8)), dict(x=(8192, 40, -8)),
       dict(desc=dict(flags=4), gate=(8194, 0, 0))]


@pytest.mark.parametrize("over", BAD + [dict(h0=1026), dict(h=1026), dict(saved=(1 << 20) + 2), dict(desc=dict(offsets=4100)),
                                        dict(desc=dict(n_seq=1, n_steps=40000), y=(8192, 40000 * 8, 8)), dict(y=None), dict(y=(8192, 40, 7)), dict(y=(8192, 39, 8)), dict(y=(8192, 0, 8))])
def test_scan_refuses(over):
    assert call(**over) == 1 and b"scan" in snn.lib().snn_last_error(None)


@pytest.mark.parametrize("over", BAD + [
    dict(y=None), dict(saved=None), dict(dh=1026), dict(dh0=1026), dict(dx=(8192, 40, 7)), dict(dgate=(8192, 39, 8)), dict(desc=dict(flags=8)),
    dict(desc=dict(flags=4)), dict(desc=dict(flags=4), work=1 << 21, bytes=8),
    dict(desc=dict(flags=4), work=(1 << 21) + 4, bytes=1 << 30)])
def test_scan_grad_refuses(over):
    assert call(grad=True, **over) == 1 and b"scan" in snn.lib().snn_last_error(None)


def test_null_descriptions():
    n = C.c_int64()
    assert snn.lib().snn_leaky_scan(None, None, None, None, None, None, None, None, 0, None) == 1
    assert snn.lib().snn_leaky_scan_saved(None, C.byref(n)) == 1
    d = snn._SCAN.pack(0, 0, 3, 100, 7, 0)
    assert snn.lib().snn_leaky_scan_saved(d, None) == 1
    # a state for every block of every sequence, whatever the lengths
    assert snn.lib().snn_leaky_scan_saved(d, C.byref(n)) == 0 and n.value >= 3 * 2 * 7


# ---- GPU ------------------------------------------------------------------------------
def check(kind, b, t, d, channel=False, logit=True, leaky=True, seed=0, layout="bt", grads=True, gate=None, x=None):
    import torch
    rng = np.random.default_rng(seed + 7 * t + d)

    def rows(v):
        """the same values in another layout"""
        if layout == "tb":
            return v.transpose(0, 1).contiguous().transpose(0, 1)
        if layout == "wide":  # rows inside wider ones, at an odd element
            w = torch.empty(b, t, d + 5, dtype=v.dtype, device="cuda")
            w[:, :, 3:3 + d] = v
            return w[:, :, 3:3 + d]
        return v

    if gate is None:
        gate = gate_of(rng, (d,), "f32", logit) if channel else rows(gate_of(rng, (b, t, d), kind, logit))
    if x is None:
        x = rows(make(rng, (b, t, d), kind))
    h0, dy, dh = make(rng, (b, d), "f32"), rows(make(rng, (b, t, d), kind)), make(rng, (b, d), "f32")
    how = dict(logit=logit, leaky=leaky)
    want = ref.scan(host(gate), host(x), host(h0), host(dy), host(dh), kind="f32" if channel else kind, **how)
    y, h, saved = snn.leaky_scan(gate, x, h0, save=True, **how)
    ref.close(host(y), *want["y"], kind, "y")
    ref.close(host(h), *want["h"], "f32", "h")
    y2, h2 = snn.leaky_scan(gate, x, h0, **how)
    assert same(y2, y) and same(h2, h)
    if not grads:
        return
    dgate, dx, dh0 = snn.leaky_scan_grad(gate, x, dy, saved, dh=dh, **how)
    ref.close(host(dx), *want["dx"], kind, "dx")
    ref.close(host(dgate), *want["dgate"], "f32" if channel else kind, "dgate")
    ref.close(host(dh0), *want["dh0"], "f32", "dh0")
    again = snn.leaky_scan_grad(gate, x, dy, saved, dh=dh, **how)
    assert all(same(p, q) for p, q in zip(again, (dgate, dx, dh0)))


@pytest.mark.gpu
@pytest.mark.parametrize("b,t,d", [(1, 1, 1), (3, 1, 64), (2, 2, 33), (5, 7, 100), (1, 63, 8), (2, 64, 40), (1, 65, 130),
                                   (3, 128, 66), (1, 129, 31), (2, 300, 257), (4, 1030, 24), (70, 20, 5), (1, 2500, 64)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("channel", [False, True])
def test_scan(kind, b, t, d, channel):
    check(kind, b, t, d, channel)


@pytest.mark.gpu
@pytest.mark.parametrize("b,t,d", [(1, 12288, 8), (1, 13001, 33), (2, 14003, 6), (1, 6145, 70), (1, 40000, 3)])
@pytest.mark.parametrize("kind,channel,logit,leaky", [("f32", False, True, True), ("f32", True, False, False),
                                                      ("bf16", False, True, False), ("bf16", True, True, True),
                                                      ("f16", False, False, True)])
def test_scan_long(b, t, d, kind, channel, logit, leaky):
    """Sequences long enough to be cut into chunks."""
    check(kind, b, t, d, channel, logit, leaky)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[0, 30000, 0, 1, 17000, 0], [0, 0, 40000], [16, 25001, 129], [12300, 12300],
                                     [6500] * 30 + [0, 3, 70000] + [1] * 3])
@pytest.mark.parametrize("channel", [False, True])
def test_packed_long(lengths, channel):
    """The same of packed sequences, with empty ones among them and rows of no sequence around them."""
    import torch
    rng = np.random.default_rng(len(lengths))
    d, before, behind = 5, 1000, 700
    off = np.cumsum([before] + lengths)
    rows, b = int(off[-1]) + behind, len(lengths)
    offsets = torch.from_numpy(off).cuda()
    gate = gate_of(rng, (d,) if channel else (rows, d), "f32", True)
    x, dy = make(rng, (rows, d), "f32"), make(rng, (rows, d), "f32")
    x[:before], x[-behind:] = float("nan"), float("nan")
    h0, dh = make(rng, (b, d), "f32"), make(rng, (b, d), "f32")
    out = torch.full((rows, d), 7.0, device="cuda")
    how = dict(logit=True, leaky=True, offsets=offsets)
    y, h, saved = snn.leaky_scan(gate, x, h0, save=True, out=out, **how)
    assert (y[:before] == 7).all() and (y[-behind:] == 7).all()
    dgate, dx, dh0 = snn.leaky_scan_grad(gate, x, dy, saved, dh=dh, **how)
    value, bound, size = 0.0, 0.0, 0.0
    for s in range(b):
        r = slice(int(off[s]), int(off[s + 1]))
        want = ref.scan(host(gate) if channel else host(gate[r])[None], host(x[r])[None], host(h0[s:s + 1]),
                        host(dy[r])[None], host(dh[s:s + 1]), True, True, "f32")
        ref.close(host(y[r])[None], *want["y"], "f32", "y")
        ref.close(host(h[s:s + 1]), *want["h"], "f32", "h")
        ref.close(host(dx[r])[None], *want["dx"], "f32", "dx")
        ref.close(host(dh0[s:s + 1]), *want["dh0"], "f32", "dh0")
        if channel:
            value, bound, size = value + want["dgate"][0], bound + want["dgate"][1], size + np.abs(want["dgate"][0])
        else:
            ref.close(host(dgate[r])[None], *want["dgate"], "f32", "dgate")
    if channel:
        ref.close(host(dgate), value, bound + (b + 4) * ref.U * size + rows * ref.U * bound, "f32", "dgate")


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("leaky", [False, True])
@pytest.mark.parametrize("channel", [False, True])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["bt", "tb", "wide"])
def test_scan_forms(kind, channel, logit, leaky, layout):
    check(kind, 3, 150, 70, channel, logit, leaky, layout=layout)
    check(kind, 2, 5, 70, channel, logit, leaky, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_scan_many_sequences(kind):
    check(kind, 3000, 3, 40)
    check(kind, 1500, 70, 12, channel=True)


@pytest.mark.gpu
def test_scan_negative_and_growing_gates():
    """Gates are any numbers where they are given as decays."""
    import torch
    rng = np.random.default_rng(2)
    gate = torch.from_numpy(rng.uniform(-1.05, 1.05, (2, 90, 40)).astype(np.float32)).cuda()
    check("f32", 2, 90, 40, logit=False, leaky=False, gate=gate)
    check("f32", 2, 90, 40, logit=False, leaky=True, gate=gate)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [4, 200, 700])
def test_scan_extreme_logits(t):
    """Gates of +-inf hold and reset the state exactly; a NaN stays in its channel and behind its step."""
    import torch
    inf = float("inf")
    for kind in ("f32", "bf16"):
        rng = np.random.default_rng(t)
        gate, x = make(rng, (2, t, 64), kind), make(rng, (2, t, 64), kind)
        h0 = make(rng, (2, 64), "f32")
        gate[:, :, 0] = inf    # holds h0
        gate[:, :, 1] = -inf   # passes x
        gate[:, t // 2, 2] = -inf
        gate[:, :, 3] = 60.0
        gate[:, :, 4] = -200.0
        x[:, t // 2 - 1, 2] = 1e30  # forgotten at the reset
        y, h = snn.leaky_scan(gate, x, h0, logit=True, leaky=True)
        assert torch.equal(h[:, 0], h0[:, 0]) and torch.equal(y[:, :, 1], x[:, :, 1])
        assert torch.equal(y[:, t // 2, 2], x[:, t // 2, 2])
        assert torch.equal(y[:, :, 4], x[:, :, 4])
        assert torch.isfinite(y).all()
        x[1, t // 2, 5] = float("nan")
        y2, _, saved = snn.leaky_scan(gate, x, h0, logit=True, leaky=True, save=True)
        bad = torch.isnan(y2)
        assert bad[1, t // 2:, 5].all() and bad.sum() == t - t // 2
        dy = make(rng, (2, t, 64), kind)
        _, dx, dh0 = snn.leaky_scan_grad(gate, x, dy, saved, logit=True, leaky=True)
        assert torch.isfinite(dx).all() and torch.isfinite(dh0).all()  # x does not enter them


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("channel", [False, True])
@pytest.mark.parametrize("d", [33, 64])
@pytest.mark.parametrize("lengths", [[5], [0, 1, 0, 2, 64, 0], [63, 65, 1, 128, 300, 0], [1] * 300, [1200, 3, 0, 40]])
def test_packed(kind, channel, d, lengths):
    import torch
    rng = np.random.default_rng(len(lengths) + d)
    before, behind = 3, 6  # rows of no sequence
    off = np.cumsum([before] + lengths)
    rows = int(off[-1]) + behind
    offsets = torch.from_numpy(off).cuda()
    gate = gate_of(rng, (d,), "f32", True) if channel else gate_of(rng, (rows, d), kind, True)
    x, dy = make(rng, (rows, d), kind), make(rng, (rows, d), kind)
    x[:before], x[-behind:], dy[:before], dy[-behind:] = (float("nan"),) * 4
    if not channel:
        gate[:before], gate[-behind:] = float("nan"), float("nan")
    b = len(lengths)
    h0, dh = make(rng, (b, d), "f32"), make(rng, (b, d), "f32")
    out = torch.full((rows, d), 7.0, dtype=dt(kind), device="cuda")
    how = dict(logit=True, leaky=True, offsets=offsets)
    y, h, saved = snn.leaky_scan(gate, x, h0, save=True, out=out, **how)
    assert (y[:before] == 7).all() and (y[-behind:] == 7).all()
    dgate, dx, dh0 = snn.leaky_scan_grad(gate, x, dy, saved, dh=dh, **how)
    sums = [0.0, 0.0, 0.0]
    for s in range(b):
        r = slice(int(off[s]), int(off[s + 1]))
        g = host(gate) if channel else host(gate[r])[None]
        want = ref.scan(g, host(x[r])[None], host(h0[s:s + 1]), host(dy[r])[None], host(dh[s:s + 1]), True, True,
                        "f32" if channel else kind)
        ref.close(host(y[r])[None], *want["y"], kind, "y")
        ref.close(host(h[s:s + 1]), *want["h"], "f32", "h")
        ref.close(host(dx[r])[None], *want["dx"], kind, "dx")
        ref.close(host(dh0[s:s + 1]), *want["dh0"], "f32", "dh0")
        if channel:
            sums = [p + q for p, q in zip(sums, (want["dgate"][0], want["dgate"][1], np.abs(want["dgate"][0])))]
        else:
            ref.close(host(dgate[r])[None], *want["dgate"], kind, "dgate")
    if channel:  # the sequences' sums are joined by b more additions
        ref.close(host(dgate), sums[0], sums[1] + (b + 4) * ref.U * sums[2] + rows * ref.U * sums[1], "f32", "dgate")


@pytest.mark.gpu
def test_packed_bad_offsets_stay_inside():
    """Offsets are data on the device: what points outside the rows is cut to them."""
    import torch
    rng = np.random.default_rng(3)
    x, gate = make(rng, (40, 20), "f32"), gate_of(rng, (40, 20), "f32", True)
    off = torch.tensor([-50, 10, 5, 1 << 50, 20], device="cuda")
    y, h, saved = snn.leaky_scan(gate, x, logit=True, offsets=off, save=True)
    one, last = snn.leaky_scan(gate[None, :10], x[None, :10], logit=True)
    assert torch.equal(y[:5], one[0, :5]) and torch.equal(h[:1], last)
    assert (h[1] == 0).all() and (h[3] == 0).all()  # empty
    snn.leaky_scan_grad(gate, x, x, saved, logit=True, offsets=off)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("t,n", [(1, 100), (3, 64), (150, 45), (400, 1100), (13000, 70), (64, 80000)])
@pytest.mark.parametrize("channel,leaky", [(True, False), (True, True), (False, True)])
def test_raster(kind, t, n, channel, leaky):
    """The packed spikes of a run as input: the same as the unpacked ones."""
    import torch
    rng = np.random.default_rng(n)
    spikes = rng.random((2, t, n)) < 0.1
    words = np.zeros((2, t, (n + 31) // 32 * 32), np.uint8)
    words[:, :, :n] = spikes
    packed = np.packbits(words, axis=-1, bitorder="little").view(np.uint32)
    xw = torch.from_numpy(packed.view(np.int32)).cuda()
    xf = torch.from_numpy(spikes.astype(np.float32)).to(dt(kind)).cuda()
    gate = gate_of(rng, (n,), "f32", False) if channel else gate_of(rng, (2, t, n), kind, False)
    dy = make(rng, (2, t, n), kind)
    y, h, saved = snn.leaky_scan(gate, xw, leaky=leaky, dtype=dt(kind), save=True)
    y1, h1, saved1 = snn.leaky_scan(gate, xf, leaky=leaky, save=True)
    assert same(y, y1) and same(h, h1)
    dgate, dx, dh0 = snn.leaky_scan_grad(gate, xw, dy, saved, leaky=leaky)
    dgate1, _, dh1 = snn.leaky_scan_grad(gate, xf, dy, saved1, leaky=leaky)
    assert dx is None and same(dgate, dgate1) and same(dh0, dh1)
    yu, _ = snn.leaky_scan(gate, xw.view(torch.uint32), leaky=leaky, dtype=dt(kind))
    assert same(yu, y)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_state_in_place_and_in_pieces(kind):
    """Steps one by one, and pieces, with the state carried in place, follow the whole scan."""
    import torch
    rng = np.random.default_rng(21)
    b, t, d = 3, 40, 77
    gate, x = make(rng, (b, t, d), kind, 2.0, 1.0), make(rng, (b, t, d), kind)
    h0 = make(rng, (b, d), "f32")
    want = ref.scan(host(gate), host(x), host(h0), logit=True, leaky=True, kind=kind)
    for piece in (1, 3, 9, 40):
        state = h0.clone()
        for i in range(0, t, piece):
            y, h = snn.leaky_scan(gate[:, i:i + piece], x[:, i:i + piece], state, logit=True, leaky=True, h_out=state)
            assert h is state
            ref.close(host(y), want["y"][0][:, i:i + piece], want["y"][1][:, i:i + piece], kind)
        ref.close(host(state), *want["h"], "f32")


@pytest.mark.gpu
def test_partial_gradients_and_missing_ones():
    import torch
    rng = np.random.default_rng(4)
    gate, x, dy = make(rng, (2, 100, 48), "f32"), make(rng, (2, 100, 48), "f32"), make(rng, (2, 100, 48), "f32")
    dh = make(rng, (2, 48), "f32")
    _, _, saved = snn.leaky_scan(gate, x, logit=True, save=True)
    full = snn.leaky_scan_grad(gate, x, dy, saved, dh=dh, logit=True)
    for need in range(1, 8):
        k = dict(need_gate=bool(need & 1), need_x=bool(need & 2), need_h0=bool(need & 4))
        part = snn.leaky_scan_grad(gate, x, dy, saved, dh=dh, logit=True, **k)
        for i in range(3):
            assert (part[i] is None) if not need >> i & 1 else torch.equal(part[i], full[i])
    zero = snn.leaky_scan_grad(gate, x, torch.zeros_like(dy), saved, dh=dh, logit=True)
    none = snn.leaky_scan_grad(gate, x, None, saved, dh=dh, logit=True)
    assert all(torch.equal(p, q) for p, q in zip(zero, none))
    with pytest.raises(snn.SnnError):
        snn.leaky_scan_grad(gate, x, None, saved, logit=True)
    with pytest.raises(snn.SnnError):
        snn.leaky_scan_grad(gate, x, dy, saved[:-1], logit=True)
    with pytest.raises(snn.SnnError):
        snn.leaky_scan(gate.bfloat16(), x)
    with pytest.raises(snn.SnnError):
        snn.leaky_scan(gate, x[:, :, ::2])
    with pytest.raises(snn.SnnError):
        snn.leaky_scan(gate, x, h0=dh[:1])


@pytest.mark.gpu
def test_gradient_against_differences():
    """y and h are linear in x and h0: a change of them moves sum(y dy) + sum(h dh) by exactly its product with
    the gradient; both sides of the difference carry the forward's bound."""
    import torch
    rng = np.random.default_rng(8)
    b, t, d = 2, 130, 70
    gate, x, dy = make(rng, (b, t, d), "f32"), make(rng, (b, t, d), "f32"), make(rng, (b, t, d), "f32")
    h0, dh = make(rng, (b, d), "f32"), make(rng, (b, d), "f32")
    ex, eh = make(rng, (b, t, d), "f32"), make(rng, (b, d), "f32")
    for leaky in (False, True):
        how = dict(logit=True, leaky=leaky)
        y, h, saved = snn.leaky_scan(gate, x, h0, save=True, **how)
        _, dx, dh0 = snn.leaky_scan_grad(gate, x, dy, saved, dh=dh, **how)
        y2, h2 = snn.leaky_scan(gate, x + ex, h0 + eh, **how)
        moved = ((host(y2) - host(y)) * host(dy)).sum() + ((host(h2) - host(h)) * host(dh)).sum()
        ex_, eh_ = host(x + ex) - host(x), host(h0 + eh) - host(h0)  # the change after rounding
        want = (ex_ * host(dx)).sum() + (eh_ * host(dh0)).sum()
        r1 = ref.scan(host(gate), host(x), host(h0), host(dy), host(dh), kind="f32", **how)
        r2 = ref.scan(host(gate), host(x + ex), host(h0 + eh), kind="f32", **how)
        slack = sum((r["y"][1] * np.abs(host(dy))).sum() + (r["h"][1] * np.abs(host(dh))).sum() for r in (r1, r2))
        slack += (r1["dx"][1] * np.abs(ex_)).sum() + (r1["dh0"][1] * np.abs(eh_)).sum()
        slack += 2.0 ** -23 * ((np.abs(host(y)) + np.abs(host(y2))) * np.abs(host(dy))).sum() + 2.0 ** -23 * abs(want)
        assert abs(moved - want) <= slack
        # the gate: central differences in 64 bits of one direction, error of third order in the step
        e = rng.standard_normal((b, t, d))

        def loss(z):
            r = ref.scan(z, host(x), host(h0), **how)
            return (r["y"][0] * host(dy)).sum() + (r["h"][0] * host(dh)).sum()

        dgate, _, _ = snn.leaky_scan_grad(gate, x, dy, saved, dh=dh, **how)
        slope = (loss(host(gate) + 1e-4 * e) - loss(host(gate) - 1e-4 * e)) / 2e-4
        slack = ((r1["dgate"][1] + 2.0 ** -24 * np.abs(r1["dgate"][0])) * np.abs(e)).sum()
        assert abs(slope - (host(dgate) * e).sum()) <= slack + 1e-6 * np.abs(r1["dgate"][0] * e).sum()


@pytest.mark.gpu
def test_empty_calls():
    import torch
    z = torch.zeros
    y, h = snn.leaky_scan(z(3, 0, 8, device="cuda"), z(3, 0, 8, device="cuda"), torch.ones(3, 8, device="cuda"))
    assert y.shape == (3, 0, 8) and (h == 1).all()
    y, h, saved = snn.leaky_scan(z(0, 5, 8, device="cuda"), z(0, 5, 8, device="cuda"), save=True)
    assert y.shape == (0, 5, 8) and h.shape == (0, 8)
    g, dx, dh0 = snn.leaky_scan_grad(torch.ones(8, device="cuda"), z(0, 5, 8, device="cuda"),
                                     z(0, 5, 8, device="cuda"), saved)
    assert (g == 0).all() and dx.shape == (0, 5, 8) and dh0.shape == (0, 8)
    ones = torch.ones(3, 8, device="cuda")
    _, _, saved = snn.leaky_scan(z(3, 0, 8, device="cuda"), z(3, 0, 8, device="cuda"), ones, save=True)
    _, _, dh0 = snn.leaky_scan_grad(z(3, 0, 8, device="cuda"), z(3, 0, 8, device="cuda"), None, saved, dh=2 * ones)
    assert (dh0 == 2).all()


@pytest.mark.gpu
def test_captured_and_eager_on_streams():
    """Two captured training steps and an eager one on three streams, replayed with new inputs."""
    import torch
    rng = np.random.default_rng(31)
    sets = []
    for b, t, d, channel in ((2, 200, 64, False), (3, 90, 100, True)):
        gate = gate_of(rng, (d,), "f32", True) if channel else make(rng, (b, t, d), "f32")
        x, dy, h0 = make(rng, (b, t, d), "f32"), make(rng, (b, t, d), "f32"), make(rng, (b, d), "f32")

        def step(gate=gate, x=x, dy=dy, h0=h0, **k):
            y, h, saved = snn.leaky_scan(gate, x, h0, logit=True, save=True, **k)
            return (y, h) + snn.leaky_scan_grad(gate, x, dy, saved, logit=True, **k)

        step()
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=s):
            out = step()
        sets.append((g, s, step, out, (x, dy, h0)))
    for trial in range(3):
        for *_, ins in sets:
            for v in ins:
                v.copy_(make(rng, v.shape, "f32"))
        torch.cuda.synchronize()
        for g, s, *_ in sets:
            with torch.cuda.stream(s):
                g.replay()
        side = torch.cuda.Stream()
        eager = [step(stream=side) for _, _, step, _, _ in sets]
        torch.cuda.synchronize()
        for (_, _, _, out, _), e in zip(sets, eager):
            assert all(torch.equal(p, q) for p, q in zip(out, e))


@pytest.mark.gpu
def test_rows_past_32_bit_offsets():
    """A packed tensor of more than 2^31 elements: its last sequence is read and written where it lies."""
    import torch
    d, rows = 1024, (1 << 21) + 200
    x = torch.empty(rows, d, dtype=torch.bfloat16, device="cuda")
    y = torch.empty(rows, d, dtype=torch.bfloat16, device="cuda")
    x[-150:].normal_()
    y[-150:] = 0
    off = torch.tensor([rows - 150, rows], device="cuda")
    gate = torch.full((d,), 0.9, device="cuda")
    snn.leaky_scan(gate, x, offsets=off, out=y)
    want = ref.scan(host(gate), host(x[-150:])[None], np.zeros((1, d)), kind="f32")
    ref.close(host(y[-150:])[None], *want["y"], "bf16")


@pytest.mark.gpu
def test_drive_scan_chain():
    """Bytes of the stream -> drive rows -> leaky scan, and the gradient back into the table, as one step; and
    the traces of a network's own raster."""
    import torch
    b, t, d = 4, 300, 200
    tok = torch.from_numpy(snn.stream(b * t, seed=9).reshape(b, t)).cuda()
    rng = np.random.default_rng(6)
    table, tau, dy = make(rng, (256, d), "f32"), make(rng, (d,), "f32", 1.0, 2.0), make(rng, (b, t, d), "f32")
    x = snn.embed(tok, table, scale=0.25)
    y, h, saved = snn.leaky_scan(tau, x, logit=True, leaky=True, save=True)
    dtau, dx, _ = snn.leaky_scan_grad(tau, x, dy, saved, logit=True, leaky=True)
    dtable = snn.embed_grad(tok, dx, 256, scale=0.25)
    xr = ref.embed(tok.cpu().numpy().astype(np.int64), host(table), 0.25)
    want = ref.scan(host(tau), xr, np.zeros((b, d)), host(dy), None, True, True)
    ref.close(host(y), *want["y"], "f32", "y")
    ref.close(host(dtau), *want["dgate"], "f32", "dtau")
    v, bound = ref.embed_grad(tok.cpu().numpy().astype(np.int64), want["dx"][0], 256, 0.25)
    # each term of a row's sum carries the scan's bound and its rounding
    eb, _ = ref.embed_grad(tok.cpu().numpy().astype(np.int64), want["dx"][1] + ref.U * np.abs(want["dx"][0]), 256, 0.25)
    ref.close(host(dtable), v, bound + 1.01 * eb, "f32", "dtable")

    net = snn.Network(device=0, phase_offset=5000)
    net.build_columns(snn.topology(n_columns=2))
    net.set_corpus(snn.stream(2000, seed=3))
    raster, counts = net.run(120, raster=True, counts=True)
    assert counts.sum() > 0
    decay = torch.full((net.N,), float(np.exp(-1 / 20)), device="cuda")
    trace, last = snn.leaky_scan(decay, torch.from_numpy(raster.view(np.int32)).cuda()[None])
    bits = np.unpackbits(raster.view(np.uint8), axis=1, bitorder="little")[:, :net.N].astype(np.float64)
    want = ref.scan(host(decay), bits[None], np.zeros((1, net.N)))
    ref.close(host(trace), *want["y"], "f32", "trace")
    net.close()
