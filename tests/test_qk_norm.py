"""snn_qk_norm and snn_qk_norm_grad against their 64-bit forms."""
import ctypes as C

import numpy as np
import pytest

import snn_b200 as snn

KINDS = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step of a rounding


def host(t):
    return t.detach().cpu().double().numpy()


def turn(x, angle, adjacent, back):
    """Pairs of x's [.., heads, d] first elements turned by angle [.., pairs]."""
    x = x.copy()
    n = angle.shape[-1]
    if n:
        i, j = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if adjacent else (slice(0, n), slice(n, 2 * n))
        c, s = np.cos(angle)[..., None, :], np.sin(angle)[..., None, :] * (-1 if back else 1)
        a, b = x[..., i].copy(), x[..., j].copy()
        x[..., i], x[..., j] = a * c - b * s, a * s + b * c
    return x


def reference(x, w, angle, eps, unit, adjacent, dy=None):
    """(y) or (dx, dw)"""
    n = 1 if unit else x.shape[-1]
    r = 1 / np.sqrt((x ** 2).sum(-1, keepdims=True) / n + eps)
    w = np.ones(x.shape[-1]) if w is None else w
    if dy is None:
        return turn(x * r * w, angle, adjacent, False)
    z = turn(dy, angle, adjacent, True)
    dw = (z * x * r).reshape(-1, x.shape[-1]).sum(0)
    z = z * w
    return r * (z - x * r * (z * x * r).sum(-1, keepdims=True) / n), dw


def close(got, want, kind, size):
    """One rounding to the type, and 2^-20 of `size`, the magnitudes that the value is made of: a sum of up to 512 squares
    by lanes (9 levels and 8 in a row: 17 roundings of 2^-24, halved by the root), a division and a root, the products
    with weight, cosine and sine (whose angle of at most a turn is rounded to 2^-25 turns: 2^-22), one subtraction."""
    got = np.asarray(got, np.float64)
    small = 2.0 ** -25 if kind == "f16" else 0.0
    assert got.shape == want.shape and np.isfinite(got).all()
    assert (np.abs(got - want) <= HALF[kind] * np.abs(want) * 1.001 + size * 2.0 ** -20 + small).all()


def test_formula_against_differences():
    """Gradients against central differences: third order in a step of 1e-5 and 2^-52 / 1e-5 from cancellation."""
    rng = np.random.default_rng(0)
    x, w, dy, angle = rng.standard_normal((2, 3, 6)), rng.standard_normal(6), rng.standard_normal((2, 3, 6)), rng.standard_normal((2, 2))
    for unit in (False, True):
        for adjacent in (False, True):
            dx, dw = reference(x, w, angle, 1e-3, unit, adjacent, dy)
            for arr, d, f in ((x, dx, lambda v: reference(v, w, angle, 1e-3, unit, adjacent)), (w, dw, lambda v: reference(x, v, angle, 1e-3, unit, adjacent))):
                for at in np.ndindex(arr.shape):
                    e = np.zeros_like(arr)
                    e[at] = 1e-5
                    assert abs(((f(arr + e) - f(arr - e)) * dy).sum() / 2e-5 - d[at]) < 1e-7 * (1 + abs(d[at]))


# ---- refusals (CPU) ----------------------------------------------------------------
def call(grad=False, desc=(), **over):
    d = dict(type=0, flags=0, n_seq=1, n_steps=10, hq=2, hk=1, dim=8, rot=4, pos=10, eps=1e-6)
    d.update(desc)
    r = {n: ((i + 1) << 20, 160, 16, 8) for i, n in enumerate(("q", "k", "yq", "yk", "dyq", "dyk", "dq", "dk"))}
    a = dict(wq=1 << 24, wk=1 << 24, positions=1 << 25, freqs=1 << 26, dwq=1 << 27, dwk=1 << 27, work=1 << 28, bytes=1 << 30)
    for k, v in over.items():
        (r if k in r else a)[k] = v
    ro = {k: snn._HEADS.pack(v[0] or 0, *v[1:]) if v else None for k, v in r.items()}
    de, L = snn._QK.pack(*d.values()), snn.lib()
    if grad:
        return L.snn_qk_norm_grad(de, ro["q"], ro["k"], a["wq"], a["wk"], a["positions"], a["freqs"], ro["dyq"], ro["dyk"],
                                  ro["dq"], ro["dk"], a["dwq"], a["dwk"], a["work"], a["bytes"], None)
    return L.snn_qk_norm(de, ro["q"], ro["k"], a["wq"], a["wk"], a["positions"], a["freqs"], ro["yq"], ro["yk"], None)


BAD = [dict(desc=dict(type=3)), dict(desc=dict(flags=4)), dict(desc=dict(n_seq=-1)), dict(desc=dict(n_steps=-1)),
       dict(desc=dict(n_seq=1 << 20, n_steps=1 << 20)), dict(desc=dict(hq=-1)), dict(desc=dict(hk=65537)), dict(desc=dict(dim=0)),
       dict(desc=dict(dim=513)), dict(desc=dict(rot=3)), dict(desc=dict(rot=10)), dict(desc=dict(rot=-2)), dict(desc=dict(pos=8)),
       dict(desc=dict(eps=-1.0)), dict(desc=dict(eps=float("nan"))), dict(q=None), dict(k=None), dict(q=((1 << 20) + 2, 160, 16, 8)),
       dict(k=(1 << 20, 160, -16, 8)), dict(wq=2), dict(wk=(1 << 24) + 1), dict(positions=None), dict(positions=(1 << 25) + 4),
       dict(freqs=None), dict(freqs=(1 << 26) + 2)]


@pytest.mark.parametrize("over", BAD + [dict(yq=None), dict(yk=None), dict(yq=(1 << 20, 160, 16, 7)), dict(yq=(1 << 20, 160, 15, 8)),
                                        dict(yk=(1 << 20, 160, 7, 8))])
def test_refuses(over):
    assert call(**over) == 1 and b"qk_norm" in snn.lib().snn_last_error(None)


@pytest.mark.parametrize("over", BAD + [dict(dyq=None), dict(dyk=None), dict(dq=None), dict(dk=(1 << 20, 160, 7, 8)), dict(work=None),
                                        dict(work=(1 << 28) + 16), dict(bytes=8), dict(dwq=2)])
def test_grad_refuses(over):
    assert call(grad=True, **over) == 1 and b"qk_norm" in snn.lib().snn_last_error(None)


def test_null_description():
    n = C.c_int64()
    assert snn.lib().snn_qk_norm_grad_workspace(None, C.byref(n)) == 1
    assert snn.lib().snn_qk_norm_grad_workspace(snn._QK.pack(0, 0, 1, 5, 1, 1, 8, 0, 9, 0.0), None) == 1


# ---- GPU ------------------------------------------------------------------------------
def check(kind, lead, hq, hk, d, rot, unit=False, adjacent=False, weights=True, far=False, layout="fused", eps=1e-6, seed=0):
    import torch
    dt = getattr(torch, KINDS[kind])
    rng = np.random.default_rng(seed + d + rot)

    def t(*shape, mean=0.0):
        return torch.from_numpy((rng.standard_normal(shape) + mean).astype(np.float32)).cuda()

    row = t(*lead, (hq + hk) * d + (1 if layout == "odd" else 0)).to(dt)
    o = 1 if layout == "odd" else 0
    q, k = row[..., o:o + hq * d].unflatten(-1, (hq, d)), row[..., o + hq * d:].unflatten(-1, (hk, d))
    if layout == "tb":
        q, k = (v.transpose(0, 1).contiguous().transpose(0, 1) for v in (q, k))
    wq, wk = (t(d, mean=1.0), t(d, mean=1.0)) if weights else (None, None)
    pos = torch.randint(0, (1 << 31) - 1 if far else 5000, lead, device="cuda", dtype=torch.int64 if far else torch.int32)
    freqs = 10000.0 ** (-torch.arange(rot // 2, device="cuda").float() * 2 / max(rot, 1))
    rotation = dict(positions=pos, freqs=freqs) if rot else {}
    how = dict(unit=unit, adjacent=adjacent, eps=eps)
    dyq, dyk = t(*lead, hq, d).to(dt), t(*lead, hk, d).to(dt)
    angle = host(pos)[..., None] * host(freqs)
    yq, yk = snn.qk_norm(q, k, wq, wk, **rotation, **how)
    dq, dk, dwq, dwk = snn.qk_norm_grad(q, k, dyq, dyk, wq, wk, **rotation, **how)
    for x, w, y, dy, dx, dw in ((q, wq, yq, dyq, dq, dwq), (k, wk, yk, dyk, dk, dwk)):
        x, w, dy = host(x), None if w is None else host(w), host(dy)
        want = reference(x, w, angle, eps, unit, adjacent)
        size = np.sqrt((want ** 2).sum(-1, keepdims=True))
        close(host(y), want, kind, size)
        wdx, wdw = reference(x, w, angle, eps, unit, adjacent, dy)
        n = 1 if unit else d
        r = 1 / np.sqrt((x ** 2).sum(-1, keepdims=True) / n + eps)
        zw = np.sqrt((dy ** 2).sum(-1, keepdims=True)) * (1 if w is None else np.abs(w).max())
        close(host(dx), wdx, kind, r * zw * 4)
        if w is None:
            assert dw is None
        else:  # summed over all rows and heads in f32, in parts: at most 2^-20 of the magnitudes again
            z = turn(dy, angle, adjacent, True)
            close(host(dw), wdw, "f32", 4 * np.abs(z * x * r).reshape(-1, d).sum(0))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d,rot", [(1, 0), (2, 2), (5, 4), (7, 2), (32, 32), (64, 0), (100, 50), (128, 64), (128, 128), (130, 130),
                                   (256, 64), (257, 256), (510, 20), (512, 512)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_dims(kind, d, rot, adjacent):
    check(kind, (9,), 3, 2, d, rot, adjacent=adjacent)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("layout", ["fused", "odd", "tb"])
@pytest.mark.parametrize("unit,weights", [(True, False), (False, True), (True, True)])
def test_layouts(kind, layout, unit, weights):
    check(kind, (3, 50), 4, 2, 64, 32, unit=unit, weights=weights, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows", [1, 1183, 1185, 9471, 20001])
def test_rows(kind, rows):
    check(kind, (rows,), 2, 1, 24, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("adjacent", [False, True])
def test_far_positions(adjacent):
    check("f32", (300,), 1, 1, 64, 64, far=True, adjacent=adjacent)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
def test_zero_rows_and_one_side(kind):
    """A head of zeros has the norm sqrt(eps); either side may be missing, and there may be no row."""
    import torch
    x = torch.zeros(4, 2, 8, dtype=getattr(torch, KINDS[kind]), device="cuda")
    yq, none = snn.qk_norm(x, None, eps=1e-2)
    assert none is None and (yq == 0).all()
    none, yk = snn.qk_norm(None, x, eps=1e-2)
    assert none is None and (yk == 0).all()
    dy, w = torch.ones_like(x), torch.ones(8, device="cuda")
    dq, dk, dwq, dwk = snn.qk_norm_grad(x, None, dy, None, w, eps=1e-2)
    assert dk is None and dwk is None and (dwq == 0).all() and torch.allclose(dq.float(), torch.full_like(dq, 10).float())
    dq, dk, dwq, dwk = snn.qk_norm_grad(x[:0], x[:0], dy[:0], dy[:0], w, w)
    assert dq.shape == (0, 2, 8) and (dwq == 0).all() and (dwk == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
def test_in_place_streams_and_graphs(kind):
    import torch
    dt = getattr(torch, KINDS[kind])
    q, k = torch.randn(500, 4, 64, device="cuda").to(dt), torch.randn(500, 2, 64, device="cuda").to(dt)
    w = torch.rand(64, device="cuda")
    rotation = dict(positions=torch.arange(500, device="cuda"), freqs=torch.rand(16, device="cuda"))
    yq, yk = snn.qk_norm(q, k, w, None, **rotation)
    a, b = q.clone(), k.clone()
    ra, rb = snn.qk_norm(a, b, w, None, **rotation, out=(a, b))
    assert ra is a and torch.equal(a, yq) and torch.equal(b, yk)
    first = snn.qk_norm_grad(q, k, yq, yk, w, w, **rotation)
    dyq, dyk = yq.clone(), yk.clone()
    again = snn.qk_norm_grad(q, k, dyq, dyk, w, w, **rotation, out=(dyq, dyk))
    assert again[0] is dyq and all(torch.equal(x, y) for x, y in zip(first, again))  # and equal bits
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    sq, sk = snn.qk_norm(q, k, w, None, **rotation, stream=side)
    side.synchronize()
    assert torch.equal(sq, yq) and torch.equal(sk, yk)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gq, gk = snn.qk_norm(q, k, w, None, **rotation)
    q.copy_(q.flip(0))
    graph.replay()
    assert torch.equal(gq, snn.qk_norm(q, k, w, None, **rotation)[0])


@pytest.mark.gpu
def test_gradient_of_weights_that_are_ones():
    """In C a weight may be NULL and have a gradient all the same."""
    import torch
    q, dy = torch.randn(40, 3, 24, device="cuda"), torch.randn(40, 3, 24, device="cuda")
    dx, dw, work = torch.empty_like(q), torch.empty(24, device="cuda"), torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    desc = snn._QK.pack(0, 0, 1, 40, 3, 0, 24, 0, 9, 1e-6)
    rows = [snn._HEADS.pack(t.data_ptr(), 0, 72, 24) for t in (q, dy, dx)]
    assert snn.lib().snn_qk_norm_grad(desc, rows[0], None, None, None, None, None, rows[1], None, rows[2], None, dw.data_ptr(), None,
                                      work.data_ptr(), work.numel(), torch.cuda.current_stream().cuda_stream) == 0
    want = snn.qk_norm_grad(q, None, dy, None, torch.ones(24, device="cuda"))
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[2])


@pytest.mark.gpu
def test_binding_refuses():
    import torch
    q, k = torch.randn(6, 4, 8, device="cuda"), torch.randn(6, 2, 8, device="cuda")
    p, f = torch.arange(6, device="cuda"), torch.ones(2, device="cuda")
    for bad in (lambda: snn.qk_norm(None, None), lambda: snn.qk_norm(q.cpu(), k), lambda: snn.qk_norm(q, k[:5]),
                lambda: snn.qk_norm(q, k.half()), lambda: snn.qk_norm(q, k[..., :7]), lambda: snn.qk_norm(q.double(), None),
                lambda: snn.qk_norm(q, k, q_weight=torch.ones(7, device="cuda")), lambda: snn.qk_norm(q, k, positions=p),
                lambda: snn.qk_norm(q, k, positions=p, freqs=torch.ones(5, device="cuda")),
                lambda: snn.qk_norm(q, k, positions=p[:5], freqs=f), lambda: snn.qk_norm(q, k, positions=p.float(), freqs=f),
                lambda: snn.qk_norm(q.transpose(1, 2), None), lambda: snn.qk_norm(q, k, out=(k, k)),
                lambda: snn.qk_norm_grad(q, k, q, None), lambda: snn.qk_norm_grad(q, k, q.half(), k)):
        with pytest.raises(snn.SnnError):
            bad()


@pytest.mark.parametrize("over", [dict(k=None), dict(dyk=None), dict(wk=2), dict(dwk=2), dict(work=None), dict(bytes=8)])
def test_grad_refuses_before_it_writes(over):
    """No weight's gradient is written, of queries that are not there either, when an argument is refused (without a GPU
    any launch would be another error)."""
    assert call(grad=True, desc=dict(hq=0), **over) == 1
