"""snn_adamw against the formula in 64 bits, and against the same roundings."""
import numpy as np
import pytest

import snn_b200 as snn

KINDS = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def table(**over):
    t = np.zeros(1, snn._ADAMW_TENSOR)
    for k, v in dict(p=1 << 20, g=1 << 21, m=1 << 22, v=1 << 23, ms=1 << 24, vs=1 << 25, copy=0, n=100, g_type=0, copy_type=0).items():
        t[k] = over.get(k, v)
    return t


def call(t, count=1, bits=32, **over):
    r = dict(lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.01, scale=1.0, step=1, dev=0)
    r.update(over)
    return snn.lib().snn_adamw(t.ctypes.data, count, bits, snn._ADAMW_RULE.pack(*r.values()), None)


@pytest.mark.parametrize("tensor,how", [
    (dict(n=-1), {}), (dict(n=1 << 41), {}), (dict(g_type=3), {}), (dict(p=0), {}), (dict(m=0), {}), (dict(v=0), {}),
    (dict(p=(1 << 20) + 2), {}), (dict(g=(1 << 21) + 1), {}), (dict(g_type=1, g=(1 << 21) + 1), {}), (dict(m=(1 << 22) + 2), {}),
    (dict(ms=0), dict(bits=8)), (dict(vs=0), dict(bits=8)), (dict(ms=(1 << 24) + 2), dict(bits=8)),
    (dict(copy=1 << 26), {}), (dict(copy=(1 << 26) + 1, copy_type=1), {}), ({}, dict(bits=16)), ({}, dict(count=-1)),
    ({}, dict(b1=1.0)), ({}, dict(b2=-0.1)), ({}, dict(eps=-1.0)), ({}, dict(step=0)), ({}, dict(dev=4))])
def test_refuses(tensor, how):
    assert call(table(**tensor), **how) == 1 and b"adamw" in snn.lib().snn_last_error(None)


def test_refuses_null_and_nothing_to_do():
    assert snn.lib().snn_adamw(None, 1, 32, snn._ADAMW_RULE.pack(1, 0, 0, 0, 0, 1, 1, 0), None) == 1
    assert snn.lib().snn_adamw(table().ctypes.data, 1, 32, None, None) == 1
    assert snn.lib().snn_adamw(None, 0, 32, snn._ADAMW_RULE.pack(1, 0, 0, 0, 0, 1, 1, 0), None) == 0
    assert call(table(n=0)) == 0 and call(table(g=0)) == 0  # a tensor without elements or gradient


def hold(x, squared):
    """8-bit form of a moment: e4m3 values and scales for blocks of 256 (numpy f32)"""
    import torch
    y = np.sqrt(x) if squared else x
    pad = np.zeros((y.size + 255) // 256 * 256, np.float32)
    pad[:y.size] = y.ravel()
    pad = pad.reshape(-1, 256)
    scale = np.abs(pad).max(1) * np.float32(1 / np.float32(448))
    with np.errstate(all="ignore"):
        z = np.where(scale[:, None] > 0, pad / scale[:, None], np.float32(0))
    if squared:
        z = np.where(pad > 0, np.maximum(z, np.float32(2.0 ** -9)), z)
    return torch.from_numpy(z.ravel()[:y.size].reshape(x.shape).astype(np.float32)).to(torch.float8_e4m3fn), scale


def step32(p, g, m, v, n, lr, b1, b2, eps, wd, scale):
    """one operation at a time in f32, as the kernel takes them"""
    f = np.float32
    g = g * f(scale)
    m = m * f(b1) + g * f(1 - b1)
    v = v * f(b2) + g * g * f(1 - b2)
    p = p * f(1 - lr * wd) - m / (np.sqrt(v) * f(1 / np.sqrt(1 - b2 ** n)) + f(eps)) * f(lr / (1 - b1 ** n))
    return p, m, v


SHAPES = [(3, 5), (1,), (256,), (257, 33), (0,), (4097,), (2048, 2), (7,)]
HOW = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1, grad_scale=0.25)


def make(shapes, kind, seed=0):
    import torch
    rng = np.random.default_rng(seed)
    dt = getattr(torch, KINDS[kind])
    p = [torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda() for s in shapes]
    gs = [[torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(dt).cuda() for s in shapes] for _ in range(3)]
    return p, gs


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("copy", [None, "bf16", "f16"])
def test_steps(kind, bits, copy):
    """Three steps: the same bits as the formula's operations in f32, one rounding each."""
    import torch
    p, gs = make(SHAPES, kind)
    copies = None if copy is None else [torch.zeros(s, dtype=getattr(torch, KINDS[copy]), device="cuda") for s in SHAPES]
    want = [(x.cpu().numpy(), np.zeros(s, np.float32), np.zeros(s, np.float32)) for x, s in zip(p, SHAPES)]
    opt = snn.AdamW(p, bits=bits, copies=copies)
    how = dict(n=0, lr=HOW["lr"], b1=0.9, b2=0.99, eps=HOW["eps"], wd=0.1, scale=0.25)
    for n, g in enumerate(gs, 1):
        opt.step(g, n, **HOW)
        for i in range(len(SHAPES)):
            x, m, v = step32(want[i][0], g[i].float().cpu().numpy(), want[i][1], want[i][2], **(how | {"n": n}))
            if bits == 8 and x.size:
                (m8, ms), (v8, vs) = hold(m, False), hold(v, True)
                for got, w in ((opt.m[i], m8), (opt.v[i], v8)):
                    assert torch.equal(got.cpu().float(), w.float())
                assert (opt.m_scale[i].cpu().numpy() == ms).all() and (opt.v_scale[i].cpu().numpy() == vs).all()
                m = (m8.float().numpy().ravel() * np.repeat(ms, 256)[:m.size]).reshape(m.shape)
                v = (v8.float().numpy().ravel() * np.repeat(vs, 256)[:v.size]).reshape(v.shape)
                v = v * v
            elif bits == 32:
                assert (opt.m[i].cpu().numpy() == m).all() and (opt.v[i].cpu().numpy() == v).all()
            want[i] = (x, m, v)
            assert (p[i].cpu().numpy() == x).all()
            if copy:
                assert torch.equal(copies[i], p[i].to(copies[i].dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_against_64_bits(bits):
    """One step from the same moments against the formula in 64 bits: 12 roundings of 2^-24 on the way to the update;
    of the parameter itself the factor's (2^-25, just below 1), the product's and the difference's: 2.5 x 2^-24."""
    import torch
    p, gs = make([(1000, 7)], "f32", 3)
    before = p[0].cpu().double().numpy()
    opt = snn.AdamW(p, bits=bits)
    opt.step(gs[0], 5, **HOW)
    g = gs[0][0].cpu().double().numpy() * 0.25
    m, v = 0.1 * g, 0.01 * g * g
    u = HOW["lr"] * m / (1 - 0.9 ** 5) / (np.sqrt(v / (1 - 0.99 ** 5)) + 1e-6)
    want = before * (1 - 1e-3) - u
    assert (np.abs(p[0].cpu().double().numpy() - want) <= 2.5 * 2.0 ** -24 * np.abs(before) + 16 * 2.0 ** -24 * np.abs(u)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [47, 49, 401])
def test_many_tensors_and_odd_addresses(bits, count):
    """More tensors than a launch takes, at addresses of every alignment, some without a gradient."""
    import torch
    rng = np.random.default_rng(count)
    n = [int(x) for x in rng.integers(1, 700, count)]
    flat, flat_g = torch.randn(sum(n) + count, device="cuda"), torch.randn(sum(n) + count, device="cuda").bfloat16()
    at = np.concatenate([[0], np.cumsum(np.array(n) + 1)])
    p = [flat[a:a + k] for a, k in zip(at, n)]
    g = [None if i % 7 == 3 else flat_g[a:a + k] for i, (a, k) in enumerate(zip(at, n))]
    before, q = flat.clone(), [x.clone() for x in p]
    one = [snn.AdamW([x], bits=bits) for x in q]
    opt = snn.AdamW(p, bits=bits)
    opt.step(g, 1, lr=0.1)
    for i, x in enumerate(q):
        one[i].step([None if g[i] is None else g[i].clone()], 1, lr=0.1)
        assert torch.equal(p[i], x) and torch.equal(opt.m[i].float(), one[i].m[0].float()) and torch.equal(opt.v[i].float(), one[i].v[0].float())
        assert g[i] is not None or torch.equal(x, before[at[i]:at[i] + n[i]])
        assert flat[at[i] + n[i]] == before[at[i] + n[i]]  # what lies between tensors


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    """A captured step with its number on the device, replayed, is the steps themselves; and a call on another stream."""
    import torch
    p, gs = make([(300,), (2049,)], "bf16", 4)
    q = [x.clone() for x in p]
    a, b = snn.AdamW(p, bits=bits), snn.AdamW(q, bits=bits)
    n = torch.zeros(1, dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n.add_(1)
        a.step(gs[0], n, **HOW)
    side = torch.cuda.Stream()
    for i in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        b.step(gs[0], i, stream=side if i == 2 else None, **HOW)
        side.synchronize()
    for x, y in zip(p, q):  # pow on the device and on the host may differ in the last place of 64 bits
        assert ((x - y).abs() <= 2.0 ** -22 * (y.abs() + HOW["lr"])).all()


@pytest.mark.gpu
def test_zero_and_infinite_gradients():
    import torch
    for bits in (32, 8):
        p = [torch.ones(600, device="cuda")]
        opt = snn.AdamW(p, bits=bits)
        opt.step([torch.zeros(600, device="cuda")], 1, lr=0.1, weight_decay=0.5)
        assert torch.equal(p[0], torch.full_like(p[0], np.float32(1 - 0.05))) and (opt.m[0].float() == 0).all()
        g = torch.ones(600, device="cuda")
        g[300] = float("nan")
        before = p[0].clone()
        opt.step([g], 2)
        assert p[0].isnan().sum() == 1 and p[0][300].isnan() and (p[0][:300] != before[:300]).all()
        if bits == 8:  # the block that the NaN is in says so, the others go on
            assert opt.m_scale[0].isnan().tolist() == [False, True, False]


@pytest.mark.gpu
def test_binding_refuses():
    import torch
    p = [torch.zeros(10, device="cuda"), torch.zeros(4, 4, device="cuda")]
    base = torch.zeros(20, device="cuda")
    for bad in (lambda: snn.AdamW([]), lambda: snn.AdamW(p, bits=16), lambda: snn.AdamW([p[0], p[0]]),
                lambda: snn.AdamW([base[:12], base[8:]]), lambda: snn.AdamW([p[0].half()]), lambda: snn.AdamW([p[0].cpu()]),
                lambda: snn.AdamW([p[1].t()[:, :2]]), lambda: snn.AdamW(p, copies=[None]),
                lambda: snn.AdamW(p, copies=[None, torch.zeros(4, 4, device="cuda")]),
                lambda: snn.AdamW(p, moments=([p[0]], [p[0]], [], []))):
        with pytest.raises(snn.SnnError):
            bad()
    opt = snn.AdamW(p)
    moved = snn.AdamW([torch.zeros(3, device="cuda")])
    moved.params[0].data = torch.ones(3, device="cuda")
    for bad in (lambda: moved.step([torch.ones(3, device="cuda")], 1), lambda: opt.step([p[0]], 1), lambda: opt.step([p[0], p[0]], 1), lambda: opt.step([p[0].cpu(), p[1]], 1),
                lambda: opt.step([p[0], p[1].t()[:2]], 1), lambda: opt.step([p[0].double(), p[1]], 1), lambda: opt.step(p, 0),
                lambda: opt.step(p, torch.ones(1, device="cuda"))):
        with pytest.raises(snn.SnnError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_what_has_been_replaced_or_moved_is_refused(bits):
    """A step writes parameters, moments, scales and copies: none of them through an address that is no longer theirs."""
    import torch
    p = [torch.ones(300, device="cuda"), torch.ones(7, 5, device="cuda")]
    opt = snn.AdamW(p, bits=bits, copies=[None, torch.zeros(7, 5, device="cuda").half()])
    g = [torch.ones(300, device="cuda"), torch.ones(7, 5, device="cuda")]
    opt.step(g, 1)
    for name in ("m", "v", "copies", "params") + (("m_scale", "v_scale") if bits == 8 else ()):
        entries = getattr(opt, name)
        for change in ("entry", "memory", "list", "none", "length"):
            before, t = [x.clone() for x in p], entries[1]
            was = t.data
            if change == "entry":
                entries[1] = t.clone()
            elif change == "memory":
                t.data = t.clone()
            elif change == "list":
                setattr(opt, name, [None if x is None else x.clone() for x in entries])
            elif change == "none":
                entries[1] = None
            else:
                entries.append(t)
            with pytest.raises(snn.SnnError):
                opt.step(g, 2)
            assert all(torch.equal(a, b) for a, b in zip(before, p))
            t.data = was
            entries[1:] = [t]
            setattr(opt, name, entries)
    opt.copies[:] = opt.copies[::-1]
    with pytest.raises(snn.SnnError):
        opt.step(g, 2)
    opt.copies[:] = opt.copies[::-1]
    opt.m[1].copy_(opt.m[1].clone())
    opt.step(g, 2)
    assert (p[1] != 1).all()
