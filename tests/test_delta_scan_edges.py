"""snn_delta_scan and snn_delta_scan_grad at the borders of what their chunks take: gates that forget everything,
sequences cut into segments, workspaces.  64-bit forms and bounds in delta_ref."""
import ctypes as C
import itertools

import numpy as np
import pytest

import delta_ref as ref
import snn_b200 as snn
from test_delta_scan import KINDS, call, host, make

GRADS = ("dq", "dk", "dv", "dgate", "dbeta", "dh0")


# ---- gates that forget -----------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("t", [5, 9, 150])
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("low", [-1e2, -103.9, -104.5, -1e4, -1e13, -1e15, -1e30, "lowest"])
def test_finite_gates_that_forget(kind, t, logit, low):
    """A gate far below zero, down to the type's lowest value, is a decay of 0 and nothing else: what comes after it
    decays by its own gates, and it gets no gradient."""
    import torch
    x, s0, dy, dh = make(21, (2, t), 1, 2, 24, 20, kind, logit)
    lowest = torch.finfo(x[3].dtype).min
    at = [0, 3, 4] if t < 64 else [0, 3, 4, 40, 63, 64, 100, 149]
    for i in at:
        x[3][0, i] = lowest if low == "lowest" else max(low, lowest)
    want = ref.run(*map(host, x), host(s0), dy=host(dy), dh=host(dh), kind=kind, logit=logit)
    y, h = snn.delta_scan(*x, s0, logit=logit)
    ref.close(host(y), want["y"], kind, "y")
    ref.close(host(h), want["h"], kind, "h")
    y, h, saved = snn.delta_scan(*x, s0, logit=logit, save=True)
    ref.close(host(y), want["y"], kind, "y")
    ref.close(host(h), want["h"], kind, "h")
    for name, g in zip(GRADS, snn.delta_scan_grad(*x, dy, saved, dh=dh, logit=logit)):
        ref.close(host(g), want[name], kind, name)
        if name == "dgate" and low not in (-1e2, -103.9):
            assert (g[0, at] == 0).all()


# ---- sequences cut into segments ---------------------------------------------------------

def sizes(packed, n_seq, n_steps, heads, dk, dv, saved):
    desc, n = snn._DELTA.pack(1, 0, n_seq, n_steps, heads, heads, dk, dv, 8 if packed else 0, 1.0, 0), C.c_int64()
    assert snn.lib().snn_delta_scan_workspace(desc, saved, C.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("n_seq,mean,heads,dk,dv", [(64, 8192, 1, 128, 16), (1, 16384, 16, 128, 128), (3, 2500, 1, 20, 36),
                                                   (50, 5000, 1, 128, 8), (12, 20000, 2, 96, 100), (64, 16400, 1, 64, 1)])
def test_workspace_of_segments(packed, n_seq, mean, heads, dk, dv):
    """A segment is 8 chunks of 64 steps at least, and a sequence has one that is not full at most: a state and the
    product of its steps each, whether the sequences are packed or not."""
    n_steps = mean * n_seq if packed else mean
    cut = sizes(packed, n_seq, n_steps, heads, dk, dv, 1)
    assert 0 < cut <= (mean * n_seq // 512 + n_seq) * heads * dk * (dv + dk) * 4 + 512
    # no more beside it than what is kept of all chunks (keys and queries, T and P: 40 kB and 1 kB of factors at most)
    assert sizes(packed, n_seq, n_steps, heads, dk, dv, 0) - cut <= (mean * n_seq // 64 + n_seq) * heads * 90000


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dk,dv", [(40, 33), (64, 100), (100, 7)])
@pytest.mark.parametrize("packed", [False, True])
def test_segments_of_odd_rows(kind, dk, dv, packed):
    """Values whose rows and heads lie at addresses of any alignment, packed sequences that begin at odd rows."""
    import torch
    lengths = [2101, 2499]
    if packed:
        off = np.concatenate([[1], 1 + np.cumsum(lengths)])
        x, s0, _, _ = make(31, (int(off[-1]) + 2,), 1, 2, dk, dv, kind, n_seq=2)
    else:
        off = None
        x, s0, _, _ = make(32, (2, 2101), 1, 2, dk, dv, kind)
    how = dict(scale=0.3)
    want = ref.run(*map(host, x), host(s0), offsets=None if off is None else off.tolist(), kind=kind, **how)
    y, h = snn.delta_scan(*x, s0, offsets=None if off is None else torch.tensor(off, device="cuda"), **how)
    ref.close(host(y), want["y"], kind, "y")
    ref.close(host(h), want["h"], kind, "h")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("lengths", [[2500], [64 * 36 + 1] * 3, [9000, 0, 3, 64 * 40, 64 * 23]])
def test_segments_with_the_state_in_place(kind, lengths):
    """h_out may be h0: the same bits as with another h, where sequences are cut, short ones and ones whose
    last segment is one chunk among them."""
    import torch
    off = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), device="cuda")
    x, s0, _, _ = make(33, (sum(lengths),), 1, 2, 64, 128, kind, n_seq=len(lengths))
    if lengths[:1] == lengths[-1:]:  # equal ones as a dense batch too
        dense = [v.unflatten(0, (len(lengths), -1)) for v in x]
        y, h = snn.delta_scan(*dense, s0)
        for _ in range(3):
            state = s0.clone()
            y2, h2 = snn.delta_scan(*dense, state, h_out=state)
            assert h2 is state and torch.equal(y2, y) and torch.equal(state, h)
    y, h = snn.delta_scan(*x, s0, offsets=off)
    for _ in range(3):
        state = s0.clone()
        y2, _ = snn.delta_scan(*x, state, offsets=off, h_out=state)
        assert torch.equal(y2, y) and torch.equal(state, h)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[2100 + 37 * i for i in range(40)], [0] * 20 + [70000] + [1] * 10, [64 * 700, 1, 640, 639, 641, 0]])
def test_segments_of_many_packed_sequences(lengths):
    """Many sequences, and very unequal ones, cut by their rows' place: the same as each sequence alone."""
    import torch
    off = np.concatenate([[700], 700 + np.cumsum(lengths)])
    x, s0, _, _ = make(34, (int(off[-1]) + 1000,), 1, 1, 32, 16, "f32", n_seq=len(lengths))
    y, h = snn.delta_scan(*x, s0, offsets=torch.tensor(off, device="cuda"))
    assert (y[:700] == 0).all() and (y[off[-1]:] == 0).all()
    _, h1, _ = snn.delta_scan(*x, s0, offsets=torch.tensor(off, device="cuda"), save=True)
    assert torch.equal(h1, h)
    for i, n in enumerate(lengths):
        if n == 0:
            assert torch.equal(h[i], s0[i])
            continue
        want = ref.run(*(host(v[off[i]:off[i + 1]][-300:]) for v in x), np.zeros((1, 1, 32, 16)), offsets=[0, min(n, 300)])
        alone = snn.delta_scan(*(v[off[i]:off[i + 1]][None] for v in x), s0[i:i + 1])
        # two ways of cutting: each is off the 64-bit form by what `far` says of its last 300 steps, which forget the rest
        far = max(want["h"][1], want["y"][1])
        assert (y[off[i]:off[i + 1]] - alone[0][0]).abs().max() <= 8 * far and (h[i] - alone[1][0]).abs().max() <= 8 * far


# ---- no sequence ---------------------------------------------------------------------------
NOTHING = {n: None for n in ("h0", "h", "dh", "dh0", "saved", "work")} | {n: (None, 0, 16, 8) for n in ("q", "k", "v", "y", "dy", "dq", "dk", "dv")}


@pytest.mark.parametrize("grad", [False, True])
def test_a_batch_of_no_sequence(grad):
    """Tensors without elements have no address: a dense batch of no sequence is nothing to do."""
    over = NOTHING | {n: (None, 400, 4) for n in ("gate", "beta", "dgate", "dbeta")}
    assert call(grad=grad, desc=dict(n_seq=0), bytes=0, sbytes=0, **over) == 0
    assert call(grad=grad, desc=dict(n_seq=1), bytes=0, sbytes=0, **over) == 1
    # rows of no sequence want neither saved nor a workspace
    assert call(grad=grad, desc=dict(n_seq=0, n_steps=500, off=4096), bytes=0, sbytes=0, saved=None, work=None) == 0
    if grad:  # (gradients of the final states of none)
        assert call(grad=True, desc=dict(n_seq=0), bytes=0, sbytes=0, **(over | dict(dy=None))) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 20])
def test_a_batch_of_no_sequence_through_the_binding(t):
    import torch
    x, s0, dy, dh = make(1, (0, t), 2, 4, 8, 12, "bf16")
    y, h, saved = snn.delta_scan(*x, s0, save=True)
    assert y.shape == (0, t, 4, 12) and h.shape == (0, 4, 8, 12)
    assert [tuple(g.shape) for g in snn.delta_scan_grad(*x, dy, saved, dh=dh)] == [
        (0, t, 2, 8), (0, t, 2, 8), (0, t, 4, 12), (0, t, 4), (0, t, 4), (0, 4, 8, 12)]
    assert snn.delta_scan_grad(*x, None, saved, dh=dh)[5].shape == s0.shape
    assert snn.delta_scan(*x)[0].shape == (0, t, 4, 12)


@pytest.mark.parametrize("over", [dict(saved=None), dict(saved=(1 << 30) + 8), dict(sbytes=64), dict(work=None), dict(bytes=64)])
def test_grad_refuses_before_it_writes(over):
    """Nothing has been launched, not even the zeros of rows of no sequence, when an argument is refused (without a GPU
    any launch would be another error)."""
    assert call(grad=True, desc=dict(off=4096, flags=snn.SCAN_ZERO, n_seq=3), **over) == 1


# ---- magnitudes ----------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("values,gradients", [(2.0 ** 80, 1.0), (2.0 ** 112, 1.0), (1.0, 2.0 ** 80), (1.0, 2.0 ** 112), (2.0 ** 55, 2.0 ** 50),
                                              (2.0 ** -40, 2.0 ** -40)])
def test_magnitudes_of_the_types(kind, values, gradients):
    """Values, states and gradients up to the magnitudes that bf16 and f32 have."""
    x, s0, dy, dh = make(41, (2, 150), 1, 2, 40, 36, kind)
    x[2], s0, dy, dh = x[2] * values, s0 * values, dy * gradients, dh * gradients
    x[0] = x[0] / 8
    want = ref.run(*map(host, x), host(s0), dy=host(dy), dh=host(dh), kind=kind)
    y, h, saved = snn.delta_scan(*x, s0, save=True)
    ref.close(host(y), want["y"], kind, "y")
    ref.close(host(h), want["h"], kind, "h")
    for name, g in zip(GRADS, snn.delta_scan_grad(*x, dy, saved, dh=dh)):
        ref.close(host(g), want[name], kind, name)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 90])
def test_states_beyond_f16(size):
    """States are f32 beside f16 tensors too; answers that are too large for f16 are infinite."""
    x, s0, _, _ = make(42, (2, 150), 1, 2, 40, 36, "f16")
    want = ref.run(*map(host, x), host(s0 * size), kind="f16")
    y, h = snn.delta_scan(*x, s0 * size)
    ref.close(host(h), want["h"], "f16", "h")
    assert not np.isnan(host(y)).any()


# ---- gradients of bf16 tensors: U and R in two pieces ------------------------------------------
def roundings(pieces):
    """delta_ref.rounded for S, D, U and R in turn (its order): 8 bits of S and D, 8 or 16 of U and R."""
    calls = itertools.count()

    def rounded(x, kind):
        bits = 8 if next(calls) % 4 < 2 or pieces == 1 else 16
        m, e = np.frexp(x)
        return np.ldexp(np.rint(np.ldexp(m, bits)), e - bits)
    return rounded


@pytest.mark.gpu
def test_pieces_of_bf16_gradients(monkeypatch):
    """The errors' 2-norms, over 512 to 65,536 elements of them steady to some per cent, are those of the model whose U
    and R have two pieces and not one: nearer to the first, which is 1.3 to 1.4 times less."""
    x, s0, dy, dh = make(51, (1, 256), 2, 2, 64, 64, "bf16")
    a = [host(v)[0] for v in x]
    how = dict(dy=host(dy)[0], dh=host(dh)[0])
    want = ref.scan(*a, host(s0)[0], **how)
    bf16 = lambda v: np.ldexp(np.rint(np.ldexp(np.frexp(v)[0], 8)), np.frexp(v)[1] - 8)  # noqa: E731
    off = {}
    for pieces in (1, 2):
        monkeypatch.setattr(ref, "rounded", roundings(pieces))
        got = ref.model(*a, host(s0)[0], kind="bf16", **how)
        off[pieces] = {n: np.linalg.norm(bf16(got[n]) - want[n]) for n in GRADS[:5]}
    _, _, saved = snn.delta_scan(*x, s0, save=True)
    for name, g in zip(GRADS[:5], snn.delta_scan_grad(*x, dy, saved, dh=dh)):
        err = np.linalg.norm(host(g)[0] - want[name])
        if name == "dv":  # (made before they are kept: its own rounding alone)
            assert err <= 1.05 * off[2][name]
        else:
            assert off[1][name] > 1.2 * off[2][name] and err < (off[1][name] * off[2][name]) ** 0.5, (name, err, off)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("v,h0,dy,dh,q,late", [
    (2.0 ** 100, 2.0 ** -75, 1.0, 1.0, 1.0, 0.0),     # large values meet a state that is next to nothing
    (2.0 ** 100, 2.0 ** -75, 2.0 ** -30, 1.0, 1.0, 70),  # .. after some chunks without values
    (1.0, 1.0, 2.0 ** 90, 2.0 ** -80, 1.0, 0.0),      # and backwards
    (1.0, 1.0, 2.0 ** -70, 2.0 ** 60, 2.0 ** -20, 0.0),  # small gradients of answers beside large ones of states
    (1.0, 2.0 ** 60, 2.0 ** -60, 1.0, 1.0, 140)])
def test_magnitudes_far_apart(kind, v, h0, dy, dh, q, late):
    """A scale that brings out what is small does not lose what is large beside it."""
    x, s0, g, d1 = make(43, (1, 200), 1, 1, 40, 36, kind)
    x[2], s0, g, d1, x[0] = x[2] * v, s0 * h0, g * dy, d1 * dh, x[0] * q
    if late:
        x[2][:, :int(late)] = 0
    want = ref.run(*map(host, x), host(s0), dy=host(g), dh=host(d1), kind=kind)
    y, h, saved = snn.delta_scan(*x, s0, save=True)
    ref.close(host(y), want["y"], kind, "y")
    ref.close(host(h), want["h"], kind, "h")
    for name, grad in zip(GRADS, snn.delta_scan_grad(*x, g, saved, dh=d1)):
        ref.close(host(grad), want[name], kind, name)


@pytest.mark.gpu
@pytest.mark.parametrize("rate", [-60.0, -80.0])
def test_large_states_and_rates_next_to_nothing(rate):
    x, s0, _, _ = make(44, (1, 200), 1, 1, 40, 36, "bf16", logit=True)
    x[4][:] = rate
    s0 = s0 * 2.0 ** 60
    want = ref.run(*map(host, x), host(s0), kind="bf16", logit=True)
    y, h = snn.delta_scan(*x, s0, logit=True)
    ref.close(host(y), want["y"], "bf16", "y")
    ref.close(host(h), want["h"], "bf16", "h")
