"""Leaky scans at the edges of what their arguments allow, each through the kernels that the sizes choose."""
import pytest

import snn_b200 as snn
from test_leaky_scan import dt

SMS = 148


def plan(b, t, d, kind, grad, packed=False):
    """The kernels that a scan of these sizes takes (t: rows in all where packed): steps, chunks, cluster, tiles,
    small (4-warp tiles) or warps."""
    width, tile = 32 if kind == "f32" else 64, 64 if grad else 128
    mean = t // max(b, 1) if packed else t
    if not grad and mean <= 8:
        return "steps"
    ctiles = -(-d // width)
    workers = min(b, max(32, 32 * SMS // ctiles))
    most = (160 if ctiles <= 8 else 48) if packed else 36 if grad else 16
    if mean >= (6144 if grad else 12288) and ctiles * b <= most:
        return "chunks"
    if ctiles * workers < (8 if packed else 2) * SMS and tile < mean:
        return "cluster"
    n = ctiles * workers
    return "tiles" if n < 3 * SMS or (not grad and n < 8 * SMS) else "small" if n < 8 * SMS else "warps"


# ---- states of 0 and decays beyond 1 ------------------------------------------------
SILENT = [("chunks", "chunks", 1, 20000, 10), ("cluster", "cluster", 1, 700, 70), ("tiles", "tiles", 320, 300, 9),
          ("tiles", "small", 500, 200, 20), ("warps", "warps", 1300, 100, 12), ("steps", "small", 600, 7, 12)]


@pytest.mark.gpu
@pytest.mark.parametrize("fwd,bwd,b,t,d", SILENT)
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("channel", [False, True])
def test_silent_channels_stay_silent(fwd, bwd, b, t, d, kind, channel):
    """Decays beyond 1 whose products overflow f32 within a warp's steps (400), a tile's (3) or a chunk's (1.125; all
    exact in bf16): a state of 0 stays 0 until the one input, at the last step, and the gradient of the one output,
    the first, reaches no later step.  Everything is exact."""
    import torch
    assert (plan(b, t, d, kind, False), plan(b, t, d, kind, True)) == (fwd, bwd)
    decays = torch.tensor([1.125, 3.0, 400.0, -3.0, 0.5, 1.0, -400.0, 2.0], device="cuda")
    row = decays.repeat(-(-d // 8))[:d]
    gate = row.clone() if channel else row.to(dt(kind)).expand(b, t, d)
    x = torch.zeros(b, t, d, dtype=dt(kind), device="cuda")
    dy = torch.zeros_like(x)
    x[:, -1] = 1.5
    dy[:, 0] = 2.0
    y, h, saved = snn.leaky_scan(gate, x, save=True)
    assert (y[:, :-1] == 0).all() and (y[:, -1] == 1.5).all() and (h == 1.5).all()
    dgate, dx, dh0 = snn.leaky_scan_grad(gate, x, dy, saved)
    assert (dx[:, 0] == 2).all() and (dx[:, 1:] == 0).all() and (dgate == 0).all()
    assert torch.equal(dh0, (2 * row).expand(b, d))
