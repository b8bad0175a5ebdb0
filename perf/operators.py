"""What is measured of the token-drive and leaky-scan operators.

embed            out[i] = scale * table[token[i]]
embed_grad       dtable[v] = scale * sum of dy[i] over the positions i with token v
leaky_scan       h_t = a_t h_{t-1} + u_t along each sequence, u = x or (1 - a) x
leaky_scan_grad  the same and its gradients (forward + backward of one training step)

`own = False` computes them in their plain form (elementary torch operations in
32 bits, rounded once), `own = True` through this repository's entry points.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INT = {"u8": torch.uint8, "i32": torch.int32, "i64": torch.int64}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "u8": 1, "i32": 4, "i64": 8}
VOCAB = 20999  # code points the synthetic stream draws from: U+4E00..U+9FFF and seven ASCII characters


def _own():
    if "snn_b200" not in sys.modules:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pure-snn-language_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import snn_b200  # noqa: F401
    return sys.modules["snn_b200"]


def listed():
    return [
        # the drive of one step for 64 parallel byte streams: latency
        {"name": "embed-step", "op": "embed", "n": 64, "vocab": 256, "d": 1000, "tok": "u8", "table": "bf16", "out": "bf16"},
        # a batch of code points into one column of 1,000 neurons, f32 master table
        {"name": "embed-codepoints", "op": "embed", "n": 16384, "vocab": VOCAB, "d": 1000, "tok": "i64", "table": "f32", "out": "bf16"},
        # a quarter of the 1 MB corpus as bytes
        {"name": "embed-corpus", "op": "embed", "n": 262144, "vocab": 256, "d": 2048, "tok": "u8", "table": "bf16", "out": "bf16"},
        # gradient of a short batch of bytes: launch latency
        {"name": "embed_grad-short", "op": "embed_grad", "n": 512, "vocab": 256, "d": 500, "tok": "u8", "dy": "f32", "out": "f32"},
        # gradient of a code-point batch: most of the vocabulary does not occur
        {"name": "embed_grad-codepoints", "op": "embed_grad", "n": 16384, "vocab": VOCAB, "d": 1000, "tok": "i32", "dy": "bf16", "out": "f32"},
        # gradient of a corpus of bytes: few rows with very many positions each
        {"name": "embed_grad-corpus", "op": "embed_grad", "n": 262145, "vocab": 256, "d": 2048, "tok": "u8", "dy": "bf16", "out": "bf16"},
        # one step of 64 streams with their state in place
        {"name": "scan-step", "op": "scan", "b": 64, "t": 1, "d": 2048, "x": "bf16", "gate": "step", "logit": True, "leaky": True, "packed": False},
        # the leaky traces of all 55,000 neurons over 1,000 steps of the spike raster
        {"name": "scan-raster", "op": "scan", "b": 1, "t": 1000, "d": 55000, "x": "bits", "gate": "channel", "logit": False, "leaky": False, "packed": False},
        # one long f32 sequence over a column of 1,000 neurons
        {"name": "scan-long", "op": "scan", "b": 1, "t": 50021, "d": 1000, "x": "f32", "gate": "step", "logit": True, "leaky": True, "packed": False},
        # a training step on short windows, gates given as decays
        {"name": "scan_grad-windows", "op": "scan_grad", "b": 32, "t": 100, "d": 500, "x": "f16", "gate": "step", "logit": False, "leaky": False, "packed": False},
        # a training step on documents of unequal length, an odd channel count, learnable time constants
        {"name": "scan_grad-documents", "op": "scan_grad", "b": 24, "t": 40003, "d": 1001, "x": "bf16", "gate": "channel", "logit": True, "leaky": True, "packed": True},
        # a training step of a large batch
        {"name": "scan_grad-batch", "op": "scan_grad", "b": 16, "t": 4096, "d": 2048, "x": "bf16", "gate": "step", "logit": True, "leaky": True, "packed": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "scan", "scan_grad"])
    if op in ("embed", "embed_grad"):
        d = _log(rng, 32, 4096)
        n = min(_log(rng, 1, 400000), (1 << 29) // d)
        vocab = rng.choice([256, _log(rng, 2, 40000)])
        tok = rng.choice(["u8", "i32", "i64"]) if vocab <= 256 else rng.choice(["i32", "i64"])
        case = {"op": op, "n": n, "vocab": vocab, "d": d, "tok": tok}
        case.update({"table" if op == "embed" else "dy": rng.choice(list(DT)), "out": rng.choice(list(DT))})
        return case
    d = _log(rng, 16, 8192)
    t = _log(rng, 1, 60000)
    b = min(_log(rng, 1, 256), max(1, (1 << 26) // (d * t)))
    t = max(1, min(t, (1 << 26) // (d * b)))
    gate = rng.choice(["step", "step", "channel"])
    x = rng.choice(["f32", "bf16", "f16"] + (["bits"] if gate == "channel" and op == "scan" else []))
    packed = x != "bits" and rng.random() < 0.4
    return {"op": op, "b": b, "t": t * b if packed else t, "d": d, "x": x, "gate": gate,
            "logit": rng.random() < 0.6, "leaky": rng.random() < 0.5, "packed": packed}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tokens(case, g):
    """Zipf(1.1) ranks, each rank a token through a permutation: how bytes and code points occur in the stream."""
    p = torch.arange(1, case["vocab"] + 1, device="cuda", dtype=torch.float64) ** -1.1
    cdf = torch.cumsum(p / p.sum(), 0)
    u = torch.rand(case["n"], generator=g, device="cuda", dtype=torch.float64)
    rank = torch.searchsorted(cdf, u).clamp_(max=case["vocab"] - 1)
    return torch.randperm(case["vocab"], generator=g, device="cuda")[rank].to(INT[case["tok"]])


def prepare(case, seed):
    g = _generator(seed)

    def normal(*shape, dt="f32", mean=0.0, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(DT[dt])

    s = {"case": case}
    if case["op"] in ("embed", "embed_grad"):
        s["tokens"] = _tokens(case, g)
        s["scale"] = math.sqrt(case["d"])
        if case["op"] == "embed":
            s["table"] = normal(case["vocab"], case["d"], dt=case["table"], std=0.02)
        else:
            s["dy"] = normal(case["n"], case["d"], dt=case["dy"])
        return s
    b, t, d = case["b"], case["t"], case["d"]
    lead = (t,) if case["packed"] else (b, t)
    if case["packed"]:
        cuts = torch.randint(0, t + 1, (b + 1,), generator=g, device="cuda").sort().values
        cuts[0], cuts[-1] = 0, t
        s["offsets"] = cuts
    gshape, gtype = ((d,), "f32") if case["gate"] == "channel" else (lead + (d,), case["x"])
    # time constants from a fraction of a step to 400 steps
    if case["logit"]:
        s["gate"] = normal(*gshape, mean=2.5, std=1.5).clamp_(max=6.0).to(DT[gtype])
    else:
        s["gate"] = (1 - torch.exp(normal(*gshape, mean=-2.5, std=1.2).clamp_(-6.0, 0.0))).to(DT[gtype])
    if case["x"] == "bits":  # about 2 % of the neurons spike at a step
        spikes = torch.rand(lead + ((d + 31) // 32, 32), generator=g, device="cuda") < 0.02
        word = (spikes.long() << torch.arange(32, device="cuda")).sum(-1)
        s["x"] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
    else:
        s["x"] = normal(*lead, d, dt=case["x"])
    s["h0"] = normal(b, d)
    if case["op"] == "scan_grad":
        s["dy"] = normal(*lead, d, dt=case["x"])
        s["dh"] = normal(b, d)
    return s


def run(s):
    if own:
        return _run_own(s)
    return _run_plain(s)


def _run_own(s):
    snn, c = _own(), s["case"]
    if c["op"] == "embed":
        return snn.embed(s["tokens"], s["table"], scale=s["scale"], dtype=DT[c["out"]])
    if c["op"] == "embed_grad":
        return snn.embed_grad(s["tokens"], s["dy"], c["vocab"], scale=s["scale"], dtype=DT[c["out"]])
    how = {"logit": c["logit"], "leaky": c["leaky"], "offsets": s.get("offsets")}
    if c["op"] == "scan":
        y, h = snn.leaky_scan(s["gate"], s["x"], s["h0"], **how)
        return {"y": y, "h": h}
    y, h, saved = snn.leaky_scan(s["gate"], s["x"], s["h0"], save=True, **how)
    dgate, dx, dh0 = snn.leaky_scan_grad(s["gate"], s["x"], s["dy"], saved, dh=s["dh"], **how)
    return {"y": y, "h": h, "dgate": dgate, "dx": dx, "dh0": dh0}


def _doubling(a, u):
    """h_t = a_t h_{t-1} + u_t along dim 1 from h = 0: spans of 1, 2, 4, .. steps are joined."""
    span, t = 1, u.shape[1]
    while span < t:
        u = torch.cat([u[:, :span], u[:, span:] + a[:, span:] * u[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return u


def _bits(words, d):
    b = (words.unsqueeze(-1) >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1
    return b.reshape(words.shape[:-1] + (-1,))[..., :d].float()


def _run_plain(s):
    c = s["case"]
    if c["op"] == "embed":
        return (s["table"][s["tokens"].long()].float() * s["scale"]).to(DT[c["out"]])
    if c["op"] == "embed_grad":
        acc = torch.zeros(c["vocab"], c["d"], device="cuda")
        acc.index_add_(0, s["tokens"].long(), s["dy"].float())
        return (acc * s["scale"]).to(DT[c["out"]])
    d, packed, h0, ydt = c["d"], c["packed"], s["h0"], torch.float32 if c["x"] == "bits" else DT[c["x"]]
    x = _bits(s["x"], d) if c["x"] == "bits" else s["x"].float()
    gate = s["gate"].float()
    a, k = (torch.sigmoid(gate), torch.sigmoid(-gate)) if c["logit"] else (gate, 1 - gate)
    if c["gate"] == "channel":
        a_all, k = a.expand(x.shape), k.expand(x.shape)
    else:
        a_all = a
    if packed:  # one row of sequences: a sequence's first step takes its state as input and keeps nothing of the one before
        x, a_all, k = x[None], a_all[None], k[None]
        off = s["offsets"]
        some = off[1:] > off[:-1]
        first, last = torch.where(some, off[:-1], 0), torch.where(some, off[1:] - 1, 0)
        zero = torch.zeros((), device="cuda")
        start = torch.where(some[:, None], a_all[0, first] * h0, zero)
    u = k * x if c["leaky"] else x
    at = a_all.clone()
    if packed:
        u = u.clone() if u is x else u
        u[0].index_add_(0, first, start)
        at[0].index_fill_(0, first, 0.0)  # row 0 is a first row too
    else:
        u = u.clone() if u is x else u
        u[:, 0] += a_all[:, 0] * h0
    h = _doubling(at, u)
    end = torch.where(some[:, None], h[0, last], h0) if packed else h[:, -1]
    y = h.to(ydt)
    if c["op"] == "scan":
        return {"y": y[0] if packed else y, "h": end.clone()}
    dy = s["dy"].float()
    if packed:
        dy = dy[None].clone()
        dy[0].index_add_(0, last, torch.where(some[:, None], s["dh"], zero))
    else:
        dy = dy.clone() if dy is s["dy"] else dy
        dy[:, -1] += s["dh"]
    after = torch.cat([at[:, 1:], torch.zeros_like(at[:, :1])], 1)
    g = _doubling(after.flip(1), dy.flip(1)).flip(1)
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    if packed:
        before[0].index_fill_(0, first, 0.0)
        before[0].index_add_(0, first, torch.where(some[:, None], h0, zero))
        dh0 = torch.where(some[:, None], a_all[0, first] * g[0, first], s["dh"])
    else:
        before[:, 0] = h0
        dh0 = a_all[:, 0] * g[:, 0]
    da = g * (before - x if c["leaky"] else before)
    if c["logit"]:
        da = da * (a_all * k)
    dx = g * k if c["leaky"] else g
    if c["gate"] == "channel":
        dgate = da.sum((0, 1))
    else:
        dgate = (da[0] if packed else da).to(DT[c["x"]])
    return {"y": y[0] if packed else y, "h": end.clone(), "dgate": dgate, "dx": (dx[0] if packed else dx).to(DT[c["x"]]), "dh0": dh0}


def work(case):
    if case["op"] in ("embed", "embed_grad"):
        n, v, d = case["n"], case["vocab"], case["d"]
        if case["op"] == "embed":
            p = np.arange(1, v + 1, dtype=np.float64) ** -1.1
            rows = float((1 - (1 - p / p.sum()) ** n).sum())  # rows expected to occur
            moved = rows * d * SIZE[case["table"]] + n * d * SIZE[case["out"]]
        else:
            moved = n * d * SIZE[case["dy"]] + v * d * SIZE[case["out"]]
        return {"bytes": moved + n * SIZE[case["tok"]], "flops": n * d}
    rows = case["t"] if case["packed"] else case["b"] * case["t"]
    e, state = rows * case["d"], 4 * case["b"] * case["d"]
    x = 1 / 8 if case["x"] == "bits" else SIZE[case["x"]]
    y = 4 if case["x"] == "bits" else x
    gate, gates = (0, 4 * case["d"]) if case["gate"] == "channel" else (x, 0)
    moved = e * (gate + x + y) + 2 * state + gates
    flops = 4 * e
    if case["op"] == "scan_grad":
        moved += e * (gate + x + y + x + gate) + 2 * state + 2 * gates
        flops += 8 * e
    return {"bytes": moved, "flops": flops}


def exact(case, seed):
    """From the definition in 64 bits, a step at a time."""
    s = prepare(case, seed)
    if case["op"] == "embed":
        return s["scale"] * s["table"].double().index_select(0, s["tokens"].long())
    if case["op"] == "embed_grad":  # rows sorted by token, runs of them as differences of running sums
        tok, order = torch.sort(s["tokens"].long(), stable=True)
        count = torch.bincount(tok, minlength=case["vocab"])
        upto = torch.cumsum(count, 0)
        out = torch.empty(case["vocab"], case["d"], dtype=torch.float64, device="cuda")
        width = max(1, (1 << 27) // max(1, case["n"]))
        for c0 in range(0, case["d"], width):
            run_sum = torch.zeros(case["n"] + 1, min(width, case["d"] - c0), dtype=torch.float64, device="cuda")
            torch.cumsum(s["dy"][:, c0:c0 + width].double()[order], 0, out=run_sum[1:])
            out[:, c0:c0 + width] = run_sum[upto] - run_sum[upto - count]
        return out * s["scale"]
    d = case["d"]
    if case["packed"]:
        off = s["offsets"].tolist()
    else:
        off = [i * case["t"] for i in range(case["b"] + 1)]
    length = [e - b for b, e in zip(off, off[1:])]
    if max(length) > 70000:
        return None
    # all sequences advance together, the longest first, so that the ones with a step t are the first rows
    order = sorted(range(case["b"]), key=lambda i: -length[i])
    begin = torch.tensor([off[i] for i in order], device="cuda")
    active = np.searchsorted(-np.array([length[i] for i in order]), -np.arange(max(length)), side="left").tolist()
    idx = torch.tensor(order, device="cuda")

    def flat(v):
        return v.reshape(-1, v.shape[-1])

    x_all = flat(s["x"])
    rows = x_all.shape[0]
    per_step = case["gate"] == "step"
    gate_all = flat(s["gate"]) if per_step else s["gate"].double()
    shift = torch.arange(d, device="cuda")

    def x_at(r):
        if case["x"] == "bits":
            return ((x_all[r][:, shift // 32].long() >> (shift % 32)) & 1).double()
        return x_all[r].double()

    def decay(z):
        if case["logit"]:
            return 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
        return z, 1 - z

    const = None if per_step else decay(gate_all)
    h = s["h0"].double()[idx]
    hist = torch.empty(rows, d, dtype=torch.float64, device="cuda")
    for t, m in enumerate(active):
        r = begin[:m] + t
        a, k = decay(gate_all[r].double()) if per_step else const
        xt = x_at(r)
        h[:m] = a * h[:m] + (k * xt if case["leaky"] else xt)
        hist[r] = h[:m]
    end = torch.empty_like(h)
    end[idx] = h
    shape = s["x"].shape[:-1] + (d,)
    out = {"y": hist.reshape(shape), "h": end}
    if case["op"] == "scan":
        return out
    dx = torch.empty(rows, d, dtype=torch.float64, device="cuda")
    dgate = torch.empty(rows, d, dtype=torch.float64, device="cuda") if per_step else torch.zeros(d, dtype=torch.float64, device="cuda")
    dy_all, h0 = flat(s["dy"]), s["h0"].double()[idx]
    carry = s["dh"].double()[idx]
    for t in reversed(range(len(active))):
        m = active[t]
        r = begin[:m] + t
        a, k = decay(gate_all[r].double()) if per_step else const
        g = dy_all[r].double() + carry[:m]
        past = hist[r - 1] if t else h0[:m]
        da = g * (past - x_at(r)) if case["leaky"] else g * past
        if case["logit"]:
            da = da * a * k
        if per_step:
            dgate[r] = da
        else:
            dgate += da.sum(0)
        dx[r] = k * g if case["leaky"] else g
        carry[:m] = a * g
    dh0 = torch.empty_like(carry)
    dh0[idx] = carry
    return out | {"dgate": dgate.reshape(shape) if per_step else dgate, "dx": dx.reshape(shape), "dh0": dh0}
