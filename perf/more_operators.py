"""What is measured of the delta-rule scan, the norms of queries and keys, and the AdamW step.

delta_scan       S' = a_t S, u = b_t (v_t - S'^T k_t), S = S' + k_t u^T, y_t = scale S^T q_t along each sequence
delta_scan_grad  the same and its gradients (forward + backward of one training step)
qk_norm          y = x / sqrt(mean x^2 + eps) * w for each head of q and k (unit: the sum in place of the
                 mean), then the position rotation of pairs
qk_norm_grad     its gradients (dq, dk and those of the weights)
adamw            one AdamW step over many tensors, moments in 32 or 8 bits

`own = False` computes them in their plain form (elementary torch operations in
32 bits, rounded once), `own = True` through this repository's entry points.
"""
import math
import os
import sys

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
VOCAB = 20999  # code points the synthetic stream draws from
BLOCK = 256    # elements of a scale of 8-bit moments


def _own():
    if "snn_b200" not in sys.modules:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pure-snn-language_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import snn_b200  # noqa: F401
    return sys.modules["snn_b200"]


def listed():
    return [
        # one token of 64 parallel byte streams, the state carried in place: latency
        {"name": "delta-step", "op": "delta", "b": 64, "t": 1, "hk": 8, "h": 8, "dk": 128, "dv": 128, "x": "bf16", "logit": False, "packed": False},
        # a batch of prompts, two value heads to a key head
        {"name": "delta-prompts", "op": "delta", "b": 8, "t": 2048, "hk": 8, "h": 16, "dk": 128, "dv": 128, "x": "bf16", "logit": False, "packed": False},
        # one long document
        {"name": "delta-long", "op": "delta", "b": 1, "t": 16384, "hk": 16, "h": 16, "dk": 128, "dv": 128, "x": "f16", "logit": True, "packed": False},
        # windows of 100 steps of a small net in f32, states and their gradients carried
        {"name": "delta_grad-windows", "op": "delta_grad", "b": 32, "t": 100, "hk": 4, "h": 4, "dk": 50, "dv": 60, "x": "f32", "logit": True, "packed": False},
        # documents of unequal length packed into one batch
        {"name": "delta_grad-documents", "op": "delta_grad", "b": 12, "t": 20003, "hk": 4, "h": 8, "dk": 96, "dv": 100, "x": "bf16", "logit": False, "packed": True},
        # a training batch
        {"name": "delta_grad-batch", "op": "delta_grad", "b": 8, "t": 4096, "hk": 16, "h": 16, "dk": 128, "dv": 128, "x": "bf16", "logit": False, "packed": False},
        # one token of 64 streams
        {"name": "norm-step", "op": "norm", "n": 64, "hq": 16, "hk": 8, "d": 128, "rot": 64, "x": "bf16", "unit": False, "pairs": "halves"},
        # a quarter of the corpus: heads of a small model, unit keys for the delta rule
        {"name": "norm-corpus", "op": "norm", "n": 65536, "hq": 16, "hk": 16, "d": 128, "rot": 128, "x": "bf16", "unit": True, "pairs": "halves"},
        # gradients of a training batch of code points, heads of an odd multiple, f32
        {"name": "norm_grad-batch", "op": "norm_grad", "n": 32768, "hq": 15, "hk": 5, "d": 100, "rot": 50, "x": "f32", "unit": False, "pairs": "adjacent"},
        # drive table, time constants and readout of one column: latency
        {"name": "adamw-column", "op": "adamw", "vocab": 256, "d": 500, "layers": 1, "bits": 32, "grad": "f32", "copy": False},
        # a model of 24 layers over the code points, 16-bit gradients and 16-bit copies for the next forward pass
        {"name": "adamw-model", "op": "adamw", "vocab": VOCAB, "d": 1000, "layers": 24, "bits": 32, "grad": "bf16", "copy": True},
        # the same with moments in 8 bits
        {"name": "adamw-model8", "op": "adamw", "vocab": VOCAB, "d": 1000, "layers": 24, "bits": 8, "grad": "bf16", "copy": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["delta", "delta", "delta_grad", "delta_grad", "norm", "norm_grad", "adamw"])
    x = rng.choice(list(DT))
    if op in ("norm", "norm_grad"):
        d = rng.choice([32, 64, 100, 128, _log(rng, 4, 256)])
        hk = _log(rng, 1, 16)
        hq = hk * rng.choice([1, 2, 4])
        n = min(_log(rng, 1, 65536), max(1, (1 << 27) // (d * (hq + hk))))
        return {"op": op, "n": n, "hq": hq, "hk": hk, "d": d, "rot": 2 * rng.randint(0, d // 2), "x": x,
                "unit": rng.random() < 0.5, "pairs": rng.choice(["halves", "adjacent"])}
    if op == "adamw":
        return {"op": op, "vocab": rng.choice([256, _log(rng, 2, VOCAB)]), "d": _log(rng, 8, 1000), "layers": rng.randint(1, 24),
                "bits": rng.choice([32, 8]), "grad": x, "copy": rng.random() < 0.5}
    dk, dv = rng.choice([64, 128, _log(rng, 8, 128)]), rng.choice([64, 128, _log(rng, 8, 200)])
    hk = rng.choice([1, 2, 4, 8, 16])
    h = hk * rng.choice([1, 1, 2, 3])
    most = (1 << 32) if op == "delta" else (1 << 31)
    t = _log(rng, 1, 16384)
    b = min(_log(rng, 1, 64), max(1, most // (h * dk * dv * t)))
    t = max(1, min(t, most // (h * dk * dv * b)))
    packed = rng.random() < 0.4
    return {"op": op, "b": b, "t": t * b if packed else t, "hk": hk, "h": h, "dk": dk, "dv": dv, "x": x,
            "logit": rng.random() < 0.5, "packed": packed}


def _shapes(case):
    """Tensors of a model over `vocab` tokens: the drive table, for each layer a projection, a readout, a norm's
    weights and the time constants, and the bias of the answer (of an odd size)."""
    d = case["d"]
    return [(case["vocab"], d)] + [(d, d), (d, d), (d,), (d // 4 + 1,)] * case["layers"] + [(2 * d + 1,)]


def _room(shape):
    """Elements of a buffer that a tensor takes: whole blocks, so that each begins with a scale of its own."""
    return (math.prod(shape) + BLOCK - 1) // BLOCK * BLOCK


def _parts(case, x, scales):
    """The tensors, or their scales, in a buffer of all."""
    shapes = _shapes(case)
    if x.numel() == 0:
        return [x] * len(shapes)
    rooms = x.split([_room(z) // (BLOCK if scales else 1) for z in shapes])
    return list(rooms) if scales else [r[:math.prod(z)].view(z) for r, z in zip(rooms, shapes)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dt="f32", mean=0.0, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(DT[dt])

    s = {"case": case}
    if case["op"] in ("norm", "norm_grad"):
        n, hq, hk, d = case["n"], case["hq"], case["hk"], case["d"]
        # queries, keys and values of one projection, a row each
        row = normal(n, (hq + 2 * hk) * d, dt=case["x"], std=2.0)
        s["q"] = row[:, :hq * d].view(n, hq, d)
        s["k"] = row[:, hq * d:(hq + hk) * d].view(n, hk, d)
        if not case["unit"]:
            s["wq"], s["wk"] = normal(d, mean=1.0, std=0.1), normal(d, mean=1.0, std=0.1)
        if case["rot"]:
            s["positions"] = torch.randint(0, 100000, (1,), generator=g, device="cuda") + torch.arange(n, device="cuda")
            s["freqs"] = 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda").float() / case["rot"])
        if case["op"] == "norm_grad":
            s["dyq"], s["dyk"] = normal(n, hq, d, dt=case["x"]), normal(n, hk, d, dt=case["x"])
        return s
    if case["op"] == "adamw":
        # a buffer for all parameters, one for all first moments and so on, of which the tensors are parts
        n = sum(_room(z) for z in _shapes(case))
        s["all"] = {"p": normal(n, std=0.02)}
        s["all"]["m"], s["all"]["ms"] = _hold(normal(n, std=3e-4), case["bits"], False)
        s["all"]["v"], s["all"]["vs"] = _hold(normal(n, std=1e-3).square_(), case["bits"], True)
        if case["copy"]:
            s["all"]["copies"] = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
        for i, x in s["all"].items():
            s[i] = _parts(case, x, x.numel() < n)
        s["g"] = [normal(*z, dt=case["grad"], std=1e-3) for z in _shapes(case)]
        s["how"] = {"lr": 3e-4, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01, "grad_scale": 0.5}
        s["step"] = 1000
        if own:  # the optimizer that a program makes once, over its tensors
            s["opt"] = _own().AdamW(s["p"], bits=case["bits"], copies=s.get("copies"), moments=(s["m"], s["v"], s["ms"], s["vs"]))
        return s
    b, t, hk, h, dk, dv, x = (case[i] for i in ("b", "t", "hk", "h", "dk", "dv", "x"))
    lead = (t,) if case["packed"] else (b, t)
    if case["packed"]:  # documents of 0.3 to 1.7 of the mean length
        w = torch.rand(b, generator=g, device="cuda").double() * 1.4 + 0.3
        cuts = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), (torch.cumsum(w, 0) / w.sum() * t).long()])
        cuts[-1] = t
        s["offsets"] = cuts
        s["longest"] = int((cuts[1:] - cuts[:-1]).max())
    s["q"] = normal(*lead, hk, dk)
    s["k"] = normal(*lead, hk, dk)
    for i in ("q", "k"):
        s[i] = (s[i] / s[i].square().sum(-1, keepdim=True).sqrt().clamp_min(1e-6)).to(DT[x])
    s["v"] = normal(*lead, h, dv, dt=x)
    # memories from a few steps to some hundred, rates around a half
    if case["logit"]:
        s["gate"], s["beta"] = normal(*lead, h, dt=x, mean=3.5, std=1.2), normal(*lead, h, dt=x)
    else:
        s["gate"] = (-torch.exp(normal(*lead, h, mean=-3.5, std=1.0))).to(DT[x])
        s["beta"] = torch.rand(lead + (h,), generator=g, device="cuda").to(DT[x])
    s["scale"] = dk ** -0.5
    s["h0"] = normal(b, h, dk, dv, std=0.3)
    if case["op"] == "delta_grad":
        s["dy"], s["dh"] = normal(*lead, h, dv, dt=x), normal(b, h, dk, dv, std=0.1)
    return s


def run(s):
    if own:
        return _run_own(s)
    if s["case"]["op"] == "adamw":
        return _adamw(s)
    if s["case"]["op"] in ("norm", "norm_grad"):
        return _norm(s)
    return _delta(s)


def _run_own(s):
    snn, c = _own(), s["case"]
    if c["op"] == "adamw":
        s["opt"].step(s["g"], s["step"], **s["how"])
        return s["all"]
    if c["op"] in ("norm", "norm_grad"):
        how = {"positions": s.get("positions"), "freqs": s.get("freqs"), "unit": c["unit"], "adjacent": c["pairs"] == "adjacent"}
        if c["op"] == "norm":
            q, k = snn.qk_norm(s["q"], s["k"], s.get("wq"), s.get("wk"), **how)
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = snn.qk_norm_grad(s["q"], s["k"], s["dyq"], s["dyk"], s.get("wq"), s.get("wk"), **how)
        return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    a = (s["q"], s["k"], s["v"], s["gate"], s["beta"])
    how = {"scale": s["scale"], "logit": c["logit"], "offsets": s.get("offsets")}
    if c["op"] == "delta":
        y, h = snn.delta_scan(*a, s["h0"], **how)
        return {"y": y, "h": h}
    y, h, saved = snn.delta_scan(*a, s["h0"], save=True, **how)
    dq, dk, dv, dgate, dbeta, dh0 = snn.delta_scan_grad(*a, s["dy"], saved, dh=s["dh"], **how)
    return {"y": y, "h": h, "dq": dq, "dk": dk, "dv": dv, "dgate": dgate, "dbeta": dbeta, "dh0": dh0}


# ---- plain forms ---------------------------------------------------------------
def _blocks(x):
    """[blocks, BLOCK] of a tensor's elements, zeros behind the last."""
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _hold(x, bits, squared):
    """A moment as it is held: itself, or e4m3 values and a scale for each BLOCK elements, the largest magnitude
    over 448; of second moments the root is held, and a value above zero as 2^-9 at least."""
    if bits == 32:
        return x, torch.empty(0, device=x.device)
    y = _blocks(x.sqrt() if squared else x)
    scale = y.abs().amax(1) / 448
    z = torch.where(scale[:, None] > 0, y / scale[:, None], 0.0)
    if squared:
        z = torch.where(y > 0, z.clamp_min(2.0 ** -9), z)
    return z.reshape(-1)[:x.numel()].view(x.shape).to(torch.float8_e4m3fn), scale


def _held(x, scale, squared):
    if x.dtype == torch.float32:
        return x
    y = (_blocks(x.float()) * scale[:, None]).reshape(-1)[:x.numel()].view(x.shape)
    return y * y if squared else y


def _adamw(s):
    how, step, bits = s["how"], s["step"], s["case"]["bits"]
    b1, b2 = how["betas"]
    size = how["lr"] / (1 - b1 ** step)
    root = 1 / math.sqrt(1 - b2 ** step)
    for i, (p, g) in enumerate(zip(s["p"], s["g"])):
        g = g.float() * how["grad_scale"]
        m = _held(s["m"][i], s["ms"][i], False) * b1 + g * (1 - b1)
        v = _held(s["v"][i], s["vs"][i], True) * b2 + g * g * (1 - b2)
        p.copy_(p * (1 - how["lr"] * how["weight_decay"]) - m / (v.sqrt() * root + how["eps"]) * size)
        for x, old, old_scale, squared in ((m, s["m"][i], s["ms"][i], False), (v, s["v"][i], s["vs"][i], True)):
            x, scale = _hold(x, bits, squared)
            old.copy_(x)
            old_scale.copy_(scale)
        if "copies" in s:
            s["copies"][i].copy_(p)
    return s["all"]


def _turn(s, x, back):
    """The pairs (a, b) of x's first `rot` elements turned by their angles."""
    c = s["case"]
    if not c["rot"]:
        return x
    angle = s["positions"].double()[:, None] * s["freqs"].double()
    co, si = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if back:
        si = -si
    r = c["rot"]
    if c["pairs"] == "halves":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * co - b * si, a * si + b * co], -1)
    else:
        a, b = x[..., :r:2], x[..., 1:r:2]
        turned = torch.stack([a * co - b * si, a * si + b * co], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _norm(s):
    c = s["case"]
    grad, out = c["op"] == "norm_grad", {}
    for i in ("q", "k"):
        x, w = s[i].float(), s.get("w" + i)
        total = x.square().sum(-1, keepdim=True)
        n = 1 if c["unit"] else c["d"]
        r = 1 / torch.sqrt(total / n + 1e-6)
        if not grad:
            y = x * r
            out[i] = _turn(s, y if w is None else y * w, False).to(s[i].dtype)
            continue
        z = _turn(s, s["dy" + i].float(), True)
        y = x * r
        if w is not None:
            out["dw" + i] = (z * y).sum((0, 1))
            z = z * w
        out["d" + i] = (r * (z - y * ((z * y).sum(-1, keepdim=True) / n))).to(s[i].dtype)
    if grad:
        return {i: out.get(i) for i in ("dq", "dk", "dwq", "dwk")}
    return out


def _inverse(a):
    """(1 + a)^-1 of strictly lower triangular a [.., 64, 64]: the blocks of 1, 2, 4, .. on the diagonal in turn."""
    n = a.shape[-1]
    inv = torch.ones(a.shape[:-2] + (n, 1, 1), device=a.device)
    while inv.shape[-1] < n:
        w, m = inv.shape[-1], inv.shape[-3] // 2
        blocks = a.view(a.shape[:-2] + (m, 2 * w, m, 2 * w)).diagonal(dim1=-4, dim2=-2).movedim(-1, -3)
        up, low = inv[..., 0::2, :, :], inv[..., 1::2, :, :]
        off = -(low @ blocks[..., w:, :w] @ up)
        inv = torch.cat([torch.cat([up, torch.zeros_like(up)], -1), torch.cat([off, low], -1)], -2)
    return inv[..., 0, :, :]


def _delta(s):
    c = s["case"]
    grad, x, names = c["op"] == "delta_grad", DT[c["x"]], ("q", "k", "v", "gate", "beta", "h0")
    leaf = {i: s[i].float() for i in names}
    if grad:
        leaf = {i: v.detach().clone().requires_grad_() for i, v in leaf.items()}
    with torch.set_grad_enabled(grad):
        y, h = _delta_forward(s, c, leaf)
        y = y.to(x)
    if not grad:
        return {"y": y, "h": h}
    got = torch.autograd.grad([y, h], [leaf[i] for i in names], [s["dy"], s["dh"]])
    out = {"y": y.detach(), "h": h.detach(), "dh0": got[5]}
    return out | {"d" + i: d.to(x) for i, d in zip(names[:5], got)}


def _delta_forward(s, c, leaf):
    """Chunks of 64 steps: (1 + A) U = b (V - G K S) by the inverse, Y = G Q S + P U, S <- G_end S + (K')^T U."""
    b, h, group, n = c["b"], c["h"], c["h"] // c["hk"], 64
    t = s["longest"] if c["packed"] else c["t"]
    pad = -t % n
    if c["packed"]:  # rows of every sequence beside one another, padded to the longest
        first, length = s["offsets"][:-1], s["offsets"][1:] - s["offsets"][:-1]
        step = torch.arange(t + pad, device="cuda")
        there = step < length[:, None]
        at = torch.where(there, first[:, None] + step, 0)

    def rows(v):
        """[b, h, chunks, 64, ..] of a tensor of rows, zeros behind the last."""
        if c["packed"]:
            v = torch.where(there.view(there.shape + (1,) * (v.dim() - 1)), v[at], 0.0)
        else:
            v = torch.nn.functional.pad(v, (0, 0) * (v.dim() - 2) + (0, pad))
        v = v.transpose(1, 2)
        return v.reshape(v.shape[:2] + (-1, n) + v.shape[3:])

    q, k = (rows(leaf[i]).repeat_interleave(group, 1) for i in ("q", "k"))
    v = rows(leaf["v"])
    if c["logit"]:
        log_a, rate = rows(torch.nn.functional.logsigmoid(leaf["gate"])), rows(torch.sigmoid(leaf["beta"]))
    else:
        log_a, rate = rows(leaf["gate"]), rows(leaf["beta"])
    upto = log_a.double().cumsum(-1)
    low = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    between = torch.where(low, (upto[..., :, None] - upto[..., None, :]).masked_fill(~low, 0.0).exp().float(), 0.0)
    since, until = upto.exp().float()[..., None], (upto[..., -1:] - upto).exp().float()[..., None]
    whole = since[..., -1:, :]
    inv = _inverse((rate[..., None] * between * (k @ k.mT)).tril(-1))
    mix = between * (q @ k.mT)
    state, ys = leaf["h0"], []
    for i in range(k.shape[2]):
        u = inv[:, :, i] @ (rate[:, :, i, :, None] * (v[:, :, i] - since[:, :, i] * (k[:, :, i] @ state)))
        ys.append(since[:, :, i] * (q[:, :, i] @ state) + mix[:, :, i] @ u)
        state = whole[:, :, i] * state + (until[:, :, i] * k[:, :, i]).mT @ u
    y = (torch.cat(ys, 2) * s["scale"]).transpose(1, 2)
    return (y[there] if c["packed"] else y[:, :t]), state


# ---- sizes -----------------------------------------------------------------------
def work(case):
    if case["op"] in ("norm", "norm_grad"):
        e = case["n"] * (case["hq"] + case["hk"]) * case["d"]
        more = case["n"] * 8 if case["rot"] else 0
        moved = e * SIZE[case["x"]] * (3 if case["op"] == "norm_grad" else 2)
        return {"bytes": moved + more, "flops": (20 if case["op"] == "norm_grad" else 8) * e}
    if case["op"] == "adamw":
        e = sum(math.prod(z) for z in _shapes(case))
        moments = 4 if case["bits"] == 8 else 16
        return {"bytes": e * (8 + SIZE[case["grad"]] + moments + (2 if case["copy"] else 0)), "flops": 15 * e}
    b, hk, h, dk, dv = (case[i] for i in ("b", "hk", "h", "dk", "dv"))
    rows = case["t"] if case["packed"] else b * case["t"]
    size, state = SIZE[case["x"]], 4 * b * h * dk * dv
    read, write = rows * (2 * hk * dk + h * dv + 2 * h), rows * h * dv
    moved, flops = (read + write) * size + 2 * state, 6 * rows * h * dk * dv
    if case["op"] == "delta_grad":  # reads its inputs again and dy, writes gradients of the inputs' forms
        moved += (read + write + read) * size + 2 * state
        flops += 14 * rows * h * dk * dv
    return {"bytes": moved, "flops": flops}


# ---- 64 bits -----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    if case["op"] in ("norm", "norm_grad"):
        return _exact_norm(s)
    return _exact_delta(s)


def _exact_adamw(s):
    """The buffers as a whole, the room between the tensors left as it was."""
    how, step, bits, was = s["how"], s["step"], s["case"]["bits"], s["all"]
    b1, b2 = how["betas"]
    n = was["p"].numel()
    g, inside = (torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(2))
    begin = 0
    for x in s["g"]:
        g[begin:begin + x.numel()] = x.double().flatten() * how["grad_scale"]
        inside[begin:begin + x.numel()] = 1
        begin += (x.numel() + BLOCK - 1) // BLOCK * BLOCK
    inside = inside.bool()

    def old(name, squared):
        x = was[name].double()
        if bits == 8:
            x = (x.view(-1, BLOCK) * was[name + "s"].double()[:, None]).flatten()
            x = x * x if squared else x
        return x

    out = {}
    m, v = b1 * old("m", False) + (1 - b1) * g, b2 * old("v", True) + (1 - b2) * g ** 2
    mean, var = m / (1 - b1 ** step), v / (1 - b2 ** step)
    p = was["p"].double()
    new = p - how["lr"] * (mean / (var ** 0.5 + how["eps"]) + how["weight_decay"] * p)
    out["p"] = torch.where(inside, new, p)
    if "copies" in was:
        out["copies"] = torch.where(inside, new, was["copies"].double())
    for name, x in (("m", m), ("v", v)):
        if bits == 32:
            out[name], out[name + "s"] = torch.where(inside, x, was[name].double()), was[name + "s"].double()
            continue
        x = torch.where(inside, x ** 0.5 if name == "v" else x, 0.0).view(-1, BLOCK)
        scale = x.abs().max(1).values / 448
        z = x / torch.where(scale == 0, 1.0, scale)[:, None]
        if name == "v":
            z = torch.where((x > 0) & (z < 2.0 ** -9), 2.0 ** -9, z)
        z = z.flatten().to(torch.float8_e4m3fn).double()
        out[name], out[name + "s"] = torch.where(inside, z, was[name].double()), scale
    return out


def _exact_norm(s):
    """Each head's row times a matrix of rotations given as complex numbers; gradients by the Jacobian's product."""
    c, out = s["case"], {}
    d, r, count = c["d"], c["rot"], 1 if c["unit"] else c["d"]
    if r:
        i = torch.arange(r, device="cuda")
        one, two = (i[:r // 2], i[r // 2:]) if c["pairs"] == "halves" else (i[::2], i[1::2])
        phase = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double().unsqueeze(1) * s["freqs"].double())

    def rotated(x, sign):
        x = x.clone()
        if r:
            z = torch.complex(x[:, :, one], x[:, :, two]) * (phase if sign > 0 else phase.conj()).unsqueeze(1)
            x[:, :, one], x[:, :, two] = z.real, z.imag
        return x

    for i in ("q", "k"):
        x = s[i].double()
        length = ((x * x).sum(2, keepdim=True) / count + 1e-6).sqrt()
        w = s["w" + i].double() if "w" + i in s else torch.ones(d, dtype=torch.float64, device="cuda")
        if c["op"] == "norm":
            out[i] = rotated(x / length * w, 1)
        else:
            e = rotated(s["dy" + i].double(), -1)
            out["dw" + i] = torch.einsum("nhd,nhd->d", e, x / length) if "w" + i in s else None
            e = e * w
            out["d" + i] = e / length - x * torch.einsum("nhd,nhd->nh", e, x).unsqueeze(2) / (count * length ** 3)
    return out


def _exact_delta(s):
    """A step at a time; backward from states kept every 64 steps."""
    c = s["case"]
    b, h, dk, dv, group = c["b"], c["h"], c["dk"], c["dv"], c["h"] // c["hk"]
    if c["packed"]:
        off = s["offsets"].tolist()
    else:
        off = [i * c["t"] for i in range(b + 1)]
    length = torch.tensor([e - a for a, e in zip(off, off[1:])], device="cuda")
    first = torch.tensor(off[:-1], device="cuda")
    steps, rows = int(length.max()), off[-1]

    def flat(v, lead):
        return v.reshape((rows,) + v.shape[lead:])

    lead = 1 if c["packed"] else 2
    q, k, v, gate, beta = (flat(s[i], lead) for i in ("q", "k", "v", "gate", "beta"))

    def at(t):
        """Row numbers of step t (a spare row where a sequence has ended), and which sequences go on."""
        on = t < length
        return torch.where(on, first + t, 0), on

    def inputs(t):
        r, on = at(t)
        z, w = gate[r].double(), beta[r].double()
        a, rate = (1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(-w))) if c["logit"] else (z.exp(), w)
        return r, on, q[r].double().repeat_interleave(group, 1), k[r].double().repeat_interleave(group, 1), v[r].double(), a, rate

    def forward(t, state):
        r, on, qt, kt, vt, a, rate = inputs(t)
        old = a[..., None, None] * state
        miss = vt - torch.einsum("bhkv,bhk->bhv", old, kt)
        new = old + kt[..., :, None] * (rate[..., None] * miss)[..., None, :]
        return r, on, qt, torch.where(on[:, None, None, None], new, state)

    state, kept = s["h0"].double(), []
    y = torch.zeros(rows + 1, h, dv, dtype=torch.float64, device="cuda")
    for t in range(steps):
        if c["op"] == "delta_grad" and t % 64 == 0:
            kept.append(state)
        r, on, qt, state = forward(t, state)
        y[torch.where(on, r, rows)] = torch.einsum("bhkv,bhk->bhv", state, qt) * s["scale"]
    shape = (rows,) if c["packed"] else (b, c["t"])
    out = {"y": y[:rows].reshape(shape + (h, dv)), "h": state}
    if c["op"] == "delta":
        return out
    dy, carry = flat(s["dy"], lead), s["dh"].double()
    dq, dkey = (torch.zeros(rows + 1, c["hk"], dk, dtype=torch.float64, device="cuda") for _ in range(2))
    dval = torch.zeros(rows + 1, h, dv, dtype=torch.float64, device="cuda")
    dgate, dbeta = (torch.zeros(rows + 1, h, dtype=torch.float64, device="cuda") for _ in range(2))
    for block in reversed(range(len(kept))):
        states = [kept[block]]
        for t in range(block * 64, min(steps, block * 64 + 64)):
            states.append(forward(t, states[-1])[3])
        for t in reversed(range(block * 64, min(steps, block * 64 + 64))):
            before, after = states[t - block * 64], states[t - block * 64 + 1]
            r, on, qt, kt, vt, a, rate = inputs(t)
            to = torch.where(on, r, rows)
            e = dy[r].double() * s["scale"]
            d = carry + qt[..., :, None] * e[..., None, :]
            old = a[..., None, None] * before
            miss = vt - torch.einsum("bhkv,bhk->bhv", old, kt)
            du = torch.einsum("bhkv,bhk->bhv", d, kt)
            dmiss = rate[..., None] * du
            dold = d - kt[..., :, None] * dmiss[..., None, :]
            key = rate[..., None] * torch.einsum("bhkv,bhv->bhk", d, miss) - torch.einsum("bhkv,bhv->bhk", old, dmiss)
            dq[to] = torch.einsum("bhkv,bhv->bhk", after, e).view(b, -1, group, dk).sum(2)
            dkey[to] = key.view(b, -1, group, dk).sum(2)
            dval[to] = dmiss
            da, dr = (dold * before).sum((2, 3)), (du * miss).sum(2)
            dgate[to] = da * a * (1 - a) if c["logit"] else da * a
            dbeta[to] = dr * rate * (1 - rate) if c["logit"] else dr
            carry = torch.where(on[:, None, None, None], a[..., None, None] * dold, carry)
    for name, d in (("dq", dq), ("dk", dkey), ("dv", dval), ("dgate", dgate), ("dbeta", dbeta)):
        out[name] = d[:rows].reshape(shape + d.shape[1:])
    return out | {"dh0": carry}
