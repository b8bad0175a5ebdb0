"""The operators together, as a layer is trained: token drive, norms of queries and keys, delta-rule scan, readout, their
gradients and an AdamW step, against the same layer in 64 bits by autograd; and the trained layer a token at a time."""
import pytest

import snn_b200 as snn


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_train_and_answer(bits):
    import torch
    torch.manual_seed(0)
    b, t, h, d, vocab = 3, 80, 2, 32, 256
    width = 3 * h * d
    tok = torch.from_numpy(snn.stream(b * t, seed=3)).cuda().view(b, t)
    table = torch.randn(vocab, width, device="cuda")
    wq, wk = torch.rand(d, device="cuda") + 0.5, torch.rand(d, device="cuda") + 0.5
    gate, beta = torch.randn(vocab, h, device="cuda") + 3, torch.randn(vocab, h, device="cuda")
    freqs = 100.0 ** (-torch.arange(d // 2, device="cuda").float() / d)
    pos = torch.arange(t, device="cuda").expand(b, t).contiguous()
    dy = torch.randn(b, t, h, d, device="cuda")
    params = [table, wq, wk, gate, beta]

    def drive(tk):
        x = snn.embed(tk, table).unflatten(-1, (3 * h, d))
        return x[..., :h, :], x[..., h:2 * h, :], x[..., 2 * h:, :]

    def layer(tk, p, state=None, **save):
        q, k, v = drive(tk)
        qn, kn = snn.qk_norm(q, k, wq, wk, p, freqs, unit=True)
        g, r = snn.embed(tk, gate), snn.embed(tk, beta)
        return (q, k, v, qn, kn, g, r), snn.delta_scan(qn, kn, v, g, r, state, logit=True, **save)

    (q, k, v, qn, kn, g, r), (y, hh, saved) = layer(tok, pos, save=True)
    dqn, dkn, dv, dg, dr, dh0 = snn.delta_scan_grad(qn, kn, v, g, r, dy, saved, logit=True)
    dq, dk, dwq, dwk = snn.qk_norm_grad(q, k, dqn, dkn, wq, wk, pos, freqs, unit=True)
    dx = torch.cat([dq, dk, dv], 2).flatten(-2)
    grads = [snn.embed_grad(tok, dx, vocab), dwq, dwk, snn.embed_grad(tok, dg, vocab), snn.embed_grad(tok, dr, vocab)]

    leaf = [p.double().requires_grad_() for p in params]
    x = leaf[0][tok.long()].unflatten(-1, (3 * h, d))

    def norm(z, w):
        z = z / (z.square().sum(-1, keepdim=True) + 1e-6).sqrt() * w
        a = pos.double()[..., None, None] * freqs.double()
        u, w2 = z[..., :d // 2], z[..., d // 2:]
        return torch.cat([u * a.cos() - w2 * a.sin(), u * a.sin() + w2 * a.cos()], -1)

    qq, kk, vv = norm(x[:, :, :h], leaf[1]), norm(x[:, :, h:2 * h], leaf[2]), x[:, :, 2 * h:]
    a, rate = leaf[3][tok.long()].sigmoid(), leaf[4][tok.long()].sigmoid()
    S, ys = torch.zeros(b, h, d, d, dtype=torch.float64, device="cuda"), []
    for i in range(t):
        S = a[:, i, :, None, None] * S
        u = rate[:, i, :, None] * (vv[:, i] - torch.einsum("bhkv,bhk->bhv", S, kk[:, i]))
        S = S + kk[:, i, :, :, None] * u[:, :, None, :]
        ys.append(torch.einsum("bhkv,bhk->bhv", S, qq[:, i]))
    want = torch.autograd.grad(torch.stack(ys, 1), leaf, dy.double())

    # f32 throughout; the operators' own bounds are some 2^-18 of the largest magnitudes, summed over up to 240 tokens of a row
    def near(got, to):
        return (got.double() - to).abs().max() <= 2.0 ** -14 * to.abs().max()

    assert near(y, torch.stack(ys, 1)) and near(hh, S)
    for name, got, to in zip(("table", "wq", "wk", "gate", "beta"), grads, want):
        assert near(got, to), name

    before = [p.clone() for p in params]
    opt = snn.AdamW(params, bits=bits)
    opt.step(grads, 1, lr=1e-3)
    for p, was, gr in zip(params, before, grads):
        # the first step is lr against the gradient's sign, whatever its size (above eps), and the decay
        there = gr.abs() > 1e-4
        assert there.any() and ((p - was * (1 - 1e-5) + 1e-3 * gr.sign())[there].abs() <= 2e-6 * (1 + was[there].abs())).all()

    # the layer with its new weights, a token at a time with the state in place, and all at once
    _, (y1, h1) = layer(tok, pos)
    state = torch.zeros(b, h, d, d, device="cuda")
    for i in range(t):
        tk, p = tok[:, i:i + 1].contiguous(), pos[:, i:i + 1].contiguous()
        q, k, v = drive(tk)
        qn, kn = snn.qk_norm(q, k, wq, wk, p, freqs, unit=True)
        yi, _ = snn.delta_scan(qn, kn, v, snn.embed(tk, gate), snn.embed(tk, beta), state, logit=True, h_out=state)
        assert near(yi[:, 0], y1[:, i].double())
    assert near(state, h1.double())
