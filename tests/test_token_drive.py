"""snn_embed and snn_embed_grad against their 64-bit forms (leaky_ref)."""
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


def tokens_of(rng, n, vocab, kind, spread="zipf"):
    import torch
    if spread == "one":
        t = np.full(n, vocab - 1)
    elif spread == "each":
        t = np.arange(n) % vocab
    else:
        t = np.minimum(rng.zipf(1.3, n) - 1, vocab - 1)
    return torch.from_numpy(t.astype(kind)).cuda()


def make(rng, shape, kind, std=1.0):
    import torch
    return torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(dt(kind)).cuda()


# ---- refusals (no GPU needed: the checks come first) --------------------------
def embed_args(**over):
    a = dict(tokens=4096, tok=8, n=4, table=8192, ttype=0, vocab=256, dim=8, tstride=8, scale=1.0,
             out=16384, otype=0, ostride=8, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over", [
    dict(tokens=None), dict(tok=3), dict(tok=9, tokens=4098), dict(n=-1), dict(n=(1 << 30) + 1),
    dict(table=None), dict(table=8194), dict(ttype=3), dict(vocab=0), dict(vocab=1 << 31), dict(dim=0), dict(dim=(1 << 22) + 1, tstride=1 << 23, ostride=1 << 23),
    dict(tstride=-1), dict(out=None), dict(otype=7), dict(otype=1, out=16385), dict(ostride=7)])
def test_embed_refuses(over):
    assert snn.lib().snn_embed(*embed_args(**over)) == 1
    assert b"embed" in snn.lib().snn_last_error(None)


def grad_args(**over):
    a = dict(tokens=4096, tok=8, n=4, dy=8192, dtype=0, dim=8, dstride=8, scale=1.0, out=16384,
             otype=0, vocab=256, ostride=8, acc=0, work=1 << 20, bytes=1 << 40, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over", [
    dict(tokens=None), dict(tok=0), dict(n=-1), dict(dy=None), dict(dtype=8), dict(dim=0), dict(dstride=-1),
    dict(out=None), dict(otype=-1), dict(vocab=0), dict(ostride=7), dict(work=None), dict(work=(1 << 20) + 8),
    dict(bytes=64)])
def test_embed_grad_refuses(over):
    assert snn.lib().snn_embed_grad(*grad_args(**over)) == 1
    assert b"embed" in snn.lib().snn_last_error(None)


def test_workspace_size():
    size = C.c_int64(-1)
    assert snn.lib().snn_embed_grad_workspace(100000, 256, 64, C.byref(size)) == 0
    assert size.value >= 2 * 8 * 100000
    assert snn.lib().snn_embed_grad_workspace(1000, 256, 64, None) == 1
    assert snn.lib().snn_embed_grad_workspace(-1, 256, 64, C.byref(size)) == 1


def test_binding_refuses_host_tensors():
    import torch
    tok, table = torch.zeros(4, dtype=torch.uint8), torch.zeros(256, 8)
    with pytest.raises(snn.SnnError):
        snn.embed(tok, table)
    with pytest.raises(snn.SnnError):
        snn.embed_grad(tok, torch.zeros(4, 8), 256)


# ---- forward ---------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("n,vocab,dim,tok", [
    (0, 5, 8, "uint8"), (1, 1, 1, "uint8"), (1, 256, 1000, "uint8"), (7, 3, 33, "int32"), (64, 256, 500, "uint8"),
    (1000, 20999, 8, "int64"), (333, 257, 1001, "int32"), (50, 70000, 4100, "int64"), (20000, 256, 12, "uint8")])
@pytest.mark.parametrize("tk,ok", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f32"),
                                   ("bf16", "f16"), ("f16", "f16")])
def test_embed(n, vocab, dim, tok, tk, ok):
    import torch
    rng = np.random.default_rng(n + dim)
    t = tokens_of(rng, n, vocab, tok)
    table = make(rng, (vocab, dim), tk)
    got = snn.embed(t, table, scale=0.37, dtype=dt(ok))
    want = (table.float() * np.float32(0.37))[t.long()].to(dt(ok))  # one product, one rounding
    assert got.shape == (n, dim) and got.dtype == dt(ok)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_embed_outside_tokens_and_shapes():
    import torch
    rng = np.random.default_rng(1)
    t = torch.tensor([[0, -1, 9], [10, 3, 1 << 40]], device="cuda")
    table = make(rng, (10, 24), "f32")
    got = snn.embed(t, table, scale=2.0)
    assert got.shape == (2, 3, 24)
    ref.close(host(got), ref.embed(t.cpu().numpy(), host(table), 2.0), 0.0, "f32")
    assert (got[0, 1] == 0).all() and (got[1, 0] == 0).all() and (got[1, 2] == 0).all()
    table[4] = float("nan")  # a zero row is zero whatever the table holds
    table[3, 5] = float("inf")
    again = snn.embed(t, table, scale=0.0)
    assert torch.isnan(again[1, 1, 5]) and (again[0, 1] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,width,at", [(24, 40, 8), (24, 37, 3), (33, 35, 1), (256, 264, 4)])
def test_embed_strides(dim, width, at):
    """Rows inside wider ones: what lies beside them stays."""
    import torch
    rng = np.random.default_rng(dim)
    wide = make(rng, (300, width), "bf16")
    table = wide[:, at:at + dim]
    out = torch.full((70, width), 7.0, dtype=torch.bfloat16, device="cuda")
    t = tokens_of(rng, 70, 300, "int32")
    got = snn.embed(t, table, out=out[:, at:at + dim])
    assert torch.equal(got, table[t.long()])
    assert (out[:, :at] == 7).all() and (out[:, at + dim:] == 7).all()
    with pytest.raises(snn.SnnError):
        snn.embed(t, table, out=out[:, at:at + dim].float())[0]
        snn.embed(t, table, dtype=torch.float32, out=out[:, at:at + dim])


@pytest.mark.gpu
def test_embed_into_an_output_of_another_type():
    """`out` sets the type where dtype is not given; a given one has to be out's."""
    import torch
    rng = np.random.default_rng(12)
    t, table = tokens_of(rng, 70, 300, "int32"), make(rng, (300, 24), "bf16")
    out = torch.full((70, 24), 7.0, device="cuda")
    assert snn.embed(t, table, out=out) is out and torch.equal(out, table[t.long()].float())
    with pytest.raises(snn.SnnError):
        snn.embed(t, table, dtype=torch.bfloat16, out=out)


# ---- gradient --------------------------------------------------------------------
GRAD = [
    (1, 1, 1, "uint8", "zipf"), (2, 256, 8, "uint8", "one"), (31, 2, 33, "int32", "each"),
    (33, 256, 500, "uint8", "zipf"), (511, 256, 64, "uint8", "one"), (512, 257, 100, "int32", "zipf"),
    (2049, 20999, 24, "int64", "zipf"), (5000, 256, 1001, "uint8", "zipf"), (4096, 4096, 16, "int32", "each"),
    (4097, 70000, 12, "int64", "each"), (30000, 3, 130, "int32", "zipf"), (70001, 256, 40, "uint8", "zipf"),
    (140000, 20999, 8, "int64", "zipf"), (70000, 5, 6, "int32", "one"), (9000, 300, 2050, "int32", "zipf")]


@pytest.mark.gpu
@pytest.mark.parametrize("n,vocab,dim,tok,spread", GRAD)
@pytest.mark.parametrize("dk,ok", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_embed_grad(n, vocab, dim, tok, spread, dk, ok):
    import torch
    rng = np.random.default_rng(n + dim)
    t = tokens_of(rng, n, vocab, tok, spread)
    dy = make(rng, (n, dim), dk)
    got = snn.embed_grad(t, dy, vocab, scale=0.3, dtype=dt(ok))
    want, bound = ref.embed_grad(t.cpu().numpy().astype(np.int64), host(dy), vocab, 0.3)
    ref.close(host(got), want, bound, ok)
    assert torch.equal(got, snn.embed_grad(t, dy, vocab, scale=0.3, dtype=dt(ok)))  # the same bits again
    seen = torch.zeros(vocab, dtype=torch.bool, device="cuda")
    seen[t.long()] = True
    assert (got[~seen] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ok", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,vocab,dim", [(0, 40, 9), (600, 40, 9), (9000, 1000, 64), (40000, 256, 24)])
def test_embed_grad_accumulates(n, vocab, dim, ok):
    import torch
    rng = np.random.default_rng(n + 5)
    t = torch.from_numpy(rng.integers(-3, vocab // 2, n).astype(np.int64)).cuda()
    dy = make(rng, (n, dim), "f32")
    out = make(rng, (vocab, dim + 4), ok)
    before = out.clone()
    got = snn.embed_grad(t, dy, out=out[:, :dim], accumulate=True)
    want, bound = ref.embed_grad(t.cpu().numpy(), host(dy), vocab, 1.0, base=host(before[:, :dim]))
    ref.close(host(got), want, bound, ok)
    assert torch.equal(out[:, dim:], before[:, dim:]) and torch.equal(out[vocab // 2:], before[vocab // 2:])


@pytest.mark.gpu
@pytest.mark.parametrize("ok", ["f32", "bf16"])
@pytest.mark.parametrize("n,vocab,dim,width", [(0, 5000, 24, 40), (300, 50, 9, 12), (3000, 50, 33, 40), (3000, 6000, 24, 32),
                                               (50000, 700, 17, 18), (40000, 20, 256, 264)])
def test_embed_grad_into_wider_rows(n, vocab, dim, width, ok):
    """Rows of `out` inside wider ones: all of its own are written, what lies beside them stays."""
    import torch
    rng = np.random.default_rng(n + dim)
    t = torch.from_numpy(rng.integers(0, max(vocab // 2, 1), n).astype(np.int32)).cuda()
    dy = make(rng, (n, dim), "bf16")
    wide = torch.full((vocab, width), 7.0, dtype=dt(ok), device="cuda")
    got = snn.embed_grad(t, dy, out=wide[:, width - dim:])
    want, bound = ref.embed_grad(t.cpu().numpy(), host(dy), vocab, 1.0)
    ref.close(host(got), want, bound, ok)
    assert (wide[:, :width - dim] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,vocab,dim", [(500, 300, 24), (4000, 9000, 25), (40000, 6000, 40), (0, 7000, 8)])
def test_embed_grad_at_an_odd_element(n, vocab, dim):
    """A gradient, dy and table that begin at an odd element of a buffer."""
    import torch
    rng = np.random.default_rng(n)
    t = torch.from_numpy(rng.integers(0, vocab, n)).cuda()
    dy = make(rng, (n * dim + 1,), "bf16")[1:].view(n, dim)
    flat = torch.full((vocab * dim + 2,), 7.0, dtype=torch.bfloat16, device="cuda")
    got = snn.embed_grad(t, dy, out=flat[1:-1].view(vocab, dim))
    want, bound = ref.embed_grad(t.cpu().numpy(), host(dy), vocab, 1.0)
    ref.close(host(got), want, bound, "bf16")
    assert flat[0] == 7 and flat[-1] == 7
    assert torch.equal(snn.embed(t, got), got[t])


@pytest.mark.gpu
def test_embed_grad_of_no_valid_token():
    import torch
    t = torch.full((3000,), -1, dtype=torch.int32, device="cuda")
    dy = torch.full((3000, 16), float("nan"), device="cuda")
    out = torch.full((50, 16), 3.0, device="cuda")
    assert (snn.embed_grad(t, dy, out=out) == 0).all()
    out.fill_(3.0)
    assert (snn.embed_grad(t, dy, out=out, accumulate=True) == 3).all()
    assert (snn.embed_grad(t[:0], dy[:0], 50) == 0).all()
    # a NaN reaches its own row alone
    t[7] = 4
    got = snn.embed_grad(t, dy, 50)
    assert torch.isnan(got[4]).all() and (got[:4] == 0).all() and (got[5:] == 0).all()


@pytest.mark.gpu
def test_embed_grad_strided_and_broadcast_dy():
    import torch
    rng = np.random.default_rng(9)
    t = tokens_of(rng, 700, 90, "int32")
    wide = make(rng, (700, 41), "bf16")
    for dy in (wide[:, 3:36], wide[:, 8:40], make(rng, (1, 32), "f32").expand(700, 32)):
        got = snn.embed_grad(t, dy, 90)
        want, bound = ref.embed_grad(t.cpu().numpy(), host(dy), 90, 1.0)
        ref.close(host(got), want, bound, "f32")


@pytest.mark.gpu
def test_two_graphs_streams_and_eager_calls():
    """Two captured calls and eager ones, on different streams, replayed with new inputs: no shared state."""
    import torch
    rng = np.random.default_rng(11)
    sets = []
    for k, (n, vocab, dim) in enumerate([(5000, 256, 64), (3000, 20999, 72)]):
        t, dy = tokens_of(rng, n, vocab, "int32"), make(rng, (n, dim), "f32")
        table = make(rng, (vocab, dim), "f32")
        snn.embed_grad(t, dy, vocab)  # warm
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=s):
            out, grad = snn.embed(t, table, scale=3.0), snn.embed_grad(t, dy, vocab, scale=0.5)
        sets.append((g, s, t, dy, table, vocab, out, grad))
    for trial in range(3):
        for g, s, t, dy, table, vocab, out, grad in sets:
            t.copy_(tokens_of(rng, t.numel(), vocab, "int32"))
            dy.copy_(make(rng, dy.shape, "f32"))
        torch.cuda.synchronize()
        for g, s, *_ in sets:
            with torch.cuda.stream(s):
                g.replay()
        side = torch.cuda.Stream()
        eager = snn.embed_grad(sets[0][2], sets[0][3], sets[0][5], scale=0.5, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(eager, sets[0][7])
        for g, s, t, dy, table, vocab, out, grad in sets:
            assert torch.equal(out, table[t.long()] * 3.0)
            want, bound = ref.embed_grad(t.cpu().numpy(), host(dy), vocab, 0.5)
            ref.close(host(grad), want, bound, "f32")


@pytest.mark.gpu
def test_two_host_threads():
    """Calls of two threads, each on its own stream, and of both on one stream."""
    import threading
    import torch
    rng = np.random.default_rng(13)
    sets = []
    for n, vocab, dim in ((9000, 256, 96), (7000, 5000, 40)):
        t, dy = tokens_of(rng, n, vocab, "int32"), make(rng, (n, dim), "f32")
        sets.append((t, dy, vocab, snn.embed_grad(t, dy, vocab), torch.cuda.Stream()))
    torch.cuda.synchronize()
    one = torch.cuda.Stream()
    for shared in (False, True):
        wrong = []

        def work(t, dy, vocab, want, stream):
            for _ in range(40):
                got = snn.embed_grad(t, dy, vocab, stream=one if shared else stream)
                (one if shared else stream).synchronize()
                if not torch.equal(got, want):
                    wrong.append(vocab)

        threads = [threading.Thread(target=work, args=s) for s in sets]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
        assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [50000, 200000])
def test_result_is_ready_for_the_next_kernel(vocab):
    """Runs that never cross pieces (each token once): what follows on the stream sees every row."""
    import torch
    n, dim = 40000, 256
    t = torch.randperm(vocab, device="cuda")[:n]
    dy = torch.randn(n, dim, device="cuda")
    want = torch.zeros(vocab, dim, device="cuda")
    want[t] = dy
    for _ in range(20):
        assert torch.equal(snn.embed_grad(t, dy, vocab), want)


@pytest.mark.gpu
def test_rows_past_32_bit_offsets():
    """A table of more than 2^31 elements (2^32 bytes in bf16), its last rows read and written."""
    import torch
    vocab, dim = 70000, 32000
    table = torch.empty(vocab, dim, dtype=torch.bfloat16, device="cuda")
    table[-2:] = torch.arange(2 * dim, device="cuda").view(2, dim).to(torch.bfloat16)
    t = torch.tensor([vocab - 1, vocab - 2, vocab - 1], device="cuda", dtype=torch.int32)
    out = snn.embed(t, table)
    assert torch.equal(out, table[t.long()])
    table[-3:] = 0
    got = snn.embed_grad(t, out, out=table, accumulate=True)
    assert torch.equal(got[-1], (out[0].float() * 2).to(torch.bfloat16)) and torch.equal(got[-2], out[1])
    assert (got[-3] == 0).all()
