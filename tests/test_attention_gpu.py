"""Attention on the GPU (forward, backward, masks, cap, bias) against its definition in 64 bits."""
import itertools

import pytest
import torch

import attention_ref as R
from lego_b200 import ops

pytestmark = pytest.mark.gpu


def make(seed, B, Sq, Sk, Hq, Hk, D, dtype, spread=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    return ((n(B, Sq, Hq, D) * spread).to(dtype), n(B, Sk, Hk, D).to(dtype), n(B, Sk, Hk, D).to(dtype),
            (n(B, Sq, Hq, D) * 0.05).to(dtype))


def check(q, k, v, do, **how):
    want = R.attention(q, k, v, do, **how)
    o, lse = ops.attention_fwd(q, k, v, **how)
    assert R.far_off(o, want["o"]) <= 1, "o"
    assert R.far_off(lse, want["lse"]) <= 1, "lse"
    if do is not None:
        for name, g in zip(("dq", "dk", "dv"), ops.attention_bwd(do, q, k, v, o, lse, **how)):
            assert g.is_contiguous()
            assert R.far_off(g, want[name]) <= 1, name
    assert ops.device_status() == 0


def slopes_of(H):
    return 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H)


def documents_of(seed, B, Sk, kind):
    g = torch.Generator().manual_seed(seed)
    if kind == "packed":                       # runs, padded at the end of every other row
        rows = []
        for b in range(B):
            cuts = sorted(torch.randint(0, Sk + 1, (4,), generator=g).tolist())
            ids = torch.zeros(Sk, dtype=torch.int32)
            for c in cuts:
                ids[c:] += 1
            if b % 2 == 0:
                ids[Sk - Sk // 5:] = -1
            rows.append(ids)
        return torch.stack(rows).cuda()
    if kind == "scattered":                    # any order, some padding in between
        return (torch.randint(-1, 4, (B, Sk), generator=g, dtype=torch.int32)).cuda()
    if kind == "none":                         # a row of padding only
        ids = torch.full((B, Sk), -3, dtype=torch.int32)
        ids[1:] = 7
        return ids.cuda()
    raise KeyError(kind)


SIZES = [(1, 1), (1, 77), (77, 77), (128, 128), (129, 257), (255, 256), (256, 255), (200, 64), (300, 640), (513, 513)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Sq,Sk", SIZES)
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(Sq, Sk, causal, dtype):
    check(*make(Sq * 7 + Sk, 2, Sq, Sk, 2, 1, 64, dtype), causal=causal)


@pytest.mark.parametrize("D", [8, 32, 56, 64, 72, 80, 96, 120, 128])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (6, 2), (5, 5)])
def test_head_layouts(D, Hq, Hk):
    check(*make(D, 2, 150, 201, Hq, Hk, D, torch.bfloat16), causal=True)


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (80, torch.float16)])
@pytest.mark.parametrize("softcap,bias", [(20.0, False), (0.0, True), (5.0, True)])
@pytest.mark.parametrize("causal", [False, True])
def test_cap_and_bias(D, dtype, softcap, bias, causal):
    q, k, v, do = make(3, 2, 270, 333, 4, 2, D, dtype, spread=6.0)
    check(q, k, v, do, causal=causal, softcap=softcap, slopes=slopes_of(4) if bias else None)


@pytest.mark.parametrize("kind", ["packed", "scattered", "none"])
@pytest.mark.parametrize("Sq,Sk", [(300, 300), (140, 519), (1, 65), (700, 700)])
@pytest.mark.parametrize("causal,softcap", [(False, 0.0), (True, 0.0), (True, 15.0)])
def test_documents(kind, Sq, Sk, causal, softcap):
    q, k, v, do = make(5, 3, Sq, Sk, 2, 1, 64, torch.bfloat16)
    check(q, k, v, do, causal=causal, documents=documents_of(Sq, 3, Sk, kind), softcap=softcap)


@pytest.mark.parametrize("Sq,Sk", [(300, 300), (100, 450), (450, 100)])
def test_prefix(Sq, Sk):
    q, k, v, do = make(6, 5, Sq, Sk, 4, 2, 72, torch.float16)
    prefix = torch.tensor([0, 1, 128, Sk, 10 ** 6], dtype=torch.int32, device="cuda")
    check(q, k, v, do, causal=True, prefix=prefix)
    check(q, k, v, do, causal=True, prefix=torch.tensor([-5, 40, 77, 129, 255], dtype=torch.int32, device="cuda"),
          slopes=slopes_of(4))


def test_prefix_within_documents():
    q, k, v, do = make(7, 2, 400, 400, 2, 2, 64, torch.bfloat16)
    check(q, k, v, do, causal=True, prefix=torch.tensor([150, 399], dtype=torch.int32, device="cuda"),
          documents=documents_of(2, 2, 400, "packed"))


def test_scale():
    q, k, v, do = make(8, 1, 130, 130, 2, 2, 128, torch.bfloat16)
    check(q, k, v, do, scale=0.31)
    check(q, k, v, do, scale=-0.05, causal=True)
    check(q, k, v, do, scale=0.0)


def test_large_scores():
    """Rows whose largest score grows from tile to tile, far beyond what exp takes without the running maximum."""
    q, k, v, do = make(9, 1, 260, 700, 2, 1, 64, torch.bfloat16)
    k = (k.float() * torch.linspace(0.1, 30, 700, device="cuda")[None, :, None, None]).to(k.dtype)
    check(q, k, v, do)
    check(q, k.flip(1).contiguous(), v, do, causal=True)


@pytest.mark.parametrize("order", list(itertools.permutations(range(3))))
def test_strides(order):
    """Token, head and batch axes in any order of memory, heads cut out of a wider tensor."""
    B, S, H, D = 2, 190, 3, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    sizes = (B, S, H)

    def one():
        wide = torch.randn(*[sizes[a] + 1 for a in order], D + 16, generator=g, device="cuda").half()
        back = [order.index(a) for a in range(3)]
        return wide.permute(*back, 3)[:B, :S, :H, 8:8 + D]

    q, k, v = one(), one(), one()
    assert q.data_ptr() % 16 == 0 and not q.is_contiguous()
    do = one()
    o, lse = ops.attention_fwd(q, k, v, True)
    o2, lse2 = ops.attention_fwd(q.contiguous(), k.contiguous(), v.contiguous(), True)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    a = ops.attention_bwd(do, q, k, v, o, lse, True)
    b = ops.attention_bwd(do.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(), o, lse, True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    check(q, k, v, do, causal=True)


def test_unaligned_and_expanded_inputs():
    base = torch.randn(2 * 100 * 2 * 64 + 1, device="cuda").half()
    q = base[1:].view(2, 100, 2, 64)                                  # starts 2 bytes off
    k = torch.randn(2, 100, 1, 64, device="cuda").half().expand(2, 100, 2, 64)   # a shared head, stride 0
    v = torch.randn(2, 100, 2, 128, device="cuda").half()[..., ::2]   # every other value
    do = torch.randn(1, 1, 1, 64, device="cuda").half().expand(2, 100, 2, 64)
    check(q, k, v, do, causal=True)


def test_padding_may_hold_anything():
    """NaN and infinities in the tokens of negative documents reach no result; their own rows are zeros."""
    B, S, H, D = 2, 333, 2, 64
    q, k, v, do = make(11, B, S, S, H, H, D, torch.bfloat16)
    docs = documents_of(4, B, S, "packed")
    docs[1, 40:60] = -1
    docs[1, 256:] = -2
    pad = docs < 0
    for x, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (do, float("-inf"))):
        x[pad] = bad
    check(q, k, v, do, causal=True, documents=docs)
    o, lse = ops.attention_fwd(q, k, v, True, None, docs)
    assert (o[pad] == 0).all() and torch.isinf(lse.permute(0, 2, 1)[pad]).all()
    dq, dk, dv = ops.attention_bwd(do, q, k, v, o, lse, True, None, docs)
    assert (dq[pad] == 0).all() and (dk[pad] == 0).all() and (dv[pad] == 0).all()


def test_small_and_large_gradients_in_fp16():
    """The gradient's size may be anything the type holds: neither what underflows nor what overflows in
    between is lost."""
    q, k, v, do = make(12, 1, 520, 520, 2, 1, 64, torch.float16)
    for by in (2.0 ** -9, 1.0, 2.0 ** 12):
        check(q, k, v, (do.float() * by).half(), causal=True)
    check(q, k, (v.float() * 200).half(), do, causal=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_capped_gradients_lose_little_more_than_their_rounding(dtype):
    """Scores of deviation 4 under a cap, documents of many lengths.  In the norm over all values, dq's own
    rounding is 1; the rounding of the weights in the forward pass, which reaches dq through o, makes it 1.07; score
    gradients of 16 bits would make it 1.46 (sums of independent roundings, from the formulas in 64 bits)."""
    q, k, v, do = make(28, 1, 2000, 2000, 4, 4, 64, dtype)
    q = (4 * q.float()).to(dtype)
    docs = documents_of(9, 1, 2000, "packed")
    how = dict(causal=True, documents=docs, softcap=30.0)
    o, lse, low = ops._attention_fwd(q, k, v, True, None, docs, 30.0, None, None, True)
    dq, _, _ = ops.attention_bwd(do, q, k, v, o, lse, o_low=low, **how)
    want = R.attention(q, k, v, do, **how)["dq"][0]
    least = (want.to(dtype).double() - want).norm()
    assert (dq.double() - want).norm() <= 1.25 * least


def test_gradient_against_differences():
    """<dO, O(x + h r) - O(x - h r)> / 2h in 64 bits is the kernel's gradient along r, to the bound of its rounding."""
    q, k, v, do = make(13, 1, 90, 120, 2, 1, 64, torch.float16)
    how = dict(causal=True, softcap=10.0, slopes=slopes_of(2))
    o, lse = ops.attention_fwd(q, k, v, **how)
    grads = ops.attention_bwd(do, q, k, v, o, lse, **how)
    bounds = R.attention(q, k, v, do, **how)
    g = torch.Generator(device="cuda").manual_seed(2)
    for i, (x, name) in enumerate(zip((q, k, v), ("dq", "dk", "dv"))):
        r = torch.randn(x.shape, generator=g, device="cuda").double()

        def at(h):
            args = [t.double() for t in (q, k, v)]
            args[i] = args[i] + h * r
            B, Sq, Hq, D = q.shape
            s = D ** -0.5 * args[0].permute(0, 2, 1, 3) @ args[1].permute(0, 2, 1, 3).mT
            s = 10.0 * torch.tanh(s / 10.0)
            far = (torch.arange(Sq, device="cuda")[:, None] + 30 - torch.arange(120, device="cuda")[None, :])
            s = (s - slopes_of(2).double()[None, :, None, None] * far.abs()).masked_fill(far < 0, float("-inf"))
            return ((torch.softmax(s, -1) @ args[2].permute(0, 2, 1, 3)).permute(0, 2, 1, 3) * do.double()).sum()

        h = 1e-5
        along = ((at(h) - at(-h)) / (2 * h)).item()
        room = (bounds[name][1] * r.abs()).sum().item()
        assert abs((grads[i].double() * r).sum().item() - along) <= room + 1e-6 * abs(along) + 1e-8


def test_autograd_through_the_public_call():
    q, k, v, do = make(14, 2, 130, 130, 4, 2, 64, torch.bfloat16)
    for x in (q, k, v):
        x.requires_grad_()
    o, lse = ops.attention(q, k, v, causal=True, return_lse=True)
    assert o.requires_grad and not lse.requires_grad
    o.backward(do)
    want = R.attention(q.detach(), k.detach(), v.detach(), do, causal=True)
    for x, name in ((q, "dq"), (k, "dk"), (v, "dv")):
        assert R.far_off(x.grad, want[name]) <= 1
    with torch.no_grad():
        assert not ops.attention(q, k, v).requires_grad
    o2, lse2 = ops.attention(q.detach(), k.detach(), v, causal=True, return_lse=True)
    assert torch.equal(o2, o) and torch.equal(lse2, lse)
    (dv,) = torch.autograd.grad(o2, v, do)
    assert torch.equal(dv, v.grad)
    # lse alone carries no gradient, and nothing fails when only it is used
    assert ops.attention(q, k, v, return_lse=True)[1].grad_fn is None


def test_gradients_of_gradients_are_refused():
    """With a graph of the backward pass its results are the same, and going through it raises."""
    q, k, v, do = make(29, 1, 40, 40, 2, 1, 64, torch.bfloat16)
    pos, f = torch.arange(40, device="cuda"), ops.rotary_frequencies(64, device="cuda")
    for x in (q, k, v):
        x.requires_grad_()
    for call in (lambda: ops.attention(q, k, v, causal=True), lambda: ops.rotary(q, None, pos, f)):
        plain, = torch.autograd.grad(call(), q, do)
        once, = torch.autograd.grad(call(), q, do, create_graph=True)
        assert torch.equal(plain, once) and not plain.requires_grad
        with pytest.raises(RuntimeError):
            torch.autograd.grad(once.float().sum(), q)


def test_same_bits_every_run_and_on_another_stream():
    q, k, v, do = make(15, 2, 700, 700, 4, 1, 128, torch.bfloat16)
    docs = documents_of(9, 2, 700, "packed")
    first = None
    side = torch.cuda.Stream()
    for n in range(4):
        with torch.cuda.stream(side if n % 2 else torch.cuda.current_stream()):
            if n % 2:
                side.wait_stream(torch.cuda.default_stream())
            o, lse = ops.attention_fwd(q, k, v, True, None, docs)
            got = (o, lse, *ops.attention_bwd(do, q, k, v, o, lse, True, None, docs))
        torch.cuda.synchronize()
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_two_streams_at_once():
    """Calls of two streams that overlap: each has its own workspace and gives the bits it gives alone."""
    jobs = []
    for n, (shape, how) in enumerate((((2, 900, 900, 4, 2, 64), dict(causal=True, softcap=20.0)),
                                      ((1, 70, 5000, 2, 1, 128), dict(causal=True)))):
        x = make(40 + n, *shape, torch.float16 if n else torch.bfloat16)
        jobs.append((x, how, torch.cuda.Stream()))

    def once(x, how):
        q, k, v, do = x
        o, lse = ops.attention_fwd(q, k, v, **how)
        return (o, lse, *ops.attention_bwd(do, q, k, v, o, lse, **how))

    alone = [once(x, how) for x, how, _ in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for n, (x, how, stream) in enumerate(jobs):
            with torch.cuda.stream(stream):
                got[n].append(once(x, how))
    torch.cuda.synchronize()
    for n in range(2):
        assert all(torch.equal(a, b) for out in got[n] for a, b in zip(alone[n], out))
    assert ops.device_status() == 0


def test_captured_and_replayed():
    """Forward and backward in a graph, replayed with new values in the same buffers, two graphs in turn."""
    shapes = [(1, 200, 200, 2, 1, 64), (2, 140, 300, 4, 2, 128)]
    graphs = []
    for n, s in enumerate(shapes):
        bufs = [x.clone() for x in make(20 + n, *s, torch.bfloat16)]
        ops.attention_bwd(bufs[3], *bufs[:3], *ops.attention_fwd(*bufs[:3], True), True)   # the first call sets up
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, lse = ops.attention_fwd(*bufs[:3], True)
            out = (o, lse, *ops.attention_bwd(bufs[3], *bufs[:3], o, lse, True))
        graphs.append((graph, bufs, out, s))
    for seed in (30, 31):
        for graph, bufs, _, s in graphs:
            for b, x in zip(bufs, make(seed, *s, torch.bfloat16)):
                b.copy_(x)
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, bufs, out, _ in graphs:
            o, lse = ops.attention_fwd(*bufs[:3], True)
            want = (o, lse, *ops.attention_bwd(bufs[3], *bufs[:3], o, lse, True))
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_captured_training_step():
    """Forward and gradients through autograd inside a capture, while another graph of the same leaves is alive."""
    q, k, v, do = make(26, 1, 300, 300, 4, 2, 64, torch.bfloat16)
    for x in (q, k, v):
        x.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = ops.attention(q, k, v, causal=True)
        want = torch.autograd.grad(alive, (q, k, v), do, retain_graph=True)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = ops.attention(q, k, v, causal=True)
        got = torch.autograd.grad(o, (q, k, v), do)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, alive) and all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(alive, (q, k, v), do), want))


def test_a_nan_is_seen():
    """A NaN in a key makes the rows that see it NaN, whichever column it stands in, and no row of an earlier tile."""
    for at in (200, 201, 202, 203, 204, 205):
        q, k, v, _ = make(27, 1, 260, 260, 1, 1, 64, torch.bfloat16)
        k[0, at, 0, 5] = float("nan")
        for how in (dict(), dict(softcap=9.0)):
            o, lse = ops.attention_fwd(q, k, v, True, **how)
            assert torch.isnan(o[0, at:]).all() and torch.isnan(lse[0, 0, at:]).all()
            assert torch.isfinite(o[0, :at]).all() and torch.isfinite(lse[0, 0, :at]).all()


def test_from_a_thread_of_its_own():
    """A thread that has made no CUDA call yet, as autograd's is in a process that only trains: it has no
    current context, which building the tensor maps needs."""
    import threading
    q, k, v, do = make(41, 1, 140, 140, 2, 1, 64, torch.bfloat16)
    o, lse = ops.attention_fwd(q, k, v, True)
    want = (o, lse, *ops.attention_bwd(do, q, k, v, o, lse, True))
    got = []

    def work():
        got.extend(ops.attention_bwd(do, q, k, v, o, lse, True))
        got.extend(ops.attention_fwd(q, k, v, True))

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert len(got) == 5 and all(torch.equal(a, b) for a, b in zip(got[3:] + got[:3], want))


def test_host_tensors():
    q, k, v, do = (x.cpu() for x in make(40, 1, 60, 90, 2, 1, 64, torch.float16))
    o, lse = ops.attention_fwd(q, k, v, True)
    assert not o.is_cuda and not lse.is_cuda
    o2, lse2 = ops.attention_fwd(q.cuda(), k.cuda(), v.cuda(), True)
    assert torch.equal(o, o2.cpu()) and torch.equal(lse, lse2.cpu())
    g = ops.attention_bwd(do, q, k, v, o, lse, True)
    g2 = ops.attention_bwd(do.cuda(), q.cuda(), k.cuda(), v.cuda(), o2, lse2, True)
    assert all(torch.equal(a, b.cpu()) for a, b in zip(g, g2))


def test_empty_calls():
    z = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")   # noqa: E731
    o, lse = ops.attention_fwd(z(2, 0, 2, 64), z(2, 5, 2, 64), z(2, 5, 2, 64))
    assert o.shape == (2, 0, 2, 64) and lse.shape == (2, 2, 0)
    q = torch.ones(2, 3, 2, 64, dtype=torch.float16, device="cuda")
    o, lse = ops.attention_fwd(q, z(2, 0, 2, 64), z(2, 0, 2, 64))
    assert (o == 0).all() and torch.isinf(lse).all()
    dq, dk, dv = ops.attention_bwd(q, q, z(2, 0, 2, 64), z(2, 0, 2, 64), o, lse)
    assert (dq == 0).all() and dk.shape == (2, 0, 2, 64)
    assert ops.attention(z(0, 3, 2, 64), z(0, 5, 1, 64), z(0, 5, 1, 64)).shape == (0, 3, 2, 64)


@pytest.mark.parametrize("Sq,Sk,Hq,Hk", [(1, 9000, 8, 2), (3, 5001, 2, 2), (130, 4097, 4, 1), (4097, 130, 4, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_few_tiles_and_long_loops(Sq, Sk, Hq, Hk, causal):
    """Calls whose loops are cut into pieces and joined: plain, with pieces a mask leaves empty, with scores that
    grow from piece to piece."""
    q, k, v, do = make(51, 1, Sq, Sk, Hq, Hk, 64, torch.bfloat16)
    check(q, k, v, do, causal=causal)
    if Sq <= Sk:
        docs = torch.arange(Sk, dtype=torch.int32, device="cuda")[None] // 700
        docs[:, -40:] = docs[0, 40]          # the last queries' document is one of the first, and these
        check(q, k, v, do, causal=causal, documents=docs, softcap=9.0)
    k = (k.float() * torch.linspace(0.1, 20, Sk, device="cuda")[None, :, None, None]).to(k.dtype)
    check(q, k, v, do, causal=causal, slopes=slopes_of(Hq))


@pytest.mark.parametrize("Sq,Sk,D,dtype", [(2047, 2047, 128, torch.bfloat16), (1025, 4100, 64, torch.float16)])
def test_longer(Sq, Sk, D, dtype):
    q, k, v, do = make(50, 1, Sq, Sk, 4, 1, D, dtype)
    check(q, k, v, do, causal=True)
    check(q, k, v, do, causal=True, documents=documents_of(3, 1, Sk, "packed"), softcap=8.0)
