"""Paths that short eager calls do not enter: captured calls of every kind, batches past a block's threads, offsets past
31 bits."""
import pytest
import torch

import attention_ref as R
from lego_b200 import ops

pytestmark = pytest.mark.gpu


def make(seed, B, Sq, Sk, Hq, Hk, D, dtype, by=0.05):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    return ((n(B, Sq, Hq, D) * 1.5).to(dtype), n(B, Sk, Hk, D).to(dtype), n(B, Sk, Hk, D).to(dtype),
            (n(B, Sq, Hq, D) * by).to(dtype))


def step(bufs, docs, softcap):
    q, k, v, do = bufs
    o, lse, low = ops._attention_fwd(q, k, v, True, None, docs, softcap, None, None, True)
    return (o, lse, *ops.attention_bwd(do, q, k, v, o, lse, True, None, docs, softcap, o_low=low))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 300, 300, 4, 2, 64), (1, 70, 5000, 2, 1, 128), (1, 2100, 2100, 1, 1, 64)])
@pytest.mark.parametrize("docs", [False, True])
def test_captured_calls_of_every_kind(docs, shape, dtype):
    """Two graphs that are replayed in turn, loops cut into pieces and not: with large gradients, then with small ones in
    the same buffers, then with other documents.  Nothing of a replay reaches the next: the bits are an eager call's."""
    B, Sk = shape[0], shape[2]
    graphs = []
    for n in range(2):
        bufs = [x.clone() for x in make(n, *shape, dtype)]
        ids = torch.zeros(B, Sk, dtype=torch.int32, device="cuda") if docs else None
        step(bufs, ids, 20.0 * n)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(bufs, ids, 20.0 * n)
        graphs.append((graph, bufs, ids, out))
    for turn, by in enumerate((1000.0, 1e-3, 0.05)):
        for n, (_, bufs, ids, _) in enumerate(graphs):
            for b, x in zip(bufs, make(10 * turn + n, *shape, dtype, by)):
                b.copy_(x)
            if docs:
                ids.copy_(torch.arange(Sk, device="cuda")[None].expand(B, -1) // (Sk // (turn + 2)))
                ids[:, Sk - 9 * turn:] = -1
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for n, (_, bufs, ids, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, step(bufs, ids, 20.0 * n)))
    assert ops.device_status() == 0


@pytest.mark.parametrize("B", [129, 513, 1100])
def test_many_sequences(B):
    """More sequences than the threads that add up their lengths, in the main kernel and in the join."""
    g = torch.Generator(device="cuda").manual_seed(B)
    lengths = torch.randint(-1, 260, (B,), generator=g, device="cuda").to(torch.int32)
    lengths[::3] = 0
    lengths[-1] = 4000                     # in many runs, past all the others
    lengths[B // 2] = 2500
    page, Hk, D = 32, 2, 64
    n = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()   # noqa: E731
    kc, vc, q = n(200, page, Hk, D), n(200, page, Hk, D), n(B, 1, 2, D)
    table = torch.randint(0, 200, (B, 126), generator=g, device="cuda").to(torch.int32)
    o = ops.tree_attention(q, kc, vc, table, lengths)
    assert R.far_off(o, R.tree(q, kc, vc, table, lengths, None)) <= 1
    assert ops.device_status() == 0


def test_rotary_past_31_bits():
    """Results past 2^31 values, inputs a stride of more than that apart."""
    S = (1 << 24) + 5
    f = ops.rotary_frequencies(128, device="cuda")
    x = torch.zeros(1, S, 1, 128, dtype=torch.float16, device="cuda")
    x[0, -300:] = torch.randn(300, 1, 128, device="cuda").half()
    pos = torch.arange(S, device="cuda")
    y = ops.rotary(x, None, pos, f)
    assert torch.equal(y[:, -300:], ops.rotary(x[:, -300:].clone(), None, pos[-300:], f))
    assert not y[:, :-300].any()
    del y
    two = x.flatten().as_strided((2, 3, 1, 128), ((1 << 31) + 128, 128, 128, 1))
    two.normal_()
    assert torch.equal(ops.rotary(two, None, pos[:3], f), ops.rotary(two.contiguous(), None, pos[:3], f))


@pytest.mark.parametrize("docs", [False, True])
def test_attention_inputs_past_31_bits(docs):
    """Batches, tokens or heads more than 2^31 values apart (padding is read by plain loads, the rest by tensor maps)."""
    far = torch.zeros((1 << 31) + (1 << 17), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.tensor([[0, 0, 0, -1], [1, -1, 1, 1]], dtype=torch.int32, device="cuda") if docs else None
    do = torch.randn(2, 4, 2, 64, generator=g, device="cuda").bfloat16()
    for axis in range(3):
        strides = [512, 128, 64]
        step = (1 << 31) // ((2, 4, 2)[axis] - 1) // 8 * 8
        strides[axis] = step
        dense = [torch.randn(2, 4, 2, 64, generator=g, device="cuda").bfloat16() for _ in range(3)]
        tensors = []
        for n, x in enumerate(dense):
            t = far[n * 8192:].as_strided((2, 4, 2, 64), (*strides, 1))
            t.copy_(x)
            tensors.append(t)
        assert tensors[0].stride(axis) == step

        def once(q, k, v):
            o, lse, low = ops._attention_fwd(q, k, v, True, None, ids, 0.0, None, None, True)
            return (o, lse, *ops.attention_bwd(do, q, k, v, o, lse, True, None, ids, o_low=low))

        assert all(torch.equal(a, b) for a, b in zip(once(*tensors), once(*dense)))
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_results_past_31_bits(dtype):
    """2^18 short calls in one: q, o, do and dq of more than 2^31 values."""
    B, H, D = (1 << 18) + 3, 64, 128
    q, do = (torch.zeros(B, 1, H, D, dtype=dtype, device="cuda") for _ in range(2))
    k, v = (torch.zeros(B, 2, 1, D, dtype=dtype, device="cuda") for _ in range(2))
    small = make(4, 5, 1, 2, H, 1, D, dtype)
    for big, x in zip((q, k, v, do), small):
        big[-5:] = x
    o, lse = ops.attention_fwd(q, k, v)
    want, want_lse = ops.attention_fwd(*small[:3])
    assert torch.equal(o[-5:], want) and torch.equal(lse[-5:], want_lse) and not o[:-5].any()
    dq, dk, dv = ops.attention_bwd(do, q, k, v, o, lse)
    # five key tiles alone are summed in pieces, 2^18 of them are not: dk and dv go by the definition
    want_dq = ops.attention_bwd(small[3], *small[:3], want, want_lse)[0]
    exact = R.attention(*small)
    assert torch.equal(dq[-5:], want_dq) and not dq[:-5].any()
    for got, name in ((dk, "dk"), (dv, "dv")):
        assert R.far_off(got[-5:], exact[name]) <= 1 and not got[:-5].any()
    assert ops.device_status() == 0
