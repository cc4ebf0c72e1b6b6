"""Attention of drafted trees over a paged cache against its definition in 64 bits."""
import pytest
import torch

import attention_ref as R
from lego_b200 import ops

pytestmark = pytest.mark.gpu


def cache(seed, lengths, T, page, Hk, D, dtype, spare=2, extra=0):
    """Pages in shuffled order; whatever no sequence owns, and all places past a sequence's end, are NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [max(0, -(-(n + T) // page)) if n >= 0 else 0 for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), max(1, max(need) + extra)), -1, dtype=torch.int32, device="cuda")
    pages = sum(need) + spare
    k = torch.full((pages, page, Hk, D), float("nan"), device="cuda", dtype=dtype)
    v = k.clone()
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        for i in range(n):
            rows = min(page, lengths[b] + T - i * page)
            pg = table[b, i].long()
            k[pg, :rows] = torch.randn(rows, Hk, D, generator=g, device="cuda").to(dtype)
            v[pg, :rows] = torch.randn(rows, Hk, D, generator=g, device="cuda").to(dtype)
    return k, v, table


def tree_parents(seed, B, T):
    g = torch.Generator().manual_seed(seed)
    rows = [[-1] + [int(torch.randint(-1, t, (1,), generator=g)) for t in range(1, T)] for _ in range(B)]
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


def check(seed, lengths, T, Hq, Hk, D, page, dtype, parents="tree", spread=1.5, **how):
    B = len(lengths)
    k, v, table = cache(seed, lengths, T, page, Hk, D, dtype)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = (torch.randn(B, T, Hq, D, generator=g, device="cuda") * spread).to(dtype)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    par = tree_parents(seed, B, T) if parents == "tree" else parents
    o = ops.tree_attention(q, k, v, table, lens, par, **how)
    assert R.far_off(o, R.tree(q, k, v, table, lens, par, **how)) <= 1
    assert ops.device_status() == 0
    return q, k, v, table, lens, par, o


def slopes_of(H):
    return 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [1, 7, 16, 64, 100])
def test_one_token(page, dtype):
    check(page, [0, 1, 63, 64, 65, 200, -1], 1, 8, 2, 64, page, dtype, parents=None)


@pytest.mark.parametrize("T", [1, 2, 5, 16, 17, 33, 64])
@pytest.mark.parametrize("Hq,Hk,D", [(4, 4, 64), (8, 1, 128), (5, 1, 80), (16, 2, 8)])
def test_trees(T, Hq, Hk, D):
    check(T + D, [0, 3, 130, 257], T, Hq, Hk, D, 16, torch.bfloat16)


def test_chain_is_the_default_and_matches_causal_attention():
    T, n, Hq, Hk, D = 20, 300, 4, 2, 64
    q, k, v, table, lens, _, o = check(5, [n], T, Hq, Hk, D, 32, torch.float16, parents=None)
    chain = torch.arange(-1, T - 1, dtype=torch.int32, device="cuda")[None]
    assert torch.equal(ops.tree_attention(q, k, v, table, lens, chain), o)
    kk, vv = (c[table[0].long()].flatten(0, 1)[None, :n + T].contiguous() for c in (k, v))
    a = ops.attention(q, kk, vv, causal=True)
    want = R.attention(q, kk, vv, causal=True)["o"]
    assert R.far_off(a, want) <= 1 and R.far_off(o, want) <= 1


@pytest.mark.parametrize("softcap,bias", [(20.0, False), (0.0, True), (5.0, True)])
def test_cap_and_bias(softcap, bias):
    check(8, [0, 17, 200], 12, 6, 2, 64, 16, torch.float16, spread=6.0, softcap=softcap, slopes=slopes_of(6) if bias else None)
    check(9, [700], 1, 6, 2, 128, 16, torch.bfloat16, parents=None, spread=6.0, softcap=softcap,
          slopes=slopes_of(6) if bias else None)


def test_unused_tokens_and_sequences():
    par = torch.tensor([[-1, 0, 5, 2, -7], [-1, -1, 1, 9, 2], [4, 0, 1, 2, 3]], dtype=torch.int32, device="cuda")
    *_, o = check(10, [40, -1, 3], 5, 4, 2, 64, 16, torch.bfloat16, parents=par)
    assert (o[0, 2:] == 0).all() and (o[1] == 0).all() and (o[2] == 0).all()
    assert (o[0, :2] != 0).any()


def test_missing_pages_hold_nothing():
    """Page numbers outside the cache and lengths past the table hide keys; nothing is read for them."""
    q, k, v, table, lens, par, _ = check(11, [100, 64, 5], 3, 4, 2, 64, 16, torch.float16)
    table[0, 2] = -1
    table[0, 4] = 10 ** 6
    table[2, :] = 2 ** 31 - 1
    o = ops.tree_attention(q, k, v, table, lens, par)
    assert R.far_off(o, R.tree(q, k, v, table, lens, par)) <= 1
    assert (o[2] == 0).all()
    k, v = k.nan_to_num(0.5), v.nan_to_num(0.5)
    long = torch.tensor([10 ** 9, 2 ** 31 - 1, 0], dtype=torch.int32, device="cuda")
    o = ops.tree_attention(q, k, v, table[:, :4].contiguous(), long, None)
    n = 4 * 16
    for b in (0, 1):
        one = R.tree(q[b:b + 1], k, v, table[b:b + 1, :4], torch.tensor([n], device="cuda"), None)
        assert R.far_off(o[b:b + 1], (one[0], one[1])) <= 1


def test_long_and_ragged():
    check(12, [5000, 1, 0, 2900], 1, 8, 2, 64, 64, torch.bfloat16, parents=None)
    check(13, [4097, 300], 9, 4, 1, 128, 48, torch.float16)


def test_strides():
    """Caches of shape [pages, Hk, page, D] and keys interleaved with values, seen through their strides."""
    q, k, v, table, lens, par, o = check(14, [90, 33], 4, 4, 2, 64, 16, torch.float16)
    kt = k.transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.stack([k, v], dim=1)
    assert torch.equal(ops.tree_attention(q, kt, v, table, lens, par), o)
    assert torch.equal(ops.tree_attention(q, both[:, 0], both[:, 1], table, lens, par), o)
    wide = torch.randn(2, 4, 4, 96, device="cuda").half()
    wide[..., 16:80] = q
    assert torch.equal(ops.tree_attention(wide[..., 16:80], k, v, table, lens, par), o)


def test_graph_two_streams_and_same_bits():
    q, k, v, table, lens, par, o = check(15, [1000, 77, 400], 6, 8, 2, 64, 16, torch.bfloat16)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.tree_attention(q, k, v, table, lens, par)
        graphs.append((graph, y))
    lens.sub_(5)
    want = ops.tree_attention(q, k, v, table, lens, par)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs[0][0].replay()
    with torch.cuda.stream(side):
        graphs[1][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want)
    lens.add_(5)
    assert torch.equal(ops.tree_attention(q, k, v, table, lens, par), o)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        y = ops.tree_attention(q, k, v, table, lens, par)
    torch.cuda.synchronize()
    assert torch.equal(y, o)


def test_offsets_past_32_bits():
    """The last page of a cache of more than 2^32 bytes and 2^31 values."""
    D, Hk, page = 128, 8, 64
    pages = (1 << 31) // (D * Hk * page) + 3
    k = torch.zeros(pages, page, Hk, D, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    small_k, small_v, _ = cache(16, [120], 1, page, Hk, D, torch.float16, spare=0)
    k[-2:], v[-2:] = small_k.nan_to_num(0), small_v.nan_to_num(0)
    q = torch.randn(1, 1, 16, D, device="cuda").half()
    lens = torch.tensor([120], dtype=torch.int32, device="cuda")
    far = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device="cuda")
    near = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.tree_attention(q, k, v, far, lens), ops.tree_attention(q, small_k, small_v, near, lens))


def test_host_tensors_and_empty():
    q, k, v, table, lens, par, o = check(17, [50], 3, 4, 2, 64, 16, torch.float16)
    y = ops.tree_attention(*(t.cpu() for t in (q, k, v, table, lens, par)))
    assert not y.is_cuda and torch.equal(y, o.cpu())
    assert ops.tree_attention(q[:0], k, v, table[:0], lens[:0], par[:0]).shape == (0, 3, 4, 64)


def test_a_serving_run():
    """Train-side attention of a prompt, then its cache pages and drafted tokens: rotary positions, cache
    places and tree attention together give what attention over the whole text gives, path by path."""
    g = torch.Generator(device="cuda").manual_seed(4)
    Hq, Hk, D, n, page = 4, 2, 64, 75, 16
    f = ops.rotary_frequencies(D, device="cuda")
    par, depth = [-1, 0, 0, 1, 2], [0, 1, 1, 2, 2]
    T = len(par)
    raw = lambda m, H: torch.randn(1, m, H, D, generator=g, device="cuda").bfloat16()   # noqa: E731
    q, k, v = raw(n + T, Hq), raw(n + T, Hk), raw(n + T, Hk)
    pos = torch.tensor(list(range(n)) + [n + d for d in depth], device="cuda")
    qr, kr = ops.rotary(q, k, pos, f)
    table = torch.tensor([[3, 0, 5, 1, 4]], dtype=torch.int32, device="cuda")
    kc, vc = (torch.full((6, page, Hk, D), float("nan"), device="cuda").bfloat16() for _ in range(2))
    at = torch.arange(n + T, device="cuda")
    kc[table[0, at // page].long(), at % page], vc[table[0, at // page].long(), at % page] = kr[0], v[0]
    o = ops.tree_attention(qr[:, n:].contiguous(), kc, vc, table, torch.tensor([n], dtype=torch.int32, device="cuda"),
                           torch.tensor([par], dtype=torch.int32, device="cuda"), softcap=12.0, slopes=slopes_of(Hq))
    for t in range(T):
        path, up = [], t
        while up >= 0:
            path, up = [n + up] + path, par[up]
        idx = torch.tensor(list(range(n)) + path, device="cuda")
        how = dict(causal=True, softcap=12.0, slopes=slopes_of(Hq))
        a = ops.attention(qr[:, idx], kr[:, idx], v[:, idx], **how)
        want, room = R.attention(qr[:, idx], kr[:, idx], v[:, idx], **how)["o"]
        assert R.far_off(a, (want, room)) <= 1
        assert R.far_off(o[:, t:t + 1], (want[:, -1:], room[:, -1:])) <= 1
