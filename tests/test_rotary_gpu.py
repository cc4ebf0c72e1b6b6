"""Rotary positions on the GPU against complex rotation in 64 bits: one rounding of the result and the
32-bit sine, cosine and products (a few 2^-24 of the pair's size) is all that may differ."""
import pytest
import torch

from lego_b200 import ops

pytestmark = pytest.mark.gpu


def turned(x, positions, freqs, pairs, scale=1.0, inverse=False):
    R = 2 * freqs.numel()
    pos = positions if positions.dim() == 2 else positions[None].expand(x.shape[0], -1)
    angle = pos.double()[..., None] * freqs
    by = torch.polar(torch.full_like(angle, scale), -angle if inverse else angle)[:, :, None, :]
    y = x.double().clone()
    head = y[..., :R].clone()
    z = head.unflatten(-1, (2, R // 2)).movedim(-2, -1) if pairs == "half" else head.unflatten(-1, (R // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * by)
    y[..., :R] = (z.movedim(-1, -2) if pairs == "half" else z).flatten(-2)
    size = x.double().abs()
    size[..., :R] = abs(scale) * x[..., :R].double().abs().amax(-1, keepdim=True) * 2
    return y, size


def close(got, want):
    y, size = want
    u = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    assert got.shape == y.shape
    assert ((got.double() - y).abs() <= u * y.abs() + 2.0 ** -21 * size + tiny).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("B,S,Hq,Hk,D,R", [(1, 1, 1, 1, 2, 2), (2, 77, 4, 2, 64, 64), (3, 5, 3, 1, 80, 40), (1, 1300, 2, 2, 128, 128),
                                           (2, 9, 5, 5, 36, 12), (70, 1, 32, 8, 128, 64), (1, 3, 1, 1, 1024, 1024), (2, 8, 2, 1, 100, 50)])
def test_turns(dtype, pairs, B, S, Hq, Hk, D, R):
    g = torch.Generator(device="cuda").manual_seed(D + S)
    q = torch.randn(B, S, Hq, D, generator=g, device="cuda").to(dtype)
    k = torch.randn(B, S, Hk, D, generator=g, device="cuda").to(dtype)
    f = ops.rotary_frequencies(R, 500000.0, device="cuda")
    pos = torch.randint(0, 1 << 20, (B, S), generator=g, device="cuda", dtype=torch.int32)
    yq, yk = ops.rotary(q, k, pos, f, pairs=pairs)
    close(yq, turned(q, pos, f, pairs))
    close(yk, turned(k, pos, f, pairs))
    assert torch.equal(yq[..., R:], q[..., R:])
    one = ops.rotary(q, None, pos.long(), f, pairs=pairs)
    assert torch.equal(one, yq)


@pytest.mark.parametrize("pairs", ["half", "interleaved"])
def test_gradient_turns_back(pairs):
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(2, 50, 4, 64, generator=g, device="cuda").bfloat16().requires_grad_()
    k = torch.randn(2, 50, 2, 64, generator=g, device="cuda").bfloat16().requires_grad_()
    f = ops.rotary_frequencies(48, device="cuda")
    pos = torch.arange(50, device="cuda") + 4000
    yq, yk = ops.rotary(q, k, pos, f, pairs=pairs, scale=1.25)
    gq, gk = torch.randn_like(yq), torch.randn_like(yk)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk), retain_graph=True)
    for got, grad in ((dq, gq), (dk, gk)):
        want, size = turned(grad, pos, f, pairs, 1.25, True)
        close(got, (want, size))
    (only,) = torch.autograd.grad(yk, k, gk)            # one of the two outputs used
    assert torch.equal(only, dk)
    # and against differences: the map is linear, so <g, y(x + r) - y(x)> = <dx, r> up to rounding
    r = torch.randn(q.shape, generator=g, device="cuda").double()
    along = (gq.double() * (turned(q.double() + r, pos, f, pairs, 1.25)[0] - turned(q.double(), pos, f, pairs, 1.25)[0])).sum()
    room = (2.0 ** -8 * turned(gq, pos, f, pairs, 1.25, True)[1] * r.abs()).sum()
    assert abs(along - (dq.double() * r).sum()) <= room


def test_far_positions_and_no_frequency_lost():
    x = torch.randn(1, 4, 1, 128, device="cuda")
    pos = torch.tensor([0, 1, 2 ** 30, -(2 ** 31)], device="cuda", dtype=torch.int32)
    f = ops.rotary_frequencies(128, device="cuda")
    y = ops.rotary(x, None, pos, f)
    close(y, turned(x, pos, f, "half"))
    assert torch.equal(y[:, 0], x[:, 0])                # position 0 turns nothing


def test_strides_and_alignment():
    g = torch.Generator(device="cuda").manual_seed(5)
    fused = torch.randn(2, 30, 3, 4, 64, generator=g, device="cuda").half()     # q, k, v of one projection
    q, k = fused[:, :, 0], fused[:, :, 1]
    pos = torch.arange(30, device="cuda")
    f = ops.rotary_frequencies(64, device="cuda")
    a = ops.rotary(q, k, pos, f)
    b = ops.rotary(q.contiguous(), k.contiguous(), pos, f)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    off = torch.randn(2 * 30 * 4 * 64 + 3, generator=g, device="cuda").half()[3:].view(2, 30, 4, 64)
    assert torch.equal(ops.rotary(off, None, pos, f), ops.rotary(off.clone(), None, pos, f))
    t = q.transpose(1, 2).contiguous().transpose(1, 2)                          # heads before tokens in memory
    assert torch.equal(ops.rotary(t, None, pos, f), a[0])
    shared = q[:1, :, :1].expand(2, 30, 4, 64)
    assert torch.equal(ops.rotary(shared, None, pos, f), ops.rotary(shared.contiguous(), None, pos, f))
    cols = torch.randn(2, 30, 4, 128, generator=g, device="cuda").half()[..., ::2]
    assert torch.equal(ops.rotary(cols, None, pos, f), ops.rotary(cols.contiguous(), None, pos, f))
    every_other = torch.arange(60, device="cuda")[::2]
    assert torch.equal(ops.rotary(q, None, every_other, f), ops.rotary(q, None, every_other.clone(), f))


@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("D,R", [(64, 64), (64, 32), (80, 40), (88, 8), (24, 16), (28, 20)])
def test_every_width_of_loads(pairs, D, R):
    """Starts on 2, 4, 8 and 16 byte boundaries, part of the head copied: the same bits as from a fresh tensor."""
    g = torch.Generator(device="cuda").manual_seed(6)
    pos, f = torch.arange(9, device="cuda"), ops.rotary_frequencies(R, device="cuda")
    for dtype in (torch.bfloat16, torch.float32):
        for off in (1, 2, 4, 8):
            x = torch.randn(2 * 9 * 3 * D + off, generator=g, device="cuda").to(dtype)[off:].view(2, 9, 3, D)
            y = ops.rotary(x, None, pos, f, pairs=pairs)
            assert torch.equal(y, ops.rotary(x.clone(), None, pos, f, pairs=pairs))
            assert torch.equal(y[..., R:], x[..., R:])


def test_graph_stream_host_and_empty():
    x = torch.randn(1, 40, 2, 64, device="cuda").bfloat16()
    pos, f = torch.arange(40, device="cuda"), ops.rotary_frequencies(64, device="cuda")
    want = ops.rotary(x, None, pos, f)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.rotary(x, None, pos, f)
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want * 2)
    assert torch.equal(ops.rotary(x.cpu(), None, pos.cpu(), f.cpu()), y.cpu())
    assert ops.rotary(x[:, :0], None, pos[:0], f).shape == (1, 0, 2, 64)
    q, k = ops.rotary(x, x[:, :, :0], pos, f)
    assert torch.equal(q, y) and k.shape == (1, 40, 0, 64)
