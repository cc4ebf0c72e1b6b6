"""What the attention operators refuse, and the frequencies: on the host, before any launch."""
import ctypes as C
import math

import pytest
import torch

from lego_b200 import _abi, ops


def t(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


Q, K = t(2, 5, 4, 64), t(2, 7, 2, 64)


@pytest.mark.parametrize("args,how", [
    ((t(2, 5, 64), K, K), {}),
    ((t(2, 5, 4, 64, dtype=torch.float32), K, K), {}),
    ((Q, t(2, 7, 2, 64, dtype=torch.bfloat16), K), {}),
    ((Q, K, t(2, 6, 2, 64)), {}),
    ((Q, t(3, 7, 2, 64), t(3, 7, 2, 64)), {}),
    ((Q, t(2, 7, 3, 64), t(2, 7, 3, 64)), {}),
    ((Q, t(2, 7, 0, 64), t(2, 7, 0, 64)), {}),
    ((t(2, 5, 4, 60), t(2, 7, 2, 60), t(2, 7, 2, 60)), {}),
    ((t(2, 5, 4, 136), t(2, 7, 2, 136), t(2, 7, 2, 136)), {}),
    ((Q, K, K), dict(prefix=ints(2))),
    ((Q, K, K), dict(causal=True, prefix=ints(3))),
    ((Q, K, K), dict(causal=True, prefix=ints(2).long())),
    ((Q, K, K), dict(documents=ints(2, 5))),
    ((t(2, 9, 4, 64), K, K), dict(documents=ints(2, 7))),
    ((Q, K, K), dict(softcap=-1.0)),
    ((Q, K, K), dict(softcap=math.inf)),
    ((Q, K, K), dict(scale=math.nan)),
    ((Q, K, K), dict(slopes=torch.zeros(2))),
    ((Q, K, K), dict(slopes=torch.zeros(4, dtype=torch.float64))),
    ((Q, K, K), dict(slopes=torch.zeros(4, requires_grad=True))),
])
def test_attention(args, how):
    with pytest.raises(ValueError):
        ops.attention(*args, **how)


@pytest.mark.parametrize("change", [
    dict(q=t(2, 3, 64)), dict(q=t(2, 3, 4, 64, dtype=torch.float32)), dict(k=t(9, 16, 2, 64, dtype=torch.bfloat16)),
    dict(v=t(9, 8, 2, 64)), dict(q=t(2, 3, 5, 64)), dict(q=t(2, 3, 4, 72)), dict(q=t(2, 65, 4, 64), parents=None),
    dict(q=t(2, 0, 4, 64), parents=None), dict(table=ints(2, 4).long()), dict(table=ints(3, 4)), dict(table=ints(2, 0)),
    dict(lengths=ints(3)), dict(lengths=ints(2).long()), dict(parents=ints(2, 4)), dict(softcap=-2.0),
    dict(scale=math.inf), dict(slopes=torch.zeros(2)), dict(k=t(0, 16, 2, 64), v=t(0, 16, 2, 64)),
    dict(q=t(2, 3, 4, 64).requires_grad_()),
])
def test_tree_attention(change):
    a = dict(q=t(2, 3, 4, 64), k=t(9, 16, 2, 64), v=t(9, 16, 2, 64), table=ints(2, 4), lengths=ints(2), parents=ints(2, 3))
    a.update(change)
    how = {n: a.pop(n) for n in ("softcap", "scale", "slopes") if n in a}
    with pytest.raises(ValueError):
        ops.tree_attention(a["q"], a["k"], a["v"], a["table"], a["lengths"], a["parents"], **how)


@pytest.mark.parametrize("q,k,pos,f,how", [
    (t(2, 5, 64), None, ints(2, 5), 8, {}),
    (t(2, 5, 1, 64, dtype=torch.float64), None, ints(2, 5), 8, {}),
    (Q, t(2, 6, 1, 64), ints(2, 5), 8, {}),
    (Q, t(2, 5, 1, 64, dtype=torch.float32), ints(2, 5), 8, {}),
    (Q, None, ints(5, 2), 8, {}),
    (Q, None, torch.zeros(2, 5), 8, {}),
    (Q, None, ints(5), 33, {}),
    (Q, None, ints(5), 0, {}),
    (Q, None, ints(5), 8, dict(pairs="thirds")),
    (Q, None, ints(5), 8, dict(scale=math.inf)),
])
def test_rotary(q, k, pos, f, how):
    with pytest.raises(ValueError):
        ops.rotary(q, k, pos, torch.zeros(f, dtype=torch.float64), **how)
    with pytest.raises(ValueError):
        ops.rotary(Q, None, ints(5), torch.zeros(8), **{})


def attention_desc(**change):
    d = _abi.Attention(dtype=_abi.F16, causal=1, batch=1, q_len=4, k_len=4, q_heads=2, k_heads=1, head_dim=64, scale=0.1)
    for s in (d.q_stride, d.k_stride, d.v_stride):
        s[:] = (512, 128, 64)
    for n, v in change.items():
        setattr(d, n, v)
    return d


def test_the_c_entry_points_return_their_reasons():
    lib = _abi.lib()
    assert lib.lego_attention_workspace_bytes(C.byref(attention_desc()), 1) >= 0
    assert lib.lego_attention_workspace_bytes(None, 0) == -1
    for change, status in ((dict(dtype=2), -8), (dict(batch=0), -4), (dict(q_len=0), -4), (dict(head_dim=136), -6),
                           (dict(head_dim=12), -6), (dict(q_heads=3, k_heads=2), -6), (dict(softcap=-1.0), -6),
                           (dict(scale=math.nan), -6), (dict(scale=1e38), -6), (dict(softcap=1e-35, scale=1.0), -6),
                           (dict(causal=0, prefix=4096), -6),
                           (dict(q_len=5, documents=4096), -6), (dict(q_len=1 << 40), -6)):
        assert lib.lego_attention_workspace_bytes(C.byref(attention_desc(**change)), 0) == status, change
    odd = attention_desc()
    odd.k_stride[1] = 65
    assert lib.lego_attention_workspace_bytes(C.byref(odd), 0) == -7
    d = attention_desc()
    args = [4096] * 6
    assert lib.lego_attention_fwd(C.byref(d), 0, *args[1:], 4096, 1 << 20, None) == -1
    assert lib.lego_attention_fwd(C.byref(d), 4098, *args[1:], 4096, 1 << 20, None) == -7
    assert lib.lego_attention_bwd(C.byref(d), *[4096] * 11, 0, None) == -6
    assert lib.lego_attention_bwd(C.byref(d), *[4096] * 10, None, 1 << 30, None) == -1

    r = _abi.Rotary(dtype=_abi.F16, pairs=0, position_bytes=4, batch=1, length=4, head_dim=64, rotary_dim=64, scale=1.0)
    r.heads[:] = (1, 0)
    bad = [4096, None, 4096, None, 4096, 4096, None]
    for change, status in ((dict(dtype=5), -8), (dict(pairs=2), -8), (dict(position_bytes=2), -8), (dict(batch=-1), -4),
                           (dict(rotary_dim=63), -6), (dict(rotary_dim=66), -6), (dict(head_dim=2000, rotary_dim=8), -6)):
        s = _abi.Rotary.from_buffer_copy(r)
        for n, v in change.items():
            setattr(s, n, v)
        assert lib.lego_rotary(C.byref(s), *bad) == status, change
    assert lib.lego_rotary(C.byref(r), None, None, 4096, None, 4096, 4096, None) == -1
    assert lib.lego_rotary(C.byref(r), 4097, None, 4096, None, 4096, 4096, None) == -7

    w = _abi.TreeAttention(dtype=_abi.BF16, batch=1, drafted=1, q_heads=2, k_heads=1, head_dim=64, pages=4, page_size=16,
                           max_pages=2, table_stride=2, scale=0.1)
    for s in (w.q_stride, w.k_stride, w.v_stride):
        s[:] = (512, 128, 64)
    assert lib.lego_tree_attention_workspace_bytes(C.byref(w)) >= 0
    for change, status in ((dict(dtype=2), -8), (dict(batch=0), -4), (dict(drafted=65), -6), (dict(drafted=0), -4),
                           (dict(pages=0), -4), (dict(page_size=0), -4), (dict(table_stride=1), -6), (dict(head_dim=4), -6),
                           (dict(q_heads=3, k_heads=2), -6), (dict(softcap=math.inf), -6),
                           (dict(page_size=1 << 20, max_pages=1 << 20, table_stride=1 << 20), -6)):
        s = _abi.TreeAttention.from_buffer_copy(w)
        for n, v in change.items():
            setattr(s, n, v)
        assert lib.lego_tree_attention_workspace_bytes(C.byref(s)) == status, change
    assert lib.lego_tree_attention(C.byref(w), None, *[4096] * 8, 1 << 30, None) == -1
    assert lib.lego_tree_attention(C.byref(w), 4097, *[4096] * 8, 1 << 30, None) == -7


def test_frequencies():
    f = ops.rotary_frequencies(8, 10000.0)
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    assert torch.allclose(ops.rotary_frequencies(8, scaling="linear", factor=4.0), f / 4, rtol=1e-15)
    ntk = ops.rotary_frequencies(8, scaling="ntk", factor=4.0)
    assert abs(ntk[0] - 1) < 1e-15 and abs(ntk[-1] - f[-1] / 4) < 1e-15
    b = ops.rotary_frequencies(8, scaling="bands", factor=4.0, original_length=1000, low=1.0, high=32.0)
    turns = 1000 * f / (2 * math.pi)
    assert b[0] == f[0] and abs(b[-1] - f[-1] / 4) < 1e-18       # 159 turns: kept; 0.16 turns: stretched
    keep = (turns[1] - 1) / 31
    assert abs(b[1] - f[1] * (keep + (1 - keep) / 4)) < 1e-16
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, base=0.0), dict(dim=8, factor=0.5), dict(dim=8, scaling="bent"),
                dict(dim=8, scaling="bands", low=4.0, high=4.0), dict(dim=8, scaling="bands", original_length=0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**bad)


LEARNED = torch.ones(4, requires_grad=True)


@pytest.mark.parametrize("given", ["slopes", "scale", "softcap"])
@pytest.mark.parametrize("learns", [(), (0,), (1,), (0, 1, 2)])
def test_a_learned_constant_of_attention_is_refused(given, learns):
    """Whatever else learns: with a q that does the call goes through an autograd function, and one that took the
    constant would give it no gradient."""
    how = {given: LEARNED if given == "slopes" else LEARNED[0]}
    args = [x.clone().requires_grad_(i in learns) for i, x in enumerate((Q, K, K))]
    with pytest.raises(ValueError, match=given):
        ops.attention(*args, **how)
    with pytest.raises(ValueError, match=given):
        ops.attention_fwd(*args, **how)
    with pytest.raises(ValueError, match=given):
        ops.attention_bwd(Q, *args, Q, torch.zeros(2, 4, 5), **how)
    with pytest.raises(ValueError, match=given):
        how = dict(dict(softcap=0.0, slopes=None, scale=None), **how)
        ops.LEGOAttention.apply(*args, False, None, None, how["softcap"], how["slopes"], how["scale"])


@pytest.mark.parametrize("learns", [(), (0,), (1,), (0, 1)])
def test_learned_frequencies_are_refused(learns):
    f = torch.ones(8, dtype=torch.float64, requires_grad=True)
    q, k = (x.clone().requires_grad_(i in learns) for i, x in enumerate((Q, t(2, 5, 2, 64))))
    with pytest.raises(ValueError, match="freqs"):
        ops.rotary(q, k, ints(5), f)
    with pytest.raises(ValueError, match="freqs"):
        ops.LEGORotary.apply(q, None, ints(5), f, "half", 1.0)
    with pytest.raises(ValueError, match="scale"):
        ops.rotary(q, k, ints(5), f.detach(), scale=LEARNED[0])


def test_learned_constants_of_tree_attention_are_refused():
    for given in ("slopes", "scale", "softcap"):
        with pytest.raises(ValueError, match=given):
            ops.tree_attention(t(2, 3, 4, 64), t(9, 16, 2, 64), t(9, 16, 2, 64), ints(2, 4), ints(2),
                               **{given: LEARNED if given == "slopes" else LEARNED[0]})


@pytest.mark.parametrize("which", range(4))
def test_forward_mode_derivatives_are_refused(which):
    """A dual tensor asks for a derivative without requiring a gradient: a result without a tangent would be a
    derivative of zero."""
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        def dual(i, x):
            return forward_ad.make_dual(x, torch.ones_like(x)) if i == which else x

        refused = pytest.raises(ValueError, match="forward-mode")
        for learns in (False, True):
            q = Q.clone().requires_grad_(learns)
            args = [dual(i, x) for i, x in enumerate((q, K, K, torch.zeros(4)))]
            with refused:
                ops.attention(*args[:3], slopes=args[3])
            with refused:
                ops.attention_fwd(*args[:3], slopes=args[3])
            with refused:
                ops.LEGOAttention.apply(*args[:3], False, None, None, 0.0, args[3], None)
            if which < 3:
                pair = [dual(i, x) for i, x in enumerate((q, t(2, 5, 2, 64), torch.ones(8, dtype=torch.float64)))]
                with refused:
                    ops.rotary(*pair[:2], ints(5), pair[2])
                with refused:
                    ops.LEGORotary.apply(*pair[:2], ints(5), pair[2], "half", 1.0)
        with refused:
            ops.attention_bwd(dual(0, Q), Q, K, K, dual(1, Q), dual(2, torch.zeros(2, 4, 5)), o_low=dual(3, Q))
        with refused:
            ops.tree_attention(dual(0, t(2, 3, 4, 64)), dual(1, t(9, 16, 2, 64)), dual(2, t(9, 16, 2, 64)), ints(2, 4),
                               ints(2), slopes=dual(3, torch.zeros(4)))
