"""Measured cases of the attention operators: rotary positions, attention with a cap / distance bias /
document and prefix masks (forward and backward), and attention of drafted token trees over a paged cache.

``run`` computes a case in plain torch operations, or, with ``own`` set, through ``lego_b200.ops``."""
import math
import random

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---- the cases --------------------------------------------------------------------------------


def listed():
    return [
        # one new token of each of 64 sequences, far into their contexts: a launch's latency counts
        dict(name="rotary decode", op="rotary", type="bf16", B=64, S=1, Hq=32, Hk=8, D=128, R=128, pairs="half", far=131072, train=False),
        # a prompt of odd length; only half of each head turns, neighbouring values are the pairs
        dict(name="rotary partial", op="rotary", type="fp16", B=3, S=2047, Hq=16, Hk=16, D=64, R=32, pairs="interleaved", far=4096, train=False),
        # a training step's queries and keys, forward and gradients
        dict(name="rotary train", op="rotary", type="bf16", B=2, S=8192, Hq=32, Hk=8, D=128, R=128, pairs="half", far=8192, train=True),
        # a short bidirectional call
        dict(name="attention short", op="attention", type="fp16", B=2, Sq=77, Sk=77, Hq=4, Hk=4, D=64, causal=False, prefix=False, docs=0, softcap=0.0, slopes=False, train=False, ragged=1),
        # a long prompt, eight query heads on one key head
        dict(name="attention prompt", op="attention", type="bf16", B=1, Sq=16384, Sk=16384, Hq=8, Hk=1, D=128, causal=True, prefix=False, docs=0, softcap=0.0, slopes=False, train=False, ragged=2),
        # a causal training step with shared key heads
        dict(name="attention train", op="attention", type="bf16", B=2, Sq=4096, Sk=4096, Hq=32, Hk=8, D=128, causal=True, prefix=False, docs=0, softcap=0.0, slopes=False, train=True, ragged=3),
        # documents packed into one row, padded at its end, scores capped
        dict(name="attention packed", op="attention", type="fp16", B=1, Sq=8191, Sk=8191, Hq=16, Hk=16, D=64, causal=True, prefix=False, docs=11, softcap=30.0, slopes=False, train=True, ragged=4),
        # prompts that see themselves both ways, answers that look back, a bias by distance, a head width between the powers of two
        dict(name="attention prefix", op="attention", type="bf16", B=3, Sq=1999, Sk=1999, Hq=8, Hk=2, D=80, causal=True, prefix=True, docs=0, softcap=0.0, slopes=True, train=True, ragged=5),
        # one sequence, one token
        dict(name="tree one token", op="tree", type="bf16", B=1, T=1, L=1000, Hq=32, Hk=8, D=128, page=64, softcap=0.0, slopes=False, ragged=0),
        # a batch of sequences of very different lengths, one token each
        dict(name="tree batch", op="tree", type="bf16", B=64, T=1, L=8192, Hq=32, Hk=8, D=128, page=64, softcap=0.0, slopes=False, ragged=6),
        # drafted trees of 37 tokens, capped scores, pages that end inside every tile
        dict(name="tree drafts", op="tree", type="fp16", B=8, T=37, L=16384, Hq=16, Hk=8, D=64, page=48, softcap=50.0, slopes=False, ragged=7),
        # few very long contexts, short drafts, a bias by distance
        dict(name="tree long", op="tree", type="bf16", B=2, T=8, L=131072, Hq=64, Hk=8, D=128, page=16, softcap=0.0, slopes=True, ragged=8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "attention", "attention", "tree", "tree"])
    Hk = rng.choice([1, 2, 3, 4, 8])
    Hq = Hk * rng.choice([1, 2, 4, 5, 8])
    if op == "rotary":
        D = rng.choice([32, 64, 80, 96, 128])
        t = rng.choice(["fp16", "bf16", "fp32"])
        tokens = (2 * 8192 * 40 * 128) // ((Hq + Hk) * D * (2 if t == "fp32" else 1))
        S = _log(rng, 1, min(8192, tokens))
        B = _log(rng, 1, max(1, min(64, tokens // S)))
        return dict(op=op, type=t, B=B, S=S, Hq=Hq, Hk=Hk, D=D, R=rng.choice([D, D // 2]),
                    pairs=rng.choice(["half", "interleaved"]), far=_log(rng, 512, 131072), train=rng.random() < 0.4)
    if op == "attention":
        D = rng.choice([32, 64, 72, 80, 96, 128])
        most = 32 * 4096 * 4096                                  # scores of a call
        Sk = _log(rng, 16, min(8192, math.isqrt(most // Hq)))
        Sq = Sk if rng.random() < 0.7 else _log(rng, 1, Sk)
        B = _log(rng, 1, max(1, min(32, most // (Sq * Sk * Hq))))
        causal = rng.random() < 0.8
        return dict(op=op, type=rng.choice(["fp16", "bf16"]), B=B, Sq=Sq, Sk=Sk, Hq=Hq, Hk=Hk, D=D, causal=causal,
                    prefix=causal and rng.random() < 0.25, docs=rng.choice([0, 0, 2, 5, 17]) if Sk > 64 else 0,
                    softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3, train=rng.random() < 0.6,
                    ragged=rng.randrange(1 << 20))
    D = rng.choice([64, 80, 128])
    L = _log(rng, 32, 65536)
    B = _log(rng, 1, max(1, min(128, (2 * 131072 * 8) // (L * Hk))))
    T = 1 if rng.random() < 0.4 else rng.randrange(2, 65)
    return dict(op=op, type=rng.choice(["fp16", "bf16"]), B=B, T=T, L=L, Hq=Hq, Hk=Hk, D=D, page=rng.choice([16, 32, 48, 64, 128]),
                softcap=rng.choice([0.0, 0.0, 30.0]), slopes=rng.random() < 0.3, ragged=rng.randrange(1 << 20))


# ---- lengths and masks of a case (they follow from the case, the values from the seed) -----------


def _documents(case):
    """Document numbers [B][Sk]: consecutive runs, -1 on padding at a row's end."""
    r = random.Random(case["ragged"])
    rows = []
    for _ in range(case["B"]):
        Sk, n = case["Sk"], case["docs"]
        end = Sk - r.randrange(0, max(1, Sk // 16))
        cuts = sorted(r.randrange(1, end + 1) for _ in range(n - 1))
        row, at = [], 0
        for d, cut in enumerate(cuts + [end]):
            row += [d] * (cut - at)
            at = max(at, cut)
        rows.append(row + [-1] * (Sk - len(row)))
    return rows


def _prefixes(case):
    r = random.Random(case["ragged"] + 1)
    return [r.randrange(0, case["Sk"] + 1) for _ in range(case["B"])]


def _lengths(case):
    """Cached tokens before the drafted ones."""
    r = random.Random(case["ragged"])
    return [case["L"]] + [r.randrange(case["L"] // 8, case["L"] + 1) for _ in range(case["B"] - 1)]


def _parents(case):
    r = random.Random(case["ragged"] + 2)
    return [[-1] + [r.randrange(max(0, t - 6), t) for t in range(1, case["T"])] for _ in range(case["B"])]


def _pairs(case):
    """Visible (query, key) pairs of one head, over the batch."""
    B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
    docs = _documents(case) if case["docs"] else [[0] * Sk] * B
    prefixes = _prefixes(case) if case["prefix"] else [0] * B
    off, total = Sk - Sq, 0
    for b in range(B):
        starts, ends, at = {}, {}, 0
        for j, d in enumerate(docs[b]):
            starts.setdefault(d, j)
            ends[d] = j + 1
        for i in range(Sq):
            d = docs[b][i + off]
            if d < 0:
                continue
            hi = max(min(ends[d], i + off + 1), min(ends[d], prefixes[b])) if case["causal"] else ends[d]
            total += max(0, hi - starts[d])
    return total


# ---- inputs -------------------------------------------------------------------------------------


def _slopes(H):
    return 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["type"]]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * by).to(t)

    B, Hq, Hk, D = case["B"], case["Hq"], case["Hk"], case["D"]
    s = dict(case=case)
    if case["op"] == "rotary":
        S, R = case["S"], case["R"]
        s["q"], s["k"] = normal(B, S, Hq, D), normal(B, S, Hk, D)
        first = torch.randint(0, max(1, case["far"] - S) + 1, (B, 1), generator=g, device="cuda", dtype=torch.int32)
        s["positions"] = first + torch.arange(S, device="cuda", dtype=torch.int32)
        s["freqs"] = 500000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
        if case["train"]:
            s["dq"], s["dk"] = normal(B, S, Hq, D, by=0.05), normal(B, S, Hk, D, by=0.05)
            s["q"].requires_grad_()
            s["k"].requires_grad_()
        return s
    s["slopes"] = _slopes(Hq) if case["slopes"] else None
    if case["op"] == "attention":
        Sq, Sk = case["Sq"], case["Sk"]
        # with a cap the raw scores spread into the range where it bends them
        s["q"], s["k"], s["v"] = normal(B, Sq, Hq, D, by=4.0 if case["softcap"] else 1.5), normal(B, Sk, Hk, D), normal(B, Sk, Hk, D)
        s["documents"] = torch.tensor(_documents(case), dtype=torch.int32, device="cuda") if case["docs"] else None
        s["prefix"] = torch.tensor(_prefixes(case), dtype=torch.int32, device="cuda") if case["prefix"] else None
        if case["train"]:
            s["do"] = normal(B, Sq, Hq, D, by=0.05)
            for n in "qkv":
                s[n].requires_grad_()
        return s
    T, page = case["T"], case["page"]
    lengths = _lengths(case)
    need = [-(-(n + T) // page) for n in lengths]
    order = torch.randperm(sum(need) + 1, generator=g, device="cuda").to(torch.int32)  # a page that none uses among them
    table, at = torch.zeros(B, max(need), dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s["q"] = normal(B, T, Hq, D, by=4.0 if case["softcap"] else 1.5)
    s["k_cache"], s["v_cache"] = normal(sum(need) + 1, page, Hk, D), normal(sum(need) + 1, page, Hk, D)
    s["page_table"], s["lengths"] = table, torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["parents"] = torch.tensor(_parents(case), dtype=torch.int32, device="cuda") if T > 1 else None
    return s


# ---- one pass -----------------------------------------------------------------------------------


def run(s):
    return {"rotary": _run_rotary, "attention": _run_attention, "tree": _run_tree}[s["case"]["op"]](s)


def _run_rotary(s):
    c = s["case"]
    if own:
        from lego_b200 import ops
        q, k = ops.rotary(s["q"], s["k"], s["positions"], s["freqs"], pairs=c["pairs"])
        if not c["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    with torch.no_grad():
        angle = s["positions"].double()[:, :, None, None] * s["freqs"]
        cos, sin = angle.cos().float(), angle.sin().float()
        out = {"q": _turn(s["q"], cos, sin, c), "k": _turn(s["k"], cos, sin, c)}
        if c["train"]:
            out["dq"], out["dk"] = _turn(s["dq"], cos, -sin, c), _turn(s["dk"], cos, -sin, c)
        return out


def _turn(x, cos, sin, c):
    R, f = c["R"], x.float()
    y = f.clone()
    if c["pairs"] == "half":
        a, b = f[..., :R // 2], f[..., R // 2:R]
        y[..., :R // 2], y[..., R // 2:R] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = f[..., 0:R:2], f[..., 1:R:2]
        y[..., 0:R:2], y[..., 1:R:2] = a * cos - b * sin, b * cos + a * sin
    return y.to(x.dtype)


def _run_attention(s):
    c = s["case"]
    if own:
        from lego_b200 import ops
        o = ops.attention(s["q"], s["k"], s["v"], causal=c["causal"], prefix=s["prefix"], documents=s["documents"],
                          softcap=c["softcap"], slopes=s["slopes"])
        if not c["train"]:
            return {"o": o}
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    with torch.no_grad():
        return _plain_attention(s, c)


def _visible(s, c):
    """[B, Sq, Sk] (or with ones in front): which key a query sees; its position is that of the last Sq tokens."""
    Sq, Sk = c["Sq"], c["Sk"]
    i = torch.arange(Sk - Sq, Sk, device="cuda")[:, None]
    j = torch.arange(Sk, device="cuda")[None, :]
    see = torch.ones(1, Sq, Sk, dtype=torch.bool, device="cuda")
    if c["causal"]:
        see = see & (j <= i)
        if s["prefix"] is not None:
            see = see | (j < s["prefix"][:, None, None])
    if s["documents"] is not None:
        d = s["documents"]
        see = see & (d[:, Sk - Sq:, None] == d[:, None, :]) & (d[:, None, :] >= 0)
    return see


def _plain_attention(s, c):
    B, Sq, Sk, Hq, Hk, D = (c[n] for n in ("B", "Sq", "Sk", "Hq", "Hk", "D"))
    G, scale = Hq // Hk, D ** -0.5

    def heads(x):  # [B, Hk, G * S, D]: the query heads of one key head as rows of one product
        n = x.shape[2] // Hk
        return x.float().permute(0, 2, 1, 3).reshape(B, Hk, n * x.shape[1], D)

    def back(x, H, like):
        return x.reshape(B, H, -1, D).permute(0, 2, 1, 3).to(like.dtype)

    q, k, v = heads(s["q"]), heads(s["k"]), heads(s["v"])
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).view(B, Hk, G, Sq, Sk)
    bend = None
    if c["softcap"]:
        p = p.div_(c["softcap"]).tanh_()
        bend = 1 - p * p if c["train"] else None
        p = p.mul_(c["softcap"])
    if s["slopes"] is not None:
        far = (torch.arange(Sk - Sq, Sk, device="cuda")[:, None] - torch.arange(Sk, device="cuda")[None, :]).abs().float()
        p -= s["slopes"].view(1, Hk, G, 1, 1) * far
    p.masked_fill_(~_visible(s, c)[:, None, None], float("-inf"))
    p -= p.amax(-1, keepdim=True).clamp_min_(torch.finfo(torch.float32).min)
    p.exp_()
    p /= p.sum(-1, keepdim=True).clamp_min_(torch.finfo(torch.float32).tiny)
    p = p.view(B, Hk, G * Sq, Sk)
    of = torch.matmul(p, v)
    out = {"o": back(of, Hq, s["q"])}
    if c["train"]:
        do = heads(s["do"])
        out["dv"] = back(torch.matmul(p.transpose(-1, -2), do), Hk, s["v"])
        ds = torch.matmul(do, v.transpose(-1, -2))
        ds -= (do * of).sum(-1, keepdim=True)
        ds *= p
        if bend is not None:
            ds *= bend.view_as(ds)
        ds *= scale
        out["dq"] = back(torch.matmul(ds, k), Hq, s["q"])
        out["dk"] = back(torch.matmul(ds.transpose(-1, -2), q), Hk, s["k"])
    return out


def _run_tree(s):
    c = s["case"]
    if own:
        from lego_b200 import ops
        return {"o": ops.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"], s["parents"],
                                        softcap=c["softcap"], slopes=s["slopes"])}
    B, T, Hq, Hk, D, page = (c[n] for n in ("B", "T", "Hq", "Hk", "D", "page"))
    G, n = Hq // Hk, s["page_table"].shape[1] * page
    k = s["k_cache"][s["page_table"].long()].view(B, n, Hk, D).float().transpose(1, 2)
    v = s["v_cache"][s["page_table"].long()].view(B, n, Hk, D).float().transpose(1, 2)
    q = s["q"].float().view(B, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * T, D)
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(D ** -0.5).view(B, Hk, G, T, n)
    if c["softcap"]:
        p = p.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    # ancestors by squaring the parent relation: a token sees itself, its parent, the parent's parent, ...
    ancestors = torch.eye(T, device="cuda").expand(B, T, T)
    if s["parents"] is not None:
        up = (s["parents"][:, :, None] == torch.arange(T, device="cuda")).float() + ancestors
        for _ in range(max(1, (T - 1).bit_length())):
            up = torch.matmul(up, up).clamp_max(1.0)
        ancestors = up
    depth = (ancestors.sum(-1) - 1).long()
    j = torch.arange(n, device="cuda")
    slot = j[None, :] - s["lengths"][:, None]                       # [B, n]: the drafted token in this place, if any
    drafted = torch.gather(ancestors, 2, slot.clamp(0, T - 1)[:, None, :].expand(B, T, n)) > 0
    see = (slot < 0)[:, None, :] | (drafted & ((slot >= 0) & (slot < T))[:, None, :])
    if s["slopes"] is not None:
        at = torch.where(slot < 0, j[None, :], s["lengths"][:, None] + torch.gather(depth, 1, slot.clamp(0, T - 1)))
        far = (s["lengths"][:, None] + depth)[:, :, None] - at[:, None, :]
        p -= s["slopes"].view(1, Hk, G, 1, 1) * far.abs().float()[:, None, None]
    p.masked_fill_(~see[:, None, None], float("-inf"))
    p -= p.amax(-1, keepdim=True)
    p.exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hk, G * T, n), v)
    return {"o": o.view(B, Hk, G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(s["q"].dtype)}


# ---- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    e = 4 if case["type"] == "fp32" else 2
    B, Hq, Hk, D = case["B"], case["Hq"], case["Hk"], case["D"]
    if case["op"] == "rotary":
        values = B * case["S"] * (Hq + Hk) * D
        ways = 2 if case["train"] else 1
        return {"bytes": ways * 2 * values * e + B * case["S"] * 4 + case["R"] * 4, "flops": ways * 3 * values * case["R"] // D}
    if case["op"] == "attention":
        q, k = B * case["Sq"] * Hq * D * e, B * case["Sk"] * Hk * D * e
        ints = (B * case["Sk"] * 4 if case["docs"] else 0) + (B * 4 if case["prefix"] else 0) + (Hq * 4 if case["slopes"] else 0)
        pairs = _pairs(case) * Hq
        if not case["train"]:
            return {"bytes": 2 * q + 2 * k + ints, "flops": 4 * D * pairs}
        return {"bytes": 2 * q + 2 * k + (3 * q + 2 * k) + (q + 2 * k) + ints, "flops": 14 * D * pairs}
    T, lengths = case["T"], _lengths(case)
    seen = sum(lengths) + T * B
    ints = B * 4 + sum(-(-(n + T) // case["page"]) for n in lengths) * 4 + (B * T * 4 if T > 1 else 0) + (Hq * 4 if case["slopes"] else 0)
    return {"bytes": 2 * seen * Hk * D * e + 2 * B * T * Hq * D * e + ints, "flops": 4 * D * Hq * T * seen}


# ---- the definition, in 64 bits ---------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "attention": _exact_attention, "tree": _exact_tree}[case["op"]](s, case)


def _exact_rotary(s, c):
    """Each pair as a complex number, turned by exp(i * position * frequency)."""
    R = c["R"]
    angle = s["positions"].to(torch.float64).unsqueeze(-1) * s["freqs"]
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None, :]

    def one(x, by):
        y = x.to(torch.float64).clone()
        head = y[..., :R]
        z = head.unflatten(-1, (2, R // 2)).movedim(-2, -1) if c["pairs"] == "half" else head.unflatten(-1, (R // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * by)
        y[..., :R] = (z.movedim(-1, -2) if c["pairs"] == "half" else z).flatten(-2)
        return y

    out = {"q": one(s["q"], turn), "k": one(s["k"], turn)}
    if c["train"]:
        out["dq"], out["dk"] = one(s["dq"], turn.conj()), one(s["dk"], turn.conj())
    return out


def _exact_attention(s, c):
    """Head by head: softmax of the visible scores, and the derivatives of <o, do>."""
    B, Sq, Sk, Hq, Hk, D = (c[n] for n in ("B", "Sq", "Sk", "Hq", "Hk", "D"))
    if B * Hq * Sq * Sk > 2.2e9:
        return None
    f = {n: s[n].double() for n in ("q", "k", "v") + (("do",) if c["train"] else ())}
    out = {"o": torch.zeros_like(f["q"])}
    if c["train"]:
        out |= {"dq": torch.zeros_like(f["q"]), "dk": torch.zeros_like(f["k"]), "dv": torch.zeros_like(f["v"])}
    at_q, at_k = torch.arange(Sq, device="cuda") + (Sk - Sq), torch.arange(Sk, device="cuda")
    gap = at_q.unsqueeze(1) - at_k
    for b in range(B):
        hidden = gap < 0 if c["causal"] else torch.zeros_like(gap, dtype=torch.bool)
        if c["prefix"]:
            hidden = hidden & ~(at_k < s["prefix"][b]).unsqueeze(0)
        if c["docs"]:
            d = s["documents"][b]
            hidden = hidden | (d[at_q].unsqueeze(1) != d) | (d < 0)
        for h in range(Hq):
            q, k, v = f["q"][b, :, h], f["k"][b, :, h // (Hq // Hk)], f["v"][b, :, h // (Hq // Hk)]
            z = q @ k.mT / math.sqrt(D)
            t = torch.tanh(z / c["softcap"]) if c["softcap"] else None
            z = c["softcap"] * t if c["softcap"] else z
            if c["slopes"]:
                z = z - s["slopes"][h].double() * gap.abs()
            z = torch.where(hidden, -math.inf, z)
            w = torch.softmax(z, -1).nan_to_num(0.0)
            out["o"][b, :, h] = o = w @ v
            if c["train"]:
                do = f["do"][b, :, h]
                dz = w * (do @ v.mT - (o * do).sum(-1, keepdim=True))
                dz = dz * (1 - t * t) / math.sqrt(D) if c["softcap"] else dz / math.sqrt(D)
                out["dq"][b, :, h] = dz @ k
                out["dk"][b, :, h // (Hq // Hk)] += dz.mT @ q
                out["dv"][b, :, h // (Hq // Hk)] += w.mT @ do
    return out


def _exact_tree(s, c):
    """Sequence by sequence, over the tokens that each drafted token descends from."""
    T, Hq, Hk, D, page = (c[n] for n in ("T", "Hq", "Hk", "D", "page"))
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lengths, parents = _lengths(c), _parents(c)
    for b, n in enumerate(lengths):
        pages = s["page_table"][b, :-(-(n + T) // page)].long()
        k, v = (s[x][pages].flatten(0, 1)[:n + T].double().repeat_interleave(Hq // Hk, 1) for x in ("k_cache", "v_cache"))
        see, depth = torch.zeros(T, n + T, dtype=torch.bool), []
        for t in range(T):
            see[t, :n] = True
            see[t, n + t] = True
            up = parents[b][t]
            depth.append(depth[up] + 1 if up >= 0 else 0)
            if up >= 0:
                see[t, n:] |= see[up, n:]
        z = torch.einsum("thd,nhd->htn", s["q"][b].double(), k) / math.sqrt(D)
        if c["softcap"]:
            z = c["softcap"] * torch.tanh(z / c["softcap"])
        if c["slopes"]:
            at = torch.tensor(list(range(n)) + [n + x for x in depth], device="cuda")
            z = z - s["slopes"].double()[:, None, None] * (at[n:, None] - at[None, :]).abs()
        z = torch.where(see.cuda(), z, -math.inf)
        o[b] = torch.einsum("htn,nhd->thd", torch.softmax(z, -1), v)
    return {"o": o}
