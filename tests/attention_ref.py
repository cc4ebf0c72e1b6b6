"""Attention, rotary positions and tree attention in 64 bits, with bounds on how far a kernel that
multiplies 16-bit operands into 32-bit sums may be off, value by value.

u = eps / 2 of the type is the error of one rounding.  A kernel rounds the weights P (and the score
gradients dS) to the type before the second product and the result once, so

    |o - O|   <= (u + t) P |V| + u |O|                       t: error of the weights in 32 bits
    |dv - dV| <= (u + t) P' |dO| + u |dV|
    |ds - dS| <= u |dS| + e_S,   |dq - dQ| <= scale (u |dS| + e_S) |K| + u |dQ|,  dK likewise.

t: a score is a sum of D products, off by at most D eps32 sum |q k| scale, and a weight by twice that
relatively (its own score and the sum's); a cap or a bias adds a few roundings of its size.
e_S: P (t |dP - delta| + error of dP and delta), dP a sum of D products, delta = sum dO O with O
rounded to the type.  fp16 weights below its normal range are off by up to 2^-25 absolutely.
A weight under 2^-126 may be zero in 32 bits: up to 2^14 such terms, each times factors under 2^10, make
at most 2^-126 2^14 2^10 = 2^-102, less than FLOOR."""
import torch

EPS32 = 2.0 ** -23
FLOOR = 2.0 ** -100


def visible(Sq, Sk, causal, prefix, documents, device):
    i = torch.arange(Sq, device=device)[:, None] + (Sk - Sq)
    j = torch.arange(Sk, device=device)[None, :]
    see = torch.ones(1, Sq, Sk, dtype=torch.bool, device=device)
    if causal:
        see = (j <= i)[None]
        if prefix is not None:
            see = see | (j < prefix.to(device)[:, None, None])
    if documents is not None:
        d = documents.to(device)
        see = see & (d[:, Sk - Sq:, None] == d[:, None, :]) & (d[:, None, :] >= 0)
    return see


def attention(q, k, v, do=None, causal=False, prefix=None, documents=None, softcap=0.0, slopes=None, scale=None):
    """{"o", "lse", "dq", "dk", "dv"} as (value, bound) pairs, float64; gradients by autograd."""
    dev, eps = q.device, torch.finfo(q.dtype).eps / 2
    B, Sq, Hq, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    G = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    see = visible(Sq, Sk, causal, prefix, documents, dev)[:, None].expand(B, Hq, Sq, Sk)
    ok_q, ok_k = see.any(-1).any(1), see.any(-2).any(1)            # [B, Sq], [B, Sk]

    def lift(x, ok):                                               # values nobody may use count as zeros
        return torch.where(ok[:, :, None, None], x.double(), 0.0).detach()

    qd, kd, vd = (lift(x, ok).requires_grad_() for x, ok in ((q, ok_q), (k, ok_k), (v, ok_k)))

    def heads(x):
        x = x.permute(0, 2, 1, 3)
        return x.repeat_interleave(Hq // x.shape[1], 1)

    s = scale * heads(qd) @ heads(kd).mT
    far = ((torch.arange(Sq, device=dev)[:, None] + Sk - Sq) - torch.arange(Sk, device=dev)[None, :]).abs().double()
    bend = torch.ones_like(s)
    if softcap:
        t = torch.tanh(s / softcap)
        s, bend = softcap * t, (1 - t * t).detach()
    if slopes is not None:
        s = s - slopes.double().to(dev)[None, :, None, None] * far
    s = s.masked_fill(~see, float("-inf"))
    some = see.any(-1, keepdim=True)
    p = torch.where(some, torch.softmax(s.masked_fill(~some, 0.0), -1), 0.0)
    o = p @ heads(vd)
    with torch.no_grad():
        size = abs(scale) * (heads(qd).abs() @ heads(kd).abs().mT)
        t = 2 * (D + 4) * EPS32 * size.max().item() + 16 * EPS32 + 8 * EPS32 * softcap
        if slopes is not None:
            t += 4 * EPS32 * slopes.max().item() * far.max().item()
        small = 2.0 ** -25 if q.dtype == torch.float16 else FLOOR
        lse = torch.where(some[..., 0], torch.logsumexp(s, -1), -float("inf"))
        l = torch.exp(lse - s.amax(-1)).nan_to_num(1.0)[..., None]
        back = lambda x: x.permute(0, 2, 1, 3)                     # noqa: E731
        fold = lambda x: x.reshape(B, Hk, G, *x.shape[2:]).sum(2).permute(0, 2, 1, 3)   # noqa: E731
        va = heads(vd).abs()
        out = {"o": (back(o), back((eps + t) * (p @ va) + small / l * (see.double() @ va) + eps * o.abs()) + small),
               "lse": (lse, t + 4 * EPS32 * lse.nan_to_num(0, 0, 0).abs() + EPS32)}
    if do is None:
        return {n: (a.detach(), b) for n, (a, b) in out.items()}
    dod = lift(do, ok_q)
    dq, dk, dv = torch.autograd.grad(back(o), (qd, kd, vd), dod)
    with torch.no_grad():
        dh, da = heads(dod), heads(dod).abs()
        dp, dpa = dh @ heads(vd).mT, da @ va.mT
        delta, deltaa = (dh * o).sum(-1, keepdim=True), (da * (eps * o.abs() + out["o"][1].permute(0, 2, 1, 3))).sum(-1, keepdim=True)
        ds = (p * (dp - delta) * bend).abs()
        es = p * (t * (dp - delta).abs() + (D + 4) * EPS32 * (dpa + (da * o.abs()).sum(-1, keepdim=True)) + deltaa) * bend
        es = es + p * (dp - delta).abs() * 16 * EPS32
        ds = eps * ds + es
        # weights and score gradients in fp16: scaled so that what falls below its range is below 2^-13 of the largest
        # possible, itself under 2^-25 of the scale; the absolute rest is counted against the largest products
        tiny = 2.0 ** -24 * da.max().item() * va.max().item() * D * 2.0 ** -13 if q.dtype == torch.float16 else 0.0
        ds = ds + tiny * see
        out["dq"] = dq, abs(scale) * back(ds @ heads(kd).abs()) + eps * dq.abs() + small
        out["dk"] = dk, abs(scale) * fold(ds.mT @ heads(qd).abs()) + eps * dk.abs() + small
        out["dv"] = dv, fold(((eps + t) * p + small * 2.0 ** -13 * see).mT @ da) + eps * dv.abs() + small
    return {n: (a.detach(), b) for n, (a, b) in out.items()}


def far_off(got, want):
    """The largest error over its bound, 0 where both agree exactly (infinities among them)."""
    value, bound = want
    got = got.double()
    if got.shape != value.shape or not torch.equal(torch.isfinite(got), torch.isfinite(value)):
        return float("inf")
    fine = torch.isfinite(value)
    if not torch.equal(got[~fine], value[~fine]):
        return float("inf")
    if not fine.any():
        return 0.0
    err = (got - value)[fine].abs()
    room = (bound.expand_as(value) if torch.is_tensor(bound) else torch.full_like(value, bound))[fine]
    return torch.where(err == 0, 0.0, err / room.clamp_min(1e-300)).max().item()


def tree(q, k_cache, v_cache, page_table, lengths, parents, softcap=0.0, slopes=None, scale=None):
    """(value, bound) of tree attention, sequence by sequence on the definition."""
    B, T, Hq, D = q.shape
    pages, page, Hk, _ = k_cache.shape
    eps = torch.finfo(q.dtype).eps / 2
    small = 2.0 ** -25 if q.dtype == torch.float16 else FLOOR
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    room = torch.zeros_like(out)
    table, lens = page_table.tolist(), lengths.tolist()
    par = parents.tolist() if parents is not None else [list(range(-1, T - 1))] * B
    for b in range(B):
        if lens[b] < 0:
            continue
        sees, depth = [], []
        for t in range(T):
            up = par[b][t]
            if up == -1:
                sees.append({t}), depth.append(0)
            elif 0 <= up < t and sees[up] is not None:
                sees.append(sees[up] | {t}), depth.append(depth[up] + 1)
            else:
                sees.append(None), depth.append(0)
        n = min(lens[b] + T, len(table[b]) * page)
        where = [(table[b][j // page], j % page) for j in range(n)]
        real = [0 <= pg < pages for pg, _ in where]
        pg = torch.tensor([p if r else 0 for (p, _), r in zip(where, real)], device=q.device, dtype=torch.long)
        sl = torch.tensor([s for _, s in where], device=q.device, dtype=torch.long)
        rl = torch.tensor(real, device=q.device, dtype=torch.bool)
        at = torch.tensor([j if j < lens[b] else lens[b] + depth[j - lens[b]] for j in range(n)], device=q.device, dtype=torch.float64)
        k, v = k_cache[pg, sl].double(), v_cache[pg, sl].double()
        for t in range(T):
            if sees[t] is None:
                continue
            see = torch.tensor([j < lens[b] or (j - lens[b]) in sees[t] for j in range(n)], device=q.device, dtype=torch.bool) & rl
            if not see.any():
                continue
            for h in range(Hq):
                kk, vv = k[see, h // (Hq // Hk)], v[see, h // (Hq // Hk)]
                qq = q[b, t, h].double()
                s = scale * kk @ qq
                tol = 2 * (D + 4) * EPS32 * (abs(scale) * kk.abs() @ qq.abs()).max().item() + 16 * EPS32 + 8 * EPS32 * softcap
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                if slopes is not None:
                    far = (lens[b] + depth[t] - at[see]).abs()
                    s = s - slopes[h].double() * far
                    tol += 4 * EPS32 * slopes[h].item() * far.max().item()
                w = torch.softmax(s, -1)
                o = w @ vv
                l = 1.0 / w.max()
                out[b, t, h] = o
                room[b, t, h] = (eps + tol) * (w @ vv.abs()) + small / l * vv.abs().sum(0) + eps * o.abs() + small
    return out, room
