"""Plain 64-bit forms of the long-support attention operators, with the error
bounds their kernels are held to. CPU or GPU tensors; test infrastructure."""

from __future__ import annotations

import math

import torch


def rounding(y, dtype: torch.dtype):
    """Largest error of rounding y to `dtype` once: half a step, which is relative for normal
    numbers and half the spacing eps x (smallest normal) below them (f16: 2^-25)."""

    f = torch.finfo(dtype)
    return f.eps / 2 * y.abs() + f.smallest_normal * f.eps / 2


def angles(coords, freqs, sections, rows):
    """(B, 1, rows, pairs) angles; rows before the placed ones have none."""

    axis = torch.tensor([a for a, m in enumerate(sections) for _ in range(m)], device=coords.device)
    c = coords.double()[..., axis] * freqs
    pad = torch.zeros(c.shape[0], rows - c.shape[1], c.shape[2], dtype=torch.float64, device=c.device)
    return torch.cat([pad, c], 1)[:, None]


def rotate(x, ang, adjacent=False):
    p = ang.shape[-1]
    at = torch.arange(p, device=x.device)
    i, j = (2 * at, 2 * at + 1) if adjacent else (at, at + p)
    y = x.clone()
    y[..., i] = x[..., i] * ang.cos() - x[..., j] * ang.sin()
    y[..., j] = x[..., j] * ang.cos() + x[..., i] * ang.sin()
    return y


def qk_norm(x, w, ang, adjacent=False, eps=1e-6):
    y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    if w is not None:
        y = y * w
    return y if ang is None else rotate(y, ang, adjacent)


def means(k, block, kv_lens=None):
    b, h, s, d = k.shape
    nb = -(-s // block)
    out = torch.zeros(b, h, nb, d, dtype=torch.float64, device=k.device)
    for i in range(b):
        n = s if kv_lens is None else int(kv_lens[i])
        for j in range(nb):
            if j * block < n:
                out[i, :, j] = k[i, :, j * block : min(n, (j + 1) * block)].double().mean(1)
    return out


def select(q, mean, topk, block, kv_rows, kv_lens=None, q_lens=None, keep_first=0, keep_own=False):
    """Row by row: forced blocks, then sorted (-score, index)."""

    b, hq, sq, d = q.shape
    hk = mean.shape[1]
    score = q.double().view(b, hk, hq // hk, sq, d).sum(2) @ mean.double().transpose(-1, -2)
    score = torch.where(score.isnan(), -math.inf, score).cpu()
    out = torch.full((b, hk, sq, topk), -1, dtype=torch.int32)
    for i in range(b):
        live = -(-(kv_rows if kv_lens is None else int(kv_lens[i])) // block)
        for h in range(hk):
            for r in range(sq if q_lens is None else int(q_lens[i])):
                forced = [j for j in range(live) if j < keep_first or (keep_own and j == r // block)]
                rest = [j for j in range(live) if j not in forced]
                s = score[i, h, r].tolist()
                kept = sorted((forced + sorted(rest, key=lambda j: (-s[j], j)))[:topk])
                out[i, h, r, : len(kept)] = torch.tensor(kept, dtype=torch.int32)
    return out


def seen_keys(index, sk, block, kv_lens=None, q_lens=None):
    """(B, Hkv, Sq, Sk) truth table of the keys each query sees."""

    b, hk, sq, topk = index.shape
    nb = -(-sk // block)
    chosen = torch.zeros(b, hk, sq, nb + 1, dtype=torch.bool, device=index.device)
    ok = (index >= 0) & (index < nb)
    chosen.scatter_(-1, torch.where(ok, index, nb).long(), True)
    seen = chosen[..., :nb].repeat_interleave(block, -1)[..., :sk]
    if kv_lens is not None:
        seen = seen & (torch.arange(sk, device=index.device) < kv_lens.view(b, 1, 1, 1))
    if q_lens is not None:
        seen = seen & (torch.arange(sq, device=index.device)[:, None] < q_lens.view(b, 1, 1, 1))
    return seen


def attention(q, k, v, index, block, scale=None, kv_lens=None, q_lens=None, dout=None, pair=False):
    """Results in 64 bits and, beside each, a bound on the kernels' error.

    u = one rounding to the inputs' type. The kernels round the weights p and, backward, ds to it
    (relative u each; in f16 also 2^-25 absolute, its subnormal step) and every result once more.
    Scores are 32-bit dot products: |error of s| <= es = (D + 4) 2^-24 scale sum |q||k| and a
    32-bit exp with the same order of error, which scales p by 1 +- 2 es + 2^-20. The backward's
    delta = do . out reads the rounded out.

    `pair`: the bound for weights that go to the matrix unit as pairs of 16-bit numbers, hi and the
    rest of it. They are off by u^2 (u for hi, u of what it leaves for the rest). What was
    drowned by u counts then: matrix steps of 16 keys add in 32 bits with an error of 2^-23 of the
    sum of magnitudes each (two products a step, 16 steps at most), the join of up to 64 parts
    with 2^-24 each and two roundings of every part's weight: 2^-17 in all. The sums of dk and dv
    over the rows take a step per 16 rows. In f16 the last half step of a pair is 2^-25 of what is
    held: p times 2^14, and ds times a power of two that leaves at least 2^12 of the bound
    max |dout| max |v| sqrt(chunks of 8 channels) + max |delta|."""

    b, hq, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    grp = hq // hk
    u = torch.finfo(q.dtype).eps / 2
    steps = 0.0
    if pair:
        u = u * u + 2.0**-17
        steps = 2.0**-22 * (sq * grp / 16 + 8)
    sub = 2.0**-25 if q.dtype == torch.float16 else 0.0
    scale = 1 / math.sqrt(d) if scale is None else scale
    seen = seen_keys(index, sk, block, kv_lens, q_lens)[:, :, None]

    # what no row sees must not matter: zeros there, whatever it holds
    used = seen.any(3).any(2)[..., None]
    q64 = torch.where(seen.any(-1)[..., None], q.double().view(b, hk, grp, sq, d), 0.0)
    k64 = torch.where(used, k.double(), 0.0)[:, :, None]
    v64 = torch.where(used, v.double(), 0.0)[:, :, None]
    s = torch.where(seen, (q64 @ k64.transpose(-1, -2)) * scale, -math.inf)
    lse = torch.logsumexp(s, -1) if sk else torch.full(s.shape[:-1], -math.inf, dtype=torch.float64, device=q.device)
    p = torch.where(seen, torch.exp(s - torch.where(lse.isinf(), 0.0, lse)[..., None]), 0.0)
    es = abs(scale) * (d + 4) * 2.0**-24 * (q64.abs() @ k64.abs().transpose(-1, -2))
    es = torch.where(seen, es, 0.0)
    worst = es.amax(-1, keepdim=True) if sk else es.sum(-1, keepdim=True)
    rel_p = 2 * worst + 2.0**-20
    out = p @ v64
    found = {"out": out, "lse": lse}
    bound = {
        "out": rounding(out, q.dtype) + (u + rel_p) * (p @ v64.abs()) + sub * (seen.double() @ v64.abs()),
        "lse": (2 * worst + 2.0**-20 * (1 + torch.where(lse.isinf(), 0.0, lse).abs())[..., None])[..., 0],
    }
    if dout is not None:
        g = torch.where(seen.any(-1)[..., None], dout.double().view(b, hk, grp, sq, d), 0.0)
        found["dv"] = (p.transpose(-1, -2) @ g).sum(2)
        bound["dv"] = rounding(found["dv"], q.dtype) + (
            ((u + steps + rel_p) * p + (2.0**-14 if pair else 1.0) * sub * seen).transpose(-1, -2) @ g.abs()).sum(2)
        dp = g @ v64.transpose(-1, -2)
        delta = (g * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        e_delta = (g.abs() * (bound["out"] + rounding(out, q.dtype))).sum(-1, keepdim=True)
        e_dp = (d + 4) * 2.0**-24 * (g.abs() @ v64.abs().transpose(-1, -2))
        floor = sub * seen
        if pair and sk:
            most = g.norm(dim=-1).max() * v64.norm(dim=-1).max() * math.ceil(d / 8) ** 0.5 + delta.abs().max()
            floor = floor * 2.0**-12 * most
        e_ds = (u + rel_p) * ds.abs() + p * (e_delta + e_dp + 2.0**-22 * delta.abs()) + floor
        found["dq"] = scale * (ds @ k64)
        found["dk"] = scale * (ds.transpose(-1, -2) @ q64).sum(2)
        bound["dq"] = rounding(found["dq"], q.dtype) + abs(scale) * (e_ds @ k64.abs())
        e_ds = e_ds + steps * ds.abs()
        bound["dk"] = rounding(found["dk"], q.dtype) + abs(scale) * (e_ds.transpose(-1, -2) @ q64.abs()).sum(2)
    for name in ("out", "lse", "dq"):
        for t in (found, bound):
            if name in t:
                t[name] = t[name].reshape(b, hq, *t[name].shape[3:])
    return found, bound
