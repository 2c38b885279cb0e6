"""Measured cases of the long-support attention operators.

Four operators, each with its plain form (elementary torch operations in 32 bits, 64 where 32 lose
what matters) and the call a user makes of `hexo_bot_b200.attention_ops`:

- rotary: rotary positions with several axes (hex coordinates of cells; time, height, width).
- qk_norm: RMS norm of every query and key head, with the position rotation in the same pass;
  "train" adds the gradients of queries, keys and both weights.
- select: block means of the keys and the blocks that each query keeps by q . mean.
- attend: softmax attention of each query over its chosen key blocks; "train" adds dq, dk, dv.

Tensors are (batch, heads, rows, head_dim) views. Lengths of a ragged batch fall linearly from the
full length, as the size-sorted rows of a serve payload do.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
COORDS = {"i16": torch.int16, "i32": torch.int32, "i64": torch.int64, "f32": torch.float32}
SIZES = {"f32": 4, "f16": 2, "bf16": 2, "i16": 2, "i32": 4, "i64": 8}
THETA = 10000.0
EPS = 1e-6


# ---- cases --------------------------------------------------------------------------------


def rotary(b, s, h, d, dtype, sections, coords="i16", prefix=0, adjacent=False, inverse=False, span=32):
    return dict(op="rotary", b=b, s=s, h=h, d=d, dtype=dtype, sections=sections, coords=coords, prefix=prefix,
                adjacent=adjacent, inverse=inverse, span=span)


def qk_norm(mode, b, s, hq, hk, d, dtype, sections, coords="i16", prefix=0, adjacent=False, span=32):
    return dict(op="qk_norm", mode=mode, b=b, s=s, hq=hq, hk=hk, d=d, dtype=dtype, sections=sections, coords=coords,
                prefix=prefix, adjacent=adjacent, span=span)


def select(b, sq, sk, hq, hk, d, dtype, block, topk, keep_first=0, keep_own=False, ragged=False, means=True):
    return dict(op="select", b=b, sq=sq, sk=sk, hq=hq, hk=hk, d=d, dtype=dtype, block=block, topk=topk,
                keep_first=keep_first, keep_own=keep_own, ragged=ragged, means=means)


def attend(mode, b, sq, sk, hq, hk, d, dtype, block, topk, ragged=False):
    return dict(op="attend", mode=mode, b=b, sq=sq, sk=sk, hq=hq, hk=hk, d=d, dtype=dtype, block=block, topk=topk,
                ragged=ragged)


def listed():
    return [
        # the cells of the main batch: 8 summary tokens without a place, then 61 cells on (q, r)
        dict(rotary(4096, 69, 8, 16, "f16", "4,4", prefix=8), name="rotary_cells"),
        # patches of a long clip on (time, height, width), the largest rotation
        dict(rotary(2, 13824, 16, 128, "bf16", "16,24,24", coords="i32", span=512), name="rotary_clip"),
        # one new token: latency
        dict(rotary(1, 1, 8, 64, "bf16", "12,20", coords="i64", span=100000), name="rotary_token"),
        # a serve group of real supports, q and k out of the packed projection
        dict(qk_norm("forward", 24, 400, 8, 8, 16, "f16", "4,4", prefix=8), name="qk_serve"),
        # a training batch of long supports with shared key heads
        dict(qk_norm("train", 8, 2440, 16, 4, 64, "bf16", "16,16", prefix=8), name="qk_train"),
        # radius-8 disk in 32 bits with an odd head size, partly rotated
        dict(qk_norm("train", 3, 217, 12, 4, 20, "f32", "3,5", coords="i32", adjacent=True), name="qk_odd"),
        # a serve batch of real supports, falling lengths
        dict(select(16, 2440, 2440, 8, 8, 16, "f16", 64, 8, keep_first=1, keep_own=True, ragged=True),
             name="select_serve"),
        # one token against the kept means of a long history
        dict(select(4, 1, 131072, 32, 8, 64, "bf16", 64, 16, keep_first=1, means=False), name="select_token"),
        # a long training sequence with shared key heads
        dict(select(1, 8192, 8192, 16, 4, 128, "bf16", 64, 16, keep_own=True), name="select_long"),
        # a serve batch of real supports, falling lengths
        dict(attend("forward", 16, 2440, 2440, 8, 8, 16, "f16", 64, 8, ragged=True), name="attend_serve"),
        # one token over a long history
        dict(attend("forward", 8, 1, 32768, 32, 8, 128, "bf16", 64, 32), name="attend_token"),
        # a long training sequence
        dict(attend("train", 1, 8192, 8192, 8, 8, 64, "bf16", 64, 16), name="attend_train"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _sections(rng, d, axes):
    pairs = rng.randint(axes, max(axes, d // 2))
    cuts = sorted(rng.sample(range(1, pairs), axes - 1)) if axes > 1 else []
    return ",".join(str(y - x) for x, y in zip([0] + cuts, cuts + [pairs]))


def draw(rng):
    op = rng.choice(["rotary", "qk_norm", "select", "attend"])
    if op in ("rotary", "qk_norm"):
        d = rng.choice([16, 16, 20, 32, 48, 64, 64, 80, 128])
        axes = rng.choice([1, 2, 2, 3])
        # whole heads rotated in equal sections half of the time, any split of the pairs otherwise
        sections = _sections(rng, d, axes)
        if rng.random() < 0.5 and d // 2 % axes == 0:
            sections = ",".join([str(d // 2 // axes)] * axes)
        dtype, coords = rng.choice(["f16", "bf16", "f32"]), rng.choice(["i16", "i32", "i64", "f32"])
        span = _log_int(rng, 8, 30000)
        h = _log_int(rng, 1, 32)
        hk = rng.choice([x for x in range(1, h + 1) if h % x == 0])
        rows = _log_int(rng, 1, max(1, 40_000_000 // (h * d) if op == "rotary" else 25_000_000 // ((h + hk) * d)))
        s = _log_int(rng, 1, rows)
        prefix = min(rng.choice([0, 0, 8]), s)
        common = dict(coords=coords, prefix=prefix, adjacent=rng.random() < 0.3, span=span)
        if op == "rotary":
            return rotary(rows // s, s, h, d, dtype, sections, inverse=rng.random() < 0.3, **common)
        return qk_norm(rng.choice(["forward", "train"]), rows // s, s, h, hk, d, dtype, sections, **common)
    hk = rng.choice([1, 2, 3, 4, 8])
    hq = hk * rng.choice([1, 1, 2, 4])
    block = rng.choice([32, 64, 64, 128])
    dtype = rng.choice(["f16", "bf16"])
    if op == "select":
        d = rng.choice([16, 32, 64, 72, 128])
        token = rng.random() < 0.3
        sk = _log_int(rng, block // 2, 100000 if token else min(10000, math.isqrt(500_000_000 * block // (hk * d))))
        sq = rng.randint(1, 4) if token else sk
        b = _log_int(rng, 1, max(1, min(2_000_000 // (sk * hk), 500_000_000 // (hk * d * sq * -(-sk // block)))))
        keep_first, keep_own = rng.randint(0, 1), sq == sk and rng.random() < 0.5
        return select(b, sq, sk, hq, hk, d, rng.choice([dtype, dtype, "f32"]), block, rng.randint(2, 24), keep_first,
                      keep_own, ragged=rng.random() < 0.5, means=not token)
    d = rng.choice([16, 24, 32, 64, 80, 128])
    token = rng.random() < 0.3
    # the plain form holds every score, so the longest row follows from the heads
    sk = _log_int(rng, block // 2, 20000 if token else min(8000, math.isqrt(400_000_000 // hq)))
    sq = rng.randint(1, 4) if token else sk
    most = min(32, 400_000_000 // (hq * sq * sk), 40_000_000 // (hk * sk * d), 4_000_000_000 // (hq * sq * block * d))
    b = _log_int(rng, 1, max(1, most))
    topk = rng.randint(1, max(1, min(16, 4_000_000_000 // (b * hq * sq * block * d))))
    return attend("forward" if token else rng.choice(["forward", "train"]), b, sq, sk, hq, hk, d, dtype, block, topk,
                  ragged=rng.random() < 0.5)


# ---- inputs -------------------------------------------------------------------------------


def _lens(case, key):
    """Live lengths of a ragged batch: they fall linearly from the full length."""
    b, s = case["b"], case[key]
    return [s - (i * s) // (2 * b) for i in range(b)]


def _blocks(case):
    return -(-case["sk"] // case["block"])


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)

    st = dict(case)
    if case["op"] in ("rotary", "qk_norm"):
        b, s, d = case["b"], case["s"], case["d"]
        sections = tuple(int(x) for x in case["sections"].split(","))
        span, n = case["span"], case["s"] - case["prefix"]
        c = torch.randint(-span, span + 1, (b, n, len(sections)), generator=g, device="cuda")
        st["coords_t"] = c.to(COORDS[case["coords"]])
        # the angle table: every axis runs through its own frequencies
        freqs = [THETA ** (-j / m) for m in sections for j in range(m)]
        st["freqs"] = torch.tensor(freqs, dtype=torch.float64, device="cuda")
        st["axis"] = torch.tensor([a for a, m in enumerate(sections) for _ in range(m)], device="cuda")
        st["parts"] = sections
        if case["op"] == "rotary":
            st["x"] = normal(b, s, case["h"], d).transpose(1, 2)
            return st
        # one packed projection row per token: q heads, k heads, v heads
        hq, hk = case["hq"], case["hk"]
        st["qkv"] = normal(b, s, (hq + 2 * hk) * d, scale=1.5)
        st["wq"], st["wk"] = (1.0 + normal(d, scale=0.2, dtype=torch.float32) for _ in range(2))
        if case["mode"] == "train":
            st["gq"] = normal(b, s, hq, d).transpose(1, 2)
            st["gk"] = normal(b, s, hk, d).transpose(1, 2)
        return st

    b, sq, sk, hq, hk, d = (case[x] for x in ("b", "sq", "sk", "hq", "hk", "d"))
    st["q"] = normal(b, sq, hq, d).transpose(1, 2)
    if case["op"] == "attend" or case["means"]:
        # neighbouring keys resemble one another, as cells of one region do: block means differ
        near = torch.randn(b, _blocks(case), 1, hk, d, generator=g, device="cuda")
        near = near.expand(-1, -1, case["block"], -1, -1).reshape(b, -1, hk, d)[:, :sk]
        st["k"] = (torch.randn(b, sk, hk, d, generator=g, device="cuda") + 0.5 * near).to(dt).transpose(1, 2)
    else:
        st["kept_means"] = normal(b, hk, _blocks(case), d, scale=0.5, dtype=torch.float32)
    st["kv_lens"] = st["q_lens"] = None
    if case["ragged"]:
        st["kv_lens"] = torch.tensor(_lens(case, "sk"), dtype=torch.int32, device="cuda")
        if sq == sk:
            st["q_lens"] = st["kv_lens"]
    if case["op"] == "select":
        return st
    st["v"] = normal(b, sk, hk, d).transpose(1, 2)
    # chosen blocks: distinct, with popular ones among them, ascending, -1 where a row has fewer
    nb, topk = _blocks(case), case["topk"]
    live = torch.tensor([-(-x // case["block"]) for x in (_lens(case, "sk") if case["ragged"] else [sk] * b)], device="cuda")
    want = torch.rand(b, hk, sq, nb, generator=g, device="cuda")
    want += 0.5 * torch.rand(b, hk, 1, nb, generator=g, device="cuda")
    want.masked_fill_(torch.arange(nb, device="cuda") >= live.view(b, 1, 1, 1), -1.0)
    val, at = want.topk(min(topk, nb), dim=-1)
    at = at.masked_fill(val < 0, nb).sort(dim=-1).values
    idx = torch.full((b, hk, sq, topk), -1, dtype=torch.int32, device="cuda")
    idx[..., : at.shape[-1]] = at.masked_fill(at == nb, -1)
    st["idx"] = idx
    if case["mode"] == "train":
        st["g"] = normal(b, sq, hq, d).transpose(1, 2)
    return st


# ---- plain forms --------------------------------------------------------------------------


def _angles(st):
    """cos and sin (b, 1, s, pairs) of every row's angles; rows before the placed ones do not turn."""
    c = st["coords_t"].double()[..., st["axis"]] * st["freqs"]
    c = torch.cat([c.new_zeros(c.shape[0], st["prefix"], c.shape[2]), c], 1)[:, None]
    return c.cos().float(), c.sin().float()


def _turn(x, cos, sin, adjacent):
    p = cos.shape[-1]
    if adjacent:
        u, v, rest = x[..., 0 : 2 * p : 2], x[..., 1 : 2 * p : 2], x[..., 2 * p :]
        turned = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
    else:
        u, v, rest = x[..., :p], x[..., p : 2 * p], x[..., 2 * p :]
        turned = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
    return torch.cat([turned, rest], -1)


def _split(st):
    """q, k views (b, h, s, d) of the packed projection."""
    hq, hk, d = st["hq"], st["hk"], st["d"]
    x = st["qkv"].view(st["b"], st["s"], hq + 2 * hk, d)
    return x[:, :, :hq].transpose(1, 2), x[:, :, hq : hq + hk].transpose(1, 2)


def _plain_qk(st):
    cos, sin = _angles(st)
    found = {}
    for name, x, w in zip("qk", _split(st), (st["wq"], st["wk"])):
        x32 = x.float()
        rstd = torch.rsqrt(x32.square().mean(-1, keepdim=True) + EPS)
        hat = x32 * rstd
        found[name] = _turn(hat * w, cos, sin, st["adjacent"]).to(x.dtype)
        if st["mode"] == "train":
            g = _turn(st["g" + name].float(), cos, -sin, st["adjacent"])
            found["dw" + name] = (g * hat).sum((0, 1, 2), dtype=torch.float64).float()
            g = g * w
            found["d" + name] = (rstd * (g - hat * (g * hat).mean(-1, keepdim=True))).to(x.dtype)
    return found


def _plain_means(k, block, kv_lens):
    b, h, s, d = k.shape
    nb = -(-s // block)
    k64 = torch.nn.functional.pad(k.double(), (0, 0, 0, nb * block - s)).view(b, h, nb, block, d)
    lens = torch.full((b,), s, device=k.device) if kv_lens is None else kv_lens.long()
    at = torch.arange(nb * block, device=k.device).view(1, 1, nb, block, 1)
    live = at < lens.view(b, 1, 1, 1, 1)
    count = live.sum(3).clamp(min=1)
    return (torch.where(live, k64, 0.0).sum(3) / count).float()


def _plain_select(st, means):
    q, block, topk = st["q"], st["block"], st["topk"]
    b, hq, sq, d = q.shape
    hk, nb = means.shape[1], means.shape[2]
    score = q.double().view(b, hk, hq // hk, sq, d).sum(2) @ means.double().transpose(-1, -2)
    score = torch.where(score.isnan(), -math.inf, score)
    at = torch.arange(nb, device=q.device)
    lens = torch.full((b,), st["sk"], device=q.device) if st["kv_lens"] is None else st["kv_lens"].long()
    live = at < ((lens + block - 1) // block).view(b, 1, 1, 1)
    forced = (at < st["keep_first"]).expand(sq, nb)
    if st["keep_own"]:
        forced = forced | (at == torch.arange(sq, device=q.device)[:, None] // block)
    score = torch.where(forced, math.inf, score)
    score = torch.where(live, score, -math.inf)
    kept = score.sort(dim=-1, descending=True, stable=True).indices[..., : min(topk, nb)]
    keep = torch.gather(live.expand_as(score), -1, kept)
    if st["q_lens"] is not None:
        keep = keep & (torch.arange(sq, device=q.device)[:, None] < st["q_lens"].view(b, 1, 1, 1))
    kept = torch.where(keep, kept, nb).sort(dim=-1).values
    out = torch.full((b, hk, sq, topk), -1, dtype=torch.int32, device=q.device)
    out[..., : kept.shape[-1]] = torch.where(kept == nb, -1, kept)
    return out


def _plain_attend(st):
    q, k, v, idx, block = st["q"], st["k"], st["v"], st["idx"], st["block"]
    b, hq, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    nb, grp = -(-sk // block), hq // hk
    scale = 1.0 / math.sqrt(d)
    chosen = torch.zeros(b, hk, sq, nb + 1, dtype=torch.bool, device=q.device)
    chosen.scatter_(-1, torch.where(idx < 0, nb, idx).long(), True)
    seen = chosen[..., :nb].repeat_interleave(block, -1)[..., :sk]
    if st["kv_lens"] is not None:
        seen = seen & (torch.arange(sk, device=q.device) < st["kv_lens"].view(b, 1, 1, 1))
    if st["q_lens"] is not None:
        seen = seen & (torch.arange(sq, device=q.device)[:, None] < st["q_lens"].view(b, 1, 1, 1))
    q32, k32, v32 = q.float().view(b, hk, grp, sq, d), k.float()[:, :, None], v.float()[:, :, None]
    p = (q32 @ k32.transpose(-1, -2)).mul_(scale)
    p.masked_fill_(~seen[:, :, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    top.masked_fill_(top == -math.inf, 0.0)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (total.log() + top).view(b, hq, sq)
    p.div_(total.masked_fill_(total == 0, 1.0))
    out = p @ v32
    found = {"out": out.view(b, hq, sq, d).to(q.dtype), "lse": lse}
    if st["mode"] == "train":
        g = st["g"].float().view(b, hk, grp, sq, d)
        found["dv"] = (p.transpose(-1, -2) @ g).sum(2).to(v.dtype)
        ds = g @ v32.transpose(-1, -2)
        ds.sub_((g * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        found["dq"] = (ds @ k32).view(b, hq, sq, d).to(q.dtype)
        found["dk"] = (ds.transpose(-1, -2) @ q32).sum(2).to(k.dtype)
    return found


def run(state):
    st = state
    if own:
        return _own_run(st)
    if st["op"] == "rotary":
        cos, sin = _angles(st)
        return _turn(st["x"].float(), cos, -sin if st["inverse"] else sin, st["adjacent"]).to(st["x"].dtype)
    if st["op"] == "qk_norm":
        return _plain_qk(st)
    if st["op"] == "select":
        if not st["means"]:
            return _plain_select(st, st["kept_means"])
        means = _plain_means(st["k"], st["block"], st["kv_lens"])
        return {"means": means, "index": _plain_select(st, means)}
    return _plain_attend(st)


# ---- the framework's calls ----------------------------------------------------------------


def _own_run(st):
    from hexo_bot_b200 import attention_ops as ops

    if st["op"] == "rotary":
        return ops.axes_rotary(st["x"], st["coords_t"], st["freqs"], st["parts"], adjacent=st["adjacent"],
                               inverse=st["inverse"])
    if st["op"] == "qk_norm":
        q, k = _split(st)
        a, rest = (q, k, st["wq"], st["wk"], st["coords_t"], st["freqs"], st["parts"]), dict(adjacent=st["adjacent"], eps=EPS)
        found = dict(zip("qk", ops.qk_norm_rotary(*a, **rest)))
        if st["mode"] == "train":
            grads = ops.qk_norm_rotary_backward(st["gq"], st["gk"], *a, **rest)
            found.update(zip(("dq", "dk", "dwq", "dwk"), grads))
        return found
    if st["op"] == "select":
        rest = dict(kv_lens=st["kv_lens"], q_lens=st["q_lens"], keep_first=st["keep_first"], keep_own=st["keep_own"])
        if not st["means"]:
            return ops.block_select(st["q"], st["kept_means"], st["topk"], st["block"], st["sk"], **rest)
        means = ops.block_means(st["k"], st["block"], kv_lens=st["kv_lens"])
        return {"means": means, "index": ops.block_select(st["q"], means, st["topk"], st["block"], st["sk"], **rest)}
    a, rest = (st["q"], st["k"], st["v"]), dict(kv_lens=st["kv_lens"], q_lens=st["q_lens"])
    out, lse = ops.block_attention(*a, st["idx"], st["block"], **rest)
    found = {"out": out, "lse": lse}
    if st["mode"] == "train":
        grads = ops.block_attention_backward(st["g"], *a, out, lse, st["idx"], st["block"], **rest)
        found.update(zip(("dq", "dk", "dv"), grads))
    return found


# ---- least work ---------------------------------------------------------------------------


def work(case):
    e = SIZES[case["dtype"]]
    b, d = case["b"], case["d"]
    if case["op"] in ("rotary", "qk_norm"):
        s = case["s"]
        places = b * (s - case["prefix"]) * len(case["sections"].split(",")) * SIZES[case["coords"]]
        if case["op"] == "rotary":
            n = b * s * case["h"] * d
            return {"bytes": 2 * n * e + places, "flops": 3 * n}
        n = b * s * (case["hq"] + case["hk"]) * d
        # forward reads x and writes y; the gradients read dy and x again and write dx
        if case["mode"] == "train":
            return {"bytes": 5 * n * e + 2 * places, "flops": 20 * n}
        return {"bytes": 2 * n * e + places, "flops": 7 * n}
    sq, hq, hk, topk, block = (case[x] for x in ("sq", "hq", "hk", "topk", "block"))
    lens = _lens(case, "sk") if case["ragged"] else [case["sk"]] * b
    rows = lens if sq == case["sk"] else [sq] * b
    index = 4 * b * hk * sq * topk
    if case["op"] == "select":
        means = 4 * b * hk * _blocks(case) * d
        scores = sum(r * -(-n // block) for r, n in zip(rows, lens)) * hk
        keys = sum(lens) * hk * d * e if case["means"] else 0
        return {"bytes": sum(rows) * hq * d * e + keys + means + index, "flops": 2 * scores * d}
    pairs = sum(r * min(topk * block, n) for r, n in zip(rows, lens)) * hq
    # each key and value that some query sees, once; each live query and output once
    seen = sum(min(r * topk * block, n) for r, n in zip(rows, lens)) * hk * d
    q, out = sum(rows) * hq * d, b * sq * hq * d
    lse = 4 * b * sq * hq
    if case["mode"] == "train":
        kv = b * case["sk"] * hk * d
        return {"bytes": (2 * q + out + 2 * seen) * e + 2 * index + lse + (3 * q + 2 * seen) * e + (out + 2 * kv) * e + lse,
                "flops": 14 * pairs * d}
    return {"bytes": (q + out + 2 * seen) * e + index + lse, "flops": 4 * pairs * d}


# ---- 64 bits ------------------------------------------------------------------------------


def _exact_phase(st):
    place = torch.zeros(st["b"], st["s"], len(st["sections"].split(",")), dtype=torch.float64, device="cuda")
    place[:, st["prefix"] :] = st["coords_t"].to(torch.float64)
    return torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), place[:, None][..., st["axis"]] * st["freqs"])


def _exact_rotation(x, phase, adjacent):
    """Pairs as complex numbers times their phase."""
    p = phase.shape[-1]
    first = torch.arange(p, device=x.device) * (2 if adjacent else 1)
    second = first + (1 if adjacent else p)
    z = torch.complex(x[..., first], x[..., second]) * phase
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_attend(st):
    """Every query gathers the keys of its own blocks; a slice of the queries at a time."""
    q, k, v = (st[n].double() for n in "qkv")
    b, hq, sq, d = q.shape
    hk, sk, block, topk = k.shape[1], k.shape[2], st["block"], st["topk"]
    grp, train = hq // hk, st["mode"] == "train"
    out, lse = torch.zeros_like(q), torch.full((b, hq, sq), -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    within = torch.arange(block, device="cuda")
    step = max(1, 30_000_000 // (topk * block * d * grp))
    for i in range(b):
        n = sk if st["kv_lens"] is None else int(st["kv_lens"][i])
        m = sq if st["q_lens"] is None else int(st["q_lens"][i])
        for h in range(hk):
            heads = slice(h * grp, (h + 1) * grp)
            for lo in range(0, m, step):
                hi = min(m, lo + step)
                at = st["idx"][i, h, lo:hi].long()
                key = (at[..., None] * block + within).flatten(1)
                ok = (at >= 0)[..., None].expand(-1, -1, block).flatten(1) & (key < n)
                key = torch.where(ok, key, 0)
                kk, vv = k[i, h][key], v[i, h][key]
                qq = q[i, heads, lo:hi]
                s = torch.einsum("grd,rtd->grt", qq, kk) / math.sqrt(d)
                s = torch.where(ok, s, -math.inf)
                lse[i, heads, lo:hi] = l = torch.logsumexp(s, -1)
                p = torch.where(ok, torch.exp(s - torch.where(l.isinf(), 0.0, l)[..., None]), 0.0)
                out[i, heads, lo:hi] = o = torch.einsum("grt,rtd->grd", p, vv)
                if train:
                    g = st["g"][i, heads, lo:hi].double()
                    ds = p * (torch.einsum("grd,rtd->grt", g, vv) - (g * o).sum(-1, keepdim=True)) / math.sqrt(d)
                    dq[i, heads, lo:hi] = torch.einsum("grt,rtd->grd", ds, kk)
                    dk[i, h].index_add_(0, key.flatten(), torch.einsum("grt,grd->rtd", ds, qq).flatten(0, 1))
                    dv[i, h].index_add_(0, key.flatten(), torch.einsum("grt,grd->rtd", p, g).flatten(0, 1))
    found = {"out": out, "lse": lse}
    if train:
        found.update(dq=dq, dk=dk, dv=dv)
    return found


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        phase = _exact_phase(st)
        return _exact_rotation(st["x"].double(), phase.conj() if case["inverse"] else phase, case["adjacent"])
    if case["op"] == "qk_norm":
        phase, found = _exact_phase(st), {}
        for name, x, w in zip("qk", _split(st), (st["wq"], st["wk"])):
            x = x.double().requires_grad_()
            w = w.double().requires_grad_()
            y = _exact_rotation(x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w, phase, case["adjacent"])
            found[name] = y.detach()
            if case["mode"] == "train":
                found["d" + name], found["dw" + name] = torch.autograd.grad(y, (x, w), st["g" + name].double())
        return found
    if case["op"] == "select":
        if not case["means"]:
            return None
        sk, block = case["sk"], case["block"]
        lens = _lens(case, "sk") if case["ragged"] else [sk] * case["b"]
        means = torch.zeros(case["b"], case["hk"], _blocks(case), case["d"], dtype=torch.float64, device="cuda")
        for i, n in enumerate(lens):
            key = st["k"][i, :, :n].double()
            whole = n // block * block
            means[i, :, : n // block] = key[:, :whole].unflatten(1, (-1, block)).mean(2)
            if n > whole:
                means[i, :, n // block] = key[:, whole:].mean(1)
        return {"means": means, "index": None}
    return _exact_attend(st)
