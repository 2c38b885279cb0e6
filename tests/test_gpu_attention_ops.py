"""Long-support attention operators on the GPU against 64-bit forms.

Bounds on the error are derived, not fitted: one rounding to the output's type
(half a step), the roundings of the weights that the kernels feed to the matrix
unit, and 32-bit arithmetic counted per term (oracle/attention_ops.py)."""

from __future__ import annotations

import math

import pytest
import torch

from hexo_bot_b200 import _lib
from hexo_bot_b200 import attention_ops as ops
from oracle import attention_ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def within(got, want, bound, name=""):
    """|got - want| <= bound everywhere; infinities and NaN in the same places."""
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs()) - bound
    worst = off.max().item() if off.numel() else 0.0
    clean = not bool(off.isnan().any()) and worst <= 0
    assert clean, f"{name}: {worst:.3e} over the bound"


# ---- rotary ---------------------------------------------------------------------------------


def turn_bound(y, x, ang, adjacent, dtype, d):
    """One rounding of the result, and 32-bit angles, products and sums."""
    mix = O.rotate(x.abs(), torch.zeros_like(ang), adjacent)
    p = ang.shape[-1]
    at = torch.arange(p, device=x.device)
    i, j = (2 * at, 2 * at + 1) if adjacent else (at, at + p)
    both = x[..., i].abs() + x[..., j].abs()
    mix[..., i], mix[..., j] = both, both
    return O.rounding(y, dtype) + 2.0**-21 * mix


ROTARY = [
    # b, h, s, d, sections, prefix, adjacent, coordinate type
    (2, 3, 7, 16, (4, 4), 2, False, torch.int16),
    (1, 1, 1, 64, (32,), 0, False, torch.int64),
    (3, 2, 33, 20, (3, 5), 0, True, torch.int32),
    (2, 5, 9, 18, (2, 3), 4, False, torch.float32),  # odd split: single channels
    (1, 2, 5, 15, (7,), 0, True, torch.int16),  # odd head size, last channel unpaired
    (2, 4, 130, 128, (16, 24, 24), 8, False, torch.int32),
    (1, 8, 70, 256, (32, 32, 32, 32), 3, True, torch.int64),
    (4, 40, 3, 96, (8, 8), 0, False, torch.int16),  # partly rotated
    (2, 2, 6, 256, (1,), 6, False, torch.int16),  # no placed row at all
    (5, 1, 1000, 8, (1, 1, 1), 0, False, torch.float32),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", ROTARY)
def test_axes_rotary(case, dtype):
    b, h, s, d, sections, prefix, adjacent, ct = case
    g = gen(11)
    x = randn(g, b, s, h, d, dtype=dtype).transpose(1, 2)
    span = 30000 if ct == torch.int16 else 5_000_000
    coords = torch.randint(-span, span, (b, s - prefix, len(sections)), generator=g, device=DEV).to(ct)
    freqs = ops.rotary_freqs(sections, device=DEV)
    ang = O.angles(coords, freqs, sections, s)
    for inverse in (False, True):
        y = ops.axes_rotary(x, coords, freqs, sections, adjacent=adjacent, inverse=inverse)
        a = -ang if inverse else ang
        want = O.rotate(x.double(), a, adjacent)
        within(y, want, turn_bound(want, x.double(), a, adjacent, dtype, d))
        assert torch.equal(y[:, :, :prefix], x[:, :, :prefix]) and torch.equal(y[..., 2 * sum(sections):],
                                                                              x[..., 2 * sum(sections):])


def test_axes_rotary_layouts_in_place_and_shared_places():
    """Contiguous, transposed, packed, broadcast and misaligned inputs give the same values; in
    place too; coordinates shared by the batch (stride 0) as well as copied ones."""
    g = gen(12)
    b, h, s, d, sec = 2, 3, 21, 32, (8, 8)
    freqs = ops.rotary_freqs(sec, device=DEV)
    coords = torch.randint(-50, 50, (1, s, 2), generator=g, device=DEV).expand(b, -1, -1)
    x = randn(g, b, h, s, d, dtype=F16)
    want = ops.axes_rotary(x, coords.contiguous(), freqs, sec)
    assert torch.equal(ops.axes_rotary(x, coords, freqs, sec), want)
    flipped = coords.flip(-1).contiguous().flip(-1)
    back = torch.empty(b, 2, s, dtype=coords.dtype, device=DEV).copy_(coords.transpose(1, 2)).transpose(1, 2)
    assert torch.equal(ops.axes_rotary(x, back, freqs, sec), want) and torch.equal(flipped, coords)
    bshd = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops.axes_rotary(bshd, coords, freqs, sec), want)
    packed = torch.cat([x, x], -1)[..., d:]
    assert torch.equal(ops.axes_rotary(packed, coords, freqs, sec), want)
    for shift in (1, 2, 4):  # bases and strides that take the narrower accesses
        wide = torch.zeros(b, h, s, d + shift, dtype=F16, device=DEV)
        wide[..., shift:] = x
        assert torch.equal(ops.axes_rotary(wide[..., shift:], coords, freqs, sec), want)
    one = x[:, :1].expand(-1, h, -1, -1)
    assert torch.equal(ops.axes_rotary(one, coords, freqs, sec), ops.axes_rotary(one.contiguous(), coords, freqs, sec))
    y = x.clone()
    assert ops.axes_rotary(y, coords, freqs, sec, out=y) is y
    assert torch.equal(y, want)
    # rows and heads outside the view are left alone
    frame = torch.full((b, h + 2, s + 2, d), 7.0, dtype=F16, device=DEV)
    ops.axes_rotary(x, coords, freqs, sec, out=frame[:, 1:-1, 1:-1])
    assert torch.equal(frame[:, 1:-1, 1:-1], want)
    frame[:, 1:-1, 1:-1] = 7.0
    assert (frame == 7.0).all()


def test_axes_rotary_unturned_channels_keep_infinities():
    x = torch.randn(1, 1, 4, 16, device=DEV)
    x[..., 12:] = torch.tensor([math.inf, -math.inf, math.nan, 1.0], device=DEV)
    coords = torch.ones(1, 4, 1, dtype=torch.int32, device=DEV)
    y = ops.axes_rotary(x, coords, ops.rotary_freqs((4,), device=DEV), (4,))
    assert torch.equal(y[..., 8:12], x[..., 8:12]) and y[..., :12].isfinite().all()
    assert torch.equal(y[..., 12:].nan_to_num(5.0), x[..., 12:].nan_to_num(5.0))


@pytest.mark.parametrize("adjacent", [False, True])
def test_axes_rotary_gradient(adjacent):
    g = gen(13)
    x = randn(g, 2, 3, 9, 20).requires_grad_()
    coords = torch.randint(-9, 9, (2, 7, 2), generator=g, device=DEV)
    freqs = ops.rotary_freqs((2, 5), device=DEV)
    w = randn(g, 2, 3, 9, 20)
    (gx,) = torch.autograd.grad(ops.axes_rotary(x, coords, freqs, (2, 5), adjacent=adjacent), x, w)
    ang = -O.angles(coords, freqs, (2, 5), 9)
    want = O.rotate(w.double(), ang, adjacent)
    within(gx, want, turn_bound(want, w.double(), ang, adjacent, F32, 20))
    # an expanded gradient, as sum() gives it
    (gx,) = torch.autograd.grad(ops.axes_rotary(x, coords, freqs, (2, 5), adjacent=adjacent).sum(), x)
    want = O.rotate(torch.ones_like(w).double(), ang, adjacent)
    within(gx, want, turn_bound(want, torch.ones_like(w).double(), ang, adjacent, F32, 20))


# ---- norm and rotation -------------------------------------------------------------------------

QK = [
    # b, hq, hk, s, d, sections, prefix, adjacent, weight type (None: no weight)
    (2, 4, 2, 9, 16, (4, 4), 1, False, F32),
    (1, 1, 1, 1, 64, (32,), 0, False, F16),
    (3, 12, 4, 217, 20, (3, 5), 0, True, F32),
    (2, 3, 1, 50, 18, (2, 3), 4, False, BF16),
    (1, 2, 2, 33, 15, (7,), 0, True, None),
    (2, 16, 4, 130, 128, (16, 24, 24), 8, False, F32),
    (1, 4, 4, 70, 256, (), 0, False, F32),  # norm alone
    (2, 5, 5, 40, 80, (10, 10), 0, False, F16),
    (1, 3, 3, 40, 72, (9, 27), 0, False, F32),
]


def qk_case(case, dtype, seed=21):
    b, hq, hk, s, d, sections, prefix, adjacent, wd = case
    g = gen(seed)
    qkv = randn(g, b, s, (hq + 2 * hk), d, dtype=dtype, scale=1.5)
    q, k = qkv[:, :, :hq].transpose(1, 2), qkv[:, :, hq : hq + hk].transpose(1, 2)
    ws = [None if wd is None else (1 + randn(g, d, scale=0.3)).to(wd) for _ in range(2)]
    coords = freqs = ang = None
    if sections:
        coords = torch.randint(-400, 400, (b, s - prefix, len(sections)), generator=g, device=DEV)
        freqs = ops.rotary_freqs(sections, device=DEV)
        ang = O.angles(coords, freqs, sections, s)
    gq, gk = randn(g, b, s, hq, d, dtype=dtype).transpose(1, 2), randn(g, b, s, hk, d, dtype=dtype).transpose(1, 2)
    return q, k, ws, coords, freqs, ang, gq, gk


def spread(t, ang, adjacent):
    """Sum of both members of each pair, at both places (unturned channels as they are)."""
    if ang is None:
        return t
    p = ang.shape[-1]
    at = torch.arange(p, device=t.device)
    i, j = (2 * at, 2 * at + 1) if adjacent else (at, at + p)
    y = t.clone()
    y[..., i] = y[..., j] = t[..., i] + t[..., j]
    return y


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", QK)
def test_qk_norm_rotary_and_gradients(case, dtype):
    b, hq, hk, s, d, sections, prefix, adjacent, wd = case
    q, k, ws, coords, freqs, ang, gq, gk = qk_case(case, dtype)
    outs = ops.qk_norm_rotary(q, k, *ws, coords, freqs, sections, adjacent=adjacent, eps=1e-5)
    grads = ops.qk_norm_rotary_backward(gq, gk, q, k, *ws, coords, freqs, sections, adjacent=adjacent, eps=1e-5)
    again = ops.qk_norm_rotary_backward(gq, gk, q, k, *ws, coords, freqs, sections, adjacent=adjacent, eps=1e-5)
    for a, c in zip(grads, again):
        assert a is c is None or torch.equal(a, c)
    n24 = 2.0**-24
    for x, w, out, gy, dx, dw in zip((q, k), ws, outs, (gq, gk), grads[:2], grads[2:]):
        x64 = x.double().requires_grad_()
        w64 = None if w is None else w.double().requires_grad_()
        want = O.qk_norm(x64, w64, ang, adjacent, 1e-5)
        rstd = (x64.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        hat = (x64 * rstd).detach()
        size = hat.abs() * (1 if w is None else w64.abs().detach())
        within(out, want.detach(), O.rounding(want.detach(), dtype) + (d + 24) * n24 * spread(size, ang, adjacent), "out")
        wants = torch.autograd.grad(want, (x64,) if w is None else (x64, w64), gy.double())
        back = spread(gy.double().abs(), ang, adjacent) * (1 if w is None else w64.abs().detach())
        mass = rstd.detach() * (back + hat.abs() * (back * hat.abs()).mean(-1, keepdim=True))
        within(dx, wants[0], O.rounding(wants[0], dtype) + (2 * d + 48) * n24 * mass, "dx")
        if w is not None:
            mass = (spread(gy.double().abs(), ang, adjacent) * hat.abs()).sum((0, 1, 2))
            within(dw, wants[1], 1.01 * O.rounding(wants[1], w.dtype) + (d + 96) * n24 * mass, "dw")


def test_qk_norm_rotary_zero_rows_and_autograd():
    case = (2, 4, 2, 9, 16, (4, 4), 1, False, F32)
    q, k, ws, coords, freqs, ang, gq, gk = qk_case(case, BF16)
    q, k = q.clone(), k.clone()
    q[:, :, 3] = 0  # a row of zeros stays zero and has gradient g w / sqrt(eps)
    qo, _ = ops.qk_norm_rotary(q, k, *ws, coords, freqs, (4, 4))
    assert (qo[:, :, 3] == 0).all() and qo.isfinite().all()
    want = ops.qk_norm_rotary_backward(gq, gk, q, k, *ws, coords, freqs, (4, 4))
    leaves = [t.detach().requires_grad_() for t in (q, k, *ws)]
    outs = ops.qk_norm_rotary(*leaves, coords, freqs, (4, 4))
    got = torch.autograd.grad(outs, leaves, (gq, gk))
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    # only one output used: the other's gradient arrives as zeros
    got = torch.autograd.grad(ops.qk_norm_rotary(*leaves, coords, freqs, (4, 4))[0].float().sum(), leaves)
    assert (got[1] == 0).all() and (got[3] == 0).all() and got[2].abs().sum() > 0


def test_qk_norm_rotary_gradient_against_differences():
    case = (1, 2, 1, 3, 8, (2, 1), 1, False, F32)
    q, k, ws, coords, freqs, ang, gq, gk = qk_case(case, F32)
    grads = ops.qk_norm_rotary_backward(gq, gk, q, k, *ws, coords, freqs, (2, 1))

    def loss(q, k, wq, wk):
        return ((O.qk_norm(q, wq, ang) * gq.double()).sum() + (O.qk_norm(k, wk, ang) * gk.double()).sum()).item()

    at = [t.double().contiguous() for t in (q, k, *ws)]
    for n, grad in enumerate(grads):
        flat = at[n].reshape(-1)
        for i in range(0, flat.numel(), 5):
            vals = []
            for h in (1e-5, -1e-5):
                moved = [t.clone() for t in at]
                moved[n].view(-1)[i] += h
                vals.append(loss(*moved))
            assert abs((vals[0] - vals[1]) / 2e-5 - grad.reshape(-1)[i].item()) <= 1e-4


# ---- block means and selection -----------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("b,h,s,d,block,lens", [
    (2, 3, 200, 16, 64, None), (3, 1, 1, 8, 32, None), (3, 2, 130, 64, 64, (130, 64, 0)), (1, 2, 77, 20, 16, (70,)),
    (2, 1, 300, 200, 128, (300, 129)), (1, 1, 50, 33, 7, None), (1, 2, 64, 256, 64, (63,))])
def test_block_means(dtype, b, h, s, d, block, lens):
    k = randn(gen(31), b, s, h, d, dtype=dtype).transpose(1, 2).clone(memory_format=torch.preserve_format)
    kl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    for i, n in enumerate(lens or ()):
        k[i, :, n:] = math.nan  # dead keys are not read
    got = ops.block_means(k, block, kv_lens=kl)
    want = O.means(k, block, kl)
    within(got, want, 1.001 * 2.0**-24 * want.abs() + 1e-45)
    odd = torch.zeros(b, h, s, d + 1, dtype=dtype, device=DEV)
    odd[..., 1:] = k
    assert torch.equal(ops.block_means(odd[..., 1:], block, kv_lens=kl), got)


SELECT = [
    # b, hq, hk, sq, sk, d, block, topk, keep_first, keep_own, kv lens, q lens
    (2, 2, 2, 100, 1000, 16, 64, 4, 0, False, None, None),
    (2, 4, 2, 130, 130, 20, 16, 3, 1, True, (130, 50), (130, 50)),
    (1, 8, 1, 70, 2000, 64, 32, 16, 2, False, (1999,), None),
    (3, 2, 2, 5, 2900, 128, 64, 8, 1, False, (2900, 65, 0), (5, 2, 0)),
    (1, 3, 3, 40, 40, 8, 64, 5, 0, False, None, None),  # more places than blocks
    (1, 1, 1, 9, 9000, 33, 8, 64, 0, False, None, None),
    (2, 2, 1, 1, 5000, 256, 64, 2, 1, True, None, None),
    (1, 2, 2, 300, 300, 16, 64, 1, 0, True, None, None),  # the forced block alone
    (1, 1, 1, 2, 40000, 16, 4, 24, 0, False, None, None),  # 10000 blocks
    (1, 4, 2, 21, 9000, 33, 8, 64, 1, True, (8999,), (20,)),  # many blocks, many queries
    (1, 1, 1, 19, 35000, 16, 4, 24, 0, False, None, None),
    (1, 2, 1, 150, 7000, 24, 64, 12, 0, False, None, None),  # 110 blocks
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", SELECT)
def test_block_select(case, dtype):
    b, hq, hk, sq, sk, d, block, topk, first, own, kl, ql = case
    g = gen(41)
    q = randn(g, b, sq, hq, d, dtype=dtype).transpose(1, 2)
    mean = randn(g, b, hk, -(-sk // block), d, scale=0.3)
    kl, ql = (None if t is None else torch.tensor(t, dtype=torch.int32, device=DEV) for t in (kl, ql))
    got = ops.block_select(q, mean, topk, block, sk, kv_lens=kl, q_lens=ql, keep_first=first, keep_own=own)
    assert torch.equal(got.cpu(), O.select(q, mean, topk, block, sk, kl, ql, first, own))


def test_block_select_close_scores():
    """Equal scores go to the lowest index, scores that only 64 bits tell apart to the larger one,
    NaN below everything; rows of zeros and infinite means included."""
    g = gen(42)
    nb, d, topk = 70, 16, 9
    q = randn(g, 1, 1, 40, d, dtype=F16)
    q[0, 0, 3] = 0
    mean = randn(g, 1, 1, nb, d)
    mean[0, 0, 20:60] = mean[0, 0, :1]  # many equal blocks
    got = ops.block_select(q, mean, topk, 64, nb * 64)
    assert torch.equal(got.cpu(), O.select(q, mean, topk, 64, nb * 64))
    assert got[0, 0, 3].tolist() == list(range(topk))
    near = mean.clone()
    near[0, 0, 20:60] *= 1 + 2.0**-23 * torch.arange(40, device=DEV)[:, None]  # one step of 32 bits apart
    assert torch.equal(ops.block_select(q, near, topk, 64, nb * 64).cpu(), O.select(q, near, topk, 64, nb * 64))
    wild = mean.clone()
    wild[0, 0, 5, 0], wild[0, 0, 6, 1], wild[0, 0, 7] = math.inf, -math.inf, math.nan
    wild[0, 0, 8] = 3e38
    assert torch.equal(ops.block_select(q, wild, topk, 64, nb * 64).cpu(), O.select(q, wild, topk, 64, nb * 64))
    tiny = mean * 1e-38
    assert torch.equal(ops.block_select(q, tiny, topk, 64, nb * 64).cpu(), O.select(q, tiny, topk, 64, nb * 64))


# ---- block-sparse attention ----------------------------------------------------------------------

ATTEND = [
    # b, hq, hk, sq, sk, d, block, topk, kv lens, q lens
    (1, 1, 1, 1, 1, 16, 64, 1, None, None),
    (2, 4, 4, 1, 700, 64, 64, 5, (700, 65), None),
    (2, 8, 2, 3, 1000, 128, 64, 11, None, None),
    (1, 40, 2, 16, 500, 32, 128, 4, None, None),
    (2, 2, 2, 17, 130, 16, 64, 2, None, None),
    (2, 2, 2, 200, 200, 16, 64, 3, (200, 70), (200, 70)),
    (3, 6, 2, 150, 333, 24, 32, 7, (333, 1, 0), (150, 9, 0)),
    (1, 4, 1, 300, 300, 40, 128, 2, None, None),
    (1, 2, 2, 260, 1000, 64, 64, 16, None, None),
    (1, 3, 1, 520, 400, 80, 64, 4, (399,), None),
    (1, 2, 1, 70, 600, 128, 128, 3, None, (33,)),
    (1, 2, 2, 90, 257, 8, 32, 64, None, None),
    (2, 3, 3, 64, 0, 16, 64, 2, None, None),  # no keys at all
    (1, 1, 1, 5000, 300, 16, 64, 2, None, None),  # several segments of queries
]


def attend_case(case, dtype, seed=51, extra=True):
    """q, k, v out of padded buffers, and an index with -1, repeated and out-of-range entries."""
    b, hq, hk, sq, sk, d, block, topk, kl, ql = case
    g = gen(seed)
    q = randn(g, b, sq, hq, d, dtype=dtype).transpose(1, 2)
    kv = randn(g, b, sk, 2, hk, d + 8, dtype=dtype)
    k, v = kv[:, :, 0, :, :d].transpose(1, 2), kv[:, :, 1, :, 8:].transpose(1, 2)
    nb = -(-sk // block)
    index = torch.randint(-1, nb + 1, (b, hk, sq, topk), generator=g, device=DEV, dtype=torch.int32)
    if extra and sq > 4:
        index[:, :, 1] = -1  # a row that sees nothing
        index[:, :, 2] = 0  # one block, named every time
        index[:, :, 3] = 2**31 - 1
        index[:, :, 4, 0] = -(2**31)
    kl, ql = (None if t is None else torch.tensor(t, dtype=torch.int32, device=DEV) for t in (kl, ql))
    dout = randn(g, b, sq, hq, d, dtype=dtype).transpose(1, 2)
    # what is masked must not matter
    for i in range(b):
        if kl is not None:
            k[i, :, int(kl[i]):] = math.nan
            v[i, :, int(kl[i]):] = math.inf
        if ql is not None:
            q[i, :, int(ql[i]):] = math.nan
            dout[i, :, int(ql[i]):] = math.nan
    return q, k, v, index, block, kl, ql, dout


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", ATTEND)
def test_block_attention(case, dtype):
    q, k, v, index, block, kl, ql, dout = attend_case(case, dtype)
    found, bound = O.attention(q, k, v, index, block, None, kl, ql, dout)
    out, lse = ops.block_attention(q, k, v, index, block, kv_lens=kl, q_lens=ql)
    within(out, found["out"], bound["out"], "out")
    within(lse, found["lse"], bound["lse"], "lse")
    grads = ops.block_attention_backward(dout, q, k, v, out, lse, index, block, kv_lens=kl, q_lens=ql)
    again = ops.block_attention_backward(dout, q, k, v, out, lse, index, block, kv_lens=kl, q_lens=ql)
    for name, got, same in zip(("dq", "dk", "dv"), grads, again):
        within(got, found[name], bound[name], name)
        assert torch.equal(got, same), name


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_block_attention_scales(scale):
    case = (1, 4, 2, 40, 150, 32, 64, 2, None, None)
    for c in (case, (1, 4, 2, 5, 150, 32, 64, 2, None, None)):
        q, k, v, index, block, kl, ql, dout = attend_case(c, BF16)
        found, bound = O.attention(q, k, v, index, block, scale, kl, ql, dout)
        out, lse = ops.block_attention(q, k, v, index, block, scale=scale)
        within(out, found["out"], bound["out"], "out")
        within(lse, found["lse"], bound["lse"], "lse")
        grads = ops.block_attention_backward(dout, q, k, v, out, lse, index, block, scale=scale)
        for name, got in zip(("dq", "dk", "dv"), grads):
            within(got, found[name], bound[name], name)


@pytest.mark.parametrize("sq", [300, 2100])
def test_block_attention_windows(sq):
    """Parts that exceed one window: several launches over heads, and over rows of one head."""
    case = (2, 8, 2, sq, 1500, 128, 32, 40, (1500, 900), (sq, sq - 77))
    q, k, v, index, block, kl, ql, dout = attend_case(case, BF16)
    found, bound = O.attention(q, k, v, index, block, None, kl, ql, dout)
    out, lse = ops.block_attention(q, k, v, index, block, kv_lens=kl, q_lens=ql)
    within(out, found["out"], bound["out"], "out")
    within(lse, found["lse"], bound["lse"], "lse")
    grads = ops.block_attention_backward(dout, q, k, v, out, lse, index, block, kv_lens=kl, q_lens=ql)
    for name, got in zip(("dq", "dk", "dv"), grads):
        within(got, found[name], bound[name], name)


def test_block_attention_unchosen_blocks_are_not_read():
    """Blocks that nobody chose may hold anything; large scores do not overflow."""
    g = gen(61)
    q, k, v = (randn(g, 1, 2, 200, 16, dtype=BF16, scale=sc) for sc in (8.0, 8.0, 1.0))
    index = torch.zeros(1, 2, 200, 2, dtype=torch.int32, device=DEV)
    index[..., 1] = 2
    want = ops.block_attention(q, k, v, index, 64)
    dout = randn(g, 1, 2, 200, 16, dtype=BF16)
    wants = ops.block_attention_backward(dout, q, k, v, *want, index, 64)
    k2, v2 = k.clone(), v.clone()
    k2[:, :, 64:128], v2[:, :, 64:128] = math.nan, math.inf
    k2[:, :, 192:], v2[:, :, 192:] = math.inf, math.nan
    got = ops.block_attention(q, k2, v2, index, 64)
    gots = ops.block_attention_backward(dout, q, k2, v2, *got, index, 64)
    assert all(torch.equal(a, b) for a, b in zip(got + gots, want + wants))
    assert all(t.isfinite().all() for t in want + wants)
    few = ops.block_attention(q[:, :, :9], k2, v2, index[:, :, :9].contiguous(), 64)
    assert few[0].isfinite().all() and (few[0] - got[0][:, :, :9]).abs().max() <= 2.0**-6 * v.abs().max()


def test_block_attention_autograd_and_accumulated_gradients():
    case = (2, 4, 2, 100, 200, 32, 64, 2, (200, 130), (100, 64))
    q, k, v, index, block, kl, ql, dout = attend_case(case, F16)
    q, k, v, dout = (t.nan_to_num(0.0, 0.0) for t in (q, k, v, dout))
    out, lse = ops.block_attention(q, k, v, index, block, kv_lens=kl, q_lens=ql)
    want = ops.block_attention_backward(dout, q, k, v, out, lse, index, block, kv_lens=kl, q_lens=ql)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o, l = ops.block_attention(*leaves, index, block, kv_lens=kl, q_lens=ql)
    assert not l.requires_grad
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(o, leaves, dout), want))
    with torch.no_grad():
        assert not ops.block_attention(*leaves, index, block)[0].requires_grad


def test_block_attention_gradient_against_differences():
    """Directional derivatives of the 64-bit forward against the kernel's gradients."""
    case = (1, 2, 1, 20, 100, 16, 32, 2, None, None)
    q, k, v, index, block, kl, ql, dout = attend_case(case, F16)
    out, lse = ops.block_attention(q, k, v, index, block)
    grads = ops.block_attention_backward(dout, q, k, v, out, lse, index, block)
    _, bound = O.attention(q, k, v, index, block, None, None, None, dout)
    g = gen(62)
    base = [t.double() for t in (q, k, v)]
    seen = O.seen_keys(index, 100, 32)[:, :, None]

    def loss(q, k, v):
        s = torch.where(seen, q.view(1, 1, 2, 20, 16) @ k[:, :, None].transpose(-1, -2) / 4, -1e300)
        p = torch.softmax(s, -1) * seen
        return ((p @ v[:, :, None]).reshape(1, 2, 20, 16) * dout.double()).sum().item()

    for n, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(base[n].shape, generator=g, device=DEV).double()
        vals = [loss(*[t + h * way if i == n else t for i, t in enumerate(base)]) for h in (1e-5, -1e-5)]
        slope = (vals[0] - vals[1]) / 2e-5
        got = (grads[n].double() * way).sum().item()
        assert abs(got - slope) <= (bound[name] * way.abs()).sum().item() + 1e-5 * abs(slope) + 1e-5


# ---- where calls run --------------------------------------------------------------------------


def chain(q, k, v, wq, wk, coords, freqs, lens):
    """The operators as an attention layer runs them."""
    q, k = ops.qk_norm_rotary(q, k, wq, wk, coords, freqs, (8, 8))
    means = ops.block_means(k, 64, kv_lens=lens)
    index = ops.block_select(q, means, 4, 64, k.shape[2], kv_lens=lens, q_lens=lens, keep_first=1, keep_own=True)
    out, lse = ops.block_attention(q, k, v, index, 64, kv_lens=lens, q_lens=lens)
    return q, k, means, index, out, lse


def chain_inputs(seed=71, b=2, hq=4, hk=2, s=520, d=32):
    g = gen(seed)
    qkv = randn(g, b, s, hq + 2 * hk, d, dtype=BF16)
    q, k, v = (t.transpose(1, 2) for t in qkv.split((hq, hk, hk), 2))
    wq, wk = 1 + randn(g, d, scale=0.2), 1 + randn(g, d, scale=0.2)
    coords = torch.randint(-20, 20, (b, s - 8, 2), generator=g, device=DEV, dtype=torch.int16)
    lens = torch.tensor([s, s - 199], dtype=torch.int32, device=DEV)
    return q, k, v, wq, wk, coords, ops.rotary_freqs((8, 8), device=DEV), lens


def test_operators_together_as_a_layer():
    """Norm and rotation, means, choice and attention after one another, forward and backward, each
    against its 64-bit form on the inputs that the one before produced."""
    ins = chain_inputs()
    q, k, v, wq, wk, coords, freqs, lens = ins
    qn, kn, means, index, out, lse = chain(*ins)
    ang = O.angles(coords, freqs, (8, 8), 520)
    n24 = 2.0**-24
    for x, w, got in ((q, wq, qn), (k, wk, kn)):
        want = O.qk_norm(x.double(), w.double(), ang)
        size = O.qk_norm(x.double(), w.double(), None).abs()
        within(got, want, O.rounding(want, BF16) + 56 * n24 * spread(size, ang, False))
    want = O.means(kn, 64, lens)
    within(means, want, 1.001 * n24 * want.abs())
    assert torch.equal(index.cpu(), O.select(qn, means, 4, 64, 520, lens, lens, 1, True))
    found, bound = O.attention(qn, kn, v, index, 64, None, lens, lens)
    within(out, found["out"], bound["out"])
    # a training step: gradients of everything that learns, through the whole layer
    leaves = [t.detach().requires_grad_() for t in (q, k, v, wq, wk)]
    outs = chain(*leaves, coords, freqs, lens)
    g = randn(gen(72), *out.shape, dtype=BF16)
    got = torch.autograd.grad(outs[4], leaves, g)
    da = ops.block_attention_backward(g, qn, kn, v, out, lse, index, 64, kv_lens=lens, q_lens=lens)
    dn = ops.qk_norm_rotary_backward(da[0], da[1], q, k, wq, wk, coords, freqs, (8, 8))
    for a, c in zip(got, (dn[0], dn[1], da[2], dn[2], dn[3])):
        assert torch.equal(a, c) and a.isfinite().all()


def test_sparse_attention_over_all_blocks_is_the_dense_operator():
    """With every block chosen the result is sb_attn_pair's with a zero bias table."""
    g = gen(73)
    b, h, s, d = 2, 4, 150, 16
    q, k, v = (randn(g, b, h, s, d, dtype=F16) for _ in range(3))
    lens = torch.tensor([150, 81], dtype=torch.int32, device=DEV)
    index = torch.arange(3, dtype=torch.int32, device=DEV).expand(b, h, s, 3).contiguous()
    out, _ = ops.block_attention(q, k, v, index, 64, kv_lens=lens, q_lens=lens)
    pair = torch.zeros(b, s, s, dtype=torch.uint8, device=DEV)
    table = torch.zeros(238, h, device=DEV)
    dense = torch.empty_like(q)
    st = torch.cuda.current_stream().cuda_stream
    _lib.check(_lib.lib().sb_attn_pair(q.data_ptr(), k.data_ptr(), v.data_ptr(), pair.data_ptr(), table.data_ptr(),
                                       lens.data_ptr(), b, h, s, d, dense.data_ptr(), st), "attn_pair")
    _, bound = O.attention(q, k, v, index, 64, None, lens, lens)
    within(out, dense.double(), 2 * bound["out"] + 2.0**-20)  # both sides round alike


def test_operators_on_another_stream():
    ins = chain_inputs()
    want = chain(*ins)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        first = chain(*ins)
        second = chain(*chain_inputs(seed=74))
        third = chain(*ins)
    side.synchronize()
    for got in (first, third):
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    assert not torch.equal(second[4], want[4])


def capture_twice(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            results.append(step())
        graphs.append(gr)
    return graphs, results


def replay_and_compare(graphs, results, leaves, sources, eager):
    for source in sources:
        with torch.no_grad():
            for leaf, t in zip(leaves, source):
                leaf.copy_(t)
        want = eager()
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for res in results:
            assert all(torch.equal(a, c) for a, c in zip(res, want))
        other = torch.cuda.Stream()  # both at once: each graph has its own workspaces
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for res in results:
            assert all(torch.equal(a, c) for a, c in zip(res, want))


def test_operators_captured_into_two_graphs():
    """Forward and backward through autograd, captured twice, replayed in turn and at once on new
    inputs."""
    ins = chain_inputs()
    leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_() for t in ins[:5]]
    g = randn(gen(76), 2, 4, 520, 32, dtype=BF16)

    def step():
        outs = chain(*leaves, *ins[5:])
        return (outs[4].detach(), *torch.autograd.grad(outs[4], leaves, g))

    graphs, results = capture_twice(step)
    replay_and_compare(graphs, results, leaves, (ins, chain_inputs(seed=75)), step)


def test_backward_functions_captured_beside_an_eager_graph():
    """The backward functions need no autograd: they are captured while an eager graph of the same
    leaves is alive (autograd's own capture is not allowed that)."""
    ins = chain_inputs()
    leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_() for t in ins[:5]]
    g = randn(gen(77), 2, 4, 520, 32, dtype=BF16)
    kept = chain(*leaves, *ins[5:])[4]

    def step():
        q, k, v, wq, wk = (t.detach() for t in leaves)
        coords, freqs, lens = ins[5:]
        qn, kn, _, index, out, lse = chain(q, k, v, wq, wk, coords, freqs, lens)
        da = ops.block_attention_backward(g, qn, kn, v, out, lse, index, 64, kv_lens=lens, q_lens=lens)
        return (out, da[2], *ops.qk_norm_rotary_backward(da[0], da[1], q, k, wq, wk, coords, freqs, (8, 8)))

    graphs, results = capture_twice(step)
    assert kept.grad_fn is not None
    replay_and_compare(graphs, results, leaves, (ins, chain_inputs(seed=78)), step)


def test_single_tokens_captured_beside_one_another():
    """The serving form (means kept, one query row) captured twice, replayed at once on new inputs."""
    g = gen(79)
    k, v = (randn(g, 2, 2, 900, 64, dtype=BF16) for _ in range(2))
    lens = torch.tensor([900, 333], dtype=torch.int32, device=DEV)
    means = ops.block_means(k, 64, kv_lens=lens)
    q = randn(g, 2, 8, 1, 64, dtype=BF16)

    def step():
        index = ops.block_select(q, means, 5, 64, 900, kv_lens=lens, keep_first=1)
        return (index, *ops.block_attention(q, k, v, index, 64, kv_lens=lens))

    graphs, results = capture_twice(step)
    sources = [(q.clone(),), (randn(g, 2, 8, 1, 64, dtype=BF16),)]
    replay_and_compare(graphs, results, (q,), sources, step)
    found, bound = O.attention(q, k, v, results[0][0], 64, None, lens)
    within(results[0][1], found["out"], bound["out"])


def test_rows_past_two_to_the_32():
    """Strides that pass 32 bits: a cache whose rows lie 2^27 elements apart."""
    rows, d, step = 40, 16, 2**27
    g = gen(81)
    buf = torch.empty((rows - 1) * step + d, dtype=F16, device=DEV)
    k = buf.as_strided((1, 1, rows, d), (0, 0, step, 1))
    k.copy_(randn(g, 1, 1, rows, d, dtype=F16))
    assert (rows - 1) * step > 2**32
    q, v = randn(g, 1, 1, 20, d, dtype=F16), k
    index = torch.tensor([0, 1], dtype=torch.int32, device=DEV).expand(1, 1, 20, 2).contiguous()
    packed = k.contiguous()
    want = ops.block_attention(q, packed, packed, index, 32)
    got = ops.block_attention(q, k, v, index, 32)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    few = [ops.block_attention(q[:, :, :3], t, t, index[:, :, :3].contiguous(), 32)[0] for t in (k, packed)]
    assert torch.equal(*few)
    dout = randn(g, 1, 1, 20, d, dtype=F16)
    grads = [ops.block_attention_backward(dout, q, t, t, *want, index, 32) for t in (k, packed)]
    assert all(torch.equal(a, c) for a, c in zip(*grads))
    assert torch.equal(ops.block_means(k, 32), ops.block_means(packed, 32))
    coords = torch.randint(-9, 9, (1, rows, 1), generator=g, device=DEV)
    freqs = ops.rotary_freqs((8,), device=DEV)
    assert torch.equal(ops.axes_rotary(k, coords, freqs, (8,), out=torch.empty_like(packed)),
                       ops.axes_rotary(packed, coords, freqs, (8,)))
    w = torch.ones(d, device=DEV)
    pq = ops.qk_norm_rotary(packed, packed, w, w, coords, freqs, (8,))
    assert torch.equal(ops._qk(packed, packed, w, w, coords, freqs, (8,), False, 1e-6)[0], pq[0])


def test_calls_from_several_host_threads():
    """A kernel's shared-memory limit is the device's: a thread that asks for less must not take it
    from one that asked for more."""
    from concurrent.futures import ThreadPoolExecutor

    g = gen(91)
    q, k, v = (randn(g, 1, 1, 300, 16, dtype=F16) for _ in range(3))
    index = torch.randint(0, 5, (1, 1, 300, 64), generator=g, device=DEV, dtype=torch.int32)
    wide = lambda: ops.block_attention(q, k, v, index, 64)[0]  # noqa: E731
    slim = lambda: ops.block_attention(q, k, v, index[..., :1].contiguous(), 64)[0]  # noqa: E731
    want = wide(), slim()
    with ThreadPoolExecutor(4) as pool:
        got = list(pool.map(lambda i: (wide, slim)[i % 2](), range(40)))
    torch.cuda.synchronize()
    assert torch.equal(wide(), want[0])
    assert all(torch.equal(t, want[i % 2]) for i, t in enumerate(got))


def test_python_refusals_on_the_gpu():
    x = torch.zeros(1, 2, 20, 16, device=DEV, dtype=F16)
    index = torch.zeros(1, 2, 20, 1, device=DEV, dtype=torch.int32)
    coords = torch.zeros(1, 20, 1, device=DEV, dtype=torch.int32)
    freqs = ops.rotary_freqs((8,), device=DEV)
    bad = [
        lambda: ops.block_attention(x.float(), x.float(), x.float(), index, 64),
        lambda: ops.block_attention(x, x, x, index, 48),
        lambda: ops.block_attention(x, x, x, index.long(), 64),
        lambda: ops.block_attention(x, x[..., :8], x, index, 64),
        lambda: ops.block_attention(x, x, x.cpu(), index, 64),
        lambda: ops.block_attention(x, x, x, index, 64, kv_lens=torch.ones(2, dtype=torch.int32, device=DEV)),
        lambda: ops.block_attention(x, x, x, index, 64, kv_lens=torch.ones(1, dtype=torch.int64, device=DEV)),
        lambda: ops.block_attention(x.transpose(2, 3), x, x, index, 64),
        lambda: ops.block_select(x, torch.zeros(1, 2, 2, 16, device=DEV), 4, 64, 20),
        lambda: ops.block_select(x, torch.zeros(1, 2, 1, 16, device=DEV), 65, 64, 20),
        lambda: ops.axes_rotary(x, coords, freqs, (4,)),
        lambda: ops.axes_rotary(x, coords, freqs.float(), (8,)),
        lambda: ops.axes_rotary(x, coords.expand(1, 20, 2), freqs, (8,)),
        lambda: ops.axes_rotary(x, torch.zeros(1, 21, 1, device=DEV), freqs, (8,)),
        lambda: ops.axes_rotary(x.double(), coords, freqs, (8,)),
        lambda: ops.axes_rotary(x, coords, freqs, (8,), out=x.float()),
        lambda: ops.qk_norm_rotary(x, x, torch.ones(8, device=DEV), None),
        lambda: ops.qk_norm_rotary(x, x, torch.ones(16, device=DEV), torch.ones(16, device=DEV, dtype=F16)),
        lambda: ops.qk_norm_rotary(x, x, None, None, eps=-1.0),
        lambda: ops.block_means(x, 0),
        lambda: ops.block_means(x, 2**32 + 64),  # a size that would wrap into another
        lambda: ops.block_select(x, torch.zeros(1, 2, 1, 16, device=DEV), 4, 2**32 + 64, 20),
        lambda: ops.block_select(x, torch.zeros(1, 2, 1, 16, device=DEV), 4, 64, 20, keep_first=2**32 + 1),
        lambda: ops.block_attention(x, x, x, index, 2**32 + 64),
        lambda: ops.block_means(x[:, :, :1].expand(1, 2, 2**31 + 20, 16), 64),
    ]
    for call in bad:
        with pytest.raises((ValueError, RuntimeError)):
            call()
    # empty calls return empty or zero results
    e = x[:, :, :0]
    assert ops.axes_rotary(e, coords[:, :0], freqs, (8,)).shape == e.shape
    assert ops.block_attention(e, x, x, index[:, :, :0].contiguous(), 64)[0].shape == e.shape
    grads = ops.block_attention_backward(e, e, x, x, e, torch.zeros(1, 2, 0, device=DEV), index[:, :, :0].contiguous(), 64)
    assert (grads[1] == 0).all() and (grads[2] == 0).all()
    dw = ops.qk_norm_rotary_backward(e, e, e, e, torch.ones(16, device=DEV), None, None, None, ())[2]
    assert (dw == 0).all()
