"""Long-support attention operators on the GPU at the edges of their range: how
little the results lose, values of every size, sizes past one window. Against
64-bit forms, with bounds derived beside them."""

from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch

from hexo_bot_b200 import attention_ops as ops
from oracle import attention_ops as O
from test_gpu_attention_ops import BF16, DEV, F16, F32, gen, randn, spread, within

pytestmark = pytest.mark.gpu

SHAPES = [
    # b, hq, hk, sq, sk, d, block, topk
    (1, 2, 2, 300, 700, 16, 64, 5),
    (2, 4, 2, 170, 500, 64, 32, 9),
    (1, 3, 1, 200, 900, 128, 128, 4),
    (1, 2, 1, 260, 333, 40, 128, 3),
    (1, 2, 2, 140, 2100, 128, 64, 20),
    (2, 8, 2, 3, 900, 64, 64, 8),
    (1, 4, 4, 1, 2000, 128, 128, 16),
    (3, 2, 1, 16, 300, 16, 32, 6),
]


def tensors(case, dtype, seed):
    b, hq, hk, sq, sk, d, block, topk = case
    g = gen(seed)
    q, dout = (randn(g, b, hq, sq, d, dtype=dtype) for _ in range(2))
    k, v = (randn(g, b, hk, sk, d, dtype=dtype) for _ in range(2))
    index = torch.randint(-1, -(-sk // block), (b, hk, sq, topk), generator=g, device=DEV, dtype=torch.int32)
    return q, k, v, index, block, dout


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", SHAPES)
def test_block_attention_output_is_rounded_once(case, dtype):
    """The softmax weights lose nothing that the result could show."""
    q, k, v, index, block, _ = tensors(case, dtype, 101)
    out, lse = ops.block_attention(q, k, v, index, block)
    found, bound = O.attention(q, k, v, index, block, pair=True)
    within(out, found["out"], bound["out"], "out")
    within(lse, found["lse"], bound["lse"], "lse")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", SHAPES)
def test_block_attention_gradients_are_rounded_once(case, dtype):
    """Softmax weights and score gradients lose nothing that dq, dk and dv could show."""
    q, k, v, index, block, dout = tensors(case, dtype, 102)
    out, lse = ops.block_attention(q, k, v, index, block)
    grads = ops.block_attention_backward(dout, q, k, v, out, lse, index, block)
    found, bound = O.attention(q, k, v, index, block, dout=dout, pair=True)
    for name, got in zip(("dq", "dk", "dv"), grads):
        within(got, found[name], bound[name], name)


def gradients_within(q, k, v, index, block, dout, **kw):
    out, lse = ops.block_attention(q, k, v, index, block, **kw)
    grads = ops.block_attention_backward(dout, q, k, v, out, lse, index, block, **kw)
    found, bound = O.attention(q, k, v, index, block, dout=dout, pair=True, **kw)
    for name, got in zip(("dq", "dk", "dv"), grads):
        within(got, found[name], bound[name], name)
    return grads


@pytest.mark.parametrize("size", [1e4, 1.0, 1e-3, 1e-4, 2e-5, 1e-6])
def test_block_attention_gradients_of_any_size_in_f16(size):
    """Weights of 1 / 8192 times gradients of any size that f16 holds."""
    g = gen(103)
    q, k, v = (randn(g, 1, 1, n, 64, dtype=F16) for n in (80, 8192, 8192))
    index = torch.arange(64, dtype=torch.int32, device=DEV).expand(1, 1, 80, 64).contiguous()
    gradients_within(q, k, v, index, 128, randn(g, 1, 1, 80, 64, dtype=F16, scale=size))


@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("rising", [False, True])
def test_block_attention_gradients_of_mixed_sizes_in_f16(rising, d, block):
    """Rows whose gradients grow or fall by 2^20 from the first to the last, over many tiles."""
    g = gen(104)
    q, dout = (randn(g, 1, 2, 900, d, dtype=torch.float32) for _ in range(2))
    k, v = (randn(g, 1, 1, 300, d, dtype=F16) for _ in range(2))
    size = torch.logspace(-12, 8, 900, base=2.0, device=DEV)
    dout = (dout * (size if rising else size.flip(0))[:, None]).to(F16)
    index = torch.randint(-1, -(-300 // block), (1, 1, 900, 4), generator=g, device=DEV, dtype=torch.int32)
    gradients_within(q.to(F16), k, v, index, block, dout)


def test_block_attention_large_score_gradients_in_f16():
    """Score gradients past 65504, whose products with small keys are not."""
    q = torch.zeros(1, 1, 20, 64, dtype=F16, device=DEV)
    k, v = (torch.zeros(1, 1, 64, 64, dtype=F16, device=DEV) for _ in range(2))
    k[:, :, 0, 0], k[:, :, 1, 0] = 0.125, -0.125
    v[:, :, 0], v[:, :, 1] = 40, -40
    index = torch.zeros(1, 1, 20, 1, dtype=torch.int32, device=DEV)
    lens = torch.tensor([2], dtype=torch.int32, device=DEV)
    grads = gradients_within(q, k, v, index, 64, torch.full_like(q, 1500.0), kv_lens=lens)
    assert all(t.isfinite().all() for t in grads)


def test_block_attention_infinite_gradients_stay_in_their_rows():
    """A row of dout with an infinity or NaN leaves dq of the other rows as it is."""
    for dtype in (F16, BF16):
        q, k, v, index, block, dout = tensors((1, 2, 2, 300, 700, 64, 64, 5), dtype, 105)
        dout[0, 0, 7, 3], dout[0, 1, 9, 0] = float("inf"), float("nan")
        out, lse = ops.block_attention(q, k, v, index, block)
        dq = ops.block_attention_backward(dout, q, k, v, out, lse, index, block)[0]
        clean = dout.nan_to_num(0.0, 0.0, 0.0)
        want = ops.block_attention_backward(clean, q, k, v, out, lse, index, block)[0]
        rows = torch.ones(1, 2, 300, dtype=torch.bool, device=DEV)
        rows[0, 0, 7] = rows[0, 1, 9] = False
        assert torch.equal(dq[rows], want[rows]) and not dq[~rows].isfinite().any()


# ---- norm and rotation ------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,hq,hk,d", [(BF16, 16, 4, 64), (F16, 3, 1, 16), (F32, 5, 3, 20), (F32, 12, 6, 8)])
def test_qk_norm_gradients_without_eps(dtype, hq, hk, d):
    """eps = 0 is allowed where no row is zero: an odd number of tokens and heads that do not fill
    a warp leave lanes without a row, which must not reach the weight gradients."""
    g = gen(111)
    q, k, gq, gk = (randn(g, 1, h, 7, d, dtype=dtype) for h in (hq, hk, hq, hk))
    w = 1 + randn(g, d, scale=0.2)
    grads = ops.qk_norm_rotary_backward(gq, gk, q, k, w, w, None, None, (), eps=0.0)
    for x, gy, dx, dw in zip((q, k), (gq, gk), grads[:2], grads[2:]):
        x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
        want = torch.autograd.grad(O.qk_norm(x64, w64, None, eps=0.0), (x64, w64), gy.double())
        hat = (x64 * x64.square().mean(-1, keepdim=True).rsqrt()).detach()
        back = gy.double().abs() * w64.detach().abs()
        rstd = x64.detach().square().mean(-1, keepdim=True).rsqrt()
        mass = rstd * (back + hat.abs() * (back * hat.abs()).mean(-1, keepdim=True))
        within(dx, want[0], O.rounding(want[0], dtype) + (2 * d + 48) * 2.0**-24 * mass, "dx")
        mass = (gy.double().abs() * hat.abs()).sum((0, 1, 2))
        within(dw, want[1], O.rounding(want[1], F32) + (d + 96) * 2.0**-24 * mass, "dw")


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_without_a_place_keep_infinities_to_themselves(dtype, adjacent):
    """Rows before the placed ones are not turned: an infinity or NaN there stays in its channel."""
    x = randn(gen(112), 2, 3, 6, 16, dtype=dtype)
    x[:, :, 0, 3], x[:, :, 1, 5], x[:, :, 2, 6] = float("inf"), float("-inf"), float("nan")
    coords = torch.ones(2, 3, 1, dtype=torch.int32, device=DEV)
    freqs = ops.rotary_freqs((8,), device=DEV)
    for inverse in (False, True):
        y = ops.axes_rotary(x, coords, freqs, (8,), adjacent=adjacent, inverse=inverse)
        assert torch.equal(y[:, :, :3].nan_to_num(5.0), x[:, :, :3].nan_to_num(5.0))
        assert y[:, :, 3:].isfinite().all()
    # behind the norm: x / inf is 0 beside NaN at the infinity itself, with and without places
    turned = ops.qk_norm_rotary(x, x[:, :1], None, None, coords, freqs, (8,), adjacent=adjacent)
    plain = ops.qk_norm_rotary(x, x[:, :1], None, None)
    for a, c in zip(turned, plain):
        assert torch.equal(a[:, :, :3].nan_to_num(5.0), c[:, :, :3].nan_to_num(5.0))
        assert int(a[:, :, :2].isnan().sum()) == 2 * a.shape[0] * a.shape[1]
    grads = ops.qk_norm_rotary_backward(x, x[:, :1], x.nan_to_num(1.0, 1.0, 1.0), x[:, :1].nan_to_num(1.0, 1.0, 1.0), None, None,
                                        coords, freqs, (8,), adjacent=adjacent)
    want = ops.qk_norm_rotary_backward(x, x[:, :1], x.nan_to_num(1.0, 1.0, 1.0), x[:, :1].nan_to_num(1.0, 1.0, 1.0), None, None,
                                       None, None, ())
    for a, c in zip(grads[:2], want[:2]):
        assert torch.equal(a[:, :, :3].nan_to_num(5.0), c[:, :, :3].nan_to_num(5.0))


@pytest.mark.parametrize("b,s,hq,hk,d,sections", [(3, 217, 12, 4, 20, (3, 5)), (8, 2440, 16, 4, 64, (16, 16)),
                                                  (64, 500, 8, 8, 128, (64,)), (2000, 37, 3, 1, 18, (2, 3))])
def test_weight_gradients_of_long_sums(b, s, hq, hk, d, sections):
    """dq_weight and dk_weight err no more than 32-bit terms summed in 64 bits do (1.5 times: both
    errors are sums of independent roundings over the channels), however many rows there are."""
    g = gen(113)
    q, k, gq, gk = (randn(g, b, h, s, d, scale=1.5) for h in (hq, hk, hq, hk))
    w = 1 + randn(g, d, scale=0.2)
    coords = torch.randint(-32, 32, (b, s, len(sections)), generator=g, device=DEV)
    freqs = ops.rotary_freqs(sections, device=DEV)
    ang = -O.angles(coords, freqs, sections, s)
    grads = ops.qk_norm_rotary_backward(gq, gk, q, k, w, w, coords, freqs, sections)
    p = sum(sections)
    for x, gy, dw in zip((q, k), (gq, gk), grads[2:]):
        found = []
        for dt in (torch.float64, F32):
            cos, sin, u, v = ang.cos().to(dt), ang.sin().to(dt), gy[..., :p].to(dt), gy[..., p : 2 * p].to(dt)
            turned = torch.cat([u * cos - v * sin, v * cos + u * sin, gy[..., 2 * p :].to(dt)], -1)
            hat = x.to(dt) * torch.rsqrt(x.to(dt).square().mean(-1, keepdim=True) + 1e-6)
            found.append((turned * hat).sum((0, 1, 2), dtype=torch.float64).to(dt))
        want, plain = found
        off, least = ((t.double() - want).norm() for t in (dw, plain))
        assert off <= 1.5 * least + 2.0**-24 * want.norm(), (off / want.norm(), least / want.norm())


PI = Fraction(31415926535897932384626433832795028841971693993751058209749445923, 10**64)


FAR = [2**20, 2**28, 2**31 - 1, 10**12, 1_700_000_000_000, 1_700_000_000_000_000, 2**52, 2**53]


@pytest.mark.parametrize("size,kind", [(n, t) for n in FAR for t in (torch.int64, F32)] + [(n, torch.int32) for n in FAR[:3]])
def test_coordinates_of_any_size(size, kind):
    """cos and sin of far positions against exact arithmetic. One turn of (1, 0): the kernel's
    reduced angle is a float of at most pi / 4 (three roundings of 2^-24), its series and their
    roundings are off by 1e-7 at most: 2^-22 in all."""
    places = torch.tensor([size, size - 1, -size, size // 3, size // 7 * 5, 1], dtype=torch.int64).to(kind)
    freqs = torch.tensor([1.0, 0.7853981633974483, 1e-4, 1 / 3], dtype=torch.float64)
    n = places.numel()
    x = torch.zeros(1, 1, n, 8, device=DEV)
    x[..., :4] = 1
    y = ops.axes_rotary(x, places.view(1, n, 1).to(DEV), freqs.to(DEV), (4,)).double().cpu()
    for i, c in enumerate(places.tolist()):
        for p, f in enumerate(freqs.tolist()):
            angle = float((Fraction(f) * Fraction(c)) % (2 * PI))
            assert abs(y[0, 0, i, p].item() - math.cos(angle)) <= 2.0**-22, (c, f)
            assert abs(y[0, 0, i, 4 + p].item() - math.sin(angle)) <= 2.0**-22, (c, f)


# ---- beside torch -----------------------------------------------------------------------------


def test_compiled_programs_call_the_operators_as_they_are():
    x = randn(gen(121), 1, 2, 6, 16)
    coords = torch.ones(1, 6, 1, dtype=torch.int32, device=DEV)
    freqs = ops.rotary_freqs((8,), device=DEV)

    def step(x):
        return ops.axes_rotary(x * 2, coords, freqs, (8,)) + 1

    assert torch.equal(torch.compile(step, backend="eager")(x), step(x))


def test_writes_into_out_are_seen_by_autograd():
    """A graph that kept a tensor which `out` overwrote refuses its backward; an `out` that needs a
    gradient is refused."""
    coords = torch.ones(1, 6, 1, dtype=torch.int32, device=DEV)
    freqs = ops.rotary_freqs((8,), device=DEV)
    x = randn(gen(122), 1, 2, 6, 16)
    w = torch.ones(16, device=DEV, requires_grad=True)
    loss = (w * x).sum()
    ops.axes_rotary(x, coords, freqs, (8,), out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    y = x.clone()
    kept = (w * y).sum()
    ops.axes_rotary(x, coords, freqs, (8,), out=torch.empty_like(x))  # another tensor: nothing changes
    kept.backward()
    leaf = torch.empty_like(x, requires_grad=True)
    with pytest.raises(ValueError, match="out="):
        ops.axes_rotary(x, coords, freqs, (8,), out=leaf)
    with torch.no_grad():
        want = ops.axes_rotary(x, coords, freqs, (8,))
        assert torch.equal(ops.axes_rotary(x, coords, freqs, (8,), out=leaf), want)
    with torch.inference_mode():
        z = x.clone()
        assert torch.equal(ops.axes_rotary(z, coords, freqs, (8,), out=z), want)


def test_rows_and_heads_that_overlap():
    """Views whose rows or heads lie one element apart (sliding windows) give what copies give."""
    base = randn(gen(123), 4000)
    coords = torch.randint(-9, 9, (1, 4, 1), generator=gen(124), device=DEV)
    freqs = ops.rotary_freqs((8,), device=DEV)
    for strides in ((0, 100, 1, 1), (0, 1, 50, 1), (0, 1, 1, 1)):
        x = base.as_strided((1, 3, 4, 16), strides)
        copy = x.clone(memory_format=torch.contiguous_format)
        assert torch.equal(ops.axes_rotary(x, coords, freqs, (8,)), ops.axes_rotary(copy, coords, freqs, (8,)))
        # behind the norm against 64 bits: narrower accesses add the squares in another order
        ang = O.angles(coords, freqs, (8,), 4)
        x64 = copy.double().requires_grad_()
        want = O.qk_norm(x64, None, ang)
        rstd = (x64.square().mean(-1, keepdim=True) + 1e-6).rsqrt().detach()
        hat = (x64.detach() * rstd).abs()
        for out in ops.qk_norm_rotary(x, x, None, None, coords, freqs, (8,)):
            within(out, want.detach(), O.rounding(want.detach(), F32) + 40 * 2.0**-24 * spread(hat, ang, False))
        (dx,) = torch.autograd.grad(want, x64, copy.double())
        back = spread(copy.double().abs(), ang, False)
        mass = rstd * (back + hat * (back * hat).mean(-1, keepdim=True))
        for got in ops.qk_norm_rotary_backward(copy, copy, x, x, None, None, coords, freqs, (8,))[:2]:
            within(got, dx, O.rounding(dx, F32) + 80 * 2.0**-24 * mass)


def test_one_token_with_its_newest_block():
    """Means kept by the program, one query, the newest block put behind the chosen ones."""
    g = gen(125)
    k, v = (randn(g, 3, 2, 900, 64, dtype=BF16) for _ in range(2))
    q = randn(g, 3, 8, 1, 64, dtype=BF16)
    lens = torch.tensor([900, 333, 64], dtype=torch.int32, device=DEV)
    means = ops.block_means(k, 64, kv_lens=lens)
    newest = ((lens - 1) // 64).view(3, 1, 1, 1).expand(3, 2, 1, 1)
    index = torch.cat([ops.block_select(q, means, 4, 64, 900, kv_lens=lens, keep_first=1), newest], -1)
    out, lse = ops.block_attention(q, k, v, index, 64, kv_lens=lens)
    want = O.select(q, means, 4, 64, 900, lens, None, 1, False)
    kept = torch.cat([want.to(DEV), newest], -1)
    assert torch.equal(index, kept) and index[1, 0, 0, -1] == 5 and index[2, 0, 0].tolist() == [0, -1, -1, -1, 0]
    found, bound = O.attention(q, k, v, kept, 64, None, lens, pair=True)
    within(out, found["out"], bound["out"], "out")
    within(lse, found["lse"], bound["lse"], "lse")


# ---- several windows ----------------------------------------------------------------------------

WINDOWS = [
    # b, hq, hk, sq, sk, d, block, topk, heads of a window (0: windows over the rows of a head)
    (2, 8, 2, 4200, 1500, 128, 32, 40, 3),
    (5, 6, 3, 4300, 700, 64, 64, 60, 7),
    (1, 4, 1, 13500, 1500, 128, 32, 40, 0),
    (1, 4, 1, 13500, 4000, 128, 128, 40, 0),
    (2, 2, 1, 33000, 500, 64, 64, 64, 0),
]


@pytest.mark.parametrize("case", WINDOWS)
def test_block_attention_over_several_windows(case):
    """Parts past 1 GB: several launches over heads, and over the rows of one head. Against 64 bits, and
    the forward against the same heads one at a time, bit for bit."""
    b, hq, hk, sq, sk, d, block, topk, heads = case
    parts = hq // hk * topk * (4 * d + 8) * sq  # of one key head, forward
    assert b * hk * parts > 2**30 and (parts > 2**30) == (heads == 0)
    assert heads == 2**30 // parts < b * hk or heads == 0
    q, k, v, index, block, dout = tensors(case[:8], BF16, 131)
    qn = torch.tensor([sq - 77 * i for i in range(b)], dtype=torch.int32, device=DEV)
    kn = torch.tensor([sk - 99 * i for i in range(b)], dtype=torch.int32, device=DEV)
    out, lse = ops.block_attention(q, k, v, index, block, kv_lens=kn, q_lens=qn)
    grads = ops.block_attention_backward(dout, q, k, v, out, lse, index, block, kv_lens=kn, q_lens=qn)
    again = ops.block_attention_backward(dout, q, k, v, out, lse, index, block, kv_lens=kn, q_lens=qn)
    assert all(torch.equal(a, c) for a, c in zip(grads, again))
    grp = hq // hk
    for i in range(b):
        for h in range(hk):
            at, qs = (slice(i, i + 1), slice(h, h + 1)), (slice(i, i + 1), slice(h * grp, (h + 1) * grp))
            one = q[qs], k[at], v[at], index[at].contiguous()
            found, bound = O.attention(*one, block, None, kn[i : i + 1], qn[i : i + 1], dout[qs], pair=True)
            within(out[qs], found["out"], bound["out"], "out")
            within(lse[qs], found["lse"], bound["lse"], "lse")
            for name, got in zip(("dq", "dk", "dv"), (grads[0][qs], grads[1][at], grads[2][at])):
                within(got, found[name], bound[name], name)
            alone = ops.block_attention(*one, block, kv_lens=kn[i : i + 1], q_lens=qn[i : i + 1])
            assert torch.equal(alone[0], out[qs]) and torch.equal(alone[1], lse[qs])
