"""Attention operators for long supports, on the C ABI (include/shrimp_b200.h).

Beside the network's biased dense attention (`sb_attn_pair`): rotary positions
with several axes, the norm of queries and keys per head with the rotation in
the same pass, and attention in which every query reads only the key blocks it
has chosen. Every tensor is a (batch, heads, rows, head_dim) view, so the heads
of a packed projection `qkv.view(B, S, 3, H, D)` are passed as
`qkv[:, :, 0].transpose(1, 2)` without a copy.

    freqs = rotary_freqs((8, 8), device="cuda")              # once: hex q and r
    q, k = qk_norm_rotary(q, k, wq, wk, coords, freqs, (8, 8))
    means = block_means(k, 64, kv_lens=lens)
    index = block_select(q, means, 8, 64, k.shape[2], kv_lens=lens, q_lens=lens, keep_first=1)
    out, lse = block_attention(q, k, v, index, 64, kv_lens=lens, q_lens=lens)

Calls run on the current stream of the tensors' device, neither synchronise nor
keep anything between calls, and may be captured into CUDA graphs. Gradients go
through autograd, or through the `*_backward` functions; a capture of autograd's
backward must not find an eager graph of the same leaves alive (torch then has
the capture wait for the other stream and fail), the functions have no such
limit. There is no forward-mode derivative, and traces (`torch.jit.trace`, `make_fx`) are refused;
`torch.compile` leaves the calls outside of its graphs. CUDA tensors only: there is no CPU fallback.
"""

from __future__ import annotations

import ctypes as C
import math
from functools import lru_cache
from typing import Optional, Sequence

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_MOST = 2**31 - 1
_PROXY = torch._C._TorchDispatchModeKey.PROXY  # the mode of make_fx
_FLOATS = {torch.float32: _lib.DT_F32, torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}
_COORDS = {torch.int64: _lib.DT_I64, torch.int32: _lib.DT_I32, torch.int16: _lib.DT_I16, torch.float32: _lib.DT_F32}


# ---- arguments ------------------------------------------------------------------------------


def _check(t: torch.Tensor, name: str, like: torch.Tensor, shape: Sequence[int], dtype=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.device != like.device:
        raise ValueError(f"{name} must be a tensor on {like.device}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _first(t: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise ValueError(f"{name} must be a (batch, heads, rows, head_dim) tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} is on {t.device}: the kernels need CUDA tensors (no CPU fallback)")
    if t.dtype not in _FLOATS:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if max(t.shape) > _MOST:
        raise ValueError(f"{name} has an axis of more than 2^31 - 1 elements")
    return t


def _int(n: int, name: str, least: int) -> int:
    """A size that the C side takes as a 32-bit integer."""
    if not least <= n <= _MOST:
        raise ValueError(f"{name} must lie in {least} to 2^31 - 1, got {n}")
    return n


def _heads(t: torch.Tensor, name: str) -> _lib.Heads:
    b, h, s, d = t.shape
    sb, sh, ss, sd = t.stride()
    if sd != 1 and d > 1:
        raise ValueError(f"{name} needs unit stride over head_dim")
    # the stride of an axis of one element says nothing
    return _lib.Heads(t.data_ptr(), sb if b > 1 else 0, sh if h > 1 else 0, ss if s > 1 else 0)


def _like(t: torch.Tensor) -> torch.Tensor:
    """A result of t's shape with unit stride over head_dim. empty_like follows t's strides, and puts
    another axis last where t's rows or heads lie one element apart (windows that overlap)."""
    y = torch.empty_like(t)
    return y if y.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _grad(t: torch.Tensor) -> torch.Tensor:
    """An incoming gradient as a view the kernels read: packed anew unless it is one already."""
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0
    ok = ok and all(s * t.element_size() % 16 == 0 for s, n in zip(t.stride()[:3], t.shape) if n > 1)
    return t if ok else t.contiguous()


def _lens(t: Optional[torch.Tensor], name: str, like: torch.Tensor) -> Optional[int]:
    if t is None:
        return None
    _check(t, name, like, (like.shape[0],), torch.int32)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _call(t: torch.Tensor, what: str, fn, *args, stream: bool = True) -> None:
    """fn(*args) with t's device as the current one, and that device's current stream as the last
    argument of calls that take one; raises on a refusal."""
    index = t.device.index
    if stream:
        args += (torch._C._cuda_getCurrentRawStream(index),)
    if index == torch._C._cuda_getDevice():
        rc = fn(*args)
    else:
        with torch.cuda.device(index):
            rc = fn(*args)
    if rc:
        _lib.check(rc, what)


def _visible(*ts) -> None:
    """Refuses calls that would lose something in silence: a trace would not see the kernel and keep
    its outputs as memory without values, a forward-mode tangent of ts would be dropped."""

    if torch._C._is_tracing() or torch._C._get_dispatch_mode(_PROXY) is not None:
        raise RuntimeError("the kernels cannot be traced: leave the call outside of the traced function")
    if forward_ad._current_level >= 0:
        if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in ts):
            raise RuntimeError("the kernels have no forward-mode derivative")


def _wants_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _frozen(coords, freqs) -> None:
    for t, name in ((coords, "coords"), (freqs, "freqs")):
        if isinstance(t, torch.Tensor) and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} gets no gradient: detach it")


# ---- rotary positions -------------------------------------------------------------------------


def rotary_freqs(sections: Sequence[int], theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """The usual angle table: axis a's pair j of m turns theta ** (-j / m) radians a step.

    float64, one entry per pair, axes in order. Any other table of that form (scaled, learned and
    frozen) serves as well; neither it nor the coordinates get a gradient."""

    table = [theta ** (-j / m) for m in sections for j in range(m)]
    return torch.tensor(table, dtype=torch.float64, device=device)


@lru_cache(maxsize=64)
def _sections(sections):
    """Pairs in all and the C array of checked section sizes."""
    if not 1 <= len(sections) <= 4 or min(sections) < 1:
        raise ValueError(f"sections must be 1 to 4 positive pair counts, got {sections}")
    return sum(sections), (C.c_int * 4)(*sections)


def _rotary(x, coords, freqs, sections, adjacent) -> Optional[_lib.Rotary]:
    b, _, s, d = x.shape
    pairs, parts = _sections(tuple(sections))
    if 2 * pairs > d:
        raise ValueError(f"{pairs} pairs do not fit head_dim {d}")
    if not isinstance(coords, torch.Tensor) or coords.dim() != 3 or coords.dtype not in _COORDS:
        raise ValueError("coords must be a (batch, placed rows, axes) tensor of int16, int32, int64 or float32")
    n = coords.shape[1]
    if n > s:
        raise ValueError(f"coords place {n} rows, x has {s}")
    _check(coords, "coords", x, (b, n, len(sections)))
    _check(freqs, "freqs", x, (pairs,), torch.float64)
    if not freqs.is_contiguous():
        raise ValueError("freqs must be contiguous")
    st = coords.stride()
    return _lib.Rotary(coords.data_ptr(), _COORDS[coords.dtype], st[0], st[1], st[2], s - n, len(sections), parts,
                       adjacent, freqs.data_ptr())


def _turn(x, coords, freqs, sections, adjacent, inverse, out=None):
    b, h, s, d = x.shape
    rot = _rotary(x, coords, freqs, sections, adjacent)
    y = _like(x) if out is None else _check(out, "out", x, x.shape, x.dtype)
    hx, hy = _heads(x, "x"), _heads(y, "out")
    _call(x, "axes_rotary", _lib.lib().sb_axes_rotary, hx, _FLOATS[x.dtype], rot, inverse, b, h, s, d, hy)
    if out is not None:
        torch.autograd.graph.increment_version(out)
    return y


class _Turn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, coords, freqs, sections, adjacent, inverse):
        ctx.save_for_backward(coords, freqs)
        ctx.rest = sections, adjacent, inverse
        return _turn(x, coords, freqs, sections, adjacent, inverse)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        sections, adjacent, inverse = ctx.rest
        return _turn(_grad(g), *ctx.saved_tensors, sections, adjacent, not inverse), None, None, None, None, None


def axes_rotary(x, coords, freqs, sections, *, adjacent=False, inverse=False, out=None):
    """x (B, H, S, D) turned by its rows' positions on several axes.

    coords (B, S - prefix, axes): the first `prefix` rows (summary tokens) have no place and stay
    as they are. sections: pairs of each axis; freqs: `rotary_freqs(sections)`. Half pairing joins
    channels (p, P + p) of the P pairs, `adjacent` (2p, 2p + 1); channels from 2P on stay.
    Coordinates and angles up to 2^53 keep 32-bit accuracy.
    `inverse` turns back. `out` may be x; it is written without autograd's knowledge and must not
    need a gradient, but graphs that kept it refuse their backward, as after torch's own writes."""

    _visible(x, coords, freqs)
    _frozen(coords, freqs)
    _first(x, "x")
    if _wants_grad(x, out):
        if out is not None:
            raise ValueError("out= is not differentiable")
        return _Turn.apply(x, coords, freqs, tuple(sections), adjacent, inverse)
    return _turn(x, coords, freqs, sections, adjacent, inverse, out)


# ---- query / key norm with the rotation ---------------------------------------------------------


def _qk_args(q, k, q_weight, k_weight, coords, freqs, sections, adjacent, eps):
    _first(q, "q")
    b, _, s, d = q.shape
    _first(k, "k")
    _check(k, "k", q, (b, k.shape[1], s, d), q.dtype)
    wd = torch.float32
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is None:
            continue
        wd = w.dtype
        if wd not in _FLOATS:
            raise ValueError(f"{name} must be float32, float16 or bfloat16")
        _check(w, name, q, (d,))
        if not w.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must share a dtype")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    rot = None if coords is None else _rotary(q, coords, freqs, sections, adjacent)
    return (b, q.shape[1], k.shape[1], s, d), _FLOATS[q.dtype], _FLOATS[wd], rot


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _qk(q, k, q_weight, k_weight, coords, freqs, sections, adjacent, eps):
    sizes, dt, wdt, rot = _qk_args(q, k, q_weight, k_weight, coords, freqs, sections, adjacent, eps)
    qo, ko = _like(q), _like(k)
    ins, outs = (_heads(q, "q"), _heads(k, "k")), (_heads(qo, "q"), _heads(ko, "k"))
    _call(q, "qk_norm_rotary", _lib.lib().sb_qk_norm_rotary, *ins, dt, _ptr(q_weight), _ptr(k_weight), wdt, eps, rot, *sizes,
          *outs)
    return qo, ko


def qk_norm_rotary_backward(dq_out, dk_out, q, k, q_weight, k_weight, coords, freqs, sections, *, adjacent=False, eps=1e-6):
    """Gradients (dq, dk, dq_weight, dk_weight) of `qk_norm_rotary` from those of its outputs; a
    weight that is None has none."""

    _visible(dq_out, dk_out, q, k, q_weight, k_weight, coords, freqs)
    sizes, dt, wdt, rot = _qk_args(q, k, q_weight, k_weight, coords, freqs, sections, adjacent, eps)
    _check(dq_out, "dq_out", q, q.shape, q.dtype)
    _check(dk_out, "dk_out", q, k.shape, q.dtype)
    dq, dk = _like(q), _like(k)
    dqw = None if q_weight is None else torch.empty_like(q_weight)
    dkw = None if k_weight is None else torch.empty_like(k_weight)
    need = C.c_size_t()
    lib = _lib.lib()
    _lib.check(lib.sb_qk_norm_rotary_backward_workspace_bytes(sizes[4], need), "qk_norm_rotary_backward")
    ws = torch.empty(need.value, dtype=torch.uint8, device=q.device)
    gs = _heads(dq_out, "dq_out"), _heads(dk_out, "dk_out")
    ins, outs = (_heads(q, "q"), _heads(k, "k")), (_heads(dq, "dq"), _heads(dk, "dk"))
    _call(q, "qk_norm_rotary_backward", lib.sb_qk_norm_rotary_backward, *gs, *ins, dt, _ptr(q_weight), _ptr(k_weight), wdt,
          eps, rot, *sizes, *outs, _ptr(dqw), _ptr(dkw), ws.data_ptr(), need.value)
    return dq, dk, dqw, dkw


class _QkNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, coords, freqs, sections, adjacent, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, coords, freqs)
        ctx.rest = sections, adjacent, eps
        return _qk(q, k, q_weight, k_weight, coords, freqs, sections, adjacent, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        sections, adjacent, eps = ctx.rest
        grads = qk_norm_rotary_backward(_grad(gq), _grad(gk), *ctx.saved_tensors, sections, adjacent=adjacent, eps=eps)
        return (*grads, None, None, None, None, None)


def qk_norm_rotary(q, k, q_weight, k_weight, coords=None, freqs=None, sections=(), *, adjacent=False, eps=1e-6):
    """RMS norm of every head of q (B, Hq, S, D) and k (B, Hk, S, D), times a weight per channel
    ((D) or None), then the rotation of `axes_rotary` (coords None: none), in one pass."""

    _visible(q, k, q_weight, k_weight, coords, freqs)
    _frozen(coords, freqs)
    _first(q, "q")
    if _wants_grad(q, k, q_weight, k_weight):
        return _QkNorm.apply(q, k, q_weight, k_weight, coords, freqs, tuple(sections), adjacent, eps)
    return _qk(q, k, q_weight, k_weight, coords, freqs, sections, adjacent, eps)


# ---- block-sparse attention ----------------------------------------------------------------------


def block_means(k, block, *, kv_lens=None):
    """(B, H, ceil(S / block), D) float32 means of the live keys (t < kv_lens[b]) of each block of
    k (B, H, S, D); 0 for a block without any. No gradient: the choice of blocks has none."""

    _visible()
    _first(k, "k")
    b, h, s, d = k.shape
    _int(block, "block", 1)
    out = torch.empty(b, h, -(-s // block), d, dtype=torch.float32, device=k.device)
    lens, hk = _lens(kv_lens, "kv_lens", k), _heads(k, "k")
    _call(k, "block_means", _lib.lib().sb_block_means, hk, _FLOATS[k.dtype], lens, b, h, s, d, block, out.data_ptr())
    return out


def block_select(q, means, topk, block, kv_rows, *, kv_lens=None, q_lens=None, keep_first=0, keep_own=False):
    """(B, Hkv, Sq, topk) int32: the key blocks each query keeps, ascending, -1 behind them.

    Score of a block: the group's query heads, summed, times its mean (`block_means`, or means that
    a serving program keeps up to date). The first `keep_first` blocks, and with `keep_own` the
    block row // block, are always kept. Rows count from 0 in every call, so for one query against a
    history `keep_own` names block 0: leave it off there, choose topk - 1 blocks and put the newest
    one behind them (`block_attention` takes any order and counts a block named twice once). Ties go
    to the lowest index."""

    _visible()
    _first(q, "q")
    b, hq, sq, d = q.shape
    if not isinstance(means, torch.Tensor) or means.dim() != 4:
        raise ValueError("means must be a (batch, kv heads, blocks, head_dim) tensor")
    _int(block, "block", 1), _int(kv_rows, "kv_rows", 0), _int(topk, "topk", 1), _int(keep_first, "keep_first", 0)
    hk = means.shape[1]
    _check(means, "means", q, (b, hk, -(-kv_rows // block), d), torch.float32)
    if not means.is_contiguous():
        raise ValueError("means must be contiguous")
    out = torch.empty(b, hk, sq, topk, dtype=torch.int32, device=q.device)
    kl, ql, hq_view = _lens(kv_lens, "kv_lens", q), _lens(q_lens, "q_lens", q), _heads(q, "q")
    _call(q, "block_select", _lib.lib().sb_block_select, hq_view, _FLOATS[q.dtype], means.data_ptr(), kl, ql, b, hq, hk, sq,
          kv_rows, d, block, topk, keep_first, keep_own, out.data_ptr())
    return out


def _attn_args(q, k, v, index, block, scale):
    _first(q, "q")
    b, hq, sq, d = q.shape
    _first(k, "k")
    hk, sk = k.shape[1], k.shape[2]
    _check(k, "k", q, (b, hk, sk, d), q.dtype)
    _check(v, "v", q, (b, hk, sk, d), q.dtype)
    if not isinstance(index, torch.Tensor) or index.dim() != 4:
        raise ValueError("index must be a (batch, kv heads, rows, topk) tensor")
    topk = index.shape[3]
    _int(block, "block", 1)
    _check(index, "index", q, (b, hk, sq, topk), torch.int32)
    if not index.is_contiguous():
        raise ValueError("index must be contiguous")
    return (b, hq, hk, sq, sk, d, block, topk), _FLOATS[q.dtype], 1.0 / math.sqrt(d) if scale is None else float(scale)


def _attn_workspace(t, sizes, backward):
    need = C.c_size_t()  # the plan counts the SMs of the device that the call runs on
    _call(t, "block_attention", _lib.lib().sb_block_attention_workspace_bytes, *sizes, backward, need, stream=False)
    return torch.empty(need.value, dtype=torch.uint8, device=t.device) if need.value else None, need.value


def _attend(q, k, v, index, block, scale, kv_lens, q_lens):
    sizes, dt, scale = _attn_args(q, k, v, index, block, scale)
    b, hq, _, sq = sizes[:4]
    out = _like(q)
    lse = torch.empty(b, hq, sq, dtype=torch.float32, device=q.device)
    ws, need = _attn_workspace(q, sizes, 0)
    kl, ql = _lens(kv_lens, "kv_lens", q), _lens(q_lens, "q_lens", q)
    hs, ho = (_heads(q, "q"), _heads(k, "k"), _heads(v, "v")), _heads(out, "out")
    _call(q, "block_attention", _lib.lib().sb_block_attention, *hs, dt, index.data_ptr(), kl, ql, *sizes, scale, ho,
          lse.data_ptr(), _ptr(ws), need)
    return out, lse


def block_attention_backward(dout, q, k, v, out, lse, index, block, *, scale=None, kv_lens=None, q_lens=None):
    """Gradients (dq, dk, dv) of `block_attention` from that of `out` and the forward's results."""

    _visible(dout, q, k, v, out, lse)
    sizes, dt, scale = _attn_args(q, k, v, index, block, scale)
    b, hq, _, sq = sizes[:4]
    _check(dout, "dout", q, q.shape, q.dtype)
    _check(out, "out", q, q.shape, q.dtype)
    _check(lse, "lse", q, (b, hq, sq), torch.float32)
    if not lse.is_contiguous():
        raise ValueError("lse must be contiguous")
    if sq == 0:
        return torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dq, dk, dv = _like(q), _like(k), _like(v)
    ws, need = _attn_workspace(q, sizes, 1)
    kl, ql = _lens(kv_lens, "kv_lens", q), _lens(q_lens, "q_lens", q)
    ins = _heads(dout, "dout"), _heads(q, "q"), _heads(k, "k"), _heads(v, "v"), _heads(out, "out")
    outs = _heads(dq, "dq"), _heads(dk, "dk"), _heads(dv, "dv")
    _call(q, "block_attention_backward", _lib.lib().sb_block_attention_backward, *ins, lse.data_ptr(), dt, index.data_ptr(),
          kl, ql, *sizes, scale, *outs, _ptr(ws), need)
    return dq, dk, dv


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, index, block, scale, kv_lens, q_lens):
        out, lse = _attend(q, k, v, index, block, scale, kv_lens, q_lens)
        ctx.save_for_backward(q, k, v, out, lse, index, kv_lens, q_lens)
        ctx.rest = block, scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        *saved, kv_lens, q_lens = ctx.saved_tensors
        block, scale = ctx.rest
        grads = block_attention_backward(_grad(g), *saved, block, scale=scale, kv_lens=kv_lens, q_lens=q_lens)
        return (*grads, None, None, None, None, None)


def block_attention(q, k, v, index, block, *, scale=None, kv_lens=None, q_lens=None):
    """(out, lse): softmax attention of each query over the live keys of its chosen blocks.

    q (B, Hq, Sq, D), k and v (B, Hkv, Sk, D) float16 or bfloat16, index (B, Hkv, Sq, topk) int32
    as `block_select` gives it (any order; entries out of range are skipped, one named twice counts
    once), block 32, 64 or 128, scale 1 / sqrt(D) by default. lse (B, Hq, Sq) float32 is the log of
    each row's sum of exp(scores) and has no gradient. Rows without keys and rows past q_lens give zeros and -inf."""

    _visible(q, k, v)
    _first(q, "q")
    if _wants_grad(q, k, v):
        return _Attend.apply(q, k, v, index, block, scale, kv_lens, q_lens)
    return _attend(q, k, v, index, block, scale, kv_lens, q_lens)


__all__ = ["rotary_freqs", "axes_rotary", "qk_norm_rotary", "qk_norm_rotary_backward", "block_means", "block_select",
           "block_attention", "block_attention_backward"]
