"""Refusals of the long-support attention operators, at the C boundary and in
Python, without a GPU; the 64-bit oracle against torch's own autograd."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from hexo_bot_b200 import _lib
from hexo_bot_b200 import attention_ops as ops
from oracle import attention_ops as O

A16 = 1 << 20  # an aligned address that no refused call reads


def heads(data=A16, b=1024, h=64, s=64):
    return _lib.Heads(data, b, h, s)


def rotary(**kw):
    f = dict(coords=A16, coords_dtype=_lib.DT_I16, batch_stride=8, row_stride=2, axis_stride=1, prefix=0, axes=2,
             sections=(4, 4), adjacent=0, freqs=A16)
    f.update(kw)
    f["sections"] = (C.c_int * 4)(*f["sections"])
    return _lib.Rotary(*f.values())


def refused(rc, code, word):
    assert rc == code, (rc, _lib.last_error())
    assert word in _lib.last_error()


def turn(x=None, dtype=_lib.DT_F16, rot=None, b=1, h=2, s=4, d=64, out=None):
    return _lib.lib().sb_axes_rotary(x or heads(), dtype, rot or rotary(), 0, b, h, s, d, out or heads(), None)


@pytest.mark.parametrize(
    "kw,code,word",
    [
        (dict(dtype=_lib.DT_I32), 2, "dtype"),
        (dict(d=0), 2, "head_dim"),
        (dict(d=257), 2, "head_dim"),
        (dict(d=14), 1, "pairs"),
        (dict(h=0), 1, "sizes"),
        (dict(b=-1), 1, "sizes"),
        (dict(b=1 << 16, s=1 << 16), 2, "2^31"),
        (dict(b=1, s=2**31 - 1), 2, "2^31"),  # a warp's rows would pass 32 bits
        (dict(x=heads(data=None)), 1, "NULL"),
        (dict(x=heads(data=A16 + 1)), 1, "aligned"),
        (dict(out=heads(data=None)), 1, "NULL"),
        (dict(rot=rotary(axes=0)), 1, "axes"),
        (dict(rot=rotary(axes=5)), 1, "axes"),
        (dict(rot=rotary(sections=(4, 0))), 1, "axis 1"),
        (dict(rot=rotary(prefix=5)), 1, "prefix"),
        (dict(rot=rotary(prefix=-1)), 1, "prefix"),
        (dict(rot=rotary(freqs=None)), 1, "freqs"),
        (dict(rot=rotary(freqs=A16 + 4)), 1, "freqs"),
        (dict(rot=rotary(coords=None)), 1, "coords"),
        (dict(rot=rotary(coords_dtype=_lib.DT_U8)), 2, "coords"),
    ],
)
def test_rotary_refusals(kw, code, word):
    refused(turn(**kw), code, word)


def test_rotary_null_table_and_empty_calls():
    refused(_lib.lib().sb_axes_rotary(heads(), 1, None, 0, 1, 2, 4, 64, heads(), None), 1, "NULL")
    assert turn(b=0) == 0 and turn(s=0) == 0


def qk(backward=False, dtype=1, wd=0, eps=1e-6, rot=None, b=1, hq=2, hk=2, s=4, d=64, ws=A16, need=1 << 30, qw=A16):
    h = heads()
    lib = _lib.lib()
    if backward:
        return lib.sb_qk_norm_rotary_backward(h, h, h, h, dtype, qw, A16, wd, eps, rot, b, hq, hk, s, d, h, h, A16, A16, ws,
                                              need, None)
    return lib.sb_qk_norm_rotary(h, h, dtype, qw, A16, wd, eps, rot, b, hq, hk, s, d, h, h, None)


@pytest.mark.parametrize(
    "kw,code,word",
    [
        (dict(dtype=3), 2, "dtype"),
        (dict(wd=4), 2, "weight"),
        (dict(qw=A16 + 2), 1, "weight"),
        (dict(eps=-1.0), 1, "eps"),
        (dict(eps=float("nan")), 1, "eps"),
        (dict(hk=-1), 1, "key heads"),
        (dict(d=300), 2, "head_dim"),
        (dict(rot=rotary(axes=7)), 1, "axes"),
        (dict(backward=True, ws=None), 4, "workspace"),
        (dict(backward=True, ws=A16 + 8), 4, "workspace"),
        (dict(backward=True, need=16), 4, "workspace"),
    ],
)
def test_qk_norm_refusals(kw, code, word):
    refused(qk(**kw), code, word)


def means(k=None, dtype=1, b=1, h=2, s=100, d=64, block=64, out=A16, lens=None):
    return _lib.lib().sb_block_means(k or heads(), dtype, lens, b, h, s, d, block, out, None)


def select(dtype=1, b=1, hq=4, hk=2, sq=8, sk=1000, d=64, block=64, topk=4, first=1, own=1, m=A16, index=A16):
    return _lib.lib().sb_block_select(heads(), dtype, m, None, None, b, hq, hk, sq, sk, d, block, topk, first, own, index,
                                      None)


@pytest.mark.parametrize(
    "call,code,word",
    [
        (lambda: means(dtype=4), 2, "dtype"),
        (lambda: means(block=0), 1, "sizes"),
        (lambda: means(s=2**31 - 1), 2, "2^31"),
        (lambda: means(s=9, block=2**31 - 1), 2, "2^31"),
        (lambda: select(sk=2**31 - 9, block=2**30), 2, "2^31"),
        (lambda: means(d=300), 2, "head_dim"),
        (lambda: means(out=None), 1, "means"),
        (lambda: means(lens=A16 + 1), 1, "misaligned"),
        (lambda: means(k=heads(data=None)), 1, "NULL"),
        (lambda: select(dtype=5), 2, "dtype"),
        (lambda: select(hq=3), 1, "key heads"),
        (lambda: select(topk=0), 2, "topk"),
        (lambda: select(topk=65), 2, "topk"),
        (lambda: select(topk=1), 1, "forced"),
        (lambda: select(first=-1), 1, "forced"),
        (lambda: select(sk=64 * 16384 + 1), 2, "blocks"),
        (lambda: select(m=None), 1, "means"),
        (lambda: select(index=None), 1, "index"),
        (lambda: select(index=A16 + 2), 1, "misaligned"),
        (lambda: select(d=0), 2, "head_dim"),
    ],
)
def test_selection_refusals(call, code, word):
    refused(call(), code, word)


def attend(backward=False, q=None, dtype=1, b=1, hq=4, hk=2, sq=100, sk=1000, d=64, block=64, topk=4, scale=0.1, ws=A16,
           need=1 << 40, index=A16, out=None):
    lib, h = _lib.lib(), heads()
    if backward:
        return lib.sb_block_attention_backward(h, q or h, h, h, out or h, A16, dtype, index, None, None, b, hq, hk, sq, sk, d,
                                               block, topk, scale, h, h, h, ws, need, None)
    return lib.sb_block_attention(q or h, h, h, dtype, index, None, None, b, hq, hk, sq, sk, d, block, topk, scale, out or h,
                                  A16, ws, need, None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize(
    "kw,code,word",
    [
        (dict(dtype=0), 2, "dtype"),
        (dict(hq=5), 1, "key heads"),
        (dict(hq=4096, hk=2), 2, "heads"),
        (dict(d=4), 2, "head_dim"),
        (dict(d=136), 2, "head_dim"),
        (dict(d=20), 2, "head_dim"),
        (dict(block=16), 2, "block"),
        (dict(sk=2**31 - 1), 2, "key rows"),
        (dict(sq=2**26 + 1), 2, "rows"),
        (dict(topk=0), 2, "topk"),
        (dict(topk=65), 2, "topk"),
        (dict(scale=float("inf")), 1, "scale"),
        (dict(q=heads(data=A16 + 8)), 1, "16-byte"),
        (dict(q=heads(s=12)), 1, "multiples of 8"),
        (dict(out=heads(data=None)), 1, "NULL"),
        (dict(index=None), 1, "index"),
        (dict(index=A16 + 1), 1, "misaligned"),
        (dict(ws=None), 4, "workspace"),
        (dict(ws=A16 + 16), 4, "workspace"),
        (dict(need=100), 4, "workspace"),
    ],
)
def test_attention_refusals(backward, kw, code, word):
    refused(attend(backward, **kw), code, word)


def test_attention_workspace_sizes():
    lib, n = _lib.lib(), C.c_size_t(7)
    assert lib.sb_block_attention_workspace_bytes(2, 4, 2, 1, 1000, 64, 64, 8, 0, n) == 0 and n.value == 0
    assert lib.sb_block_attention_workspace_bytes(0, 4, 2, 99, 1000, 64, 64, 8, 0, n) == 0 and n.value == 0
    assert lib.sb_block_attention_workspace_bytes(2, 4, 2, 999, 1000, 64, 64, 8, 0, n) == 0 and n.value > 0
    refused(lib.sb_block_attention_workspace_bytes(2, 4, 2, 9, 9, 64, 64, 8, 0, None), 1, "NULL")
    refused(lib.sb_block_attention_workspace_bytes(2, 4, 2, 9, 9, 64, 48, 8, 0, n), 2, "block")
    refused(lib.sb_qk_norm_rotary_backward_workspace_bytes(0, n), 1, "bad")


def test_python_calls_need_cuda_tensors():
    x = torch.zeros(1, 2, 4, 16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.axes_rotary(x, torch.zeros(1, 4, 2, dtype=torch.int16), ops.rotary_freqs((4, 4), device="cpu"), (4, 4))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.qk_norm_rotary(x, x, None, None)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.block_means(x, 64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.block_select(x, x, 4, 64, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.block_attention(x, x, x, torch.zeros(1, 2, 4, 1, dtype=torch.int32), 64)
    with pytest.raises(ValueError, match="batch, heads, rows"):
        ops.block_means(x[0], 64)


def test_rotary_freqs():
    f = ops.rotary_freqs((2, 3), theta=100.0, device="cpu")
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 1.0, 100 ** (-1 / 3), 100 ** (-2 / 3)], dtype=torch.float64))


def test_oracle_attention_gradients_are_autograds():
    torch.manual_seed(3)
    q = torch.randn(2, 4, 9, 8, dtype=torch.float64, requires_grad=True)
    k, v = (torch.randn(2, 2, 70, 8, dtype=torch.float64, requires_grad=True) for _ in range(2))
    index = torch.randint(-1, 4, (2, 2, 9, 3), dtype=torch.int32)
    lens = torch.tensor([70, 40])
    g = torch.randn(2, 4, 9, 8, dtype=torch.float64)
    seen = O.seen_keys(index, 70, 32, lens).repeat_interleave(2, 1)
    s = (q @ k.repeat_interleave(2, 1).transpose(-1, -2)) / 8**0.5
    p = torch.softmax(torch.where(seen, s, -1e300), -1) * seen
    out = p @ v.repeat_interleave(2, 1)
    want = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), g)))
    found, _ = O.attention(q, k, v, index, 32, None, lens, None, g)
    want["out"] = out
    for name, w in want.items():
        assert torch.allclose(found[name], w, atol=1e-12), name


def test_oracle_rotation_turns_back():
    torch.manual_seed(4)
    x = torch.randn(2, 3, 6, 12, dtype=torch.float64)
    ang = O.angles(torch.randint(-9, 9, (2, 4, 2)), ops.rotary_freqs((2, 3), device="cpu"), (2, 3), 6)
    for adjacent in (False, True):
        y = O.rotate(x, ang, adjacent)
        assert torch.allclose(O.rotate(y, -ang, adjacent), x, atol=1e-12)
        assert torch.equal(y[:, :, :2], x[:, :, :2]) and torch.equal(y[..., 10:], x[..., 10:])
