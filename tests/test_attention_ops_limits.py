"""What the long-support attention operators refuse or promise at the edges of
their use, without a GPU."""

from __future__ import annotations

import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

from hexo_bot_b200 import _lib
from hexo_bot_b200 import attention_ops as ops

X = torch.zeros(1, 2, 4, 16)
W = torch.ones(16)
COORDS = torch.zeros(1, 4, 1, dtype=torch.int32)
FREQS = ops.rotary_freqs((8,), device="cpu")
INDEX = torch.zeros(1, 2, 4, 1, dtype=torch.int32)

CALLS = {
    "axes_rotary": lambda x: ops.axes_rotary(x, COORDS, FREQS, (8,)),
    "qk_norm_rotary q": lambda x: ops.qk_norm_rotary(x, X, W, W, COORDS, FREQS, (8,)),
    "qk_norm_rotary k": lambda x: ops.qk_norm_rotary(X, x, W, W, COORDS, FREQS, (8,)),
    "qk_norm_rotary weight": lambda x: ops.qk_norm_rotary(X, X, None, x[0, 0, 0]),
    "qk_norm_rotary_backward": lambda x: ops.qk_norm_rotary_backward(X, x, X, X, W, W, COORDS, FREQS, (8,)),
    "block_attention q": lambda x: ops.block_attention(x, X, X, INDEX, 64),
    "block_attention v": lambda x: ops.block_attention(X, X, x, INDEX, 64),
    "block_attention_backward": lambda x: ops.block_attention_backward(x, X, X, X, X, X[..., 0], INDEX, 64),
}


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_tangents_are_refused(name):
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(1, 2, 4, 16), torch.ones(1, 2, 4, 16))
        with pytest.raises(RuntimeError, match="forward-mode"):
            CALLS[name](x)
        with pytest.raises(RuntimeError, match="no CPU fallback"):  # a level without tangents changes nothing
            CALLS[name](X)


@pytest.mark.parametrize("name", [*CALLS, "block_means", "block_select"])
def test_traces_are_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    calls = dict(CALLS, block_means=lambda x: ops.block_means(x, 64), block_select=lambda x: ops.block_select(x, X, 1, 64, 4))
    for trace in (lambda f: torch.jit.trace(f, (X,)), lambda f: make_fx(f)(X)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            trace(calls[name])


def workspace(backward, batch, q_heads, kv_heads, rows, dim, block, topk):
    need = C.c_size_t()
    rc = _lib.lib().sb_block_attention_workspace_bytes(batch, q_heads, kv_heads, rows, rows, dim, block, topk, backward, need)
    assert rc == 0, _lib.last_error()
    return need.value


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("batch", [1, 8])
@pytest.mark.parametrize("topk", [16, 64])
@pytest.mark.parametrize("rows", [2000, 32768, 131072, 1 << 20])
def test_workspace_of_long_calls(rows, topk, batch, backward):
    """At most 1 GB of parts, the lists of as many rows (entries and where a block's queries begin),
    8 bytes a row for flags, 8 for the backward, and its sums of dk and dv: those of one head in 32
    bits, or 400 MB for the segments of a window."""
    q_heads, kv_heads, dim, block = 32, 8, 128, 64
    bh = batch * kv_heads
    marks = min(bh * (rows // 256 + 1), 2**30 // (4 * topk * dim * 4) // 256 + bh)
    lists = marks * (2 * topk * 256 + 4 * (rows // block + 1)) + 8 * bh * rows
    sums = max(2 * (rows + block) * dim * 4, 400 << 20)
    most = (1 << 30) + lists + backward * (8 * batch * q_heads * rows + sums) + (1 << 20)
    assert workspace(backward, batch, q_heads, kv_heads, rows, dim, block, topk) <= most


def test_workspace_is_sized_on_the_tensors_device(monkeypatch):
    """The plan depends on the device's SMs: the size is asked for where the call will run."""
    current, asked = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Lib:
        def sb_block_attention_workspace_bytes(self, *args):
            asked.append(current[0])
            return 0

        def sb_block_attention(self, *args):
            return 0

        sb_block_attention_backward = sb_block_attention

    class OnGpu1(torch.Tensor):
        device = torch.device("cuda:1")
        is_cuda = True

    class Memory:
        def data_ptr(self):
            return 0

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(ops._lib, "lib", Lib)
    monkeypatch.setattr(torch, "empty", lambda *a, **k: Memory())
    monkeypatch.setattr(torch, "empty_like", lambda t: t)
    monkeypatch.setattr(ops, "_check", lambda t, *a: t)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0)
    x = torch.zeros(1, 1, 20, 16, dtype=torch.float16).as_subclass(OnGpu1)
    index = torch.zeros(1, 1, 20, 1, dtype=torch.int32)
    ops.block_attention(x, x, x, index, 64)
    ops.block_attention_backward(x, x, x, x, x, torch.zeros(1, 1, 20), index, 64)
    assert asked == [1, 1] and current == [0]


@pytest.mark.parametrize("which", ["coords", "freqs"])
def test_tables_that_need_a_gradient_are_refused(which):
    """Neither coordinates nor frequencies get one: a table that is still learned would stand still."""
    coords, freqs = torch.zeros(1, 4, 1), FREQS.clone()
    {"coords": coords, "freqs": freqs}[which].requires_grad_()
    for call in (lambda: ops.axes_rotary(X, coords, freqs, (8,)), lambda: ops.qk_norm_rotary(X, X, W, W, coords, freqs, (8,))):
        with pytest.raises(ValueError, match=f"{which} gets no gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
