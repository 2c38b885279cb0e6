"""Long-support attention operators on the GPU at the edges of their range: how
little the results lose, values of every size, sizes past one window. Against
64-bit forms, with bounds derived beside them."""

from __future__ import annotations

import pytest
import torch

from hexo_bot_b200 import attention_ops as ops
from oracle import attention_ops as O
from test_gpu_attention_ops import BF16, DEV, F16, gen, randn, within

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
