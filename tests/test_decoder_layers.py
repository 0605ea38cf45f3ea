"""Weights, scales and caches of the 8-bit operators (``mlc.ops``) as a program builds them, without a GPU."""

from __future__ import annotations

import pytest
import torch

from mlc import ops

FULL = torch.float32


@pytest.mark.parametrize("default", (torch.float16, torch.bfloat16, torch.float64))
def test_types_do_not_depend_on_the_default(default):
    """A program that builds a decoder in half precision sets torch's default type."""
    w = torch.randn(200, 272, generator=torch.Generator().manual_seed(0), dtype=FULL) * 0.02
    linear = torch.nn.Linear(272, 200, dtype=FULL)
    codes, scales = ops.quantize_weight(w)
    layer = ops.ScaledLinear.from_linear(linear)
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = ops.quantize_weight(w)
        made = ops.ScaledLinear.from_linear(linear)
        empty = ops.ScaledLinear(272, 200, bias=True)
        cache = ops.KeyValueCache(2, 3, 128, 64)
    finally:
        torch.set_default_dtype(before)
    assert got[1].dtype == FULL and torch.equal(got[1], scales)
    assert torch.equal(got[0].view(torch.uint8), codes.view(torch.uint8))
    for name, x in layer.state_dict().items():
        y = made.state_dict()[name]
        assert x.dtype == y.dtype and torch.equal(x.view(torch.uint8), y.view(torch.uint8)), name
    assert empty.scales.dtype == empty.bias.dtype == FULL
    assert cache.key_scales.dtype == cache.value_scales.dtype == FULL


def test_scales_whose_offsets_pass_32_bits_together_are_refused():
    """A row's and a block's part of an offset are below 2^31 each, but not their sum."""
    from mlc.codegen import hip_decoder as plans
    from mlc.codegen.hip_operators import Operand

    e4m3 = torch.float8_e4m3fn
    b, by = Operand((512, 4096), (4096, 1), e4m3), Operand((4, 32), (32, 1), FULL)

    def plan(a, a_scales):
        return plans.plan_product(a, a_scales, b, by, None, torch.bfloat16)

    tile, _ = plans.choose_tile(600, 512, 32, torch.bfloat16)
    rows, part = max(tile[:2]), 3 << 29  # bytes, of 2^31
    a = Operand((600, 4096), (4096, 1), e4m3)
    assert plan(a, Operand((600, 32), (part // 4 // rows, 1), FULL)).launches
    assert plan(a, Operand((600, 32), (1, part // 4 // 32), FULL)).launches
    with pytest.raises(ops.OperatorError, match="too far apart"):
        plan(a, Operand((600, 32), (part // 4 // rows, part // 4 // 32), FULL))
    # rows that have two strides count from the first of all
    a = Operand((3, 200, 4096), (300 * 4096, 4096, 1), e4m3)
    assert plan(a, Operand((3, 200, 32), (part // 8, 32, 1), FULL)).launches
    with pytest.raises(ops.OperatorError, match="too far apart"):
        plan(a, Operand((3, 200, 32), (part // 8, 1, part // 4 // 32), FULL))
