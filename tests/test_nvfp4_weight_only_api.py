"""Argument checks of the weight-only NVFP4 product (CPU: nothing here reaches a device)."""

from __future__ import annotations

import pytest
import torch

from vflash_b200 import _lib
from vflash_b200.kernels import KernelInputError, nvfp4_weight_only
from vflash_b200.native import h3_nvfp4_linear as nv

BF16 = torch.bfloat16


def operands(rows=3, n=128, k=64):
    return dict(matrix=torch.zeros(rows, k, dtype=BF16), w_packed=torch.zeros(n, k // 2, dtype=torch.uint8),
                w_scales=torch.zeros(n, k // 16, dtype=torch.uint8), alpha=torch.ones(()))


@pytest.mark.parametrize("change,match", [
    (dict(matrix=torch.zeros(3, 64)), "bf16/fp16"),
    (dict(matrix=torch.zeros(64, dtype=BF16)), "M, K"),
    (dict(matrix=torch.zeros(64, 3, dtype=BF16).T), "unit column stride"),
    (dict(matrix=torch.zeros(3, 128, dtype=BF16)), "codes"),
    (dict(w_packed=torch.zeros(128, 32, dtype=torch.int8)), "codes"),
    (dict(w_packed=torch.zeros(32, 128, dtype=torch.uint8).T), "codes"),
    (dict(w_scales=torch.zeros(128, 3, dtype=torch.uint8)), "128x4"),
    (dict(alpha=torch.ones((), dtype=torch.float64)), "alpha"),
    (dict(alpha=torch.ones(2)), "alpha"),
    (dict(bias=torch.zeros(128)), "bias"),
    (dict(bias=torch.zeros(127, dtype=BF16)), "bias"),
    (dict(out=torch.zeros(3, 128)), "output"),
    (dict(out=torch.zeros(2, 128, dtype=BF16)), "output"),
    (dict(w_packed=torch.zeros(128 * 32 + 1, dtype=torch.uint8)[1:].view(128, 32)), "aligned"),
])
def test_refusals(change, match):
    with pytest.raises(KernelInputError, match=match):
        nvfp4_weight_only(**{**operands(), **change})


def test_sizes():
    for n, k in ((64, 64), (192, 64), (128, 32), (128, 96)):
        with pytest.raises(KernelInputError, match="K % 64"):
            nvfp4_weight_only(**operands(n=n, k=k))
    assert nvfp4_weight_only(**operands(rows=0)).shape == (0, 128)


def test_c_entry_refuses_before_any_launch():
    lib = _lib.load()
    good = [256, 0, 3, 64, 256, 256, 256, None, 128, 64, 256, 128, None]
    for index, value in ((1, 2), (2, -1), (3, 63), (8, 64), (9, 32), (9, 32832), (2, 524289), (11, 127), (0, None), (4, None), (4, 264),
                         (5, 258), (6, None), (10, None)):
        bad = list(good)
        bad[index] = value
        assert lib.vfb_nvfp4_weight_only(*bad) == _lib.VFB_EINVAL, index
        assert "vfb_nvfp4_weight_only" in _lib.last_error()


def test_execution_checks(monkeypatch):
    weight = nv.NVFP4Weight(torch.zeros(128, 32, dtype=torch.uint8), torch.zeros(128, 4, dtype=torch.uint8),
                            torch.tensor(2.0), torch.tensor(4.0))
    engine = nv.NVFP4Execution()
    with pytest.raises(ValueError, match="SM100"):
        engine.weight_only_linear(torch.zeros(1, 64, dtype=BF16), weight)
    with pytest.raises(ValueError, match="frozen"):
        engine.weight_only_linear(torch.zeros(1, 32, dtype=BF16), weight)
    with pytest.raises(ValueError, match="frozen"):
        engine.weight_only_linear(torch.zeros(1, 64, dtype=torch.float64), weight)
    with pytest.raises(ValueError, match="inference"):
        engine.weight_only_linear(torch.zeros(1, 64, requires_grad=True), weight)
    monkeypatch.setattr(nv, "_require_device", lambda _: None)
    with pytest.raises(ValueError, match="bias"):
        engine.weight_only_linear(torch.zeros(1, 64, dtype=BF16), weight, torch.zeros(128))
    with pytest.raises(ValueError, match="contiguous"):
        engine.weight_only_linear(torch.zeros(1, 64, dtype=BF16), weight, torch.zeros(256, dtype=BF16)[::2])
    with pytest.raises(ValueError, match="nonempty"):
        engine.weight_only_linear(torch.zeros(0, 64, dtype=BF16), weight)
    assert engine.calls == 0

    def product(matrix, packed, scales, alpha, bias, *, checked):
        assert checked
        assert matrix.dtype == BF16 and matrix.shape == (6, 64) and alpha is weight.alpha
        return torch.ones(6, 128, dtype=BF16)

    monkeypatch.setattr(nv, "nvfp4_weight_only", product)
    assert engine.weight_only_linear(torch.zeros(2, 3, 64), weight).shape == (2, 3, 128)
    assert engine.calls == 1 and engine.rows == 6


X, CODES, SF, ALPHA, BIAS, OUT = (i << 20 for i in range(1, 7))


@pytest.mark.parametrize("changed,refused", [
    ({}, False), ({10: X}, True), ({10: X + 2 * 64}, True), ({10: X - 2 * 128 * 3 + 2}, True), ({10: X - 2 * 128 * 3}, False),
    ({10: X + 2 * 64 * 3}, False), ({10: CODES + 100}, True), ({10: SF + 511}, True), ({10: ALPHA - 4}, True),
    ({10: BIAS + 254}, True), ({10: BIAS + 256}, False), ({7: None, 10: BIAS}, False),
    ({3: 192, 11: 192, 10: X + 2 * 64}, False), ({3: 192, 11: 192, 10: X + 2 * 62}, True),  # columns of one buffer
    ({3: 192, 11: 192, 10: X - 2 * 128}, False), ({3: 192, 11: 256, 10: X + 2 * 64}, True), ({2: 1, 10: X + 2 * 64}, False)])
def test_c_entry_refuses_an_out_over_its_operands(changed, refused):
    args = [X, 0, 3, 64, CODES, SF + 2, ALPHA, BIAS, 128, 64, OUT, 128, None]  # the scales' alignment is refused later
    for index, value in changed.items():
        args[index] = value
    assert _lib.load().vfb_nvfp4_weight_only(*args) == _lib.VFB_EINVAL
    assert ("overlap" if refused else "aligned") in _lib.last_error()
