"""The weight-only NVFP4 product against 64-bit sums of the exactly decoded weights.

Bound per element: the final rounding (2^-8 of the value, bf16), fp32 sums of
exact products (K/16 + 64 dependent additions of 2^-24 each, relative to the
sum of magnitudes), the power-of-two fp16 form of the activations (2^-38 of
the row's largest magnitude times the sum of the weights' magnitudes) and one
fp32 rounding for alpha and the bias each.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import nvfp4
from vflash_b200 import _lib
from vflash_b200.kernels import KernelInputError, attention, nvfp4_quantize, nvfp4_weight_only
from vflash_b200.native.h3_attention import PackedAttention
from vflash_b200.native.h3_nvfp4_linear import NVFP4Execution, NVFP4Weight

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def weight_of(n, k, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn(n, k, generator=gen, device=DEV) * 0.02).to(BF16)
    scale = (448.0 * 6.0 / w.float().abs().max()).reshape(())
    packed, sf = nvfp4_quantize(w, scale)
    return NVFP4Weight(packed, sf.reshape(n, k // 16), (1.0 / scale).reshape(()), torch.ones((), device=DEV))


def decoded(weight):
    n, k = weight.out_features, weight.in_features
    w = nvfp4.dequantize(weight.packed.cpu().numpy(), weight.scales.cpu().numpy().reshape(-1), n, k)
    return torch.from_numpy(w).to(DEV)


def activations(rows, k, seed, dtype, gain=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, k, generator=gen, device=DEV) * gain
    x[torch.rand(rows, k, generator=gen, device=DEV) < 0.002] *= 20
    return x.to(dtype)


def check(got, x, weight, bias):
    w, xd, alpha = decoded(weight), x.double(), weight.alpha.double()
    want = alpha * (xd @ w.T)
    size = alpha * (xd.abs() @ w.abs().T)
    if bias is not None:
        want = want + bias.double()
        size = size + bias.double().abs()
    k = x.shape[1]
    bound = (2.0**-8 * want.abs() + (k / 16 + 64 + 4) * 2.0**-24 * size
             + 2.0**-38 * alpha * xd.abs().amax(dim=1, keepdim=True) * w.abs().sum(dim=1) + 1e-38)
    error = (got.double() - want).abs()
    assert got.dtype == BF16 and got.shape == want.shape
    assert (error <= bound).all(), f"{(error / bound).max().item():.2f} times the bound"
    assert _lib.device_status(clear=True) == _lib.VFB_OK


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 3, 7, 8, 9, 16, 17, 31, 33, 70])
@pytest.mark.parametrize("n,k", [(128, 64), (256, 192), (384, 1024), (128, 4160), (1152, 512)])
def test_against_the_decoded_weight(rows, n, k, dtype, with_bias):
    weight = weight_of(n, k, n + k)
    x = activations(rows, k, rows, dtype)
    bias = activations(1, n, 5, BF16)[0] if with_bias else None
    check(nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha, bias), x, weight, bias)


@pytest.mark.parametrize("n,k", [(4096, 4096), (12288, 4096), (4096, 16384), (5376, 14336)])
@pytest.mark.parametrize("rows", [1, 5])
def test_model_sizes(n, k, rows):
    weight = weight_of(n, k, 3)
    x = activations(rows, k, 4, BF16)
    check(nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha), x, weight, None)


@pytest.mark.parametrize("n,rows,k", [(128, 9, 8384), (128, 17, 4416), (128, 18, 8768), (128, 32, 16384),
                                      (128, 32, 16448), (128, 8, 32768), (256, 33, 32768), (4096, 20, 16384), (8192, 10, 7488),
                                      (16384, 4, 18880), (16384, 3, 25280)])
def test_rows_that_fill_shared_memory(n, rows, k):
    """x takes most of a block's shared memory, or its K is dealt out so that it fits."""
    weight = weight_of(n, k, 4)
    x = activations(rows, k, 6, BF16)
    check(nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha), x, weight, None)


def test_every_code_and_scale_decodes_exactly():
    """One activation of 1 per row of x: the output is that weight times alpha, exact in bf16."""
    n, k = 128, 256
    rng = np.random.default_rng(0)
    codes = rng.integers(0, 16, (n, k), dtype=np.uint8)
    scales = rng.permutation(np.arange(n * k // 16) % 127).astype(np.uint8)  # every finite e4m3 >= 0
    flat = np.zeros(n * (k // 16), dtype=np.uint8)
    flat[nvfp4.sf_offsets(n, k // 16).reshape(-1)] = scales
    weight = NVFP4Weight(torch.from_numpy(nvfp4.pack(codes)).to(DEV), torch.from_numpy(flat.reshape(n, -1)).to(DEV),
                         torch.tensor(0.5, device=DEV), torch.ones((), device=DEV))
    w = decoded(weight)
    for dtype in (BF16, FP16):
        x = torch.eye(k, dtype=dtype, device=DEV)
        got = nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha)
        assert torch.equal(got.double(), 0.5 * w.T)


def test_whole_numbers_are_exact():
    n, k = 256, 2048
    rng = np.random.default_rng(1)
    codes = rng.integers(0, 16, (n, k), dtype=np.uint8)
    weight = NVFP4Weight(torch.from_numpy(nvfp4.pack(codes)).to(DEV),
                         torch.full((n, k // 16), 0x40, dtype=torch.uint8, device=DEV),  # e4m3 2.0: whole weights
                         torch.ones((), device=DEV), torch.ones((), device=DEV))
    x = torch.randint(-8, 9, (5, k), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(BF16)
    got = nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha)
    assert torch.equal(got, (x.double() @ decoded(weight).T).to(BF16))


@pytest.mark.parametrize("gain", [1e-30, 1e-6, 1e6, 1e30])
def test_activation_ranges(gain):
    weight = weight_of(256, 512, 8)
    x = activations(4, 512, 9, BF16, gain)
    x[1] *= 1e-3  # rows of very different sizes
    x[2] = 0
    check(nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha), x, weight, None)


def test_activations_that_are_not_finite():
    weight = weight_of(256, 512, 8)
    x = activations(4, 512, 9, BF16)
    want = nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha)
    x[1, 77] = float("nan")
    x[2, 300] = float("inf")
    got = nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha)
    assert torch.equal(got[[0, 3]], want[[0, 3]])
    assert torch.isnan(got[1]).all()
    column = decoded(weight)[:, 300]
    assert torch.equal(torch.isnan(got[2]), column == 0)  # inf * 0
    assert torch.equal(got[2][column > 0] == torch.inf, torch.ones_like(column[column > 0], dtype=torch.bool))
    assert torch.equal(got[2][column < 0] == -torch.inf, torch.ones_like(column[column < 0], dtype=torch.bool))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_strides_and_alignment(dtype):
    weight = weight_of(384, 320, 2)
    wide = activations(9, 331, 3, dtype)
    out = torch.full((9, 400), 7.0, dtype=BF16, device=DEV)
    for shift in (0, 1, 3, 8):  # rows that start on any element
        x = wide[:, shift:shift + 320]
        got = nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha, out=out[:, shift:shift + 384])
        check(got, x, weight, None)
        assert torch.equal(got, nvfp4_weight_only(x.contiguous(), weight.packed, weight.scales, weight.alpha))
    assert (out[:, 8 + 384:] == 7.0).all()


def test_expanded_rows():
    weight = weight_of(128, 192, 2)
    x = activations(1, 192, 3, BF16)
    got = nvfp4_weight_only(x.expand(5, 192), weight.packed, weight.scales, weight.alpha)
    want = nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha)
    assert torch.equal(got, want.expand(5, 128))


def test_execution_keeps_leading_dimensions_and_rounds_fp32_first():
    weight = weight_of(128, 192, 2)
    x = activations(6, 192, 3, torch.float32).reshape(2, 3, 192)
    engine = NVFP4Execution()
    got = engine.weight_only_linear(x, weight)
    assert got.shape == (2, 3, 128) and engine.calls == 1 and engine.rows == 6
    check(got.reshape(6, 128), x.reshape(6, 192).to(BF16), weight, None)


def test_graph_replay_and_the_same_bits_on_two_streams():
    weight = weight_of(1024, 2048, 2)
    x = activations(3, 2048, 3, BF16)
    run = lambda: nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha)  # noqa: E731
    want = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    graph.replay()
    assert torch.equal(got, want)
    x.copy_(activations(3, 2048, 30, BF16))
    graph.replay()
    check(got, x, weight, None)
    want = run()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        outs = []
        for stream in streams:
            with torch.cuda.stream(stream):
                outs.append(run())
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_single_token_step():
    """The operators as a serving step uses them: weight-only QKV, attention over cached keys, weight-only output."""
    heads, kv, dim, hidden, batch, slot = 8, 2, 64, 512, 3, 300
    qkv, out = weight_of((heads + 2 * kv) * dim, hidden, 1), weight_of(hidden, heads * dim, 2)
    engine = NVFP4Execution()
    x = activations(batch, hidden, 3, BF16)
    lengths = [299, 1, 130]
    k_cache = activations(batch * slot, kv * dim, 4, BF16).reshape(-1, kv, dim)
    v_cache = activations(batch * slot, kv * dim, 5, BF16).reshape(-1, kv, dim)
    cu_q = torch.arange(batch + 1, dtype=torch.int32, device=DEV)
    used = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    rows = torch.arange(batch, device=DEV) * slot + used.long() - 1

    def step():
        planes = engine.weight_only_linear(x, qkv)
        q, k, v = planes.split([heads * dim, kv * dim, kv * dim], dim=-1)
        k_cache[rows] = k.reshape(batch, kv, dim)
        v_cache[rows] = v.reshape(batch, kv, dim)
        y = PackedAttention(heads, kv, causal=True)(q, k_cache.reshape(-1, kv * dim), v_cache.reshape(-1, kv * dim),
                                                    cu_q, cu_q * slot, lengths_k=used)
        return q, y, engine.weight_only_linear(y, out)

    q, y, z = step()
    check(z, y, out, None)
    want = attention(q.reshape(batch, heads, dim), k_cache, v_cache, cu_q, cu_q * slot, lengths_k=used)
    assert torch.equal(y.reshape(batch, heads, dim), want)
    for b, n in enumerate(lengths):
        keys = k_cache[b * slot:b * slot + n].double()
        values = v_cache[b * slot:b * slot + n].double()
        for h in range(heads):
            p = torch.softmax(keys[:, h // 4] @ q[b, h * dim:(h + 1) * dim].double() * dim**-0.5, dim=0)
            ref, size = p @ values[:, h // 4], p @ values[:, h // 4].abs()
            # one rounding of the output and one of every probability, and 2^-12 for all that is kept in fp32
            bound = 2.0**-8 * ref.abs() + (2.0**-8 + 2.0**-12) * size
            assert ((y[b, h * dim:(h + 1) * dim].double() - ref).abs() <= bound).all()


def test_an_out_over_the_activations_is_refused():
    weight = weight_of(128, 128, 2)
    both = activations(9, 256, 3, BF16)
    x, beside = both[:, :128], both[:, 128:]
    want = nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha)
    for out in (x, both[:, 64:192]):
        with pytest.raises(KernelInputError, match="overlap"):
            nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha, out=out)
    assert torch.equal(nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha, out=beside), want)


def without_column(weight, column):
    """The weight with zeros in one input column."""
    weight.packed[:, column // 2] &= 0xF0 if column % 2 == 0 else 0x0F
    return weight


def check_without_loss(got, x, weight):
    """``check`` without its term for what fp16 loses of small activations."""
    w, xd, alpha = decoded(weight), x.double(), weight.alpha.double()
    want, size = alpha * (xd @ w.T), alpha * (xd.abs() @ w.abs().T)
    bound = 2.0**-8 * want.abs() + (x.shape[1] / 16 + 68) * 2.0**-24 * size + 1e-38
    error = (got.double() - want).abs()
    assert (error <= bound).all(), f"{(error / bound).max().item():.2f} times the bound"
    assert _lib.device_status(clear=True) == _lib.VFB_OK


@pytest.mark.parametrize("rows", [1, 3, 8, 9, 20, 33])
@pytest.mark.parametrize("n,k,column,shift", [(128, 64, 5, 0), (256, 192, 190, 0), (384, 1024, 700, 0), (384, 1024, 1, 3),
                                              (4096, 4096, 4095, 0), (128, 16384, 9000, 0), (256, 32768, 0, 0),
                                              (16384, 512, 77, 0)])
def test_an_outlier_on_a_weight_of_zero_takes_nothing_from_the_others(rows, n, k, column, shift):
    """Only some blocks of a K that is dealt out hold the outlier; the bits are those without it."""
    weight = without_column(weight_of(n, k, 5), column)
    x = torch.zeros(rows, k + 8, dtype=BF16, device=DEV)[:, shift:shift + k]  # rows off 16 bytes where shifted
    x.copy_(activations(rows, k, 6, BF16))
    x[:, column] = 0
    want = nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha)
    check_without_loss(want, x, weight)
    for big in (1e30, -3e38, 1e9):
        x[rows // 2, column] = big
        got = nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha)
        check_without_loss(got, x, weight)
        assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [2, 12, 32])
@pytest.mark.parametrize("below", [16, 28, 29, 30, 31, 32, 33, 40, 80, 120, 150])
def test_activations_far_below_their_row_s_largest(rows, below):
    weight = without_column(weight_of(256, 384, 5), 100)
    x = activations(rows, 384, 6, BF16)
    x = torch.where(x == 0, 1, x) * 2.0**(40 - below)
    x[:, 100] = 2.0**45
    x[0, 7] = 0
    check_without_loss(nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha), x, weight)


def test_subnormal_and_largest_activations():
    weight = without_column(weight_of(128, 256, 5), 3)
    x = activations(4, 256, 6, BF16)
    x[0] = (x[0].float() * 2.0**-128).to(BF16)  # subnormal ones alone
    x[1] = (x[1].float() * 2.0**-100).to(BF16)  # far below the largest, normal
    x[1:3, 3] = 1e6
    x[2, 9] = 2.0**-60
    x[3] = (x[3].float().clamp(-4, 4) * 2.0**100).to(BF16)
    got = nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha)
    check_without_loss(got, x, weight)


@pytest.mark.parametrize("rows,n,k", [(1, 4096, 4096), (3, 256, 512), (8, 128, 16384), (9, 384, 1024), (32, 256, 4096)])
@pytest.mark.parametrize("outlier", [0.0, 2e4])
def test_activations_behind_a_gelu(rows, n, k, outlier):
    """A row's long tail towards zero, with and without an outlier on a weight of zero."""
    weight = without_column(weight_of(n, k, 5), 40)
    x = torch.nn.functional.gelu(3 * activations(rows, k, 6, torch.float32), approximate="tanh").to(BF16)
    x[:, 40] = outlier
    check_without_loss(nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha), x, weight)


@pytest.mark.parametrize("rows,n,k", [(1, 4096, 4096), (8, 128, 16384), (32, 256, 4096)])
@pytest.mark.parametrize("outlier", [0.0, 2e4])
def test_activations_over_many_orders(rows, n, k, outlier):
    """Evenly spread from 2^-43 to 1 on a logarithmic scale: enough large ones that what fp16 leaves of the small
    ones is nothing beside their sums, unless there is an outlier on a weight of zero."""
    weight = without_column(weight_of(n, k, 5), 40)
    gen = torch.Generator(device=DEV).manual_seed(7)
    x = torch.exp(-30 * torch.rand(rows, k, generator=gen, device=DEV))
    x = (x * torch.where(torch.rand(rows, k, generator=gen, device=DEV) < 0.5, -1, 1)).to(BF16)
    x[:, 40] = outlier
    check_without_loss(nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha), x, weight)


@pytest.mark.parametrize("rows", [1, 8, 20])
@pytest.mark.parametrize("k,outliers", [(64, 5), (64, 15), (512, 60), (4096, 300)])
def test_many_outliers_of_several_sizes(rows, k, outliers):
    """Up to a quarter of a row may be large numbers on weights of zero."""
    weight = weight_of(2048, k, 5)
    x = activations(rows, k, 6, BF16)
    gen = torch.Generator().manual_seed(8)
    for i, column in enumerate(torch.randperm(k, generator=gen)[:outliers].tolist()):
        without_column(weight, column)
        x[:, column] = (1e30, -2e30, 1e20, 4e29)[i % 4]
    check_without_loss(nvfp4_weight_only(x, weight.packed, weight.scales, weight.alpha), x, weight)
