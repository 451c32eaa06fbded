"""Attention over packed sequences against the 64-bit definition, per element within its derived bound."""

from __future__ import annotations

import ctypes

import pytest
import torch

from oracle.attention import reference
from vflash_b200 import _lib
from vflash_b200.kernels import KernelInputError, attention
from vflash_b200.native.h3_attention import PackedAttention

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16 = torch.bfloat16, torch.float16


def offsets(lengths, slot=0):
    at = [0]
    for n in lengths:
        at.append(at[-1] + (slot or n))
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def normal(shape, seed, dtype, gain=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=DEV) * gain).to(dtype)


def operands(lengths_q, lengths_k, heads, kv_heads, dim, dtype, slot=0, seed=0):
    total_k = slot * len(lengths_k) if slot else sum(lengths_k)
    return (normal((sum(lengths_q), heads, dim), seed, dtype, 1.5), normal((total_k, kv_heads, dim), seed + 1, dtype),
            normal((total_k, kv_heads, dim), seed + 2, dtype))


def check(got, lse, q, k, v, lengths_q, lengths_k, causal, slot=0, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out, want_lse, bound, lse_bound = reference(q, k, v, lengths_q, lengths_k, causal=causal, scale=scale, slot=slot)
    error = (got.double() - out).abs()
    assert torch.isfinite(got.float()).all()
    worst = (error / bound.clamp_min(1e-30)).max().item() if error.numel() else 0.0
    assert (error <= bound).all(), f"output error {worst:.2f} times its bound"
    if lse is not None:
        empty = want_lse == -torch.inf
        assert torch.equal(lse == -torch.inf, empty)
        assert ((lse.double() - want_lse).abs()[~empty] <= lse_bound[~empty]).all()
    assert _lib.device_status(clear=True) == _lib.VFB_OK


LENGTHS = [
    ([1], [1]),
    ([1], [2]),
    ([2], [2]),
    ([17], [17]),
    ([127], [127]),
    ([128], [128]),
    ([129], [129]),
    ([255, 256, 257], [255, 256, 257]),
    ([600], [600]),
    ([5, 0, 300, 1, 64], [5, 0, 300, 1, 64]),
    ([1, 1, 1, 1], [1, 700, 128, 129]),
    ([3, 130, 1], [400, 131, 1025]),
    ([4, 2], [0, 9]),
    ([40, 300], [7, 130]),
    ([1], [5000]),
    ([64], [3000]),
    ([300], [4000]),
    ([700, 20], [5000, 3100]),
    ([2500], [2500]),
    ([5, 1, 0, 2], [9000, 3, 40, 6000]),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [
    (2, 2, 128, BF16), (8, 2, 128, BF16), (4, 1, 64, FP16), (3, 1, 80, BF16), (7, 1, 128, FP16), (6, 3, 96, FP16),
    (2, 1, 8, BF16), (1, 1, 72, BF16), (24, 1, 64, BF16)])
@pytest.mark.parametrize("lengths_q,lengths_k", LENGTHS)
def test_against_the_definition(lengths_q, lengths_k, heads, kv_heads, dim, dtype, causal):
    q, k, v = operands(lengths_q, lengths_k, heads, kv_heads, dim, dtype)
    got, lse = attention(q, k, v, offsets(lengths_q), offsets(lengths_k), causal=causal, return_lse=True)
    assert got.shape == q.shape and got.dtype == dtype and lse.shape == (heads, q.shape[0])
    check(got, lse, q, k, v, lengths_q, lengths_k, causal)


@pytest.mark.parametrize("heads,kv_heads", [(130, 1), (256, 2), (200, 1)])
def test_groups_wider_than_a_tile(heads, kv_heads):
    q, k, v = operands([3, 70], [9, 200], heads, kv_heads, 64, BF16)
    got, lse = attention(q, k, v, offsets([3, 70]), offsets([9, 200]), causal=True, return_lse=True)
    check(got, lse, q, k, v, [3, 70], [9, 200], True)


def test_without_offsets_all_rows_are_one_sequence():
    q, k, v = operands([300], [300], 4, 2, 128, BF16)
    got = attention(q, k, v, causal=True)
    assert torch.equal(got, attention(q, k, v, offsets([300]), causal=True))
    check(got, None, q, k, v, [300], [300], True)


def test_many_sequences_of_every_length():
    gen = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 90, (700,), generator=gen).tolist()
    q, k, v = operands(lengths, lengths, 4, 2, 64, BF16)
    got, lse = attention(q, k, v, offsets(lengths), causal=True, return_lse=True)
    check(got, lse, q, k, v, lengths, lengths, True)


@pytest.mark.parametrize("peak", [1.0, 30.0])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_scores_that_grow_along_the_keys(dtype, peak):
    """The running maximum moves in every tile, by little (held back) and by much (rescaled)."""
    q, k, v = operands([200], [1500], 2, 1, 64, dtype)
    k = (k.float() * torch.linspace(0.05, peak, 1500, device=DEV)[:, None, None]).to(dtype)
    got, lse = attention(q, k, v, offsets([200]), offsets([1500]), return_lse=True)
    check(got, lse, q, k, v, [200], [1500], False)
    k = k.flip(0).contiguous()
    got, lse = attention(q, k, v, offsets([200]), offsets([1500]), return_lse=True)
    check(got, lse, q, k, v, [200], [1500], False)


@pytest.mark.parametrize("scale", [1e-3, 0.5, 3.0])
def test_scale(scale):
    q, k, v = operands([150], [333], 2, 2, 64, BF16)
    got, lse = attention(q, k, v, offsets([150]), offsets([333]), scale=scale, return_lse=True)
    check(got, lse, q, k, v, [150], [333], False, scale=scale)


@pytest.mark.parametrize("lengths", [[1, 33, 0, 256, 700, 64], [700] * 6])
@pytest.mark.parametrize("nq", [1, 2, 20])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (4, 4)])
def test_cache_slots(lengths, nq, heads, kv_heads):
    slot = 700
    lengths_q = [nq] * len(lengths)
    q, k, v = operands(lengths_q, lengths, heads, kv_heads, 128, BF16, slot=slot)
    for b, n in enumerate(lengths):  # what lies behind a slot's length is never used
        k[b * slot + n:(b + 1) * slot] = float("nan")
        v[b * slot + n:(b + 1) * slot] = float("inf")
    used = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got, lse = attention(q, k, v, offsets(lengths_q), offsets(lengths, slot), lengths_k=used, causal=True,
                         return_lse=True)
    check(got, lse, q, k, v, lengths_q, lengths, True, slot=slot)
    # lengths beyond the slot are those of the slot; negative ones are none
    used = torch.tensor([10**6, -5] + lengths[2:], dtype=torch.int32, device=DEV)
    got = attention(q, k, v, offsets(lengths_q), offsets(lengths, slot), lengths_k=used, causal=True)
    full = torch.tensor([slot, 0] + lengths[2:], dtype=torch.int32, device=DEV)
    want = attention(q, k, v, offsets(lengths_q), offsets(lengths, slot), lengths_k=full, causal=True)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("nq,heads,kv_heads,lengths,slot", [
    (1, 8, 2, [1, 5000, 0, 9000, 64, 3000], 9000), (20, 8, 2, [20, 5000, 0, 9000], 9000), (200, 8, 8, [200, 6000, 131], 6000),
    (1, 16, 2, [30000], 32768)])
def test_long_cache_slots(nq, heads, kv_heads, lengths, slot):
    """Slots whose keys are shared out over the blocks, much of them unused."""
    lengths_q = [nq] * len(lengths)
    q, k, v = operands(lengths_q, lengths, heads, kv_heads, 128, BF16, slot=slot)
    used = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got, lse = attention(q, k, v, offsets(lengths_q), offsets(lengths, slot), lengths_k=used, causal=True,
                         return_lse=True)
    check(got, lse, q, k, v, lengths_q, lengths, True, slot=slot)


def test_head_groups_whose_keys_do_not_fit_together():
    """A causal sequence so long that its jobs go a few head groups at a time, more of them than blocks."""
    q, k, v = operands([1500], [20000], 24, 12, 128, BF16)
    got, lse = attention(q, k, v, offsets([1500]), offsets([20000]), causal=True, return_lse=True)
    check(got, lse, q, k, v, [1500], [20000], True)


def test_few_sequences_with_rows_among_many_without():
    """Far more blocks are launched than there are jobs."""
    lengths = [0] * 3000
    lengths[17], lengths[2990] = 400, 2700
    q, k, v = operands(lengths, lengths, 4, 2, 64, BF16)
    got, lse = attention(q, k, v, offsets(lengths), causal=True, return_lse=True)
    check(got, lse, q, k, v, lengths, lengths, True)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim", [64, 128])
def test_hidden_keys_never_reach_a_row(bad, dim):
    lengths = [70, 200, 131]
    q, k, v = operands(lengths, lengths, 4, 2, dim, BF16)
    want = attention(q, k, v, offsets(lengths), causal=True)
    k2, v2 = k.clone(), v.clone()
    last = 70 + 200  # the last key of the second sequence: only its last row sees it
    k2[last - 1, 0, 3] = bad
    v2[last - 1, :, 5] = bad
    got = attention(q, k2, v2, offsets(lengths), causal=True)
    keep = torch.ones(sum(lengths), dtype=torch.bool, device=DEV)
    keep[last - 1] = False
    assert torch.equal(got[keep], want[keep])
    # a value alone that a row does see: its column is not finite, its others are as before
    v3 = v.clone()
    v3[70 + 128, 1, 7] = bad
    got = attention(q, k, v3, offsets(lengths), causal=True)
    column = got[70 + 128:last, 2:, 7].float()
    assert (column != column).all() if bad != bad else (column == bad).all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[70 + 128:last, 2:, 7] = False
    assert torch.equal(got[keep], want[keep])


def test_a_row_whose_scores_are_not_finite_is_not_finite():
    q, k, v = operands([300], [300], 2, 2, 64, BF16)
    for bad in (float("nan"), float("inf")):
        for column in (0, 7, 31, 64, 100, 127, 130, 299):
            k2 = k.clone()
            k2[column, 0] = bad
            q2 = q.clone()
            q2[:, 0] = q2[:, 0].abs() + 0.5  # inf keys: every score of the column is +inf
            got = attention(q2, k2, v)
            assert torch.isnan(got[:, 0].float()).all(), (bad, column)
            assert torch.isfinite(got[:, 1].float()).all()


def test_rows_behind_the_last_sequence():
    lengths = [33, 90]
    q, k, v = operands([33, 90, 60], [33, 90, 60], 4, 2, 64, BF16)
    q[123:] = float("nan")
    got, lse = attention(q, k, v, offsets(lengths), causal=True, return_lse=True)
    assert (got[123:] == 0).all() and (lse[:, 123:] == -torch.inf).all()
    check(got[:123], lse[:, :123], q[:123], k, v, lengths, lengths, True)
    mine = torch.full_like(q, 7.0)
    back = attention(q, k, v, offsets(lengths), causal=True, out=mine)
    assert back is mine and (mine[123:] == 7.0).all() and torch.equal(mine[:123], got[:123])


def test_strided_operands():
    lengths = [100, 261]
    rows, heads, kv, dim = sum(lengths), 4, 2, 64
    merged = normal((rows, (heads + 2 * kv) * dim + 8), 5, BF16)
    q = merged[:, :heads * dim].unflatten(1, (heads, dim))
    k = merged[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim))
    v = normal((kv, rows, dim), 6, BF16).transpose(0, 1)  # head-major
    out = torch.zeros(heads, rows, dim, dtype=BF16, device=DEV).transpose(0, 1)
    attention(q, k, v, offsets(lengths), causal=True, out=out)
    check(out, None, q, k, v, lengths, lengths, True)
    assert torch.equal(out, attention(q.contiguous(), k.contiguous(), v.contiguous(), offsets(lengths), causal=True))


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements: the last slot lies behind that offset."""
    kv, dim, slot, slots = 8, 128, 65536, 34
    k = torch.empty(slot * slots, kv, dim, dtype=BF16, device=DEV)
    v = torch.empty_like(k)
    assert k.numel() > 2**31
    n = 777
    k[-slot:-slot + n] = normal((n, kv, dim), 1, BF16)
    v[-slot:-slot + n] = normal((n, kv, dim), 2, BF16)
    q = normal((2, 16, dim), 3, BF16)
    cu_k = offsets([0] * slots, slot)
    lengths = torch.zeros(slots, dtype=torch.int32, device=DEV)
    lengths[-1] = n
    cu_q = torch.zeros(slots + 1, dtype=torch.int32, device=DEV)
    cu_q[-1] = 2
    got = attention(q, k, v, cu_q, cu_k, lengths_k=lengths, causal=True)
    check(got, None, q, k[-slot:-slot + n], v[-slot:-slot + n], [2], [n], True)


def test_bad_offsets_stay_inside_the_buffers():
    """Offsets that decrease or leave the buffers give some result without leaving them."""
    q, k, v = operands([200], [200], 2, 2, 64, BF16)
    for at in ([0, 500], [0, -7, 200], [0, 150, 20, 190], [5, 5, 5]):
        cu = torch.tensor(at, dtype=torch.int32, device=DEV)
        attention(q, k, v, cu, causal=True)
    torch.cuda.synchronize()
    assert _lib.device_status(clear=True) == _lib.VFB_OK


@pytest.mark.parametrize("lengths_q,lengths_k", [([600, 1, 90], [600, 1, 90]), ([1, 1, 3], [4000, 1, 2500])])
def test_graph_replay_follows_its_inputs(lengths_q, lengths_k):
    q, k, v = operands(lengths_q, lengths_k, 8, 2, 128, BF16)
    cu_q, cu_k = offsets(lengths_q), offsets(lengths_k)
    attention(q, k, v, cu_q, cu_k, causal=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, lse = attention(q, k, v, cu_q, cu_k, causal=True, return_lse=True)
    for seed, (nq, nk) in enumerate([(lengths_q, lengths_k), (lengths_q[::-1], lengths_k[::-1])]):
        for t, fresh in zip((q, k, v), operands(nq, nk, 8, 2, 128, BF16, seed=10 * seed)):
            t.copy_(fresh)
        cu_q.copy_(offsets(nq))
        cu_k.copy_(offsets(nk))
        graph.replay()
        check(got, lse, q, k, v, nq, nk, True)


def test_two_streams_at_once_and_the_same_bits_again():
    cases = []
    for seed, (nq, nk) in enumerate([([1, 1], [6000, 20]), ([900, 3], [900, 3])]):
        q, k, v = operands(nq, nk, 8, 2, 128, BF16, seed=seed)
        cases.append((q, k, v, offsets(nq), offsets(nk)))
    want = [attention(*c, causal=True) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        got = []
        for stream, c in zip(streams, cases):
            with torch.cuda.stream(stream):
                got.append(attention(*c, causal=True))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rows_and_no_keys():
    q, k, v = operands([5], [5], 2, 1, 64, BF16)
    out, lse = attention(q[:0], k[:0], v[:0], return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (2, 0)
    out, lse = attention(q, k[:0], v[:0], offsets([5]), offsets([0]), return_lse=True)
    assert (out == 0).all() and (lse == -torch.inf).all()


def test_planes_of_a_block():
    """PackedAttention on [rows, 1, heads * dim] planes, as the QKV projection returns them."""
    lengths = [100, 29]
    planes = normal((3, 129, 1, 4 * 128), 9, BF16)
    cu = offsets(lengths)
    got = PackedAttention(heads=4)(planes[0], planes[1], planes[2], cu)
    assert got.shape == planes[0].shape
    q, k, v = (planes[i].reshape(129, 4, 128) for i in range(3))
    check(got.reshape(129, 4, 128), None, q, k, v, lengths, lengths, False)
    out = torch.empty_like(planes[0])
    assert PackedAttention(heads=4)(planes[0], planes[1], planes[2], cu, out=out) is out
    assert torch.equal(out, got)


def test_block_stack_with_attention():
    """A streamed and a captured stack run attention between their linears, on samples packed into one call."""
    from tests.helpers import fp8_weight, outlier_activations
    from vflash_b200.native.h3_block_stack import FP8BlockStack, block_shapes
    from vflash_b200.native.h3_fp8_linear import RowFP8Execution
    from vflash_b200.native.h3_parallel import FP8Weight

    hidden, ffn = 256, 1024
    blocks = []
    for b in range(3):
        parts = {name: fp8_weight(n, k, 10 * b + j) for j, (name, n, k) in enumerate(block_shapes(hidden, ffn))}
        blocks.append({name: FP8Weight(c.to(DEV), s.to(DEV)) for name, (c, s) in parts.items()})
    x = outlier_activations(300, hidden, 5).to(DEV).reshape(300, 1, hidden)
    gate = torch.full((1, hidden), 1 / 32, dtype=BF16, device=DEV)
    cu = offsets([170, 130])
    attend = PackedAttention(heads=4)
    execution = RowFP8Execution("w8a8")
    want = x
    for w in blocks:
        planes = execution.qkv_linear(want, w["qkv"].codes, w["qkv"].row_scale)
        y = attention(*(p.reshape(300, 4, 64) for p in planes), cu).reshape(x.shape)
        want = execution.gate_residual_linear(y, w["attention_out"].codes, w["attention_out"].row_scale, want, gate)
        want = execution.ffn(want, w["ffn_in"].codes, w["ffn_in"].row_scale, w["ffn_out"].codes,
                             w["ffn_out"].row_scale, activation="gelu_tanh", residual=want, gate=gate)
    streamed = FP8BlockStack(blocks, hidden, ffn, DEV, chunk_bytes=1 << 20)
    assert torch.equal(streamed.forward(x, gate, attention=attend, cu_seqlens=cu), want)
    resident = FP8BlockStack(blocks, hidden, ffn, DEV, resident=True, chunk_bytes=1 << 20)
    replay = resident.capture(x, gate, attention=attend, cu_seqlens=cu)
    assert torch.equal(replay(), want)
    assert not torch.equal(streamed.forward(x, gate), want)


@pytest.mark.parametrize("at_peak", [1.0, 0.0])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("nq,nk", [(1, 131072), (3, 1000), (300, 700)])
def test_many_keys_far_below_the_peak_count(nq, nk, dtype, at_peak):
    """One key carries the maximum, all others 18 nats less: below what fp16 holds of the largest, but many."""
    q = torch.zeros(nq, 2, 64, dtype=dtype, device=DEV)
    q[..., 0] = 1
    k = torch.zeros(nk, 1, 64, dtype=dtype, device=DEV)
    k[1:, :, 0] = -18
    v = torch.ones(nk, 1, 64, dtype=dtype, device=DEV)
    v[0] = at_peak
    got, lse = attention(q, k, v, offsets([nq]), offsets([nk]), scale=1.0, return_lse=True)
    check(got, lse, q, k, v, [nq], [nk], False, scale=1.0)


def workspace_bytes(q, k, batch, causal, slots=False):
    """What the call reserves for pieces of jobs: 0 where it runs whole jobs."""
    rows, heads, dim = q.shape
    kv = k.shape[1]
    at = q.data_ptr()
    args = _lib.attention_args(
        at, k.data_ptr(), k.data_ptr(), at + q.numel() * 2, 0, heads * dim, dim, kv * dim, dim, kv * dim, dim, heads * dim, dim, rows,
        k.shape[0], heads, kv, dim, 0 if q.dtype == BF16 else 1, at, at, at if slots else 0, batch, causal, 1.0, 0, 0, 0)
    need = _lib.load().vfb_attention_workspace_bytes(ctypes.byref(args))
    assert need >= 0
    return need


CUT = [(1, 9000, 2, 1, 64, True), (3, 9001, 8, 2, 128, True), (40, 9000, 4, 4, 128, True), (300, 4001, 2, 1, 128, True),
       (300, 4001, 4, 4, 64, True), (3, 500, 8, 2, 128, False), (300, 700, 4, 4, 64, False)]  # the last ones are whole


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("nq,nk,heads,kv_heads,dim,cut", CUT)
def test_values_that_are_not_finite_where_the_keys_have_no_weight(nq, nk, heads, kv_heads, dim, cut, bad):
    """Seen keys whose exponentials vanish beside the others' still bring their NaN and infinities (0 * inf)."""
    q, k, v = operands([nq], [nk], heads, kv_heads, dim, BF16)
    assert (workspace_bytes(q, k, 1, False) > 0) == cut
    q[..., 0], k[..., 0] = 1, 0
    low = nk // 3
    k[:low, :, 0] = -1000  # at scale 1: far more than 126 binary orders below, in pieces of their own when cut
    run = lambda values: attention(q, k, values, offsets([nq]), offsets([nk]), scale=1.0, return_lse=True)  # noqa: E731
    want, want_lse = run(v)
    check(want, want_lse, q, k, v, [nq], [nk], False, scale=1.0)
    v[7, 0, 5] = bad
    v[low - 1, 0, 6] = bad
    got, lse = run(v)
    assert not torch.isfinite(got[:, :heads // kv_heads, 5:7].float()).any()
    got[:, :heads // kv_heads, 5:7] = want[:, :heads // kv_heads, 5:7]
    assert torch.equal(got, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("nq,nk,heads,kv_heads,dim,cut", CUT)
def test_values_that_are_not_finite_at_the_end_of_a_job(nq, nk, heads, kv_heads, dim, cut, bad):
    """Keys that only later rows see: taken out of the tile for the others, added back for those that see them."""
    q, k, v = operands([nq], [nk], heads, kv_heads, dim, BF16)
    assert (workspace_bytes(q, k, 1, True) > 0) == cut
    run = lambda values: attention(q, k, values, offsets([nq]), offsets([nk]), causal=True, return_lse=True)  # noqa: E731
    want, want_lse = run(v)
    check(want, want_lse, q, k, v, [nq], [nk], True)
    first = nq // 2  # the row from which on this key is seen
    v[nk - nq + first, 0, 5] = bad
    got, lse = run(v)
    column = got[first:, :heads // kv_heads, 5].float()
    assert (column != column).all() if bad != bad else (column == bad).all()
    got[first:, :heads // kv_heads, 5] = want[first:, :heads // kv_heads, 5]
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    # a key that is not finite: every row that sees it is NaN, the others are as they were
    k[nk - nq + first, 0, 3] = float("nan")
    got, _ = run(torch.where(torch.isfinite(v), v, 0))
    assert torch.isnan(got[first:, :heads // kv_heads].float()).all()
    assert torch.equal(got[:first, :, 6:], want[:first, :, 6:])


@pytest.mark.parametrize("nq,nk,heads,kv_heads,dim,cut", CUT)
def test_scores_of_minus_infinity(nq, nk, heads, kv_heads, dim, cut):
    """Keys with scores of -inf have no weight; a row that sees nothing else is 0 / 0, whether its job is cut or not."""
    q, k, v = operands([nq], [nk], heads, kv_heads, dim, BF16)
    assert (workspace_bytes(q, k, 1, False) > 0) == cut
    q[..., 0] = 1
    low = nk // 3 + 1
    k[:low, :, 0] = float("-inf")
    got, lse = attention(q, k, v, offsets([nq]), offsets([nk]), return_lse=True)
    check(got, lse, q, k[low:], v[low:], [nq], [nk - low], False)
    k[..., 0] = float("-inf")
    got, lse = attention(q, k, v, offsets([nq]), offsets([nk]), return_lse=True)
    assert torch.isnan(got.float()).all() and (lse == -torch.inf).all()


def test_an_out_over_its_operands_is_refused_and_columns_of_one_buffer_are_not():
    rows, heads, dim = 300, 4, 64
    merged = normal((rows + 1, 4, heads, dim), 3, BF16)
    q, k, v, free = (merged[:rows, i] for i in range(4))
    want = attention(q, k, v, causal=True)
    with pytest.raises(KernelInputError, match="overlap"):
        attention(q, k, v, causal=True, out=merged[1:, 0])
    with pytest.raises(KernelInputError, match="overlap"):
        attention(q, k, v, causal=True, out=merged[:rows, 2, :, :])
    assert attention(q, k, v, causal=True, out=free) is free
    assert torch.equal(free, want)


def test_a_hundred_thousand_prompts_of_one_token():
    """One key each: every row is its own value, exactly."""
    n = 100_000
    q, k, v = operands([n], [n], 4, 2, 64, BF16)
    cu = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    got, lse = attention(q, k, v, cu, causal=True, return_lse=True)
    assert torch.equal(got, v.repeat_interleave(2, dim=1))
    products = q.double() * k.double().repeat_interleave(2, dim=1) * 64**-0.5
    want, size = products.sum(dim=2).T, products.abs().sum(dim=2).T
    # 64 products summed and scaled in fp32, and four roundings (twice ln 2, its inverse, the logarithm of 1) of the result
    assert ((lse.double() - want).abs() <= (68 * size + 4 * want.abs()) * 2.0**-24 + 1e-7).all()
    assert _lib.device_status(clear=True) == _lib.VFB_OK


@pytest.mark.parametrize("keys", [0, 20000])
def test_rows_at_both_ends_of_the_largest_batch(keys):
    """2^24 - 1 sequences, all but the first and the last empty: passed over 32 at a time, and one by one by a share."""
    batch = 2**24 - 1
    nq, nk = [3, 2], [3 + keys, 2 + keys]
    q, k, v = operands(nq, nk, 4, 2, 64, BF16)
    cu_q = torch.full((batch + 1,), nq[0], dtype=torch.int32, device=DEV)
    cu_k = torch.full((batch + 1,), nk[0], dtype=torch.int32, device=DEV)
    cu_q[0] = cu_k[0] = 0
    cu_q[-1], cu_k[-1] = sum(nq), sum(nk)
    got, lse = attention(q, k, v, cu_q, cu_k, causal=True, return_lse=True)
    check(got, lse, q, k, v, nq, nk, True)


def test_a_job_longer_than_the_limit_of_a_wait():
    """600 million keys in every job: the warps that wait for a job's end wait longer than for a tile."""
    nq, nk = 146 * 256, 600_000_000
    k = torch.zeros(nk, 1, 8, dtype=BF16, device=DEV)
    k[nk // 2, 0, 0] = 40  # all the weight: the others have e^-40 each
    q = torch.zeros(nq, 1, 8, dtype=BF16, device=DEV)
    q[..., 0] = 1
    cu_q = offsets([nq])
    assert workspace_bytes(q, k, 1, False) == 0
    out = torch.zeros_like(q)
    attention(q, k, k, cu_q, offsets([nk]), scale=1.0, out=out)
    assert _lib.device_status(clear=True) == _lib.VFB_OK
    assert torch.equal(out, 40 * q)


@pytest.mark.parametrize("rows,keys,heads,cut", [(200, 200, 2, False), (700, 700, 24, False), (3, 9000, 4, True), (300, 4001, 4, True)])
@pytest.mark.parametrize("fill_tail", [0, 1])
def test_bad_offsets_write_nothing_beside_the_outputs(rows, keys, heads, cut, fill_tail):
    """Offsets and lengths that decrease, repeat or leave the buffers: what lies around out, lse and the workspace stays."""
    dim, guard = 64, 300
    q, k, v = operands([rows], [keys], heads, heads, dim, BF16)
    lists = [[0, 500_000], [0, -7, rows], [0, rows - 1, 1, rows], [5, 5, 5], [2**31 - 1, -(2**31), 2**31 - 1, 0], [rows, 0],
             [-1, rows + 1, rows, 0, rows]]
    for at in lists:
        for keys_at in (at, [x * keys // rows if abs(x) < 2**20 else x for x in at], [0] * len(at), [keys] * len(at)):
            for lengths in (None, [2**31 - 1] * (len(at) - 1), [-5] * (len(at) - 1), [1] * (len(at) - 1)):
                out = torch.full((rows + 2 * guard, heads, dim), 7.0, dtype=BF16, device=DEV)
                lse = torch.full((heads * rows + 2 * guard,), 7.0, device=DEV)
                cu_q, cu_k = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (at, keys_at))
                used = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
                args = _lib.attention_args(
                    q.data_ptr(), k.data_ptr(), v.data_ptr(), out[guard:].data_ptr(), lse[guard:].data_ptr(),
                    *(heads * dim, dim) * 4, rows, keys, heads, heads, dim, 0, cu_q.data_ptr(), cu_k.data_ptr(),
                    0 if used is None else used.data_ptr(), len(at) - 1, 1, 0.125, fill_tail, 0, 0)
                need = _lib.load().vfb_attention_workspace_bytes(ctypes.byref(args))
                if len(at) == 2 and lengths is None:
                    assert (need > 0) == cut
                workspace = torch.full((need + 512,), 99, dtype=torch.uint8, device=DEV)
                if need:
                    args.workspace, args.workspace_bytes = workspace[256:].data_ptr(), need
                _lib.check(_lib.load().vfb_attention(ctypes.byref(args), _lib.stream_handle(q.device)), "vfb_attention")
                assert (out[:guard] == 7).all() and (out[guard + rows:] == 7).all()
                assert (lse[:guard] == 7).all() and (lse[guard + heads * rows:] == 7).all()
                assert (workspace[:256] == 99).all() and (workspace[256 + need:] == 99).all()
                assert _lib.device_status(clear=True) == _lib.VFB_OK


def test_a_captured_stack_keeps_what_it_reads():
    """Inputs that only the graph still needs (the offsets of a packed batch, the gate, the weights) stay as they were."""
    import gc
    import weakref

    from tests.helpers import fp8_weight
    from vflash_b200.native.h3_block_stack import FP8BlockStack, block_shapes
    from vflash_b200.native.h3_parallel import FP8Weight

    hidden = 256
    parts = {name: fp8_weight(n, k, j) for j, (name, n, k) in enumerate(block_shapes(hidden, 1024))}
    blocks = [{name: FP8Weight(c.to(DEV), s.to(DEV)) for name, (c, s) in parts.items()}]
    x = normal((300, 1, hidden), 5, BF16)
    gate = torch.full((1, hidden), 1 / 32, dtype=BF16, device=DEV)
    cu = offsets([170, 130])
    attend = PackedAttention(heads=4)
    stack = FP8BlockStack(blocks, hidden, 1024, DEV, resident=True, chunk_bytes=1 << 20)
    want = stack.forward(x, gate, attention=attend, cu_seqlens=cu)
    replay = stack.capture(x, gate, attention=attend, cu_seqlens=cu)
    kept = [weakref.ref(t) for t in (x, gate, cu, stack)]
    del x, gate, cu, stack
    gc.collect()
    assert all(ref() is not None for ref in kept)
    others = [torch.full((n,), -1, dtype=torch.int32, device=DEV) for n in (3, 128, 300 * 128) for _ in range(50)]
    assert torch.equal(replay(), want)
    del others


def test_the_largest_number_of_keys():
    """2^31 - 1 keys and rows of both tiles of a job: key counts rounded up to tiles pass 31 bits."""
    nq, nk = 256, 2**31 - 1
    k = torch.zeros(nk, 1, 8, dtype=BF16, device=DEV)
    k[-1, 0, 0] = 40  # all the weight: the others have e^-40 each
    q = torch.zeros(nq, 1, 8, dtype=BF16, device=DEV)
    q[..., 0] = 1
    assert workspace_bytes(q, k, 1, False) > 0
    got, lse = attention(q, k, k, scale=1.0, return_lse=True)
    assert _lib.device_status(clear=True) == _lib.VFB_OK
    assert torch.equal(got, 40 * q)
    assert ((lse - 40).abs() <= 1e-4).all()  # 2^31 e^-40 is 9e-9


@pytest.mark.parametrize("dtype,size", [(FP16, 300.0), (FP16, 5000.0), (FP16, 60000.0), (BF16, 1e4), (BF16, 1e9), (BF16, 1e17)])
@pytest.mark.parametrize("nq,nk,heads,kv_heads,dim,cut", CUT)
def test_huge_scores_pick_the_largest(nq, nk, heads, kv_heads, dim, cut, dtype, size):
    """Scores far beyond 2^24 and far apart: every row is the value of its best key, and stays finite."""
    q, k, v = operands([nq], [nk], heads, kv_heads, dim, dtype)
    assert (workspace_bytes(q, k, 1, False) > 0) == cut
    q.zero_()
    k.zero_()
    gen = torch.Generator().manual_seed(4)
    sign = torch.where(torch.rand(nq, heads, generator=gen) < 0.5, -1.0, 1.0).to(DEV)
    q[..., 3] = (size * sign).to(dtype)
    # keys by their place: steps of a 64th of the size, so that neighbours are far apart in the scores too
    place = torch.randint(-64, 65, (nk, kv_heads), generator=gen).to(DEV)
    best, worst = nk // 3, nk - 2
    place[best], place[worst] = 65, -65
    k[..., 3] = (size * place / 66).to(dtype)
    got, lse = attention(q, k, v, offsets([nq]), offsets([nk]), scale=1.0, return_lse=True)
    wide = lambda row: v[row].repeat_interleave(heads // kv_heads, dim=0).expand(nq, heads, dim)  # noqa: E731
    want = torch.where(sign[..., None] > 0, wide(best), wide(worst))
    assert torch.equal(got, want)
    peak = torch.where(sign > 0, k[best, :, 3].repeat_interleave(heads // kv_heads).double(),
                       -k[worst, :, 3].repeat_interleave(heads // kv_heads).double()) * q[..., 3].abs().double()
    assert ((lse.double().T - peak).abs() <= 2.0**-22 * peak).all()  # the score and its way through log2 and back
    assert _lib.device_status(clear=True) == _lib.VFB_OK
