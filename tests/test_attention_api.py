"""Attention's argument checks: every refusal happens on the host, before any device is touched."""

from __future__ import annotations

import ctypes

import pytest
import torch

from vflash_b200 import _lib
from vflash_b200.kernels import KernelInputError, attention
from vflash_b200.native.h3_attention import PackedAttention
from vflash_b200.native.h3_block_stack import block_linears

BF16 = torch.bfloat16


def operands(dtype=BF16, rows=6, heads=4, kv=2, dim=64):
    return (torch.zeros(rows, heads, dim, dtype=dtype), torch.zeros(rows, kv, dim, dtype=dtype),
            torch.zeros(rows, kv, dim, dtype=dtype))


def cu(*at, dtype=torch.int32):
    return torch.tensor(at, dtype=dtype)


@pytest.mark.parametrize("change,match", [
    (lambda q, k, v: (q[0], k, v), "rows, heads, dim"),
    (lambda q, k, v: (q.float(), k, v), "all bf16 or all fp16"),
    (lambda q, k, v: (q, k.half(), v.half()), "all bf16 or all fp16"),
    (lambda q, k, v: (q, k, v[:5]), "one shape"),
    (lambda q, k, v: (q[:, :3], k, v), "divisible"),
    (lambda q, k, v: (q, k[:, :0], v[:, :0]), "divisible"),
    (lambda q, k, v: (q[..., :4], k[..., :4], v[..., :4]), "head dimension"),
    (lambda q, k, v: (q[..., :12].contiguous(), k[..., :12].contiguous(), v[..., :12].contiguous()),
     "head dimension"),
    (lambda q, k, v: (torch.zeros(6, 4, 136, dtype=BF16), torch.zeros(6, 2, 136, dtype=BF16),
                      torch.zeros(6, 2, 136, dtype=BF16)), "head dimension"),
    (lambda q, k, v: (q.transpose(1, 2).contiguous().transpose(1, 2), k, v), "unit stride"),
    (lambda q, k, v: (q, k[:, :1].expand(6, 2, 64), v), "strides must be multiples of 8"),
    (lambda q, k, v: (q, k, torch.zeros(6, 2 * 64 + 4, dtype=BF16)[:, :128].unflatten(1, (2, 64))), "strides must be multiples of 8"),
    (lambda q, k, v: (torch.zeros(6 * 4 * 64 + 1, dtype=BF16)[1:].view(6, 4, 64), k, v), "16-byte"),
    (lambda q, k, v: (q.requires_grad_(), k, v), "inference-only"),
])
def test_operand_refusals(change, match):
    with pytest.raises(KernelInputError, match=match):
        attention(*change(*operands()))


@pytest.mark.parametrize("kwargs,match", [
    (dict(cu_seqlens_q=cu(0, 6, dtype=torch.int64)), "int32"),
    (dict(cu_seqlens_q=cu(0)), "two entries"),
    (dict(cu_seqlens_q=cu(0, 3, 6)[::2]), "contiguous"),
    (dict(cu_seqlens_q=cu(0, 6), cu_seqlens_k=cu(0, 3, 6)), "2 entries"),
    (dict(cu_seqlens_k=cu(0, 6)), "needs cu_seqlens_q"),
    (dict(cu_seqlens_q=cu(0, 6), lengths_k=cu(1, 2)), "1 entries"),
    (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(scale=3e38), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(out=torch.zeros(6, 4, 32, dtype=BF16)), "out"),
    (dict(out=torch.zeros(6, 4, 64, dtype=torch.float16)), "out"),
])
def test_option_refusals(kwargs, match):
    with pytest.raises(KernelInputError, match=match):
        attention(*operands(), **kwargs)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_out_may_not_be_an_operand(which):
    planes = [torch.zeros(6, 4, 64, dtype=BF16) for _ in range(3)]
    with pytest.raises(KernelInputError, match="overlap"):
        attention(*planes, out=planes[which])


def test_other_key_count_needs_offsets():
    q, _, _ = operands()
    _, k, v = operands(rows=9)
    with pytest.raises(KernelInputError, match="cu_seqlens_k"):
        attention(q, k, v, cu(0, 6))


def test_host_tensors_are_refused_and_empty_ones_answered():
    with pytest.raises(KernelInputError, match="SM100"):
        attention(*operands())
    q, k, v = operands(rows=0)
    out, lse = attention(q, k, v, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)


def valid_args() -> _lib.AttentionArgs:
    a = _lib.AttentionArgs()
    for name in ("q", "k", "v", "out"):
        setattr(a, name, 256)
        setattr(a, name + "_token_stride", 256)
        setattr(a, name + "_head_stride", 64)
    a.total_q = a.total_k = 6
    a.heads, a.kv_heads, a.dim, a.batch, a.scale = 4, 2, 64, 1, 0.125
    return a


@pytest.mark.parametrize("field,value", [
    ("total_q", -1), ("total_k", 2**31), ("heads", 3), ("heads", 0), ("kv_heads", 0), ("dim", 4), ("dim", 60),
    ("dim", 136), ("dtype", 2), ("batch", 0), ("batch", 2), ("batch", 2**31 - 1), ("cu_seqlens_k", 256), ("scale", 0.0),
    ("scale", float("nan")), ("scale", 3e38), ("scale", float("inf")), ("q_token_stride", 60), ("k_head_stride", 0),
    ("v_token_stride", 250), ("out_head_stride", -64)])
def test_c_entry_refuses(field, value):
    lib = _lib.load()
    a = valid_args()
    assert lib.vfb_attention_workspace_bytes(ctypes.byref(a)) >= 0
    setattr(a, field, value)
    assert lib.vfb_attention_workspace_bytes(ctypes.byref(a)) == -1
    assert lib.vfb_attention(ctypes.byref(a), None) == _lib.VFB_EINVAL
    assert "vfb_attention" in _lib.last_error()


@pytest.mark.parametrize("field,value", [("q", None), ("out", None), ("k", None), ("v", 264), ("q", 258)])
def test_c_entry_refuses_pointers(field, value):
    a = valid_args()
    setattr(a, field, value)
    assert _lib.load().vfb_attention(ctypes.byref(a), None) == _lib.VFB_EINVAL


def test_null_args():
    assert _lib.load().vfb_attention(None, None) == _lib.VFB_EINVAL
    assert _lib.load().vfb_attention_workspace_bytes(None) == -1


def test_struct_layout_matches_header():
    a = _lib.AttentionArgs
    assert ctypes.sizeof(a) == 8 * 15 + 4 * 4 + 8 * 3 + 4 * 4 + 8 * 2
    assert a.total_q.offset == 8 * 13 and a.heads.offset == 8 * 15 and a.workspace.offset == 8 * 15 + 16 + 24 + 16


def test_packed_attention_checks():
    with pytest.raises(ValueError, match="divisible"):
        PackedAttention(heads=4, kv_heads=3)
    with pytest.raises(ValueError, match="plane"):
        PackedAttention(heads=3)(torch.zeros(2, 64), torch.zeros(2, 64), torch.zeros(2, 64))
    with pytest.raises(ValueError, match="contiguous"):
        PackedAttention(heads=1)(*[torch.zeros(2, 64, dtype=BF16)] * 3, out=torch.zeros(64, 2, dtype=BF16).T)
    with pytest.raises(ValueError, match="cu_seqlens"):
        block_linears(None, {}, None, None, cu_seqlens=cu(0, 1))


def launch_refusal(**fields) -> str:
    """What vfb_attention answers for planes that lie apart but for ``fields``, and a workspace that is missing."""
    a = valid_args()
    for i, name in enumerate(("q", "k", "v", "out")):
        setattr(a, name, (i + 1) << 26)
    a.total_k, a.cu_seqlens_q, a.cu_seqlens_k = 20000, 256, 256
    for name, value in fields.items():
        setattr(a, name, value)
    lib = _lib.load()
    assert lib.vfb_attention_workspace_bytes(ctypes.byref(a)) > 0  # so the call is refused here or there, on any machine
    assert lib.vfb_attention(ctypes.byref(a), None) == _lib.VFB_EINVAL
    return _lib.last_error()


Q, K, V, OUT = ((i + 1) << 26 for i in range(4))
ROW = 2 * 256  # bytes of a packed row of 4 heads of 64


@pytest.mark.parametrize("fields", [
    dict(out=Q), dict(out=Q + ROW), dict(out=Q - ROW), dict(out=Q + 5 * ROW), dict(out=K + 16), dict(out=V - 5 * ROW), dict(out=V + 19999 * ROW),
    dict(out=Q + ROW // 2, q_token_stride=512, out_token_stride=512),  # half a row on, the other half in the next gap
    dict(q=1 << 16, out=(1 << 16) + 128, q_head_stride=128, out_head_stride=64, q_token_stride=512),
    dict(out=1 << 16, q=(1 << 16) + 6 * 128 - 16, q_token_stride=64, q_head_stride=6 * 64, out_token_stride=64,
         out_head_stride=6 * 64),
    dict(lse=Q), dict(lse=K + 19999 * ROW + ROW // 2 - 4), dict(lse=OUT + 100)])
def test_launch_refuses_overlap(fields):
    assert "overlap" in launch_refusal(**fields)


@pytest.mark.parametrize("fields", [
    {}, dict(out=Q + 6 * ROW), dict(out=Q - 6 * ROW), dict(out=V + 20000 * ROW), dict(lse=OUT + 6 * ROW),
    # columns of one buffer beside q's, k's and v's
    dict(q=Q, k=Q + ROW, v=Q + ROW + ROW // 2, out=Q + 2 * ROW,
         **{f"{n}_token_stride": 3 * 256 for n in ("q", "k", "v", "out")}),
    dict(q=Q + 2 * ROW, k=Q + ROW, v=Q + ROW + ROW // 2, out=Q,
         **{f"{n}_token_stride": 3 * 256 for n in ("q", "k", "v", "out")}),
    # behind q inside every head, and planes of heads in turn
    dict(out=Q + 128, q_head_stride=128, out_head_stride=128, q_token_stride=512, out_token_stride=512),
    dict(out=Q + 6 * 128, q_token_stride=64, out_token_stride=64, q_head_stride=2 * 6 * 64, out_head_stride=2 * 6 * 64),
    # one row: its stride says nothing
    dict(out=Q + ROW, total_q=1)])
def test_launch_accepts_tensors_that_lie_apart(fields):
    assert "workspace" in launch_refusal(**fields)


def test_batches_that_take_too_long_to_pass_over_are_refused():
    lib = _lib.load()
    a = valid_args()
    a.cu_seqlens_q, a.batch = 256, 2**24 - 1
    assert lib.vfb_attention_workspace_bytes(ctypes.byref(a)) >= 0
    a.batch = 2**24
    assert lib.vfb_attention_workspace_bytes(ctypes.byref(a)) == -1
    assert "2^24" in _lib.last_error()
    with pytest.raises(KernelInputError, match="2\\^24"):
        attention(*operands(), torch.zeros(2**24 + 1, dtype=torch.int32))
