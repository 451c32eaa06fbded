"""Dense attention between a block's QKV projection and its output projection, on SM100.

The reference's block runs attention on the Q, K and V planes its merged
projection returns (src/vflash/native/h3_native_denoiser.py:543-550) with one
of several library backends.  ``PackedAttention`` does that step on the planes
of ``RowFP8Execution.qkv_linear`` / ``NVFP4Execution.qkv_linear`` as they are
(no copy, no head-major transpose), for one sample or for samples and prompts
of different lengths packed into one call.  It also serves prompts (causal),
pieces of prompts and single tokens that read earlier keys from a cache.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from ..kernels import attention


@dataclass(frozen=True)
class PackedAttention:
    """The head layout and mask of one block's attention.

    ``heads`` query heads share ``kv_heads`` key/value heads (default: as many),
    ``causal`` masks later keys, ``scale`` defaults to ``dim ** -0.5``.
    """

    heads: int
    kv_heads: int | None = None
    causal: bool = False
    scale: float | None = None

    def __post_init__(self):
        if self.heads < 1 or (self.kv_heads is not None and (self.kv_heads < 1 or self.heads % self.kv_heads)):
            raise ValueError("attention needs heads >= 1 divisible by kv_heads")

    def _split(self, plane: torch.Tensor, heads: int, name: str) -> torch.Tensor:
        if plane.ndim < 1 or plane.shape[-1] % heads:
            raise ValueError(f"attention {name} plane must be [..., heads * dim]")
        return plane.reshape(-1, heads, plane.shape[-1] // heads)

    def __call__(self, q, k, v, cu_seqlens_q=None, cu_seqlens_k=None, *, lengths_k=None, out=None):
        """Attention of the planes ``[..., heads * dim]`` (``kv_heads * dim`` for k and v).

        The leading dimensions are flattened to rows; the offsets and lengths
        are those of ``vflash_b200.kernels.attention``.  Returns a tensor of
        ``q``'s shape, ready for the attention output projection.
        """
        kv_heads = self.kv_heads or self.heads
        if out is not None and (out.shape != q.shape or not out.is_contiguous()):
            raise ValueError("attention out must be contiguous with q's shape")
        result = attention(self._split(q, self.heads, "q"), self._split(k, kv_heads, "k"),
                           self._split(v, kv_heads, "v"), cu_seqlens_q, cu_seqlens_k, lengths_k=lengths_k,
                           causal=self.causal, scale=self.scale,
                           out=None if out is None else self._split(out, self.heads, "out"))
        return result.reshape(q.shape) if out is None else out
