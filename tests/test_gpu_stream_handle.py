"""The current stream's handle for every way of naming a device."""

from __future__ import annotations

import pytest
import torch

from vflash_b200 import _lib

pytestmark = pytest.mark.gpu


def test_names_of_a_device():
    names = [torch.device("cuda", 0), torch.device("cuda"), "cuda:0", "cuda", 0, None]
    assert [_lib.stream_handle(name) for name in names] == [torch.cuda.current_stream().cuda_stream] * len(names)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert [_lib.stream_handle(name) for name in names] == [side.cuda_stream] * len(names)
