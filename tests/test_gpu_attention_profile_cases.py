"""The profiling cases of attention and the weight-only product run clean (small row counts)."""

from __future__ import annotations

import pytest

from vflash_b200 import profile_cases

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("argv", [
    ["attention", "--rows", "300", "--repeats", "1"],
    ["attention", "--rows", "300", "--repeats", "1", "--causal"],
    ["attention_cached", "--rows", "4096", "--repeats", "1"],
    ["weight_only", "--rows", "1", "--n", "256", "--repeats", "1"],
    ["weight_only", "--rows", "20", "--n", "256", "--repeats", "1"],
])
def test_profile_case_runs(argv):
    assert profile_cases.main(argv) == 0
