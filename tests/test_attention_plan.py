"""The attention kernel's work order covers every job and key tile once, on the CPU (tests/attention_plan_check.cpp)."""

from __future__ import annotations

import random
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def case(rng: random.Random) -> str:
    split = rng.random() < 0.7
    blocks = rng.choice([1, 2, 3, 7, 148])
    groups = rng.choice([1, 2, 8, 32])
    tokens = rng.choice([1, 5, 32, 64, 128, 256])
    causal = int(rng.random() < 0.6)
    offsets = rng.random() < 0.85
    batch = rng.choice([1, 2, 5, 40, 90]) if offsets else 1
    if tokens < 32 and batch > 5:
        groups = 2
    top_q = rng.choice([1, 3, 300] if tokens < 32 else [1, 3, 300, 2000])
    top_k = rng.choice([0, 1, 128, 700, 20000])
    nq = [rng.randint(0, top_q) for _ in range(batch)]
    nk = [rng.randint(0, top_k) for _ in range(batch)]
    if rng.random() < 0.3:
        nk = list(nq)
    if rng.random() < 0.2:  # one long request among short ones
        nk[rng.randrange(batch)] = 60000
    cu_q, cu_k = [0], [0]
    for a, b in zip(nq, nk):
        cu_q.append(cu_q[-1] + a)
        cu_k.append(cu_k[-1] + b)
    total_q, total_k = cu_q[-1] + rng.choice([0, 0, 3, 500]), cu_k[-1] + rng.choice([0, 9])
    if offsets and rng.random() < 0.1:  # offsets that nobody may rely on
        rng.shuffle(cu_q)
        total_k = max(0, total_k - 50)
    used = [rng.choice([0, x, x // 2, x + 5]) for x in nk] if rng.random() < 0.4 else [-1] * batch
    per_tile = total_q // tokens + batch + 1 if offsets else -(-total_q // tokens)
    grid = max(1, min(total_q, per_tile) * groups if rng.random() < 0.3 else rng.choice([1, 1, 148]))
    band_keys = rng.choice([1, 700, 4000, 98304])
    return " ".join(map(str, [int(split), blocks, rng.choice([6, 7]), band_keys, rng.choice([0, 0, 0, 2, 9]), grid, groups, tokens, causal, int(offsets), batch, total_q, total_k,
                              *cu_q, *cu_k, *used]))


def test_every_key_tile_is_visited_once(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ is not installed")
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", f"-I{ROOT / 'vflash_b200' / 'csrc'}",
                    str(ROOT / "tests" / "attention_plan_check.cpp"), "-o", str(exe)], check=True)
    rng = random.Random(11)
    lines = "\n".join(case(rng) for _ in range(400))
    result = subprocess.run([str(exe)], input=lines, capture_output=True, text=True, timeout=300)
    assert result.returncode == 0, result.stdout
    word, cases, cuts = result.stdout.split()
    assert word == "ok" and int(cases) == 400 and int(cuts) > 300


def build(tmp_path, source: str) -> Path:
    if shutil.which("g++") is None:
        pytest.skip("g++ is not installed")
    exe = tmp_path / source
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", f"-I{ROOT / 'vflash_b200' / 'csrc'}",
                    str(ROOT / "tests" / f"{source}.cpp"), "-o", str(exe)], check=True)
    return exe


@pytest.mark.parametrize("n,blocks,groups,tokens,top", [(1, 3, 2, 64, 900), (300, 5, 3, 64, 300), (2000, 9, 2, 16, 40),
                                                        (300000, 4, 8, 32, 2)])
def test_blocks_go_on_where_they_last_were(tmp_path, n, blocks, groups, tokens, top):
    """The same jobs as by a search from the first sequence, and each block passes over the sequences once."""
    rng = random.Random(n)
    lengths = [rng.randint(0, top) for _ in range(n)]
    result = subprocess.run([str(build(tmp_path, "attention_cursor_check"))], capture_output=True, text=True, timeout=60,
                            input=" ".join(map(str, [n, blocks, groups, tokens, *lengths])))
    assert result.returncode == 0, result.stdout
    word, jobs, passed = result.stdout.split()
    assert word == "ok" and int(jobs) >= sum(x > 0 for x in lengths) * groups
    if n > 3000:
        assert int(passed) <= blocks * (n + 1)
