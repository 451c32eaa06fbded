"""What the attention and weight-only NVFP4 operators are measured on.

Two operators that sit between the quantised linears of a transformer block:

* ``attention``: softmax attention over packed sequences (``cu_seqlens``),
  grouped heads, causal or full, from whole prompts down to single tokens that
  read a cache of earlier keys (``vflash_b200.kernels.attention``);
* ``weight_only``: the product of a few activation rows with a 4-bit NVFP4
  weight and its group scales, activations kept in 16 bits
  (``NVFP4Execution.weight_only_linear``).

``own`` selects between their plain form (elementary torch operations in
fp32, rounded once at the end) and the framework's calls.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _lengths(text: str) -> list[int]:
    return [int(part) for part in text.split(",")]


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def _attention(name, heads, kv_heads, dim, dtype, causal, queries, keys="", slot=0, lse=False):
    """``keys`` empty: the keys are the queries' own tokens; ``slot``: keys lie in cache slots of this many rows."""
    return {"name": name, "op": "attention", "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "causal": causal, "queries": queries, "keys": keys, "slot": slot, "lse": lse}


def _weight_only(name, rows, n, k, dtype, bias):
    return {"name": name, "op": "weight_only", "rows": rows, "n": n, "k": k, "dtype": dtype, "bias": bias}


_SHORT = ("113,7,300,1,64,65,128,129,31,250,18,96,77,3,211,40,5,290,133,59,1,12,199,84,"
          "256,27,101,9,160,47,222,70,2,275,33,118,66,15,181,90,6,240,52,145,23,108,19,299")
_CACHED = ("8192,5000,1,777,4096,63,2500,8191,129,6400,1024,300,7000,128,3333,64,"
           "5555,17,4097,900,8000,2048,450,6001,1500,33,7777,256,3800,2,512,7168")


def listed():
    return [
        # a diffusion block's self-attention over one sample of the benchmark's 32760 tokens
        _attention("block_full_32760", 32, 32, 128, "bf16", False, "32760"),
        # the wider block (inner width 7168): two samples of different sizes packed into one call
        _attention("block_packed_56_heads", 56, 56, 128, "bf16", False, "9997,6387"),
        # a text encoder's prompts of very different lengths, grouped heads; the row statistics are kept too
        _attention("prompt_ragged_grouped", 32, 8, 128, "bf16", True, "8192,4111,2500,1031,509,40,1", lse=True),
        # many short prompts with 64-wide heads in fp16
        _attention("prompt_short_fp16", 16, 2, 64, "fp16", True, _SHORT),
        # the smallest call: one prompt of 17 tokens, where latency is all
        _attention("prompt_17_tokens", 32, 8, 128, "bf16", True, "17"),
        # a prompt taken in pieces: 512 new tokens after 16384 cached ones
        _attention("prompt_piece_on_cache", 32, 8, 128, "bf16", True, "512", "16896"),
        # one new token for each of 32 requests whose caches hold 1 to 8192 tokens
        _attention("token_batch_cached", 32, 8, 128, "bf16", True, ",".join(["1"] * 32), _CACHED, slot=8192),
        # one new token of one request with a long cache
        _attention("token_long_cache", 32, 8, 128, "bf16", True, "1", "131072"),
        # one token through the merged QKV projection of the benchmark's block
        _weight_only("vector_qkv", 1, 12288, 4096, "bf16", True),
        # one token through its FFN output projection: few outputs, long sums
        _weight_only("vector_ffn_out", 1, 4096, 16384, "bf16", False),
        # seven rows through the wider block's packed FFN input
        _weight_only("rows_7_ffn_in", 7, 28672, 5376, "fp16", True),
        # a batch of 32 rows through the FFN input
        _weight_only("rows_32_ffn_in", 32, 16384, 4096, "bf16", False),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "piece", "token", "token", "vector", "vector"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "vector":
        return _unnamed(_weight_only("", _log_int(rng, 1, 32), 128 * _log_int(rng, 1, 224),
                                     64 * _log_int(rng, 1, 256), dtype, rng.random() < 0.5))
    heads, kv_heads = rng.choice([(32, 32), (56, 56), (32, 8), (16, 2), (12, 4), (7, 1), (40, 8), (6, 6), (24, 1)])
    dim = rng.choice([64, 80, 96, 128, 128, 128])
    if kind == "prompt":
        batch = _log_int(rng, 1, 40)
        top = _log_int(rng, 2, max(4, 12000 // batch))
        queries = ",".join(str(rng.randint(1, top)) for _ in range(batch))
        return _unnamed(_attention("", heads, kv_heads, dim, dtype, rng.random() < 0.6, queries,
                                   lse=rng.random() < 0.3))
    if kind == "piece":
        batch = rng.randint(1, 4)
        new = [_log_int(rng, 2, 900) for _ in range(batch)]
        old = [_log_int(rng, 1, 9000) for _ in range(batch)]
        return _unnamed(_attention("", heads, kv_heads, dim, dtype, rng.random() < 0.8,
                                   ",".join(map(str, new)), ",".join(str(a + b) for a, b in zip(new, old))))
    batch = _log_int(rng, 1, 64)
    slot = _log_int(rng, 16, max(32, 60000 // batch))
    keys = ",".join(str(rng.randint(1, slot)) for _ in range(batch))
    return _unnamed(_attention("", heads, kv_heads, dim, dtype, True, ",".join(["1"] * batch), keys, slot=slot))


def _unnamed(case):
    case = dict(case)
    del case["name"]
    return case


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _layout(case):
    """Lengths of queries and keys, first query row and first key row of every sequence, and the buffers' rows."""
    queries = _lengths(case["queries"])
    keys = _lengths(case["keys"]) if case["keys"] else list(queries)
    q_at = _offsets(queries)
    k_at = _offsets([case["slot"]] * len(keys) if case["slot"] else keys)
    return queries, keys, q_at, k_at


def _inputs(case, seed):
    """The data alone, the same whichever form runs on it."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "attention":
        queries, keys, q_at, k_at = _layout(case)

        def normal(rows, heads, gain=1.0):
            return (torch.randn(rows, heads, case["dim"], generator=gen, device=DEVICE) * gain).to(dtype)

        # normalised and rotated queries and keys have entries near 1; a gain on the queries makes some rows peaked
        q = normal(q_at[-1], case["heads"], 1.5)
        k = normal(k_at[-1], case["kv_heads"])
        v = normal(k_at[-1], case["kv_heads"])
        return {"q": q, "k": k, "v": v}
    rows, n, k = case["rows"], case["n"], case["k"]
    x = torch.randn(rows, k, generator=gen, device=DEVICE)
    # a few large entries, as activations after a norm and its weight have
    x = torch.where(torch.rand(rows, k, generator=gen, device=DEVICE) < 0.001, x * 20, x).to(dtype)
    w = torch.randn(n, k // 16, 16, generator=gen, device=DEVICE) * 0.02
    # NVFP4: one e4m3 scale for 16 weights, the matrix scale chosen so that the largest group scale is 448
    peak = w.abs().amax(dim=-1)
    global_scale = 448.0 * 6.0 / peak.max()
    scales = (peak * (global_scale / 6.0)).to(torch.float8_e4m3fn)
    unit = (scales.float() / global_scale).clamp_min(1e-30)
    levels = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEVICE)
    codes = torch.bucketize((w / unit[..., None]).abs(), levels).to(torch.uint8)
    codes |= (w < 0).to(torch.uint8) << 3
    codes = codes.reshape(n, k)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    bytes_ = scales.view(torch.uint8)  # [n, k / 16]
    tiled = bytes_.reshape(n // 128, 4, 32, k // 64, 4).permute(0, 3, 2, 1, 4).contiguous()
    bias = None
    if case["bias"]:
        bias = (torch.randn(n, generator=gen, device=DEVICE) * 0.1).to(torch.bfloat16)
    return {"x": x, "packed": packed.contiguous(), "scales": tiled.reshape(n, k // 16),
            "alpha": (1.0 / global_scale).reshape(()), "bias": bias}


_SCORES = 1 << 29  # the plain form holds at most this many scores (2 GB)


def _batches(queries, keys, q_at, k_at, heads):
    """The plain form's batches: neighbouring sequences padded to one size while that costs little."""
    batches, first = [], 0
    while first < len(queries):
        last = first + 1
        while last < len(queries) and (last + 1 - first) * max(queries[first:last + 1]) * max(
                keys[first:last + 1]) * heads <= _SCORES // 8:
            last += 1
        nq = torch.tensor(queries[first:last], device=DEVICE)
        nk = torch.tensor(keys[first:last], device=DEVICE)
        rows = torch.arange(max(queries[first:last]), device=DEVICE).clamp(max=nq[:, None] - 1)
        columns = torch.arange(max(keys[first:last]), device=DEVICE).clamp(max=nk[:, None] - 1)
        batches.append((rows + torch.tensor(q_at[first:last], device=DEVICE)[:, None],
                        columns + torch.tensor(k_at[first:last], device=DEVICE)[:, None], nq, nk))
        first = last
    return batches


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if case["op"] == "attention":
        queries, keys, q_at, k_at = _layout(case)
        state["cu_q"] = torch.tensor(q_at, dtype=torch.int32, device=DEVICE)
        state["cu_k"] = torch.tensor(k_at, dtype=torch.int32, device=DEVICE) if case["keys"] else None
        state["lengths_k"] = torch.tensor(keys, dtype=torch.int32, device=DEVICE) if case["slot"] else None
        if not own:
            state["batches"] = _batches(queries, keys, q_at, k_at, case["heads"])
    elif own:
        from vflash_b200.native.h3_nvfp4_linear import NVFP4Execution, NVFP4Weight

        one = torch.ones((), dtype=torch.float32, device=DEVICE)
        state["weight"] = NVFP4Weight(state["packed"], state["scales"], state["alpha"], one)
        state["execution"] = NVFP4Execution()
    return state


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "attention":
        return _run_attention(state, case)
    return _run_weight_only(state)


def _run_attention(state, case):
    if own:
        from vflash_b200.kernels import attention

        return attention(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"],
                         lengths_k=state["lengths_k"], causal=case["causal"], return_lse=case["lse"])
    q, k, v = state["q"], state["k"], state["v"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group = heads // kv_heads
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[0], heads, dtype=torch.float32, device=q.device)
    for q_at, k_at, nq, nk in state["batches"]:
        (batch, rows), keys = q_at.shape, k_at.shape[1]
        ks = k[k_at].float().permute(0, 2, 3, 1)     # [batch, kv_heads, dim, keys]
        vs = v[k_at].float().transpose(1, 2)         # [batch, kv_heads, keys, dim]
        key = torch.arange(keys, device=q.device)
        step = max(1, _SCORES // (batch * heads * keys))
        for r0 in range(0, rows, step):
            at = q_at[:, r0:r0 + step]
            r = at.shape[1]
            qs = q[at].float().reshape(batch, r, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
            scores = (qs.reshape(batch, kv_heads, group * r, dim) @ ks) * dim ** -0.5
            scores = scores.reshape(batch, heads, r, keys)
            row = torch.arange(r0, r0 + r, device=q.device)
            seen = nk[:, None].expand(batch, r)
            if case["causal"]:
                seen = torch.minimum(seen, row + 1 + (nk - nq)[:, None])
            scores.masked_fill_((key >= seen[..., None])[:, None], float("-inf"))
            peak = scores.amax(dim=-1, keepdim=True)
            p = torch.exp_(scores.sub_(peak))
            total = p.sum(dim=-1, keepdim=True)
            y = (p.reshape(batch, kv_heads, group * r, keys) @ vs).reshape(batch, heads, r, dim) / total
            real = row < nq[:, None]
            out[at[real]] = y.transpose(1, 2)[real].to(out.dtype)
            lse[at[real]] = (peak + torch.log(total))[..., 0].transpose(1, 2)[real]
    return (out, lse.T.contiguous()) if case["lse"] else out


def _run_weight_only(state):
    if own:
        return state["execution"].weight_only_linear(state["x"], state["weight"], state["bias"])
    packed = state["packed"]
    n, half = packed.shape
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).reshape(n, 2 * half)
    values = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                          device=packed.device)
    w = values[codes.int()].reshape(n, half // 8, 16)
    scales = state["scales"].reshape(n // 128, half // 32, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(n, half // 8)
    w = (w * scales.view(torch.float8_e4m3fn).float()[..., None]).reshape(n, 2 * half)
    y = (state["x"].float() @ w.T) * state["alpha"]
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(torch.bfloat16)


# --------------------------------------------------------------------------
# cost and exact values
# --------------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        queries, keys, _, _ = _layout(case)
        pairs = 0
        for nq, nk in zip(queries, keys):
            if case["causal"]:
                first = nk - nq + 1  # keys the first row sees
                pairs += nq * first + nq * (nq - 1) // 2
            else:
                pairs += nq * nk
        row = 2 * case["dim"]
        moved = (2 * sum(queries) * case["heads"] + 2 * sum(keys) * case["kv_heads"]) * row
        if case["lse"]:
            moved += 4 * sum(queries) * case["heads"]
        return {"bytes": moved, "flops": 4 * case["dim"] * case["heads"] * pairs}
    rows, n, k = case["rows"], case["n"], case["k"]
    moved = n * k // 2 + n * k // 16 + 2 * rows * k + 2 * rows * n + (2 * n if case["bias"] else 0)
    return {"bytes": moved, "flops": 2 * rows * n * k}


def exact(case, seed):
    """The outputs in 64 bits from the definitions: per head and row block for attention, per row block for the product."""
    data = _inputs(case, seed)
    if case["op"] == "attention":
        queries, keys, q_at, k_at = _layout(case)
        out = torch.zeros(data["q"].shape, dtype=torch.float64, device=DEVICE)
        lse = torch.zeros(case["heads"], q_at[-1], dtype=torch.float64, device=DEVICE)
        for b, (nq, nk) in enumerate(zip(queries, keys)):
            for h in range(case["heads"]):
                g = h * case["kv_heads"] // case["heads"]
                kk = data["k"][k_at[b]:k_at[b] + nk, g].double()
                vv = data["v"][k_at[b]:k_at[b] + nk, g].double()
                for r in range(0, nq, 8192):
                    rows = slice(q_at[b] + r, q_at[b] + min(nq, r + 8192))
                    s = torch.einsum("id,jd->ij", data["q"][rows, h].double(), kk) / math.sqrt(case["dim"])
                    if case["causal"]:
                        keep = torch.ones_like(s, dtype=torch.bool).tril(nk - nq + r)
                        s = torch.where(keep, s, -math.inf)
                    z = torch.logsumexp(s, dim=1)
                    out[rows, h] = torch.exp(s - z[:, None]) @ vv
                    lse[h, rows] = z
        return (out, lse) if case["lse"] else out
    n, k = case["n"], case["k"]
    groups = torch.arange(k // 16, device=DEVICE)
    rows = torch.arange(n, device=DEVICE)[:, None]
    # 128x4 layout: 512-byte blocks of 128 rows by 4 groups
    at = ((rows // 128) * (k // 64) + groups // 4) * 512 + (rows % 32) * 16 + (rows % 128) // 32 * 4 + groups % 4
    scale = data["scales"].reshape(-1)[at].view(torch.float8_e4m3fn).double()
    low, high = data["packed"] & 15, data["packed"] >> 4
    y = torch.zeros(case["rows"], n, dtype=torch.float64, device=DEVICE)
    for offset, code in ((0, low), (1, high)):
        e, m = (code >> 1) & 3, (code & 1).double()
        mag = torch.where(e == 0, 0.5 * m, torch.exp2(e.double() - 1) * (1 + 0.5 * m))
        w = torch.where(code >= 8, -mag, mag) * scale.repeat_interleave(8, dim=1)
        y += data["x"][:, offset::2].double() @ w.T
    y *= data["alpha"].double()
    return y if data["bias"] is None else y + data["bias"].double()
