"""Attention over packed sequences in 64 bits, with the error bound a correct kernel meets (test infrastructure only).

``reference`` computes every row from its definition over exactly the keys it
may see (nothing behind a mask is touched).  ``bound`` is per element, from the
roundings that any kernel of this contract makes, u being half a step of the
operand type (``torch.finfo(t).eps / 2``) and e = 2^-24 that of fp32:

* the output's rounding: u |o|, and half the smallest subnormal (2^-25 in fp16,
  nothing measurable in bf16) where it is subnormal;
* every exp value rounded to the type before the second product:
  u sum_j p_j |v_j| / l, plus half the smallest subnormal for each key
  (2^-25 in fp16, nothing measurable in bf16) times |v_j|, with l >= 1; a kernel
  that holds its maximum within 2^8 of the true one has room for a factor of 2^7
  in fp16 (2^15 < 65504), so 2^-32 of the largest is all that a key may lose;
* a score summed over ``dim`` products in fp32 and scaled: at most
  (dim + 4) e sum_d |q_d k_d| scale, and the same again relative to its value
  for the argument of exp, so a relative error of every exp value of twice
  that, once in the numerator and once in l;
* exp itself: 2^-17 relative (an approximation finer than that is required);
* fp32 sums over the keys, in numerator and l: (nk + 64) e each.
"""

from __future__ import annotations

import torch


def rows_of(lengths_q, lengths_k, slot: int = 0):
    q_at, k_at = [0], [0]
    for nq, nk in zip(lengths_q, lengths_k, strict=True):
        q_at.append(q_at[-1] + nq)
        k_at.append(k_at[-1] + (slot or nk))
    return q_at, k_at


def reference(q, k, v, lengths_q, lengths_k, *, causal: bool, scale: float, slot: int = 0):
    """(out, lse, out_bound, lse_bound), all float64, [total_q, heads, dim] and [heads, total_q]."""
    q_at, k_at = rows_of(lengths_q, lengths_k, slot)
    heads, dim = q.shape[1:]
    group = heads // k.shape[1]
    u, e = torch.finfo(q.dtype).eps / 2, 2.0**-24
    tiny, subnormal = (2.0**-32, 2.0**-25) if q.dtype == torch.float16 else (0.0, 0.0)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((heads, q.shape[0]), -torch.inf, dtype=torch.float64, device=q.device)
    out_bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    for b, (nq, nk) in enumerate(zip(lengths_q, lengths_k, strict=True)):
        for h in range(heads):
            qs = q[q_at[b]:q_at[b] + nq, h].double()
            ks = k[k_at[b]:k_at[b] + nk, h // group].double()
            vs = v[k_at[b]:k_at[b] + nk, h // group].double()
            if nq == 0 or nk == 0:
                continue
            first = max(0, nq - nk) if causal else 0  # the first row with a key
            if first == nq:
                continue
            rows = slice(q_at[b] + first, q_at[b] + nq)
            s = qs[first:] @ ks.T * scale
            size = qs[first:].abs() @ ks.abs().T * scale
            seen = torch.ones_like(s, dtype=torch.bool)
            if causal:
                seen = seen.tril(nk - nq + first)
            s = s.masked_fill(~seen, -torch.inf)
            z = torch.logsumexp(s, dim=1, keepdim=True)
            p = torch.exp(s - z)
            out[rows, h] = p @ vs
            lse[h, rows] = z[:, 0]
            score = ((dim + 4) * e * size).masked_fill(~seen, 0).amax(dim=1, keepdim=True)
            peak = s.masked_fill(~seen, 0).abs().amax(dim=1, keepdim=True)
            relative = 2 * (score + 4 * e * peak) + 2.0**-17 + (nk + 64) * e
            out_bound[rows, h] = (u * out[rows, h].abs() + (u + 2 * relative) * (p @ vs.abs())
                                  + tiny * (seen.double() @ vs.abs()) + subnormal + 2.0**-40)
            lse_bound[h, rows] = (relative + 4 * e * (z.abs() + peak) + 1e-7)[:, 0]
    return out, lse, out_bound, lse_bound
