"""64-bit references and error bounds for the operators that branch and trim
the INT4 cache (tree attention, commit, scored attention, eviction).

Bounds are worst-case bounds of the arithmetic, not fitted numbers.  With u32 =
2**-24, a row whose scores have magnitudes X = max_t sum_c |q_c k_tc| * sm_scale
over n visible keys of head size d:

* a score is off by at most (d + 8) * u32 * X (d products and sums in fp32, the
  scaling), so a weight by e^delta - 1 <= 2 * delta relative, and the normalised
  weight by twice that; the row's sum and output sums add (n + 64) * u32 each
  (the exponential's own error is inside the 64);
* on the tensor-core path the weights enter the second product as f16, 2**-11
  relative (one rounding), and the products
  accumulate with fp32 inputs aligned to the largest term, counted as one more
  u32 * 2 per term;
* f16 has an absolute step of 2**-24 below 2**-14, and the largest weight of a
  row is written as at least 2**7, so a weight is also off by up to 2**-31 of
  the largest (2**-20 of it times the 2**-11 above);
* the output is rounded once to its type, u_out relative.

A[c] = sum_t (p_t + 2**-20) |v_tc| over the visible keys scales the absolute
error of output column c.
"""

from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24
# unit roundoffs: 2**-p for a p-bit significand (bf16 8, f16 11, f32 24)
U_OUT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# smallest normal-range rounding step that the output type adds near zero
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25, torch.float32: 1e-38}


def random_rows(b, h, s, d, group, dtype, seed, scale=1.0):
    """Random codes and positive scales: [k_packed, k_scales, v_packed, v_scales]."""
    g = torch.Generator().manual_seed(seed)
    ng, pb = math.ceil(d / group), (group + 1) // 2
    out = []
    for _ in range(2):
        out.append(torch.randint(0, 256, (b, h, s, ng * pb), generator=g, dtype=torch.uint8))
        out.append((scale * (0.05 + 0.4 * torch.rand(b, h, s, ng, generator=g))).to(dtype))
    return out


def values(packed, scales, group, d):
    """Packed rows as float64 [..., d]."""
    ng, pb = scales.shape[-1], (group + 1) // 2
    p = packed[..., : ng * pb].cpu().unflatten(-1, (ng, pb))
    c = torch.stack((p & 15, p >> 4), -1).flatten(-2)[..., :group].double() - 8
    return (c * scales.cpu().double().unsqueeze(-1)).flatten(-2)[..., :d]


def attend(q, k, v, seen, sm_scale=None):
    """q [Hq, n, d] over k, v [Hkv, S, d] (float64), seen [n, S] bool ->
    out, weights [Hq, n, S], X [Hq, n], A [Hq, n, d]."""
    hq, n, d = q.shape
    r = hq // k.shape[0]
    kk, vv = k.repeat_interleave(r, 0), v.repeat_interleave(r, 0)
    sm = sm_scale or d ** -0.5
    x = (q @ kk.transpose(1, 2)) * sm
    big = (q.abs() @ kk.abs().transpose(1, 2)) * sm
    x = x.masked_fill(~seen, -math.inf)
    p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
    big = big.masked_fill(~seen, 0.0)
    X = big.amax(-1) if x.shape[-1] else torch.zeros(hq, n, dtype=torch.float64)
    return p @ vv, p, X, (p + 2.0 ** -20 * seen.double()) @ vv.abs()


def weight_bound(X, d, keys):
    """Relative error of a normalised weight."""
    return U32 * (4 * (d + 8) * X + 2 * (keys + 64)) * 2


def check_out(got, ref, X, A, keys):
    """got in its dtype against ref within the bound of the module's comment."""
    dt, d = got.dtype, got.shape[-1]
    rel = weight_bound(X, d, keys).unsqueeze(-1) + U32 * 2 * (keys + 64)
    if dt != torch.float32:
        rel = rel + 2.0 ** -11
    bound = U_OUT[dt] * (ref.abs() + rel * A) + rel * A + TINY[dt]
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all()
    assert bool((err <= bound).all()), f"{float((err / bound).max()):.3g} times the bound"


def tree_mask(b, n, seed):
    """Random trees: node i's parent is one of the three before it or the context."""
    g = torch.Generator().manual_seed(seed)
    m = torch.zeros(b, n, n, dtype=torch.bool)
    for x in range(b):
        for i in range(n):
            back = int(torch.randint(0, 4, (1,), generator=g))
            if 0 < back <= i:
                m[x, i] = m[x, i - back]
            m[x, i, i] = True
    return m


def evict_index(mass, keep, recent, sinks):
    """Kept token numbers by sorting (score descending, NaN last, then index)."""
    b, h, s = mass.shape
    out = torch.empty(b, h, keep, dtype=torch.int64)
    for x in range(b):
        for y in range(h):
            row = mass[x, y].double()
            mid = sorted(range(sinks, s - recent),
                         key=lambda t: (bool(row[t].isnan()), 0.0 if row[t].isnan() else -float(row[t]), t))
            chosen = mid[: keep - recent - sinks]
            out[x, y] = torch.tensor(sorted(list(range(sinks)) + chosen + list(range(s - recent, s))),
                                     dtype=torch.int64)
    return out
