"""Eviction from the INT4 cache by accumulated attention weight.

Long caches hold many tokens that no query looks at.  The attention call below
adds the weight each cached token received to a running score per KV head;
``evict_by_mass`` then cuts the cache to the tokens worth keeping.  The scores
come from decode steps (one query), or from the last queries of a prompt
before decoding starts.  The reference has no counterpart.
"""

from __future__ import annotations

import torch

from kernels.llama3._checks import (check_apart, check_out, check_query, check_rows, check_written, need_cuda,
                                    same_view)
from kvint4 import ops
from kvint4._lib import binding, result


def attention_forward_quant_gqa_scored(
    q: torch.Tensor,
    k_packed: torch.Tensor,
    k_scales: torch.Tensor,
    v_packed: torch.Tensor,
    v_scales: torch.Tensor,
    mass: torch.Tensor,
    *,
    n_q_heads: int,
    n_kv_heads: int,
    group_size: int = 32,
    is_causal: bool = False,
    decay: float = 1.0,
    mass_out: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``attention_forward_quant_gqa`` that also scores the cached tokens.

    Returns ``(out, mass_out)`` with ``mass_out[b, g, t] = decay * mass[b, g, t]
    +`` the softmax weight of token ``t``, summed over the queries and over the
    q heads of KV head ``g``.  ``mass`` is f32 ``[B, n_kv_heads, S]`` (any
    strides) and is updated in place when ``mass_out`` is not given.  ``out`` and
    another ``mass_out`` must not overlap each other nor anything that is read.
    ``is_causal``: query ``i`` sees tokens ``t <= S - sq + i``.
    """
    got = binding().scored(q, k_packed, k_scales, v_packed, v_scales, mass, n_q_heads, n_kv_heads,
                           group_size, is_causal, decay, mass_out, out)
    if got is not None:
        return result("kv4_scored_attention", got)
    # something about the arguments is not plainly right: say what
    cache = (k_packed, k_scales, v_packed, v_scales)
    check_rows("cache", *cache)
    check_query(q, k_packed, k_scales, n_q_heads, n_kv_heads, group_size)
    shape = k_packed.shape[:3]
    read = dict(zip(("q", "k_packed", "k_scales", "v_packed", "v_scales"), (q, *cache)))
    if mass_out is None:
        mass_out = mass
    elif not same_view(mass_out, mass):
        check_apart("mass_out", mass_out, {"mass": mass})
    check_written("mass_out", mass_out)
    check_apart("mass_out", mass_out, read)
    if out is not None:
        check_written("out", out)
        check_apart("out", out, {**read, "mass": mass, "mass_out": mass_out})
    need_cuda("attention_forward_quant_gqa_scored", q, *cache, mass)
    check_out("mass", mass, shape, torch.float32, q)
    check_out("mass_out", mass_out, shape, torch.float32, q)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        check_out("out", out, q.shape, q.dtype, q)
    ops.scored_attention_into(q, cache, mass, mass_out, out, group_size, is_causal, decay)
    return out, mass_out


def evict_by_mass(
    k_packed: torch.Tensor,
    k_scales: torch.Tensor,
    v_packed: torch.Tensor,
    v_scales: torch.Tensor,
    mass: torch.Tensor,
    *,
    keep: int,
    recent: int = 0,
    sinks: int = 0,
    out: tuple[torch.Tensor, ...] | None = None,
) -> tuple[torch.Tensor, ...]:
    """Cut each (sequence, KV head) of the cache to ``keep`` tokens.

    Kept are the first ``sinks`` tokens, the last ``recent`` ones and, of the
    rest, those with the highest ``mass`` (f32 ``[B, n_kv_heads, S]``; equal
    scores: the earlier token; NaN below everything), in token order.  Returns
    ``(k_packed, k_scales, v_packed, v_scales, mass, index)`` of the kept
    tokens, ``index`` int32 ``[B, n_kv_heads, keep]``; the first five are
    written into ``out`` when given (views of other capacity buffers, for
    instance: rows are moved all at once, so ``out`` must not overlap the inputs).
    """
    got = binding().evict(k_packed, k_scales, v_packed, v_scales, mass, keep, recent, sinks, out)
    if got is not None:
        return result("kv4_evict", got)
    # something about the arguments is not plainly right: say what
    cache = (k_packed, k_scales, v_packed, v_scales)
    check_rows("cache", *cache)
    b, h, s = k_packed.shape[:3]
    keep, recent, sinks = int(keep), int(recent), int(sinks)
    if recent < 0 or sinks < 0:
        raise ValueError("recent and sinks must be >= 0")
    if not recent + sinks <= keep <= s:
        raise ValueError(f"keep must lie between recent + sinks = {recent + sinks} and the {s} cached tokens")
    if any(t.shape[-1] > 1 and t.stride(-1) != 1 for t in cache):
        raise ValueError("cache rows need a unit stride in the last dimension")
    if out is not None and len(out) == 5:
        read = dict(zip(("k_packed", "k_scales", "v_packed", "v_scales", "mass"), (*cache, mass)))
        for i, o in enumerate(out):
            check_written("out", o)
            check_apart("out", o, {**read, **{f"out[{j}]": out[j] for j in range(i)}})
    need_cuda("evict_by_mass", *cache, mass)
    check_out("mass", mass, (b, h, s), torch.float32, k_packed)
    if out is None:
        out = tuple(torch.empty(b, h, keep, t.shape[-1], dtype=t.dtype, device=t.device)
                    for t in cache) + (torch.empty(b, h, keep, dtype=mass.dtype, device=mass.device),)
    else:
        if len(out) != 5:
            raise ValueError("out must be (k_packed, k_scales, v_packed, v_scales, mass)")
        for o, t in zip(out, (*cache, mass)):
            check_out("out", o, (b, h, keep, *t.shape[3:]), t.dtype, t)
            if o.dim() == 4 and o.shape[-1] > 1 and o.stride(-1) != 1:
                raise ValueError("out rows need a unit stride in the last dimension")
    index = torch.empty(b, h, keep, dtype=torch.int32, device=mass.device)
    ops.evict_into(mass, cache, out[:4], out[4], index, recent, sinks)
    return (*out, index)
