"""Attention for a tree of drafted tokens over the INT4 cache, and the commit of an accepted path.

Speculative decoding drafts N tokens per sequence that form a tree, verifies
all of them in one step, and keeps one path.  The drafted K/V rows live in a
draft buffer of the cache's own format until then, so a rejected token never
touches the cache:

    k, v of the nodes --quantize--> draft rows
    out = tree_attention_quant_gqa(q, *cache, *draft, mask, ...)
    lens = commit_draft_rows(*cache, *draft, path, accepted, context_lens=lens)

``models.llama3.tree_cache.TreeKVCache`` keeps these buffers for all layers of a model.
The reference has no counterpart (it decodes one token at a time).
"""

from __future__ import annotations

import torch

from kernels.llama3._checks import (check_apart, check_int32, check_out, check_query, check_rows, check_written,
                                    need_cuda, same_view)
from kvint4 import ops
from kvint4._lib import binding, result


def tree_attention_quant_gqa(
    q: torch.Tensor,
    k_packed: torch.Tensor,
    k_scales: torch.Tensor,
    v_packed: torch.Tensor,
    v_scales: torch.Tensor,
    draft_k_packed: torch.Tensor,
    draft_k_scales: torch.Tensor,
    draft_v_packed: torch.Tensor,
    draft_v_scales: torch.Tensor,
    tree_mask: torch.Tensor,
    *,
    n_q_heads: int,
    n_kv_heads: int,
    group_size: int = 32,
    context_lens: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of N drafted nodes per sequence: ``[B, n_q_heads, N, d_head]`` in the dtype of ``q``.

    Node ``i`` of sequence ``b`` sees the cache rows ``[0, context_lens[b])``
    (all rows when ``context_lens`` is None) and the drafted rows ``j`` with
    ``tree_mask[b, i, j]`` (bool ``[N, N]`` for the whole batch or
    ``[B, N, N]``; normally the ancestors of ``i`` and ``i`` itself).  A node
    that sees nothing gives zeros.  ``context_lens`` is int32 ``[B]`` on the
    device; an entry outside ``[0, S]`` reads as 0 and is reported by
    ``ops.device_error()`` (bit 16).  ``lse`` (f32 ``[B, n_q_heads, N]``)
    receives the log-sum-exp of each row's scores.  ``out`` (which may be ``q``
    itself) and ``lse`` must not overlap each other nor anything that is read.
    """
    got = binding().tree(q, k_packed, k_scales, v_packed, v_scales, draft_k_packed, draft_k_scales,
                         draft_v_packed, draft_v_scales, tree_mask, n_q_heads, n_kv_heads,
                         group_size, context_lens, out, lse)
    if got is not None:
        return result("kv4_tree_attention", got)
    # something about the arguments is not plainly right: say what
    cache = (k_packed, k_scales, v_packed, v_scales)
    draft = (draft_k_packed, draft_k_scales, draft_v_packed, draft_v_scales)
    check_rows("cache", *cache)
    check_rows("draft", *draft)
    check_query(q, k_packed, k_scales, n_q_heads, n_kv_heads, group_size)
    b, hq, n, d = q.shape
    if draft_k_packed.shape != (b, n_kv_heads, n, k_packed.shape[-1]):
        raise ValueError("draft rows must be [B, n_kv_heads, N, ...] with the widths of the cache")
    if draft_k_scales.shape[-1] != k_scales.shape[-1] or draft_k_scales.dtype != k_scales.dtype:
        raise ValueError("draft scales must match the cache's scales")
    if tree_mask.dtype != torch.bool or tuple(tree_mask.shape) not in ((n, n), (b, n, n)):
        raise ValueError("tree_mask must be bool [N, N] or [B, N, N]")
    names = ("k_packed", "k_scales", "v_packed", "v_scales")
    read = {**dict(zip(names, cache)), **dict(zip((f"draft_{x}" for x in names), draft)),
            "tree_mask": tree_mask, "context_lens": context_lens}
    if out is not None:
        check_written("out", out)
        check_apart("out", out, read if same_view(out, q) else {"q": q, **read})
    if lse is not None:
        check_written("lse", lse)
        check_apart("lse", lse, {"q": q, "out": out, **read})
    need_cuda("tree_attention_quant_gqa", q, *cache, *draft, tree_mask)
    if context_lens is not None:
        check_int32("context_lens", context_lens, (b,), q)
    if lse is not None:
        check_out("lse", lse, q.shape[:3], torch.float32, q)
    if out is None:
        out = torch.empty(b, hq, n, d, dtype=q.dtype, device=q.device)
    else:
        check_out("out", out, q.shape, q.dtype, q)
    if q.numel() == 0:
        return out
    ops.tree_attention_into(q, cache, draft, tree_mask, out, group_size,
                            context_lens=context_lens, lse=lse)
    return out


def commit_draft_rows(
    k_packed: torch.Tensor,
    k_scales: torch.Tensor,
    v_packed: torch.Tensor,
    v_scales: torch.Tensor,
    draft_k_packed: torch.Tensor,
    draft_k_scales: torch.Tensor,
    draft_v_packed: torch.Tensor,
    draft_v_scales: torch.Tensor,
    path: torch.Tensor,
    accepted: torch.Tensor,
    *,
    context_lens: torch.Tensor,
    lens_out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Move the accepted drafted rows behind each sequence's context; returns the new lengths.

    Cache row ``context_lens[b] + j`` becomes drafted row ``path[b, j]`` for
    ``j < accepted[b]``.  ``path`` is int32 ``[B, width]``, ``accepted`` and
    ``context_lens`` int32 ``[B]``, all on the device; the host waits for
    nothing.  Cache and drafted rows must not overlap, nor ``lens_out`` what is
    read.  A sequence whose rows do not fit is left as it was and reported
    by ``ops.device_error()`` (bit 16).
    """
    got = binding().commit(k_packed, k_scales, v_packed, v_scales, draft_k_packed, draft_k_scales,
                           draft_v_packed, draft_v_scales, path, accepted, context_lens, lens_out)
    if got is not None:
        return result("kv4_commit_rows", got)
    # something about the arguments is not plainly right: say what
    cache = (k_packed, k_scales, v_packed, v_scales)
    draft = (draft_k_packed, draft_k_scales, draft_v_packed, draft_v_scales)
    check_rows("cache", *cache)
    check_rows("draft", *draft)
    for c, f in zip(cache, draft):
        if c.dtype != f.dtype or c.shape[:2] != f.shape[:2] or c.shape[-1] != f.shape[-1]:
            raise ValueError("draft rows must match the cache in all but the token dimension")
        if (c.shape[-1] > 1 and c.stride(-1) != 1) or (f.shape[-1] > 1 and f.stride(-1) != 1):
            raise ValueError("cache and draft rows need a unit stride in the last dimension")
    b = k_packed.shape[0]
    names = ("k_packed", "k_scales", "v_packed", "v_scales")
    read = {**dict(zip((f"draft_{x}" for x in names), draft)), "path": path, "accepted": accepted}
    for name, c in zip(names, cache):
        check_written(name, c)
        check_apart(name, c, {**read, "context_lens": context_lens})
    if lens_out is not None:
        if lens_out.data_ptr() == context_lens.data_ptr():
            raise ValueError("lens_out must not be context_lens")
        check_apart("lens_out", lens_out, {**read, **dict(zip(names, cache)), "context_lens": context_lens})
    need_cuda("commit_draft_rows", *cache, *draft, path, accepted, context_lens)
    if path.dim() != 2:
        raise ValueError("path must be [B, width]")
    check_int32("path", path, (b, path.shape[1]), k_packed)
    check_int32("accepted", accepted, (b,), k_packed)
    check_int32("context_lens", context_lens, (b,), k_packed)
    if lens_out is None:
        lens_out = torch.empty_like(context_lens)
    else:
        check_int32("lens_out", lens_out, (b,), k_packed)
    ops.commit_rows(k_packed, cache, draft, path, accepted, context_lens, lens_out)
    return lens_out
