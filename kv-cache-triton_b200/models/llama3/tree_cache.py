"""KV cache of speculative decoding: contexts of different lengths and a tree of drafted tokens.

Packed INT4 buffers of a fixed capacity per layer, with the number of tokens of
each sequence on the device (``lens``), and a draft buffer per layer for the
nodes of the current tree.  One step:

    cache.begin(mask)                     # which nodes see which: bool [N, N] or [B, N, N]
    logits = model(nodes, past_key_values=cache, position_ids=cache.positions(depth), ...)
    path, accepted, token = accept_greedy(nodes, parents, logits)
    cache.commit(path, accepted)          # accepted K/V move behind the context

Nothing in a step waits for the device: lengths, paths and counts stay there
(``tree_mask``, for a new shape of tree, does wait).  What a step could not do, a
path that no longer fits the capacity for instance, ``check()`` raises.
Rejected nodes are never in the cache.  The reference decodes one token at a
time and has no counterpart.
"""

from __future__ import annotations

import math

import torch

from kernels.llama3.tree_attention_quant import commit_draft_rows, tree_attention_quant_gqa
from kvint4 import ops
from kvint4._lib import TIE_HALF_AWAY
from kvint4.cache import CAPACITY_ALIGN, _round_up


class TreeKVCache:
    """Contexts and drafted trees for ``n_layers`` layers."""

    is_compileable = False
    is_sliding = [False]

    def __init__(self, n_layers: int, batch: int, n_kv_heads: int, head_dim: int, *, capacity: int,
                 max_nodes: int, group_size: int = 32, dtype: torch.dtype = torch.bfloat16,
                 device="cuda", tie_mode: int = TIE_HALF_AWAY):
        if min(n_layers, batch, n_kv_heads, head_dim, capacity, max_nodes, group_size) <= 0:
            raise ValueError("sizes must be > 0")
        self.group_size, self.tie_mode = int(group_size), int(tie_mode)
        self.capacity, self.max_nodes = _round_up(int(capacity), CAPACITY_ALIGN), int(max_nodes)
        ng = math.ceil(head_dim / group_size)
        pw = ng * ((group_size + 1) // 2)

        def rows(t):
            return [torch.zeros(batch, n_kv_heads, t, w, dtype=x, device=device)
                    for w, x in ((pw, torch.uint8), (ng, dtype)) * 2]

        self._cache = [rows(self.capacity) for _ in range(n_layers)]
        self._draft = [rows(_round_up(self.max_nodes, 8)) for _ in range(n_layers)]
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        # true position of a sequence's next token minus its tokens in the cache
        self.offset = torch.zeros(batch, dtype=torch.int32, device=device)
        self._mask: torch.Tensor | None = None
        self._nodes = self._draft  # the draft rows of the current tree's nodes (views)

    @classmethod
    def from_cache(cls, cache, *, extra: int, max_nodes: int, tokens_seen: int | None = None):
        """Take over a prefilled ``QuantizedKVCache`` (evicted or not), with room for
        ``extra`` more tokens.  ``tokens_seen``: length of the text so far, where
        eviction made it differ from the tokens held."""
        layers = [cache._layers[i] for i in sorted(cache._layers)]
        if not layers:
            raise ValueError("the cache is empty")
        n = layers[0].seq_len
        if any(st.seq_len != n for st in layers):
            raise ValueError("layers of different lengths")
        b, h, _, _ = layers[0].k_packed_buf.shape
        ng = layers[0].k_scales_buf.shape[-1]
        self = cls(len(layers), b, h, ng * cache.group_size, capacity=n + int(extra),
                   max_nodes=max_nodes, group_size=cache.group_size,
                   dtype=layers[0].k_scales_buf.dtype, device=layers[0].k_packed_buf.device,
                   tie_mode=cache._store.tie_mode)
        for st, mine in zip(layers, self._cache):
            for src, dst in zip(st.views(), mine):
                dst[:, :, :n].copy_(src)
        self.lens.fill_(n)
        self.offset.fill_(0 if tokens_seen is None else int(tokens_seen) - n)
        return self

    # -- a step --------------------------------------------------------------
    def begin(self, mask: torch.Tensor) -> None:
        """The tree of the coming step: ``mask`` bool ``[N, N]`` or ``[B, N, N]``."""
        n = mask.shape[-1]
        if mask.dtype != torch.bool or mask.dim() not in (2, 3) or mask.shape[-2] != n:
            raise ValueError("mask must be bool [N, N] or [B, N, N]")
        if n > self.max_nodes:
            raise ValueError(f"{n} nodes, but the cache was made for {self.max_nodes}")
        if n != self._nodes[0][0].shape[2]:
            self._nodes = [[t[:, :, :n] for t in rows] for rows in self._draft]
        self._mask = mask

    def positions(self, depth: torch.Tensor) -> torch.Tensor:
        """Positions ``[B, N]`` of nodes at ``depth`` (int ``[N]`` or ``[B, N]``, 0 for the first)."""
        return (self.lens + self.offset).unsqueeze(1).long() + depth

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Quantize the nodes' K/V ``[B, n_kv, N, d]`` into the layer's draft rows, then
        attention of their queries ``[B, n_q, N, d]``."""
        if self._mask is None:
            raise ValueError("begin() a step first")
        n = self._mask.shape[-1]
        if q.shape[2] != n or k.shape[2] != n:
            raise ValueError(f"{q.shape[2]} tokens for a tree of {n} nodes")
        draft = self._nodes[layer]
        ops.append_kv(k, v, *draft, 0, self.group_size, self.tie_mode)
        return tree_attention_quant_gqa(q, *self._cache[layer], *draft, self._mask,
                                        n_q_heads=q.shape[1], n_kv_heads=k.shape[1],
                                        group_size=self.group_size, context_lens=self.lens, out=out)

    def commit(self, path: torch.Tensor, accepted: torch.Tensor) -> None:
        """Move the accepted nodes (``path`` int32 ``[B, width]``, the first
        ``accepted[b]`` of each row) of the step's tree behind each sequence's context."""
        if self._mask is None:
            raise ValueError("begin() a step first")
        new = None
        for cache, draft in zip(self._cache, self._nodes):
            new = commit_draft_rows(*cache, *draft, path, accepted, context_lens=self.lens)
        self.lens = new
        self._mask = None

    def check(self) -> None:
        """Wait for the device and raise ``RuntimeError`` if a call since the last
        check could not do its work (on this device, whoever made it)."""
        ops.check_device(self.lens.device)

    # -- what Hugging Face's model asks of a cache ----------------------------
    def get_seq_length(self, layer_idx: int = 0) -> int:
        return 0  # lengths are on the device: positions are passed to the model

    def get_mask_sizes(self, cache_position, layer_idx: int = 0) -> tuple[int, int]:
        n = cache_position if isinstance(cache_position, int) else cache_position.shape[0]
        return int(n), 0

    def get_max_cache_shape(self, layer_idx: int = 0) -> int:
        return self.capacity

    @property
    def is_initialized(self) -> bool:
        return True

    def __len__(self) -> int:
        return len(self._cache)


def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """Which nodes see which: bool ``[..., N, N]`` from ``parents`` int ``[..., N]``
    (-1: hangs on the context; a parent comes before its children)."""
    n = parents.shape[-1]
    eye = torch.eye(n, dtype=torch.bool, device=parents.device)
    up = parents.clamp(min=0).long()
    mask = eye.expand(*parents.shape, n)
    for _ in range(n):
        above = mask.gather(-2, up.unsqueeze(-1).expand(*parents.shape, n)) & (parents >= 0).unsqueeze(-1)
        grown = eye | above
        if torch.equal(grown, mask):
            break
        mask = grown
    return mask.contiguous()


def tree_depth(parents: torch.Tensor) -> torch.Tensor:
    """Depth of every node (0 for those on the context)."""
    return tree_mask(parents).sum(-1) - 1


def accept_greedy(nodes: torch.Tensor, parents: torch.Tensor, logits: torch.Tensor):
    """Follow the model's own choices down each tree.

    ``nodes`` int ``[B, N]`` (node 0 is the last token already decided),
    ``parents`` int ``[N]`` or ``[B, N]``, ``logits`` ``[B, N, vocab]``.  Returns
    ``(path, accepted, token)``: int32 ``[B, N]`` node numbers from node 0 down,
    how many of them are accepted (at least node 0), and the token that follows.
    """
    b, n = nodes.shape
    choice = logits.argmax(-1)
    parents = parents.expand(b, n)
    rows = torch.arange(b, device=nodes.device)
    at = torch.zeros(b, dtype=torch.long, device=nodes.device)
    path = torch.zeros(b, n, dtype=torch.int32, device=nodes.device)
    accepted = torch.ones(b, dtype=torch.int32, device=nodes.device)
    alive = torch.ones(b, dtype=torch.bool, device=nodes.device)
    for j in range(1, n):
        fits = (parents == at.unsqueeze(1)) & (nodes == choice[rows, at].unsqueeze(1))
        fits[:, 0] = False
        alive = alive & fits.any(1)
        at = torch.where(alive, fits.int().argmax(1), at)
        path[:, j] = torch.where(alive, at, torch.zeros_like(at)).int()
        accepted += alive.int()
    return path, accepted, choice[rows, at]
