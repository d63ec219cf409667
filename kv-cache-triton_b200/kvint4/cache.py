"""INT4 KV-cache storage with preallocated capacity and in-place append.

Layout in HBM, per layer (one tensor each for K and V):

    packed  uint8 [B, n_kv, capacity, ceil(d/G)*ceil(G/2)]
    scales  float [B, n_kv, capacity, ceil(d/G)]

Tokens ``[0, seq_len)`` are valid; ``get_quantized`` returns strided views
``[:, :, :seq_len]`` with exactly the reference's shapes.  An append
quantizes the new K and V rows straight into rows ``[seq_len, seq_len+s)``
with ONE kernel launch (``kv4_append_kv``); the reference instead quantized
into fresh tensors and concatenated the whole cache each step
(``models/llama3/kv_cache.py:76-102``), an O(S) copy per decode step.
Capacity grows geometrically (one copy of the valid prefix) when exceeded.
Capacity is kept a multiple of 64 tokens so every (batch, head) plane starts
16-byte aligned, which the TMA loads of the decode kernel require.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib, frontend, ops

CAPACITY_ALIGN = 64


def _round_up(x: int, m: int) -> int:
    return (x + m - 1) // m * m


@dataclass
class LayerStore:
    k_packed_buf: torch.Tensor
    k_scales_buf: torch.Tensor
    v_packed_buf: torch.Tensor
    v_scales_buf: torch.Tensor
    seq_len: int
    # True while the last kernel that wrote these buffers was a fused decode
    # step (kv4_append_attention): the next fused step may then start early
    # (kv4_attn_opts.early_start), since no other kernel wrote the rows it reads
    early_ok: bool = False
    # [B, n_kv, capacity] f32: attention weight each token received so far
    # (``track_mass`` stores only)
    mass_buf: torch.Tensor | None = None
    # first of the tokens that came by a path that scores nothing (``note_unscored``)
    # and that no attention has scored since
    unscored: int | None = None

    @property
    def capacity(self) -> int:
        return self.k_packed_buf.shape[2]

    def view_descs(self, n: int):
        """C-ABI descriptors of the four views ``[:, :, :n]``, built from
        descriptors of the buffers kept on the layer (no torch views)."""
        bufs = (self.k_packed_buf, self.k_scales_buf, self.v_packed_buf, self.v_scales_buf)
        cached = getattr(self, "_descs", None)
        if cached is None or cached[0] != tuple(b.data_ptr() for b in bufs):
            cached = (tuple(b.data_ptr() for b in bufs), [ops.desc(b) for b in bufs])
            self._descs = cached
        for d in cached[1]:
            d.shape[2] = n
        return cached[1]

    def views(self):
        s = self.seq_len
        return (self.k_packed_buf[:, :, :s], self.k_scales_buf[:, :, :s],
                self.v_packed_buf[:, :, :s], self.v_scales_buf[:, :, :s])


class Int4KVStore:
    """Per-layer INT4 storage shared by the Llama and GPT-2 caches."""

    def __init__(self, group_size: int = 32, *, capacity: int | None = None,
                 scale_dtype: torch.dtype | None = None, tie_mode: int = _lib.TIE_HALF_AWAY,
                 growth: float = 1.5, track_mass: bool = False, mass_decay: float = 1.0,
                 mass_window: int = 32):
        if group_size <= 0:
            raise ValueError("group_size must be > 0")
        self.group_size = int(group_size)
        self.capacity_hint = int(capacity) if capacity else 0
        self.scale_dtype = scale_dtype
        self.tie_mode = int(tie_mode)
        self.growth = float(growth)
        # score the cached tokens by the attention weight they receive: from every
        # one-token step, and from the last ``mass_window`` queries of a prompt
        self.track_mass = bool(track_mass)
        self.mass_decay = float(mass_decay)
        self.mass_window = int(mass_window)
        if self.track_mass and self.mass_window <= 0:
            raise ValueError("mass_window must be > 0")
        self._layers: dict[int, LayerStore] = {}

    # -- storage ---------------------------------------------------------
    def _alloc(self, like: torch.Tensor, b: int, h: int, cap: int, d: int) -> LayerStore:
        g = self.group_size
        ng = math.ceil(d / g)
        pw = ng * ((g + 1) // 2)
        sdt = self.scale_dtype or like.dtype
        dev = like.device
        return LayerStore(
            k_packed_buf=torch.empty(b, h, cap, pw, dtype=torch.uint8, device=dev),
            k_scales_buf=torch.empty(b, h, cap, ng, dtype=sdt, device=dev),
            v_packed_buf=torch.empty(b, h, cap, pw, dtype=torch.uint8, device=dev),
            v_scales_buf=torch.empty(b, h, cap, ng, dtype=sdt, device=dev),
            seq_len=0,
            mass_buf=torch.zeros(b, h, cap, device=dev) if self.track_mass else None,
        )

    def append(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int) -> None:
        layer = self._reserve(key_states, value_states, layer_idx)
        s = key_states.shape[2]
        if s == 0:
            return
        ops.append_kv(key_states, value_states, layer.k_packed_buf, layer.k_scales_buf,
                      layer.v_packed_buf, layer.v_scales_buf, layer.seq_len, self.group_size,
                      self.tie_mode)
        if layer.mass_buf is not None:
            layer.mass_buf[:, :, layer.seq_len:layer.seq_len + s].zero_()
        layer.seq_len += s
        layer.early_ok = False

    def append_attend(self, query: torch.Tensor, key_states: torch.Tensor,
                      value_states: torch.Tensor, layer_idx: int, out: torch.Tensor, *,
                      n_q_heads: int, n_kv_heads: int, is_causal: bool = False) -> torch.Tensor:
        """``append`` followed by attention of ``query`` over the whole layer
        cache, written to ``out`` (any strides, [B, Hq, sq, d]).  A one-token
        decode step is a single launch: the attention kernel quantizes the new
        row itself (``kv4_append_attention``).  ``track_mass`` stores score the
        tokens by one query, or by the last ``mass_window`` of several."""
        s = key_states.shape[2]
        if self.track_mass and s == 1 and query.shape[2] == 1:
            self.append(key_states, value_states, layer_idx)
            return self.attend_scored(query, layer_idx, out, is_causal=is_causal)
        layer = self._reserve(key_states, value_states, layer_idx)
        if s != 1 or self.track_mass:
            self.append(key_states, value_states, layer_idx)
            kp, ks, vp, vs = self.layer(layer_idx).views()
            frontend.attention(query, kp, ks, vp, vs, n_q_heads=n_q_heads,
                               n_kv_heads=n_kv_heads, group_size=self.group_size,
                               is_causal=is_causal, out=out)
            if self.track_mass:
                self.score_window(query, layer_idx)
            return out
        n = layer.seq_len + 1
        ops.append_attention_descs(query, key_states, value_states, layer.view_descs(n), out,
                                   self.group_size, is_causal, self.tie_mode,
                                   early_start=layer.early_ok)
        layer.seq_len = n
        layer.early_ok = True
        return out

    # -- scores of the cached tokens ----------------------------------------
    def attend_scored(self, query: torch.Tensor, layer_idx: int, out: torch.Tensor, *,
                      is_causal: bool = False) -> torch.Tensor:
        """Attention of ``query`` over the layer's cache into ``out`` that adds the
        weight each cached token received to the layer's scores."""
        layer = self.layer(layer_idx)
        if layer.mass_buf is None:
            raise ValueError("the store does not track scores (track_mass=True)")
        ops.scored_attention_into(query, layer.views(), self.mass(layer_idx), self.mass(layer_idx),
                                  out, self.group_size, is_causal, self.mass_decay)
        layer.unscored = None
        return out

    def note_unscored(self, layer_idx: int, tokens: int) -> None:
        """The layer's last ``tokens`` tokens came by a path that scores nothing."""
        layer = self.layer(layer_idx)
        if layer.mass_buf is not None and tokens > 0 and layer.unscored is None:
            layer.unscored = layer.seq_len - tokens

    def score_window(self, query: torch.Tensor, layer_idx: int) -> None:
        """Score the layer's tokens by the last ``mass_window`` queries of
        ``query`` [B, Hq, s, d], which belong to the cache's last s tokens."""
        q = query[:, :, -self.mass_window:]
        self.attend_scored(q, layer_idx, torch.empty(q.shape, dtype=q.dtype, device=q.device),
                           is_causal=True)

    def mass(self, layer_idx: int) -> torch.Tensor:
        """Scores [B, n_kv, seq_len] of a layer's tokens (a view)."""
        layer = self.layer(layer_idx)
        if layer.mass_buf is None:
            raise ValueError("the store does not track scores (track_mass=True)")
        return layer.mass_buf[:, :, :layer.seq_len]

    def evict(self, keep: int, *, recent: int = 0, sinks: int = 0) -> dict[int, torch.Tensor]:
        """Cut every layer that holds more than ``keep`` tokens to the first
        ``sinks``, the last ``recent`` and the highest scored of the rest, per KV
        head, in token order; returns the kept token numbers
        ``{layer: int32 [B, n_kv, keep]}`` of the layers that were cut.  Refused,
        with nothing cut, while tokens would be ranked that came by a path that scores
        nothing (attention under a mask) and that no attention has scored since."""
        if not 0 <= recent + sinks <= keep or recent < 0 or sinks < 0:
            raise ValueError("keep must be at least recent + sinks, all >= 0")
        kept = {}
        for layer_idx, old in self._layers.items():
            if old.seq_len > keep and old.unscored is not None and old.seq_len - old.unscored > recent:
                raise ValueError(f"layer {layer_idx}: the last {old.seq_len - old.unscored} tokens have no scores "
                                 f"(score_window() them, or keep them as recent)")
        for layer_idx, old in self._layers.items():
            if old.seq_len <= keep:
                continue
            mass = self.mass(layer_idx)
            b, h, cap, _ = old.k_packed_buf.shape
            new_cap = min(cap, _round_up(max(keep, int(keep * self.growth), self.capacity_hint,
                                             CAPACITY_ALIGN), CAPACITY_ALIGN))
            bufs = [torch.empty(b, h, new_cap, t.shape[-1], dtype=t.dtype, device=t.device)
                    for t in (old.k_packed_buf, old.k_scales_buf, old.v_packed_buf, old.v_scales_buf)]
            new = LayerStore(*bufs, seq_len=keep, mass_buf=torch.zeros(b, h, new_cap, device=mass.device),
                             unscored=None if old.unscored is None else keep - (old.seq_len - old.unscored))
            index = torch.empty(b, h, keep, dtype=torch.int32, device=mass.device)
            ops.evict_into(mass, old.views(), new.views(), new.mass_buf[:, :, :keep], index,
                           recent, sinks)
            self._layers[layer_idx] = new
            kept[layer_idx] = index
        return kept

    def _reserve(self, key_states: torch.Tensor, value_states: torch.Tensor,
                 layer_idx: int) -> LayerStore:
        """Check the new states and make room for them (valid rows unchanged)."""
        if key_states.shape != value_states.shape or key_states.dim() != 4:
            raise ValueError("key/value states must both be [B, n_kv, s, d_head]")
        if key_states.dtype not in frontend.FLOATS or value_states.dtype != key_states.dtype:
            raise ValueError("key/value states must be bf16/fp16/fp32 of the same dtype")
        frontend._need_cuda("QuantizedKVCache.append", key_states, value_states)
        b, h, s, d = key_states.shape
        layer = self._layers.get(layer_idx)
        need = (layer.seq_len if layer else 0) + s
        if layer is None:
            cap = _round_up(max(need, self.capacity_hint, CAPACITY_ALIGN), CAPACITY_ALIGN)
            layer = self._alloc(key_states, b, h, cap, d)
            self._layers[layer_idx] = layer
        else:
            kb = layer.k_packed_buf
            if kb.shape[0] != b or kb.shape[1] != h or kb.device != key_states.device:
                raise ValueError("batch/head/device of appended states must match the cache")
            if need > layer.capacity:
                cap = _round_up(max(need, int(layer.capacity * self.growth)), CAPACITY_ALIGN)
                grown = self._alloc(key_states, b, h, cap, d)
                grown.k_scales_buf = grown.k_scales_buf.to(layer.k_scales_buf.dtype)
                grown.v_scales_buf = grown.v_scales_buf.to(layer.v_scales_buf.dtype)
                n = layer.seq_len
                for src, dst in zip(
                        (layer.k_packed_buf, layer.k_scales_buf, layer.v_packed_buf,
                         layer.v_scales_buf),
                        (grown.k_packed_buf, grown.k_scales_buf, grown.v_packed_buf,
                         grown.v_scales_buf)):
                    dst[:, :, :n].copy_(src[:, :, :n])
                if grown.mass_buf is not None:
                    grown.mass_buf[:, :, :n].copy_(layer.mass_buf[:, :, :n])
                grown.seq_len, grown.unscored = n, layer.unscored
                layer = grown
                self._layers[layer_idx] = layer
        return layer

    def crop(self, max_length: int) -> None:
        """Keep the first ``max_length`` tokens of every layer (negative: drop
        that many from the end), as ``DynamicCache.crop``."""
        for st in self._layers.values():
            n = max_length if max_length >= 0 else st.seq_len + max_length
            st.seq_len = max(0, min(st.seq_len, n))
            if st.unscored is not None and st.unscored >= st.seq_len:
                st.unscored = None

    def reorder(self, beam_idx: torch.Tensor) -> None:
        """Reorder the batch dimension of every layer (beam search)."""
        for st in self._layers.values():
            idx = beam_idx.to(st.k_packed_buf.device)
            for name in ("k_packed_buf", "k_scales_buf", "v_packed_buf", "v_scales_buf"):
                setattr(st, name, getattr(st, name).index_select(0, idx).contiguous())
            if st.mass_buf is not None:
                st.mass_buf = st.mass_buf.index_select(0, idx).contiguous()
            st.early_ok = False

    def layer(self, layer_idx: int) -> LayerStore:
        st = self._layers.get(layer_idx)
        if st is None:
            raise KeyError(f"no cache state for layer {layer_idx}")
        return st

    def dequantized(self, layer_idx: int, out_dtype: torch.dtype):
        st = self.layer(layer_idx)
        kp, ks, vp, vs = st.views()
        d_head = ks.shape[-1] * self.group_size
        k = frontend.dequantize(kp, ks, self.group_size, d_head, out_dtype)
        v = frontend.dequantize(vp, vs, self.group_size, d_head, out_dtype)
        return k, v

    def nbytes(self) -> int:
        """Logical bytes held (packed + scales over the valid tokens), like the
        reference's ``nbytes`` (``models/llama3/kv_cache.py:158-166``)."""
        total = 0
        for st in self._layers.values():
            for t in st.views():
                total += t.element_size() * t.numel()
        return total

    def capacity_nbytes(self) -> int:
        """Bytes actually reserved on the device (including headroom and scores)."""
        total = 0
        for st in self._layers.values():
            for t in (st.k_packed_buf, st.k_scales_buf, st.v_packed_buf, st.v_scales_buf, st.mass_buf):
                total += t.element_size() * t.numel() if t is not None else 0
        return total
