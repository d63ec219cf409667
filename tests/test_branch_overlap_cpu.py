"""Refusals of outputs that overlap what is read or one another (no GPU needed), and
the test for overlap itself against element addresses."""

from __future__ import annotations

import random

import pytest
import torch

import branch_ref as br

F32 = torch.float32


def _addresses(t):
    at = [t.data_ptr()]
    for n, st in zip(t.shape, t.stride()):
        at = [x + t.element_size() * st * k for x in at for k in range(n)]
    return {x + e for x in at for e in range(t.element_size())}


@pytest.mark.parametrize("seed", range(8))
def test_overlap_by_addresses(seed):
    from kernels.llama3._checks import overlap
    rnd = random.Random(seed)
    buf = torch.zeros(400, dtype=torch.uint8)

    def view():
        base = buf.view(rnd.choice((torch.uint8, torch.int16, F32)))
        while True:
            shape = [rnd.randint(1, 4) for _ in range(rnd.randint(1, 4))]
            strides = [rnd.choice((0, 1, 2, 3, 4, 5, 8, 12, 16, 24, 32)) for _ in shape]
            need = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
            if need < base.numel():
                return base.as_strided(shape, strides, rnd.randint(0, base.numel() - need))

    seen = set()
    for _ in range(400):
        a, b = view(), view()
        want = bool(_addresses(a) & _addresses(b))
        assert overlap(a, b) == want
        seen.add(want)
    assert seen == {True, False}


def test_overlap_of_cache_views():
    from kernels.llama3._checks import overlap
    buf = torch.zeros(4, 2, 8, 1000, 64, dtype=torch.uint8)
    assert overlap(buf[0, :, :, :300], buf[0, :, :, 299:])
    assert not overlap(buf[0, :, :, :300], buf[0, :, :, 300:600])   # interleaved heads
    assert not overlap(buf[:, 0], buf[:, 1])
    assert not overlap(buf[0][..., :32], buf[0][..., 32:])
    assert not overlap(buf[:0], buf)


def _rows(s=8, d=64):
    return br.random_rows(1, 2, s, d, 32, torch.bfloat16, 0)


def test_eviction_refuses_its_own_buffers():
    from kernels.llama3.evict import evict_by_mass
    cache, mass = _rows(), torch.zeros(1, 2, 8)

    def out():
        return [t.clone() for t in _rows(4)] + [torch.zeros(1, 2, 4)]

    with pytest.raises(ValueError, match="CUDA"):
        evict_by_mass(*cache, mass, keep=4, out=out())
    for i, t in enumerate((*cache, mass)):
        bad = out()
        bad[i] = t[:, :, :4]
        with pytest.raises(ValueError, match="overlap"):
            evict_by_mass(*cache, mass, keep=4, out=bad)
    bad = out()
    bad[2] = bad[0]
    with pytest.raises(ValueError, match=r"overlap out\[0\]"):
        evict_by_mass(*cache, mass, keep=4, out=bad)
    bad = out()
    bad[4] = torch.zeros(1, 1, 4).expand(1, 2, 4)
    with pytest.raises(ValueError, match="expanded"):
        evict_by_mass(*cache, mass, keep=4, out=bad)
    # halves of one buffer do not overlap, although their extents do
    buf = torch.zeros(1, 2, 2, 4)
    with pytest.raises(ValueError, match="CUDA"):
        evict_by_mass(*[t[:, :, :4] for t in cache], buf[:, :, 0], keep=4, out=out()[:4] + [buf[:, :, 1]])


def test_scored_attention_refuses_overlaps():
    from kernels.llama3.evict import attention_forward_quant_gqa_scored as call
    cache, heads = _rows(), dict(n_q_heads=4, n_kv_heads=2)
    q, mass = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 9)
    with pytest.raises(ValueError, match="CUDA"):
        call(q, *cache, mass[..., :8], mass_out=mass[..., :8], **heads)
    with pytest.raises(ValueError, match="mass_out must not overlap mass"):
        call(q, *cache, mass[..., :8], mass_out=mass[..., 1:], **heads)
    with pytest.raises(ValueError, match="expanded"):
        call(q, *cache, torch.zeros(1, 1, 8).expand(1, 2, 8), **heads)
    with pytest.raises(ValueError, match="out must not overlap q"):
        call(q, *cache, mass[..., :8], out=q, **heads)


def test_tree_attention_refuses_overlaps():
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    cache, draft, heads = _rows(), _rows(3), dict(n_q_heads=4, n_kv_heads=2)
    room = torch.zeros(1, 4, 4, 64, dtype=torch.bfloat16)
    q, mask = room[:, :, :3], torch.ones(3, 3, dtype=torch.bool)
    with pytest.raises(ValueError, match="CUDA"):
        tree_attention_quant_gqa(q, *cache, *draft, mask, out=q, **heads)
    with pytest.raises(ValueError, match="out must not overlap q"):
        tree_attention_quant_gqa(q, *cache, *draft, mask, out=room[:, :, 1:], **heads)
    with pytest.raises(ValueError, match="expanded"):
        tree_attention_quant_gqa(q, *cache, *draft, mask, lse=torch.zeros(1, 1, 3).expand(1, 4, 3), **heads)


def test_commit_refuses_overlaps():
    from kernels.llama3.tree_attention_quant import commit_draft_rows
    cache, draft, path = _rows(), _rows(3), torch.zeros(1, 2, dtype=torch.int32)
    n = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="draft_k_packed"):
        commit_draft_rows(*cache, cache[0][:, :, 5:], *draft[1:], path, n[:1], context_lens=n[1:])
    with pytest.raises(ValueError, match="lens_out must not overlap accepted"):
        commit_draft_rows(*cache, *draft, path, n[:1], context_lens=n[1:], lens_out=n[:1])
    with pytest.raises(ValueError, match="lens_out must not be context_lens"):
        commit_draft_rows(*cache, *draft, path, n[:1], context_lens=n[1:], lens_out=n[1:])
    with pytest.raises(ValueError, match="CUDA"):
        commit_draft_rows(*cache, *draft, path, n[:1], context_lens=n[1:])
