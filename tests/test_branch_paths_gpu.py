"""Tree and scored attention where the work is cut differently from the small
calls of test_tree_gpu and test_evict_gpu: groups of 16 (tensor-memory tiles
whatever the size), enough rows and keys for the tiles with any group, strides
that only the kernels for any shape read; and values in places no row may see.
References and bounds as there."""

from __future__ import annotations

import math

import pytest
import torch

import branch_ref as br
from test_evict_gpu import _scored
from test_tree_gpu import _run

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 300])
def test_tiles_node_counts(n):
    _run(1, 2, 1, n, 260, 128, 16, BF16, seed=n, want_lse=True)
    _run(2, 3, 3, n, 130, 64, 16, BF16, seed=n)


@pytest.mark.parametrize("s", [0, 1, 15, 16, 31, 127, 128, 129, 255, 256, 257, 384, 1025])
def test_tiles_context_lengths(s):
    _run(1, 8, 2, 5, s, 128, 16, BF16, seed=s)
    _run(2, 8, 2, 70, s, 64, 16, BF16, seed=s)


@pytest.mark.parametrize("n", [3, 40, 70])
def test_tiles_ragged_lengths(n):
    lens = [0, 1, 127, 128, 129, 383, 699, 700]
    _run(8, 8, 2, n, 700, 128, 16, BF16, lens=lens, seed=5, want_lse=True)


@pytest.mark.parametrize("n", [6, 40, 140])
def test_tiles_rows_that_see_nothing(n):
    mask = torch.zeros(2, n, n, dtype=torch.bool)
    mask[0, 3, 2] = mask[1, n - 1, 0] = mask[1, 5] = True
    got = _run(2, 4, 2, n, 200, 128, 16, BF16, lens=[0, 0], mask=mask, seed=9, want_lse=True)
    assert bool((got[0, :, 0] == 0).all()) and bool((got[1, :, 0] == 0).all())
    # nothing at all is seen
    got = _run(2, 4, 2, n, 0, 64, 16, BF16, mask=torch.zeros(n, n, dtype=torch.bool), seed=9, want_lse=True)
    assert bool((got == 0).all())


def test_tiles_general_masks_strides_and_lengths():
    g = torch.Generator().manual_seed(10)
    _run(3, 8, 2, 50, 90, 128, 16, BF16, mask=torch.rand(50, 50, generator=g) < 0.4, seed=10)
    wide = torch.rand(1, 150, 300, generator=g) < 0.5
    _run(1, 8, 2, 150, 90, 128, 16, BF16, mask=wide[:, :, ::2], seed=11)
    _run(2, 8, 2, 33, 40, 64, 16, BF16, mask=(torch.rand(2, 33, 33, generator=g) < 0.5).transpose(1, 2), seed=12)
    _run(2, 8, 2, 12, 333, 128, 16, BF16, strided=True, seed=13)
    _run(1, 8, 1, 6, 20000, 128, 16, BF16, seed=8, want_lse=True)
    _run(40, 8, 8, 3, 512, 64, 16, BF16, lens=[(37 * i) % 513 for i in range(40)], seed=6)


@pytest.mark.parametrize("q_scale,rows_scale", [(1e-3, 1.0), (1e4, 1e-2), (1e-2, 1e3), (30.0, 3.0)])
def test_tiles_magnitudes(q_scale, rows_scale):
    _run(1, 8, 2, 7, 300, 128, 16, BF16, q_scale=q_scale, rows_scale=rows_scale, seed=16)


@pytest.mark.parametrize("d,group", [(128, 32), (128, 64), (128, 128), (64, 32), (64, 64)])
def test_much_work(d, group):
    """Enough rows and keys for tensor-memory tiles with every group."""
    lens = [1600, 0, 1599, 777]
    _run(4, 32, 8, 33, 1600, d, group, BF16, lens=lens, seed=group, want_lse=True)
    _run(2, 24, 8, 129, 700, d, group, BF16, seed=group + 1)


@pytest.mark.parametrize("dtype,sdtype", [(torch.float16, torch.float16), (torch.float16, BF16), (BF16, torch.float16)])
def test_much_work_in_half_precision(dtype, sdtype):
    _run(2, 24, 8, 65, 700, 128, 32, dtype, sdtype=sdtype, seed=3, want_lse=True)


def test_rows_off_by_a_few_bytes():
    """Rows that start where only narrow loads may read, in every type."""
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    for dtype, d, group in ((BF16, 128, 32), (torch.float32, 64, 32), (torch.float16, 40, 8)):
        b, hq, hkv, n, s = 2, 4, 2, 5, 150
        cache = br.random_rows(b, hkv, s, d, group, dtype, 1)
        draft = br.random_rows(b, hkv, n, d, group, dtype, 2)
        q = torch.randn(b, hq, n, d, generator=torch.Generator().manual_seed(3)).to(dtype)
        mask = br.tree_mask(b, n, 4)
        want = None
        for off in (0, 1, 2, 4, 8):
            def shift(t):
                buf = torch.zeros(t.numel() + 16, dtype=t.dtype, device="cuda")
                view = buf[off:off + t.numel()].view(t.shape)
                view.copy_(t)
                return view
            got = tree_attention_quant_gqa(shift(q), *[shift(t) for t in cache], *[shift(t) for t in draft],
                                           mask.cuda(), n_q_heads=hq, n_kv_heads=hkv, group_size=group)
            for x in range(b):
                k, v = (torch.cat((br.values(*cache[i:i + 2], group, d)[x], br.values(*draft[i:i + 2], group, d)[x]), 1)
                        for i in (0, 2))
                seen = torch.ones(n, s + n, dtype=torch.bool)
                seen[:, s:] = mask[x]
                ref, _, X, A = br.attend(q[x].double(), k, v, seen)
                br.check_out(got[x], ref, X, A, s + n)


# path: group and amount of work that reach each of the kernels
PATHS = {"warps": (BF16, 1, 8, 2, 12, 300, 32), "tiles": (BF16, 1, 8, 2, 12, 300, 16),
         "two row tiles": (BF16, 4, 32, 8, 40, 1300, 32), "half": (torch.float16, 1, 8, 2, 12, 300, 32),
         "any shape": (torch.float32, 1, 8, 2, 12, 300, 32)}


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e4])
def test_unseen_rows_do_not_matter(path, bad):
    """Scales that are no numbers (or too large for f16 products) in drafted rows
    that a node does not see, and past context_lens: that node's output is the
    one without them.  A node that sees such a V row gets what the row holds."""
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    from kvint4 import ops
    dtype, b, hq, hkv, n, s, group = PATHS[path]
    d = 128
    cache = [t.cuda() for t in br.random_rows(b, hkv, s, d, group, dtype, 1)]
    draft = [t.cuda() for t in br.random_rows(b, hkv, n, d, group, dtype, 2)]
    q = torch.randn(b, hq, n, d, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    mask = br.tree_mask(b, n, 4).cuda()
    mask[:, :, 7] = False      # node 7's K and V are seen by nodes 7 and 9 alone
    mask[:, 7, 7] = mask[:, 9, 7] = True
    lens = torch.tensor([s - 5, 128, 1, s - 130][:b], dtype=torch.int32, device="cuda")

    def call():
        return tree_attention_quant_gqa(q, *cache, *draft, mask, n_q_heads=hq, n_kv_heads=hkv,
                                        group_size=group, context_lens=lens)

    want = call()
    for x in range(b):
        for t in (cache[1], cache[3]):
            t[x, :, int(lens[x]):] = bad
    ops.device_error()
    assert torch.equal(call(), want)
    assert ops.device_error() == 0
    for which in (1, 3):
        kept = draft[which][:, :, 7].clone()
        draft[which][:, :, 7] = bad
        got = call()
        draft[which][:, :, 7] = kept
        others = [i for i in range(n) if i not in (7, 9)]
        assert torch.equal(got[:, :, others], want[:, :, others])
        if not math.isfinite(bad) and which == 3:
            assert not bool(torch.isfinite(got[:, :, 7]).all(-1).any())
    ops.device_error()


@pytest.mark.parametrize("sq", [2, 32, 33, 100, 129, 300])
@pytest.mark.parametrize("causal", [True, False])
def test_scored_tiles_windows(sq, causal):
    _scored(1, 8, 2, sq, 300, 128, 16, BF16, causal=causal, decay=0.9, seed=sq)
    _scored(2, 2, 2, sq, 300, 64, 16, BF16, causal=causal, decay=0.9, seed=sq)


@pytest.mark.parametrize("s", [1, 31, 32, 33, 127, 128, 129, 257, 1000, 4100])
def test_scored_tiles_lengths(s):
    _scored(1, 8, 2, 1, s, 128, 16, BF16, seed=s)
    _scored(1, 8, 2, 7, s, 64, 16, BF16, seed=s)


def test_scored_tiles_empty_rows_in_place_and_strided():
    out, _ = _scored(1, 8, 2, 40, 30, 128, 16, BF16, seed=3)
    assert bool((out[:, :, :10] == 0).all())
    _scored(2, 8, 2, 9, 222, 128, 16, BF16, in_place=True, strided=True, decay=0.25, seed=4)


@pytest.mark.parametrize("d,group", [(128, 32), (128, 128), (64, 32)])
def test_scored_much_work(d, group):
    _scored(2, 64, 8, 32, 2000, d, group, BF16, decay=0.9, seed=group)
    _scored(3, 32, 8, 65, 1300, d, group, BF16, seed=group)


@pytest.mark.parametrize("dtype,sdtype", [(torch.float16, torch.float16), (BF16, torch.float16)])
def test_scored_much_work_in_half_precision(dtype, sdtype):
    _scored(2, 64, 8, 32, 700, 128, 32, dtype, sdtype=sdtype, decay=0.9, seed=3)


@pytest.mark.parametrize("dtype,group", [(BF16, 16), (BF16, 32), (torch.float16, 32), (torch.float32, 32)])
def test_output_layout_may_differ_from_the_queries(dtype, group):
    """An output that only element-wise stores can write takes another kernel."""
    from kernels.llama3.evict import attention_forward_quant_gqa_scored
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    b, hq, hkv, s, d = 2, 8, 2, 700, 128
    for n in (1, 3, 40):
        cache = [t.cuda() for t in br.random_rows(b, hkv, s, d, group, dtype, 1)]
        draft = [t.cuda() for t in br.random_rows(b, hkv, n, d, group, dtype, 2)]
        q = torch.randn(b, hq, n, d, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
        odd = torch.full((b, hq, n, d + 1), float("nan"), dtype=dtype, device="cuda")[..., 1:]
        mask = br.tree_mask(1, n, 4)[0].cuda()
        mass = torch.zeros(b, hkv, s, device="cuda")
        tree = tree_attention_quant_gqa(q, *cache, *draft, mask, n_q_heads=hq, n_kv_heads=hkv,
                                        group_size=group, out=odd)
        k, v = (torch.cat((br.values(*cache[i:i + 2], group, d), br.values(*draft[i:i + 2], group, d)), 2)
                for i in (0, 2))
        seen = torch.ones(n, s + n, dtype=torch.bool)
        seen[:, s:] = mask.cpu()
        for x in range(b):
            ref, _, X, A = br.attend(q[x].cpu().double(), k[x], v[x], seen)
            br.check_out(tree[x], ref, X, A, s + n)
        odd = torch.full((b, hq, n, d + 1), float("nan"), dtype=dtype, device="cuda")[..., 1:]
        out, new = attention_forward_quant_gqa_scored(q, *cache, mass, n_q_heads=hq, n_kv_heads=hkv,
                                                      group_size=group, is_causal=True, out=odd)
        seen = torch.ones(n, s, dtype=torch.bool).tril(s - n)
        for x in range(b):
            ref, p, X, A = br.attend(q[x].cpu().double(), k[x, :, :s], v[x, :, :s], seen)
            br.check_out(out[x], ref, X, A, s)
            add = p.reshape(hkv, -1, s)
            rel = br.weight_bound(X, d, s).reshape(hkv, -1, 1) + br.U32 * (add.shape[1] + 8)
            want = add.sum(1)
            assert bool(((new[x].cpu().double() - want).abs()
                         <= (rel * add).sum(1) + br.U32 * 2 * want + 1e-30).all())


@pytest.mark.parametrize("dtype", [BF16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,sq", [(8, 2, 4), (16, 1, 1), (17, 1, 1), (9, 1, 1), (8, 1, 1), (6, 2, 5)])
def test_scored_few_rows(dtype, hq, hkv, sq):
    for s in (17, 100, 1000, 9001):
        _scored(2, hq, hkv, sq, s, 128, 32, dtype, causal=True, decay=0.9, seed=s)
        _scored(2, hq, hkv, sq, s, 64, 64, dtype, causal=False, decay=0.9, seed=s)


@pytest.mark.parametrize("dtype", [BF16, torch.float16, torch.float32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, 3e4])
def test_unseen_rows_do_not_matter_to_few_rows(dtype, bad):
    """As above, for calls of at most eight rows per KV head."""
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    from kvint4 import ops
    b, h, n, s, d, group = 2, 2, 7, 200, 64, 32
    cache = [t.cuda() for t in br.random_rows(b, h, s, d, group, dtype, 1)]
    draft = [t.cuda() for t in br.random_rows(b, h, n, d, group, dtype, 2)]
    q = torch.randn(b, h, n, d, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    mask = br.tree_mask(b, n, 4).cuda()
    mask[:, :, 3] = False
    mask[:, 3, 3] = mask[:, 5, 3] = True
    lens = torch.tensor([s - 3, 17], dtype=torch.int32, device="cuda")

    def call():
        return tree_attention_quant_gqa(q, *cache, *draft, mask, n_q_heads=h, n_kv_heads=h,
                                        group_size=group, context_lens=lens)

    want = call()
    for x in range(b):
        for t in (cache[1], cache[3]):
            t[x, :, int(lens[x]):] = bad
    ops.device_error()
    assert torch.equal(call(), want)
    assert ops.device_error() == 0
    for which in (1, 3):
        kept = draft[which][:, :, 3].clone()
        draft[which][:, :, 3] = bad
        got = call()
        draft[which][:, :, 3] = kept
        others = [i for i in range(n) if i not in (3, 5)]
        assert torch.equal(got[:, :, others], want[:, :, others])
        if not math.isfinite(bad) and which == 3:
            assert not bool(torch.isfinite(got[:, :, 3]).all(-1).any())
    ops.device_error()


@pytest.mark.parametrize("dtype,group", [(BF16, 32), (BF16, 16), (torch.float16, 32), (torch.float32, 32)])
def test_offsets_past_32_bits(dtype, group):
    """Sequences of a cache that lie more than 2**32 elements apart."""
    from kernels.llama3.evict import attention_forward_quant_gqa_scored, evict_by_mass
    from kernels.llama3.tree_attention_quant import commit_draft_rows, tree_attention_quant_gqa
    b, hq, hkv, n, s, d, far = 2, 8, 2, 5, 300, 128, (1 << 32) + 4096
    room = torch.empty(far + (1 << 20), dtype=torch.uint8, device="cuda")
    wide = torch.empty(far + (1 << 20), dtype=dtype, device="cuda")
    small = [t.cuda() for t in br.random_rows(b, hkv, s, d, group, dtype, 1)]
    cache = []
    for i, t in enumerate(small):  # K's and V's tensors side by side in the same buffer
        src = wide if i & 1 else room
        v = src.as_strided(t.shape, (far, s * t.shape[3], t.shape[3], 1), (i >> 1) * (1 << 19))
        v.copy_(t)
        cache.append(v)
    draft = [t.cuda() for t in br.random_rows(b, hkv, n, d, group, dtype, 2)]
    q = torch.randn(b, hq, n, d, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    mask = br.tree_mask(b, n, 4).cuda()
    lens = torch.tensor([s - 9, 100], dtype=torch.int32, device="cuda")
    heads = dict(n_q_heads=hq, n_kv_heads=hkv, group_size=group)

    def calls(c):
        mass = torch.rand(b, hkv, s, generator=torch.Generator().manual_seed(5)).cuda()
        out = [tree_attention_quant_gqa(q, *c, *draft, mask, context_lens=lens, **heads)]
        out += attention_forward_quant_gqa_scored(q[:, :, :1].contiguous(), *c, mass, **heads)
        out += attention_forward_quant_gqa_scored(q, *c, mass, is_causal=True, **heads)
        out += evict_by_mass(*c, mass, keep=100, recent=5, sinks=2)
        path = torch.tensor([[0, 2, 4], [1, 3, 0]], dtype=torch.int32, device="cuda")
        out.append(commit_draft_rows(*c, *draft, path, torch.tensor([3, 2], dtype=torch.int32, device="cuda"),
                                     context_lens=lens))
        return out + [t.clone() for t in c]

    for got, want in zip(calls(cache), calls([t.clone() for t in small])):
        assert torch.equal(got, want)


@pytest.mark.parametrize("nodes", [3, 4, 5])
@pytest.mark.parametrize("d,group", [(512, 32), (200, 8), (64, 16), (96, 32)])
def test_any_shape_row_counts(nodes, d, group):
    _run(2, 2, 2, nodes, 150, d, group, torch.float32, seed=d)
    _scored(2, 2, 2, nodes, 150, d, group, torch.float32, causal=True, seed=d)
