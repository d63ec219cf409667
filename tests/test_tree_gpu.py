"""Tree attention and path commit against 64-bit references (bounds in branch_ref)."""

from __future__ import annotations

import pytest
import torch

import branch_ref as br

pytestmark = pytest.mark.gpu


def _run(b, hq, hkv, n, s, d, group, dtype, *, lens=None, mask=None, sdtype=None, seed=0,
         q_scale=1.0, rows_scale=1.0, strided=False, want_lse=False):
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    from kvint4 import ops
    sdtype = sdtype or dtype
    cache = br.random_rows(b, hkv, s, d, group, sdtype, seed, rows_scale)
    draft = br.random_rows(b, hkv, n, d, group, sdtype, seed + 1, rows_scale)
    g = torch.Generator().manual_seed(seed + 2)
    q = (q_scale * torch.randn(b, hq, n, d, generator=g)).to(dtype)
    mask = br.tree_mask(b, n, seed + 3) if mask is None else mask
    dev = [t.cuda() for t in cache]
    if strided:  # capacity views, and q / out as [B, n, H, d] storage
        dev = []
        for t in cache:
            buf = torch.full((b, hkv, s + 70, t.shape[-1]), 255, dtype=torch.uint8).to(t.dtype).cuda()
            buf[:, :, :s] = t.cuda()
            dev.append(buf[:, :, :s])
        qd = q.transpose(1, 2).contiguous().cuda().transpose(1, 2)
        out = torch.full((b, n, hq, d), float("nan"), dtype=dtype, device="cuda").transpose(1, 2)
    else:
        qd = q.cuda()
        out = torch.full((b, hq, n, d), float("nan"), dtype=dtype, device="cuda")
    lse = torch.full((b, hq, n), float("nan"), device="cuda") if want_lse else None
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda") if lens is not None else None
    got = tree_attention_quant_gqa(qd, *dev, *[t.cuda() for t in draft], mask.cuda(),
                                   n_q_heads=hq, n_kv_heads=hkv, group_size=group,
                                   context_lens=lt, out=out, lse=lse)
    assert got is out
    torch.cuda.synchronize()
    kc, vc = br.values(*cache[:2], group, d), br.values(*cache[2:], group, d)
    kd, vd = br.values(*draft[:2], group, d), br.values(*draft[2:], group, d)
    for x in range(b):
        live = s if lens is None else lens[x]
        if not 0 <= live <= s:
            live = 0
        k, v = torch.cat((kc[x, :, :live], kd[x]), 1), torch.cat((vc[x, :, :live], vd[x]), 1)
        seen = torch.ones(n, live + n, dtype=torch.bool)
        seen[:, live:] = mask[x] if mask.dim() == 3 else mask
        ref, p, X, A = br.attend(q[x].double(), k, v, seen)
        br.check_out(got[x], ref, X, A, live + n)
        if want_lse:
            sc = (q[x].double() @ k.repeat_interleave(hq // hkv, 0).transpose(1, 2)) * d ** -0.5
            ref_lse = torch.logsumexp(sc.masked_fill(~seen, -float("inf")), -1)
            bound = br.U32 * ((d + 8) * X * 2 + 2 * (live + n + 64)) + br.U32 * 4 * ref_lse.abs()
            have = lse[x].cpu().double()
            empty = torch.isinf(ref_lse)
            assert torch.equal(torch.isinf(have), empty)
            assert bool(((have - ref_lse).abs()[~empty] <= bound[~empty]).all())
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,group", [(128, 32), (64, 64), (128, 128), (64, 16)])
def test_types_and_head_sizes(dtype, d, group):
    _run(2, 8, 2, 9, 300, d, group, dtype, seed=d + group)


@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 1), (6, 2), (7, 1), (10, 2), (64, 1)])
def test_head_ratios(hq, hkv):
    _run(1, hq, hkv, 11, 200, 128, 32, torch.bfloat16, seed=hq)


@pytest.mark.parametrize("n", [1, 2, 16, 31, 32, 33, 64, 65, 127, 128, 129, 200])
def test_node_counts(n):
    _run(1, 8, 2, n, 260, 128, 32, torch.bfloat16, seed=n)


@pytest.mark.parametrize("s", [0, 1, 15, 31, 32, 33, 127, 128, 129, 255, 256, 257, 500, 1025])
def test_context_lengths(s):
    _run(1, 8, 2, 5, s, 128, 32, torch.bfloat16, seed=s)
    _run(2, 3, 3, 5, s, 64, 32, torch.float32, seed=s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ragged_lengths(dtype):
    s = 700
    lens = [0, 1, 127, 128, 129, 383, 699, 700]
    _run(8, 8, 2, 13, s, 128, 32, dtype, lens=lens, seed=5, want_lse=True)


def test_many_units_share_the_gpu():
    # more (sequence, KV head) units than SMs, of uneven lengths
    lens = [(37 * i) % 513 for i in range(40)]
    _run(40, 8, 8, 3, 512, 64, 32, torch.bfloat16, lens=lens, seed=6)
    _run(40, 16, 8, 40, 512, 128, 64, torch.bfloat16, lens=lens, seed=7)


def test_long_context_is_split():
    _run(1, 8, 1, 6, 20000, 128, 32, torch.bfloat16, seed=8, want_lse=True)
    _run(1, 2, 1, 6, 20000, 64, 32, torch.float32, seed=8, want_lse=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_see_nothing(dtype):
    n = 40
    mask = torch.zeros(2, n, n, dtype=torch.bool)
    mask[0, 3, 7] = mask[1, 39, 0] = mask[1, 5] = True
    got = _run(2, 8, 2, n, 200, 128, 32, dtype, lens=[0, 0], mask=mask, seed=9, want_lse=True)
    assert bool((got[0, :, 0] == 0).all()) and bool((got[1, :, 0] == 0).all())


def test_mask_is_general():
    # not a tree: any pattern, and one mask for the whole batch
    g = torch.Generator().manual_seed(10)
    _run(3, 8, 2, 50, 90, 128, 32, torch.bfloat16, mask=torch.rand(50, 50, generator=g) < 0.4, seed=10)
    wide = torch.rand(1, 150, 300, generator=g) < 0.5
    _run(1, 8, 2, 150, 90, 128, 32, torch.bfloat16, mask=wide[:, :, ::2], seed=11)  # strided
    _run(2, 8, 2, 33, 40, 64, 32, torch.float32,
         mask=(torch.rand(2, 33, 33, generator=g) < 0.5).transpose(1, 2), seed=12)


def test_strided_cache_query_and_output():
    _run(2, 8, 2, 12, 333, 128, 32, torch.bfloat16, strided=True, seed=13)
    _run(2, 8, 2, 12, 333, 64, 32, torch.float16, strided=True, seed=13)


@pytest.mark.parametrize("d,group", [(96, 32), (70, 32), (256, 64), (512, 128), (40, 5), (8, 8), (1, 1)])
def test_other_sizes(d, group):
    _run(1, 4, 2, 6, 77, d, group, torch.bfloat16, seed=14)
    _run(1, 4, 2, 6, 77, d, group, torch.float32, seed=14)


def test_mixed_scale_types():
    _run(1, 8, 2, 6, 150, 128, 32, torch.bfloat16, sdtype=torch.float32, seed=15)
    _run(1, 8, 2, 6, 150, 128, 32, torch.bfloat16, sdtype=torch.float16, seed=15)
    _run(1, 8, 2, 6, 150, 128, 32, torch.float32, sdtype=torch.bfloat16, seed=15)


@pytest.mark.parametrize("q_scale,rows_scale", [(1e-3, 1.0), (1e4, 1e-2), (1e-2, 1e3), (30.0, 3.0)])
def test_magnitudes(q_scale, rows_scale):
    _run(1, 8, 2, 7, 300, 128, 32, torch.bfloat16, q_scale=q_scale, rows_scale=rows_scale, seed=16)


def test_same_bits_twice():
    a = _run(3, 8, 2, 20, 900, 128, 32, torch.bfloat16, lens=[900, 10, 400], seed=17)
    assert torch.equal(a, _run(3, 8, 2, 20, 900, 128, 32, torch.bfloat16, lens=[900, 10, 400], seed=17))


def test_bad_length_is_reported_and_reads_as_zero():
    from kvint4 import ops
    ops.device_error()
    _run(3, 8, 2, 4, 100, 128, 32, torch.bfloat16, lens=[101, -1, 100], seed=18)
    assert ops.device_error() == 16
    assert ops.device_error() == 0


def test_side_stream():
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _run(2, 8, 2, 9, 1500, 128, 32, torch.bfloat16, seed=19)


@pytest.mark.parametrize("seen", [0, 5])
def test_cuda_graph_replay(seen):
    """A captured call replays with new inputs (lengths included) in its buffers."""
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    b, hq, hkv, n, s, d = 2, 8, 2, 6, 400, 128
    q = torch.randn(b, hq, n, d, device="cuda").to(torch.bfloat16)
    cache = [t.cuda() for t in br.random_rows(b, hkv, s, d, 32, torch.bfloat16, 1)]
    draft = [t.cuda() for t in br.random_rows(b, hkv, n, d, 32, torch.bfloat16, 2)]
    mask = br.tree_mask(b, n, 3).cuda()
    lens = torch.tensor([400, 399], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)

    def call(o):
        return tree_attention_quant_gqa(q, *cache, *draft, mask, n_q_heads=hq, n_kv_heads=hkv,
                                        group_size=32, context_lens=lens, out=o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    lens.copy_(torch.tensor([seen, 250], dtype=torch.int32))
    q.mul_(0.5)
    graph.replay()
    want = call(torch.empty_like(q))
    assert torch.equal(out, want)


def test_commit_moves_the_accepted_rows():
    from kernels.llama3.tree_attention_quant import commit_draft_rows
    from kvint4 import ops
    b, h, cap, n, d = 5, 3, 90, 12, 128
    for dtype, group in ((torch.bfloat16, 32), (torch.float32, 64), (torch.float16, 5)):
        cache = [t.cuda() for t in br.random_rows(b, h, cap, d, group, dtype, 1)]
        draft = [t.cuda() for t in br.random_rows(b, h, n, d, group, dtype, 2)]
        lens = torch.tensor([0, 1, 86, 40, 90], dtype=torch.int32, device="cuda")
        acc = torch.tensor([4, 0, 4, 1, 0], dtype=torch.int32, device="cuda")
        path = torch.tensor([[0, 3, 7, 11], [0, 1, 2, 3], [1, 2, 5, 6], [11, 0, 0, 0], [0, 0, 0, 0]],
                            dtype=torch.int32, device="cuda")
        want = [t.clone() for t in cache]
        for x in range(b):
            for j in range(int(acc[x])):
                for w, f in zip(want, draft):
                    w[x, :, int(lens[x]) + j] = f[x, :, int(path[x, j])]
        views = cache
        new = commit_draft_rows(*views, *draft, path, acc, context_lens=lens)
        assert torch.equal(new, lens + acc)
        for c, w in zip(cache, want):
            assert torch.equal(c, w)
        assert ops.device_error() == 0


def test_commit_leaves_what_does_not_fit():
    from kernels.llama3.tree_attention_quant import commit_draft_rows
    from kvint4 import ops
    cache = [t.cuda() for t in br.random_rows(5, 2, 16, 64, 32, torch.bfloat16, 1)]
    draft = [t.cuda() for t in br.random_rows(5, 2, 4, 64, 32, torch.bfloat16, 2)]
    before = [t.clone() for t in cache]
    lens = torch.tensor([15, -1, 3, 3, 16], dtype=torch.int32, device="cuda")
    acc = torch.tensor([2, 1, 3, -1, 1], dtype=torch.int32, device="cuda")  # 3 > width
    path = torch.tensor([[0, 1]] * 5, dtype=torch.int32, device="cuda")
    ops.device_error()
    new = commit_draft_rows(*cache, *draft, path, acc, context_lens=lens)
    assert torch.equal(new, lens)
    for c, w in zip(cache, before):
        assert torch.equal(c, w)
    assert ops.device_error() == 16
    # a node outside the draft is skipped
    path = torch.tensor([[9, 1]] * 5, dtype=torch.int32, device="cuda")
    lens = torch.full((5,), 2, dtype=torch.int32, device="cuda")
    new = commit_draft_rows(*cache, *draft, path, torch.full_like(lens, 2), context_lens=lens)
    assert ops.device_error() == 16
    assert torch.equal(cache[0][:, :, 2], before[0][:, :, 2])
    assert torch.equal(cache[0][:, :, 3], draft[0][:, :, 1])
