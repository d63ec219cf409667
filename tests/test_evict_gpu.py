"""Scored attention and eviction against 64-bit references (bounds in branch_ref)."""

from __future__ import annotations

import pytest
import torch

import branch_ref as br

pytestmark = pytest.mark.gpu


def _scored(b, hq, hkv, sq, s, d, group, dtype, *, causal=True, decay=1.0, sdtype=None, seed=0,
            in_place=False, strided=False):
    from kernels.llama3.evict import attention_forward_quant_gqa_scored
    cache = br.random_rows(b, hkv, s, d, group, sdtype or dtype, seed)
    g = torch.Generator().manual_seed(seed + 2)
    q = torch.randn(b, hq, sq, d, generator=g).to(dtype)
    mass = torch.rand(b, hkv, s, generator=g)
    dev, md = [t.cuda() for t in cache], mass.cuda()
    if strided:
        dev = []
        for t in cache:
            buf = torch.zeros(b, hkv, s + 37, t.shape[-1], dtype=t.dtype, device="cuda")
            buf[:, :, :s] = t.cuda()
            dev.append(buf[:, :, :s])
        md = torch.zeros(b, hkv, s + 37, device="cuda")
        md[:, :, :s] = mass.cuda()
        md = md[:, :, :s]
    to = None if in_place else torch.full((b, hkv, s), float("nan"), device="cuda")
    out, new = attention_forward_quant_gqa_scored(
        q.cuda(), *dev, md, n_q_heads=hq, n_kv_heads=hkv, group_size=group, is_causal=causal,
        decay=decay, mass_out=to)
    torch.cuda.synchronize()
    assert new is (md if in_place else to)
    if not in_place:
        assert torch.equal(md.cpu(), mass)
    k, v = br.values(*cache[:2], group, d), br.values(*cache[2:], group, d)
    seen = torch.ones(sq, s, dtype=torch.bool)
    if causal:
        seen = seen.tril(s - sq)
    r = hq // hkv
    for x in range(b):
        ref, p, X, A = br.attend(q[x].double(), k[x], v[x], seen)
        br.check_out(out[x], ref, X, A, s)
        add = p.reshape(hkv, r * sq, s)
        rel = br.weight_bound(X, d, s).reshape(hkv, r * sq, 1) + br.U32 * (r * sq + 8)
        want = decay * mass[x].double() + add.sum(1)
        bound = (rel * add).sum(1) + br.U32 * 2 * want.abs() + 1e-30
        err = (new[x].cpu().double() - want).abs()
        assert bool((err <= bound).all()), f"{float((err / bound).max()):.3g} times the bound"
    return out, new


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,group", [(128, 32), (64, 32), (128, 128), (64, 16)])
def test_single_token(dtype, d, group):
    _scored(2, 8, 2, 1, 333, d, group, dtype, seed=d)


@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 1), (6, 2), (14, 2), (64, 1)])
@pytest.mark.parametrize("sq", [1, 5])
def test_head_ratios(hq, hkv, sq):
    _scored(1, hq, hkv, sq, 260, 128, 32, torch.bfloat16, decay=0.5, seed=hq)


@pytest.mark.parametrize("s", [1, 31, 32, 33, 127, 128, 129, 257, 1000, 4100])
def test_lengths(s):
    _scored(1, 8, 2, 1, s, 128, 32, torch.bfloat16, seed=s)
    _scored(1, 2, 2, 1, s, 64, 32, torch.float32, seed=s)


@pytest.mark.parametrize("sq", [2, 16, 32, 33, 64, 100, 300])
@pytest.mark.parametrize("causal", [True, False])
def test_windows(sq, causal):
    _scored(1, 8, 2, sq, 300, 128, 32, torch.bfloat16, causal=causal, decay=0.9, seed=sq)


def test_queries_before_the_first_key_see_nothing():
    # more queries than tokens: the first rows are empty and weigh nothing
    out, _ = _scored(1, 8, 2, 40, 30, 128, 32, torch.bfloat16, seed=3)
    assert bool((out[:, :, :10] == 0).all())
    _scored(1, 8, 2, 40, 30, 64, 32, torch.float32, seed=3)


def test_in_place_and_strided():
    _scored(2, 8, 2, 1, 222, 128, 32, torch.bfloat16, in_place=True, strided=True, seed=4)
    _scored(2, 8, 2, 9, 222, 64, 32, torch.float32, in_place=True, strided=True, decay=0.25, seed=4)


@pytest.mark.parametrize("d,group", [(96, 32), (70, 32), (256, 64), (512, 128), (40, 5), (1, 1)])
def test_other_sizes(d, group):
    _scored(1, 4, 2, 3, 77, d, group, torch.bfloat16, seed=5)
    _scored(1, 4, 2, 3, 77, d, group, torch.float32, seed=5)


def test_mixed_scale_types():
    _scored(1, 8, 2, 2, 150, 128, 32, torch.bfloat16, sdtype=torch.float32, seed=6)
    _scored(1, 8, 2, 2, 150, 128, 32, torch.bfloat16, sdtype=torch.float16, seed=6)


def test_many_units_and_long_contexts():
    _scored(24, 8, 8, 1, 300, 128, 32, torch.bfloat16, seed=7)
    _scored(1, 4, 1, 1, 30000, 128, 32, torch.bfloat16, seed=8)


def test_same_bits_twice_and_on_a_side_stream():
    a = _scored(2, 8, 2, 7, 2000, 128, 32, torch.bfloat16, seed=9)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = _scored(2, 8, 2, 7, 2000, 128, 32, torch.bfloat16, seed=9)
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_scores_add_up():
    """Without decay a step adds exactly Hq / Hkv * queries per KV head, up to rounding."""
    from kernels.llama3.evict import attention_forward_quant_gqa_scored
    cache = [t.cuda() for t in br.random_rows(1, 2, 500, 128, 32, torch.bfloat16, 1)]
    mass = torch.zeros(1, 2, 500, device="cuda")
    for sq in (1, 4):
        q = torch.randn(1, 8, sq, 128, device="cuda").to(torch.bfloat16)
        attention_forward_quant_gqa_scored(q, *cache, mass, n_q_heads=8, n_kv_heads=2)
    total = mass.double().sum(-1)
    assert bool(((total - 4 * 5).abs() <= 20 * 500 * br.U32 * 8).all())


# ---------------------------------------------------------------------------
def _evict(mass, keep, recent, sinks, d=128, group=32, dtype=torch.bfloat16, strided=False, out=False):
    from kernels.llama3.evict import evict_by_mass
    b, h, s = mass.shape
    cache = br.random_rows(b, h, s, d, group, dtype, 3)
    dev, md = [t.cuda() for t in cache], mass.cuda()
    if strided:
        dev = [torch.cat((t, t[:, :, :9]), 2)[:, :, :s] for t in dev]
        md = torch.stack((md, md), -1)[..., 1]
    to = None
    if out:
        to = tuple(torch.zeros(b, h, keep + 11, *t.shape[3:], dtype=t.dtype, device="cuda")[:, :, :keep]
                   for t in (*dev, md))
    *got, new, index = evict_by_mass(*dev, md, keep=keep, recent=recent, sinks=sinks, out=to)
    torch.cuda.synchronize()
    want = br.evict_index(mass, keep, recent, sinks)
    assert torch.equal(index.cpu().long(), want)
    for c, g in zip(cache, got):
        assert torch.equal(g.cpu(), c.gather(2, want.unsqueeze(-1).expand(*want.shape, c.shape[-1])))
    assert torch.equal(new.cpu().view(torch.int32), mass.gather(2, want).view(torch.int32))


@pytest.mark.parametrize("s", [1, 2, 31, 64, 1000, 1023, 1024, 1025, 2500])
def test_evict_lengths(s):
    g = torch.Generator().manual_seed(s)
    mass = torch.rand(2, 3, s, generator=g)
    for keep in sorted({0, 1, s // 3, s - 1, s}):
        _evict(mass, keep, min(keep, s // 10), 0)
        _evict(mass, keep, 0, min(keep, 4))


@pytest.mark.parametrize("s", [5000, 20001, 70000])
def test_evict_long(s):
    g = torch.Generator().manual_seed(s)
    mass = (3 * torch.randn(1, 2, s, generator=g)).exp()
    mass[torch.rand(1, 2, s, generator=g) < 0.2] = 0.0
    _evict(mass, s // 4, 64, 4, d=64)
    _evict(mass, s - 5, 1, 1, d=64)


def test_evict_ties_go_to_the_earlier_token():
    mass = torch.zeros(1, 2, 700)
    mass[0, 1] = torch.randint(0, 3, (700,), generator=torch.Generator().manual_seed(0)).float()
    for keep in (1, 100, 350, 699):
        _evict(mass, keep, 0, 0)
        _evict(mass, keep, keep // 2, 0)
    mass[0, 0, ::2] = -0.0
    _evict(mass, 300, 5, 5)


def test_evict_special_scores():
    inf, nan = float("inf"), float("nan")
    mass = torch.tensor([0.5, -inf, nan, inf, 1e-40, -1e-40, 0.0, -0.0, -3.0, nan, inf, 3e38]).repeat(4)
    mass = mass.reshape(1, 1, -1)
    for keep in range(0, 49, 3):
        _evict(mass, keep, 0, 0)
        if keep >= 5:
            _evict(mass, keep, 3, 2)
    _evict(torch.full((1, 1, 50), nan), 20, 3, 2)


@pytest.mark.parametrize("d,group,dtype", [(64, 32, torch.float16), (70, 32, torch.bfloat16),
                                           (40, 5, torch.float32), (256, 64, torch.float32)])
def test_evict_layouts(d, group, dtype):
    mass = torch.rand(2, 2, 300, generator=torch.Generator().manual_seed(1))
    _evict(mass, 100, 10, 2, d, group, dtype)
    _evict(mass, 100, 10, 2, d, group, dtype, strided=True)
    _evict(mass, 100, 10, 2, d, group, dtype, out=True)


def test_evict_then_attend():
    """The kept rows are a cache like any other."""
    from kernels.llama3.attention_quant import attention_forward_quant_gqa
    from kernels.llama3.evict import evict_by_mass
    cache = br.random_rows(1, 2, 400, 128, 32, torch.bfloat16, 5)
    mass = torch.rand(1, 2, 400, generator=torch.Generator().manual_seed(2))
    *kept, _, index = evict_by_mass(*[t.cuda() for t in cache], mass.cuda(), keep=130, recent=8, sinks=2)
    q = torch.randn(1, 8, 1, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    out = attention_forward_quant_gqa(q.cuda(), *kept, n_q_heads=8, n_kv_heads=2, group_size=32)
    idx = index.cpu().long().unsqueeze(-1)
    k = br.values(*cache[:2], 32, 128).gather(2, idx.expand(-1, -1, -1, 128))
    v = br.values(*cache[2:], 32, 128).gather(2, idx.expand(-1, -1, -1, 128))
    ref = br.attend(q[0].double(), k[0], v[0], torch.ones(1, 130, dtype=torch.bool))[0]
    assert float((out[0].cpu().double() - ref).abs().max()) < 2e-2
