"""Tree and scored attention over scales of any size, alike in all rows or many
powers of two apart, on every kernel.

Bounds: those of branch_ref, and what a power of two common to several rows leaves
out.  A kernel that holds scales in f16 multiplies them by 2^e such that the largest
of them comes to at least 2^10 (or leaves them alone where all are exact), so a value
is off by at most half of f16's smallest step, 2^-25 / 2^10 of the largest scale of
its sequence and head:

* output: sum_t p_t * 2^-35 * max scale of V <= 2^-35 * max scale of V;
* scores: sum_c |q_c| * 2^-35 * max scale of K * sm_scale =: E, hence a weight by
  e^E - 1 <= 2 E relative and a normalised one by twice that.
"""

from __future__ import annotations

import math

import pytest
import torch

import branch_ref as br

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

# batch, q heads, KV heads, nodes, context, head size, group: each reaches a kernel of its own
PATHS = {
    "up to 8 rows": (2, 2, 2, 3, 500, 128, 32),
    "up to 8 rows, d 64": (2, 4, 2, 3, 500, 64, 64),
    "warps": (2, 8, 2, 12, 300, 128, 32),
    "one row tile": (2, 8, 2, 12, 700, 128, 16),
    "one full row tile, d 64": (2, 8, 2, 30, 700, 64, 16),
    "two row tiles": (4, 32, 8, 40, 1300, 128, 32),
    "two row tiles, long": (1, 64, 8, 40, 5000, 128, 128),
    "any shape": (2, 4, 2, 5, 200, 96, 32),
}


def _spread(rows, seed, low, pattern):
    """Multiply the scales of K and V by powers of ten from 10^low to 1."""
    g = torch.Generator().manual_seed(seed)
    for i in (1, 3):
        b, h, s, ng = rows[i].shape
        if pattern == "random":
            f = 10.0 ** (low * torch.rand(b, h, s, ng, generator=g))
        elif pattern == "falling":  # the largest first
            f = 10.0 ** (low * torch.linspace(0, 1, max(s, 1))).reshape(1, 1, s, 1).expand(b, h, s, ng)
        else:  # "rising"
            f = 10.0 ** (low * torch.linspace(1, 0, max(s, 1))).reshape(1, 1, s, 1).expand(b, h, s, ng)
        rows[i] = (rows[i].float() * f).to(rows[i].dtype)
    return rows


def _limits(q, ks, vs, X, d):
    """What the two lines of the module's comment add: to outputs, to weights (relative)."""
    r = q.shape[0] // ks.shape[0]
    kmax, vmax = (t.cpu().double().abs().amax((-1, -2)).repeat_interleave(r, 0) for t in (ks, vs))
    e = q.double().abs().sum(-1) * kmax.unsqueeze(1) * 2.0 ** -35 * d ** -0.5
    return 2.0 ** -35 * vmax.reshape(-1, 1, 1), 4 * e


def _check(got, q, k, v, ks, vs, seen, keys):
    """One sequence: got [Hq, n, d]."""
    d = q.shape[-1]
    ref, p, X, A = br.attend(q.double(), k, v, seen)
    add, more = _limits(q, ks, vs, X, d)
    dt = got.dtype
    rel = (br.weight_bound(X, d, keys) + more).unsqueeze(-1) + br.U32 * 2 * (keys + 64)
    if dt != F32:
        rel = rel + 2.0 ** -11
    bound = br.U_OUT[dt] * (ref.abs() + rel * A) + rel * A + br.TINY[dt] + add * (1 + br.U_OUT[dt])
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all()
    assert bool((err <= bound).all()), f"{float((err / bound).max()):.3g} times the bound"
    return p, (br.weight_bound(X, d, keys) + more)


def _tree(shape, dtype, rows_scale=1.0, q_scale=None, spread=None, seed=0):
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    from kvint4 import ops
    b, hq, hkv, n, s, d, group = shape
    cache = br.random_rows(b, hkv, s, d, group, dtype, seed, rows_scale)
    draft = br.random_rows(b, hkv, n, d, group, dtype, seed + 1, rows_scale)
    if spread:
        cache, draft = _spread(cache, seed, *spread), _spread(draft, seed + 5, spread[0], "random")
    g = torch.Generator().manual_seed(seed + 2)
    q = ((0.5 / rows_scale if q_scale is None else q_scale) * torch.randn(b, hq, n, d, generator=g)).to(dtype)
    mask = br.tree_mask(b, n, seed + 3)
    lens = [max(0, s - 131 * i) for i in range(b)]
    ops.device_error()
    got = tree_attention_quant_gqa(q.cuda(), *[t.cuda() for t in cache], *[t.cuda() for t in draft], mask.cuda(),
                                   n_q_heads=hq, n_kv_heads=hkv, group_size=group,
                                   context_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert ops.device_error() == 0
    for x in range(b):
        c, f = [t[x, :, :lens[x]] for t in cache], [t[x] for t in draft]
        rows = [torch.cat(t, 1) for t in zip(c, f)]
        seen = torch.ones(n, lens[x] + n, dtype=torch.bool)
        seen[:, lens[x]:] = mask[x]
        _check(got[x], q[x], br.values(*rows[:2], group, d), br.values(*rows[2:], group, d), rows[1], rows[3],
               seen, lens[x] + n)


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("rows_scale", [1e-20, 1e-8, 1e-6, 1e-4, 1e5, 1e10])
def test_tree_scales(path, rows_scale):
    _tree(PATHS[path], BF16, rows_scale, seed=3)


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("low", [-3, -7, -12, -25])
@pytest.mark.parametrize("pattern", ["random", "falling", "rising"])
def test_tree_scales_apart(path, low, pattern):
    _tree(PATHS[path], BF16, q_scale=1.0, spread=(low, pattern), seed=4)


@pytest.mark.parametrize("path", ["up to 8 rows", "warps", "any shape"])
@pytest.mark.parametrize("rows_scale", [1e-4, 1e-2, 1e4])
def test_tree_scales_in_half_precision(path, rows_scale):
    _tree(PATHS[path], F16, rows_scale, q_scale=min(1e3, 0.5 / rows_scale) if rows_scale < 1 else 1e-3, seed=5)


@pytest.mark.parametrize("path", PATHS)
def test_large_rows_that_few_nodes_see(path):
    """Drafted rows 2^60 larger than the rest: the nodes that do not see them keep
    what they have without them."""
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    b, hq, hkv, n, s, d, group = PATHS[path]
    cache = [t.cuda() for t in br.random_rows(b, hkv, s, d, group, BF16, 1, 1e-6)]
    draft = [t.cuda() for t in br.random_rows(b, hkv, n, d, group, BF16, 2, 1e-6)]
    q = (1e5 * torch.randn(b, hq, n, d, generator=torch.Generator().manual_seed(3))).to(BF16).cuda()
    mask = torch.eye(n, dtype=torch.bool, device="cuda")

    def call():
        return tree_attention_quant_gqa(q, *cache, *draft, mask, n_q_heads=hq, n_kv_heads=hkv, group_size=group)

    want = call()
    draft[3][:, :, 1] *= 2.0 ** 20
    got = call()
    others = [i for i in range(n) if i != 1]
    assert torch.equal(got[:, :, others], want[:, :, others])


# ---------------------------------------------------------------------------
SCORED = {
    "one query": (2, 8, 2, 1, 700, 128, 32),
    "one query, d 64": (2, 2, 2, 1, 700, 64, 32),
    "warps": (2, 8, 2, 12, 700, 128, 32),
    "one row tile": (2, 8, 2, 12, 700, 128, 16),
    "several row tiles": (1, 8, 2, 70, 700, 128, 16),
    "tiles, d 64": (2, 8, 2, 20, 700, 64, 16),
    "much work": (2, 64, 8, 32, 2000, 128, 32),
    "any shape": (2, 4, 2, 20, 200, 96, 32),
}


def _scored(shape, rows_scale=1.0, q_scale=None, spread=None, seed=0):
    from kernels.llama3.evict import attention_forward_quant_gqa_scored
    from kvint4 import ops
    b, hq, hkv, sq, s, d, group = shape
    cache = br.random_rows(b, hkv, s, d, group, BF16, seed, rows_scale)
    if spread:
        cache = _spread(cache, seed, *spread)
    g = torch.Generator().manual_seed(seed + 2)
    q = ((0.5 / rows_scale if q_scale is None else q_scale) * torch.randn(b, hq, sq, d, generator=g)).to(BF16)
    mass = torch.rand(b, hkv, s, generator=g)
    ops.device_error()
    out, new = attention_forward_quant_gqa_scored(
        q.cuda(), *[t.cuda() for t in cache], mass.cuda(), n_q_heads=hq, n_kv_heads=hkv, group_size=group,
        is_causal=True, decay=0.5)
    assert ops.device_error() == 0
    seen = torch.ones(sq, s, dtype=torch.bool).tril(s - sq)
    for x in range(b):
        rows = [t[x] for t in cache]
        p, rel = _check(out[x], q[x], br.values(*rows[:2], group, d), br.values(*rows[2:], group, d), rows[1],
                        rows[3], seen, s)
        r = hq // hkv
        add = p.reshape(hkv, r * sq, s)
        rel = rel.reshape(hkv, r * sq, 1) + br.U32 * (r * sq + 8)
        want = 0.5 * mass[x].double() + add.sum(1)
        bound = (rel * add).sum(1) + br.U32 * 2 * want.abs() + 1e-30
        err = (new[x].cpu().double() - want).abs()
        assert bool((err <= bound).all()), f"{float((err / bound).max()):.3g} times the bound"


@pytest.mark.parametrize("path", SCORED)
@pytest.mark.parametrize("rows_scale", [1e-20, 1e-8, 1e-6, 1e-4, 1e5, 1e10])
def test_scored_scales(path, rows_scale):
    _scored(SCORED[path], rows_scale, seed=6)


@pytest.mark.parametrize("path", SCORED)
@pytest.mark.parametrize("low", [-7, -25])
@pytest.mark.parametrize("pattern", ["random", "falling"])
def test_scored_scales_apart(path, low, pattern):
    _scored(SCORED[path], q_scale=1.0, spread=(low, pattern), seed=7)


# f16 scales from 8192 on, whose products with codes f16 does not hold: a cache of
# f16 values holds scales of up to 65504 / 7
@pytest.mark.parametrize("path", ["up to 8 rows", "warps", "any shape"])
@pytest.mark.parametrize("where", ["first", "last", "draft", "all"])
def test_large_f16_scales(path, where):
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    from kvint4 import ops
    b, hq, hkv, n, s, d, group = PATHS[path]
    cache, draft = br.random_rows(b, hkv, s, d, group, F16, 1), br.random_rows(b, hkv, n, d, group, F16, 2)
    for rows, part in (("first", cache[3][:, :, :40]), ("last", cache[3][:, :, -40:]), ("draft", draft[3])):
        if where in (rows, "all"):
            part.copy_(part.float() * (9350.0 / 0.45))  # 1039 .. 9350
            cache[2][:, :, :40] |= 0x88  # codes 8 .. 15: no value past f16's largest
            cache[2][:, :, -40:] |= 0x88
            draft[2] |= 0x88
    q = torch.randn(b, hq, n, d, generator=torch.Generator().manual_seed(3)).to(F16)
    mask = br.tree_mask(b, n, 4)
    ops.device_error()
    got = tree_attention_quant_gqa(q.cuda(), *[t.cuda() for t in cache], *[t.cuda() for t in draft], mask.cuda(),
                                   n_q_heads=hq, n_kv_heads=hkv, group_size=group)
    assert ops.device_error() == 0
    for x in range(b):
        rows = [torch.cat((c[x], f[x]), 1) for c, f in zip(cache, draft)]
        seen = torch.ones(n, s + n, dtype=torch.bool)
        seen[:, s:] = mask[x]
        _check(got[x], q[x], br.values(*rows[:2], group, d), br.values(*rows[2:], group, d), rows[1], rows[3],
               seen, s + n)


@pytest.mark.parametrize("path", [p for p in PATHS if p != "any shape"])
def test_a_hidden_row_out_of_all_proportion(path):
    """A drafted row 2^180 larger than the rest takes the bits of the rows beside it, and
    nothing else: what does not see it stays as small as it was."""
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    b, hq, hkv, n, s, d, group = PATHS[path]
    cache = [t.cuda() for t in br.random_rows(b, hkv, s, d, group, BF16, 1, 1e-25)]
    draft = [t.cuda() for t in br.random_rows(b, hkv, n, d, group, BF16, 2, 1e-25)]
    draft[3][:, :, 1] = 2.0 ** 99
    q = torch.randn(b, hq, n, d, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    mask = torch.eye(n, dtype=torch.bool, device="cuda")
    got = tree_attention_quant_gqa(q, *cache, *draft, mask, n_q_heads=hq, n_kv_heads=hkv, group_size=group)
    others = [i for i in range(n) if i != 1]
    assert float(got[:, :, others].float().abs().max()) <= 8 * 0.45e-25
    assert float(got[:, :, 1].float().abs().max()) > 1e20
