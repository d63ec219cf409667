"""Half-precision queries down to f16's smallest steps, over keys large enough for
them to matter: log-sum-exp and scores as exact as for any other queries (bounds of
branch_ref; test_tree_gpu's for the log-sum-exp)."""

from __future__ import annotations

import pytest
import torch

import branch_ref as br

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _inputs(b, hq, hkv, n, s, d, group, q_scale, sdtype, seed):
    cache = br.random_rows(b, hkv, s, d, group, sdtype, seed)
    cache[1] = (cache[1].float() * (1.0 / q_scale)).clamp(max=6e4).to(sdtype)
    g = torch.Generator().manual_seed(seed + 2)
    return cache, (q_scale * torch.randn(b, hq, n, d, generator=g)).to(F16)


# rows per KV head: up to 8, up to 16, more; head sizes
SHAPES = [(2, 4, 2, 3, 300, 128, 32), (2, 8, 2, 4, 300, 64, 32), (2, 8, 2, 12, 301, 128, 64)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("q_scale", [1e-3, 1e-4, 2e-5, 1e-6, 1e4])
@pytest.mark.parametrize("sdtype", [F16, BF16])
def test_tree(shape, q_scale, sdtype):
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    b, hq, hkv, n, s, d, group = shape
    cache, q = _inputs(b, hq, hkv, n, s, d, group, q_scale, sdtype, 1)
    draft = [t[:, :, :n].contiguous() for t in cache]
    mask = torch.eye(n, dtype=torch.bool)
    lse = torch.empty(b, hq, n, device="cuda")
    got = tree_attention_quant_gqa(q.cuda(), *[t.cuda() for t in cache], *[t.cuda() for t in draft], mask.cuda(),
                                   n_q_heads=hq, n_kv_heads=hkv, group_size=group, lse=lse)
    for x in range(b):
        rows = [torch.cat((c[x], f[x]), 1) for c, f in zip(cache, draft)]
        k, v = br.values(*rows[:2], group, d), br.values(*rows[2:], group, d)
        seen = torch.cat((torch.ones(n, s, dtype=torch.bool), mask), 1)
        ref, _, X, A = br.attend(q[x].double(), k, v, seen)
        br.check_out(got[x], ref, X, A, s + n)
        sc = (q[x].double() @ k.repeat_interleave(hq // hkv, 0).transpose(1, 2)) * d ** -0.5
        want = torch.logsumexp(sc.masked_fill(~seen, -float("inf")), -1)
        bound = br.U32 * ((d + 8) * X * 2 + 2 * (s + n + 64)) + br.U32 * 4 * want.abs()
        assert bool(((lse[x].cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("shape", SHAPES + [(2, 8, 2, 1, 300, 128, 32)])
@pytest.mark.parametrize("q_scale", [1e-3, 1e-4, 2e-5, 1e-6])
def test_scored(shape, q_scale):
    from kernels.llama3.evict import attention_forward_quant_gqa_scored
    b, hq, hkv, n, s, d, group = shape
    cache, q = _inputs(b, hq, hkv, n, s, d, group, q_scale, F16, 3)
    mass = torch.zeros(b, hkv, s, device="cuda")
    out, new = attention_forward_quant_gqa_scored(q.cuda(), *[t.cuda() for t in cache], mass, n_q_heads=hq,
                                                  n_kv_heads=hkv, group_size=group, is_causal=True)
    seen = torch.ones(n, s, dtype=torch.bool).tril(s - n)
    for x in range(b):
        k, v = br.values(cache[0][x], cache[1][x], group, d), br.values(cache[2][x], cache[3][x], group, d)
        ref, p, X, A = br.attend(q[x].double(), k, v, seen)
        br.check_out(out[x], ref, X, A, s)
        add = p.reshape(hkv, -1, s)
        rel = br.weight_bound(X, d, s).reshape(hkv, -1, 1) + br.U32 * (add.shape[1] + 8)
        want = add.sum(1)
        assert bool(((new[x].cpu().double() - want).abs() <= (rel * add).sum(1) + br.U32 * 2 * want + 1e-30).all())
