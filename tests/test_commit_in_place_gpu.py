"""The commit's C entry with lens_out the same buffer as context_lens (one KV head),
over paths longer than one round of the kernel."""

from __future__ import annotations

import ctypes

import pytest
import torch

import branch_ref as br

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [5, 256, 257, 700])
def test_lengths_in_place(width):
    from kvint4 import _lib, ops
    b, cap, n, d = 3, 2000, 800, 64
    cache = [t.cuda() for t in br.random_rows(b, 1, cap, d, 32, torch.bfloat16, 1)]
    draft = [t.cuda() for t in br.random_rows(b, 1, n, d, 32, torch.bfloat16, 2)]
    lens = torch.tensor([0, 17, cap - width], dtype=torch.int32, device="cuda")
    accepted = torch.tensor([width, width - 1, width], dtype=torch.int32, device="cuda")
    path = torch.stack([torch.randperm(n, generator=torch.Generator().manual_seed(x))[:width] for x in range(b)])
    want = [t.clone() for t in cache]
    for x in range(b):
        m, at = int(accepted[x]), int(lens[x])
        for w, f in zip(want, draft):
            w[x, 0, at:at + m] = f[x, 0, path[x, :m].cuda()]
    new = lens + accepted
    path = path.int().cuda()
    ds = [ops.desc(t) for t in (*cache, *draft)]
    ops.device_error()
    rc = _lib.lib().kv4_commit_rows(*[ctypes.byref(x) for x in ds], path.data_ptr(), path.stride(0), width,
                                    accepted.data_ptr(), lens.data_ptr(), lens.data_ptr(),
                                    torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert torch.equal(lens, new)
    for c, w in zip(cache, want):
        assert torch.equal(c, w)
    assert ops.device_error() == 0
