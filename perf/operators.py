"""Cases and plain forms of the operators that branch and trim an INT4 KV cache.

Four operators over the packed cache (``packed uint8 [B, Hkv, S, d/2]``, low
nibble = even column, ``scales [B, Hkv, S, d/G]``, value = (code - 8) * scale):

* ``tree``   -- attention of N drafted nodes over each sequence's committed
  context and over those drafted nodes that a boolean mask lets them see;
* ``commit`` -- the accepted drafted rows move into the cache behind each
  sequence's context;
* ``scored`` -- attention that also adds the weight each cached token received
  to a running score per KV head;
* ``evict``  -- the cache is cut to the first tokens, the most recent ones and
  the highest scored of the rest, per KV head, in token order.

``run`` computes them in elementary torch operations in 32 bits, or, where
``own`` is true, by the calls that a user makes of this repository.
"""

import math
import os
import sys

import torch

own = False

_HEADS = {"llama8b": (32, 8, 128), "llama70b": (64, 8, 128), "gpt2": (12, 12, 64)}
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one user, a short chat, eight drafted nodes: what counts is the latency of the call
        {"name": "tree_b1_n8_s512", "op": "tree", "heads": "llama8b", "type": "bf16", "group": 32,
         "batch": 1, "nodes": 8, "context": 512, "ragged": False, "own_tree": False},
        # a batch in speculative decoding: sequences of different lengths, a tree for each
        {"name": "tree_b8_n63_s4096", "op": "tree", "heads": "llama8b", "type": "bf16", "group": 32,
         "batch": 8, "nodes": 63, "context": 4096, "ragged": True, "own_tree": True},
        # GPT-2's heads in half precision, one tree for the whole batch
        {"name": "tree_gpt2_n17_s1000", "op": "tree", "heads": "gpt2", "type": "f16", "group": 32,
         "batch": 4, "nodes": 17, "context": 1000, "ragged": False, "own_tree": False},
        # GPT-2's heads in single precision
        {"name": "tree_f32_n12_s777", "op": "tree", "heads": "gpt2", "type": "f32", "group": 32,
         "batch": 2, "nodes": 12, "context": 777, "ragged": True, "own_tree": True},
        # eight query heads to a KV head, long contexts, wide trees: the products bound it
        {"name": "tree_b4_n64_s16384", "op": "tree", "heads": "llama70b", "type": "bf16", "group": 64,
         "batch": 4, "nodes": 64, "context": 16384, "ragged": True, "own_tree": True},
        # the step after the smallest verification
        {"name": "commit_b1_n8_s512", "op": "commit", "heads": "llama8b", "type": "bf16", "group": 32,
         "batch": 1, "nodes": 8, "context": 512},
        # the step after a large batch's verification
        {"name": "commit_b32_n64_s2047", "op": "commit", "heads": "llama8b", "type": "bf16", "group": 32,
         "batch": 32, "nodes": 64, "context": 2047},
        # single-token decoding with GPT-2's heads in single precision
        {"name": "scored_f32_s1023", "op": "scored", "heads": "gpt2", "type": "f32", "group": 32,
         "batch": 2, "queries": 1, "context": 1023, "decay": 1.0},
        # single-token decoding of a batch: this repository's benchmark shape
        {"name": "scored_b16_s4096", "op": "scored", "heads": "llama8b", "type": "bf16", "group": 32,
         "batch": 16, "queries": 1, "context": 4096, "decay": 1.0},
        # the last queries of a long prompt score the whole of it before it is cut
        {"name": "scored_window_s16384", "op": "scored", "heads": "llama70b", "type": "bf16", "group": 32,
         "batch": 2, "queries": 32, "context": 16384, "decay": 0.9},
        # one user's cache is cut, at an odd length
        {"name": "evict_b1_s1537", "op": "evict", "heads": "llama8b", "type": "bf16", "group": 32,
         "batch": 1, "context": 1537, "keep": 512, "recent": 64, "sinks": 4},
        # a batch's prompts are cut to a quarter before decoding starts
        {"name": "evict_b16_s16384", "op": "evict", "heads": "llama8b", "type": "bf16", "group": 32,
         "batch": 16, "context": 16384, "keep": 4096, "recent": 256, "sinks": 4},
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("tree", "tree", "commit", "scored", "scored", "evict"))
    kind = rng.choice(("bf16", "bf16", "bf16", "f16", "f32"))
    heads = rng.choice(("llama8b", "llama70b", "gpt2")) if kind == "bf16" else "gpt2"
    group = rng.choice((32, 32, 64)) if heads == "gpt2" else rng.choice((32, 32, 64, 128))
    c = {"op": op, "heads": heads, "type": kind, "group": group}
    most = 2048 if heads == "gpt2" else 16384
    c["context"] = _spread(rng, 1 if op == "tree" else 64, most)
    if op == "tree":
        c["nodes"] = _spread(rng, 1, 64)
        c["batch"] = _spread(rng, 1, max(1, min(16, 4 * 16384 // (c["context"] + 64))))
        c["ragged"], c["own_tree"] = rng.random() < 0.5, rng.random() < 0.5
    elif op == "commit":
        c["nodes"] = _spread(rng, 1, 64)
        c["batch"] = _spread(rng, 1, max(1, min(32, 32 * 2047 // c["context"])))
    elif op == "scored":
        c["queries"] = rng.choice((1, 1, _spread(rng, 2, 32)))
        c["queries"] = min(c["queries"], c["context"])
        c["batch"] = _spread(rng, 1, max(1, min(16, 2 * 16384 // (c["context"] if c["queries"] > 1 else (c["context"] + 1) // 2))))
        c["decay"] = rng.choice((1.0, 0.9))
    else:
        c["batch"] = _spread(rng, 1, 16)
        c["recent"] = rng.randint(0, c["context"] // 8)
        c["sinks"] = rng.choice((0, 4))
        c["keep"] = rng.randint(c["recent"] + c["sinks"] + 1, max(c["recent"] + c["sinks"] + 1, c["context"] // 2))
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """The context lengths of a batch: all alike, or spread from half the context to the whole of it."""
    b, s = case["batch"], case["context"]
    if not case.get("ragged", case["op"] == "commit"):
        return [s] * b
    return [s - (s // 2) * i // b for i in range(b)]


def _quantized(x, group, dtype):
    """x as 4-bit codes, two to a byte, and the scales of its groups."""
    g = x.unflatten(-1, (-1, group))
    m = g.abs().amax(-1, keepdim=True)
    s = torch.where(m > 0, m / 7, torch.ones_like(m))
    c = (torch.round(g / s).clamp(-8, 7) + 8).to(torch.uint8).flatten(-2)
    return (c[..., 0::2] | (c[..., 1::2] << 4)).contiguous(), s.squeeze(-1).to(dtype).contiguous()


def _cache(gen, b, hkv, s, d, group, dtype):
    """Keys with outlier channels (a factor from 1/2 to 8 each) and values, quantized."""
    dev = gen.device
    f = torch.exp(torch.rand(d, generator=gen, device=dev) * math.log(16.0)) * 0.5
    k = torch.randn(b, hkv, s, d, generator=gen, device=dev) * f
    v = torch.randn(b, hkv, s, d, generator=gen, device=dev)
    return [*_quantized(k, group, dtype), *_quantized(v, group, dtype)]


def _tree_masks(gen, count, n):
    """Random trees: node 0 hangs on the context, a later one on one of the eight before it or on the
    context; a node sees its ancestors and itself."""
    dev = gen.device
    back = torch.randint(0, 9, (count, n), generator=gen, device=dev)
    mask = torch.eye(n, dtype=torch.bool, device=dev).repeat(count, 1, 1)
    at = torch.arange(count, device=dev)
    for i in range(1, n):
        parent = (i - back[:, i]).clamp(min=0)
        mask[:, i] |= mask[at, parent] & (back[:, i] > 0)[:, None]
    return mask


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    hq, hkv, d = _HEADS[case["heads"]]
    dtype, group, b, s = _TYPES[case["type"]], case["group"], case["batch"], case["context"]
    op = case["op"]
    n = case.get("nodes", 0)
    room = s + n if op == "commit" else s
    state = {"op": op, "hq": hq, "hkv": hkv, "group": group}
    state["cache"] = _cache(gen, b, hkv, room, d, group, dtype)
    if op in ("tree", "commit"):
        order = torch.randperm(b, generator=gen, device="cuda")
        lens = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]
        state["lens"] = lens.contiguous()
        state["draft"] = _cache(gen, b, hkv, n, d, group, dtype)
    if op == "tree":
        state["q"] = torch.randn(b, hq, n, d, generator=gen, device="cuda").to(dtype)
        own_tree = case["own_tree"]
        mask = _tree_masks(gen, b if own_tree else 1, n)
        state["mask"] = mask if own_tree else mask[0].contiguous()
    elif op == "commit":
        # a path from the root: increasing node numbers; the accepted count differs by sequence
        keys = torch.rand(b, n, generator=gen, device="cuda")
        state["path"] = torch.sort(keys.argsort(1)[:, : (n + 1) // 2], dim=1).values.to(torch.int32)
        state["accepted"] = _accepted(case)[order]
    elif op == "scored":
        state["q"] = torch.randn(b, hq, case["queries"], d, generator=gen, device="cuda").to(dtype)
        # what some steps like this one left: about four times the weight that this one adds
        left = (2 * torch.randn(b, hkv, s, generator=gen, device="cuda")).exp()
        state["mass"] = left * (4 * (hq // hkv) * case["queries"] / s / math.exp(2.0))
        state["decay"] = case["decay"]
    elif op == "evict":
        # a few tokens hold most of the weight; one in ten was never looked at
        m = (2 * torch.randn(b, hkv, s, generator=gen, device="cuda")).exp()
        state["mass"] = torch.where(torch.rand(b, hkv, s, generator=gen, device="cuda") < 0.1, torch.zeros_like(m), m)
        state.update(keep=case["keep"], recent=case["recent"], sinks=case["sinks"])
    return state


def _accepted(case):
    """How many nodes of the path each sequence accepts, from none to all of it."""
    b, most = case["batch"], (case["nodes"] + 1) // 2
    return torch.tensor([most - i % (most + 1) for i in range(b)], dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _values(packed, scales, group):
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).float() - 8
    return (codes.unflatten(-1, (-1, group)) * scales.float().unsqueeze(-1)).flatten(-2)


def _attend(q, k, v, seen):
    """Weights and output of q [B, Hq, n, d] over k, v [B, Hkv, S, d]; seen: broadcastable to
    [B, 1, n, S]. A row that sees nothing gives zeros."""
    b, hq, n, d = q.shape
    hkv = k.shape[1]
    x = q.float().reshape(b, hkv, hq // hkv * n, d) @ k.transpose(-1, -2) * d**-0.5
    x = x.reshape(b, hkv, hq // hkv, n, -1).masked_fill(~seen.unsqueeze(1), -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = p.reshape(b, hkv, hq // hkv * n, -1) @ v
    return p, out.reshape(b, hq, n, d).to(q.dtype)


def _plain_tree(state):
    kp, ks, vp, vs = state["cache"]
    dkp, dks, dvp, dvs = state["draft"]
    g = state["group"]
    k = torch.cat((_values(kp, ks, g), _values(dkp, dks, g)), 2)
    v = torch.cat((_values(vp, vs, g), _values(dvp, dvs, g)), 2)
    b, s, n = kp.shape[0], kp.shape[2], dkp.shape[2]
    context = (torch.arange(s, device=kp.device) < state["lens"][:, None])[:, None, None, :]
    mask = state["mask"] if state["mask"].dim() == 3 else state["mask"].unsqueeze(0)
    seen = torch.cat((context.expand(b, 1, n, s), mask.unsqueeze(1).expand(b, 1, n, n)), -1)
    return {"out": _attend(state["q"], k, v, seen)[1]}


def _plain_commit(state):
    path, accepted, lens = state["path"].long(), state["accepted"], state["lens"]
    width = path.shape[1]
    b, j = torch.nonzero(torch.arange(width, device=path.device) < accepted[:, None], as_tuple=True)
    to, src = lens.long()[b] + j, path[b, j]
    for cache, draft in zip(state["cache"], state["draft"]):
        cache[b, :, to] = draft[b, :, src]
    return {"cache": list(state["cache"]), "lens": lens + accepted}


def _plain_scored(state):
    kp, ks, vp, vs = state["cache"]
    q, g = state["q"], state["group"]
    s, n = kp.shape[2], q.shape[2]
    j, i = torch.arange(s, device=q.device), torch.arange(n, device=q.device)
    seen = (j <= s - n + i[:, None])[None, None]
    p, out = _attend(q, _values(kp, ks, g), _values(vp, vs, g), seen)
    return {"out": out, "mass": state["mass"] * state["decay"] + p.sum((2, 3))}


def _plain_evict(state):
    mass, keep, recent, sinks = state["mass"], state["keep"], state["recent"], state["sinks"]
    s = mass.shape[2]
    key = mass.clone()
    key[..., :sinks] = math.inf
    key[..., s - recent:] = math.inf
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    index = torch.sort(order, dim=-1).values
    rows = [t.gather(2, index.unsqueeze(-1).expand(*index.shape, t.shape[-1])) for t in state["cache"]]
    return {"cache": rows, "mass": mass.gather(2, index), "index": index.to(torch.int32)}


# ---------------------------------------------------------------------------
# this repository's operators
# ---------------------------------------------------------------------------
_calls = {}


def _own():
    if not _calls:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "kv-cache-triton_b200"))
        from kernels.llama3.evict import attention_forward_quant_gqa_scored, evict_by_mass
        from kernels.llama3.tree_attention_quant import commit_draft_rows, tree_attention_quant_gqa
        _calls.update(tree=tree_attention_quant_gqa, commit=commit_draft_rows,
                      scored=attention_forward_quant_gqa_scored, evict=evict_by_mass)
    return _calls


def _run_own(state):
    op = state["op"]
    call = _own()[op]
    if op == "tree":
        return {"out": call(state["q"], *state["cache"], *state["draft"], state["mask"], n_q_heads=state["hq"],
                            n_kv_heads=state["hkv"], group_size=state["group"], context_lens=state["lens"])}
    if op == "commit":
        lens = call(*state["cache"], *state["draft"], state["path"], state["accepted"], context_lens=state["lens"])
        return {"cache": list(state["cache"]), "lens": lens}
    if op == "scored":
        out, mass = call(state["q"], *state["cache"], state["mass"], n_q_heads=state["hq"], n_kv_heads=state["hkv"],
                         group_size=state["group"], is_causal=True, decay=state["decay"],
                         mass_out=torch.empty_like(state["mass"]))
        return {"out": out, "mass": mass}
    *cache, mass, index = call(*state["cache"], state["mass"], keep=state["keep"], recent=state["recent"],
                               sinks=state["sinks"])
    return {"cache": cache, "mass": mass, "index": index}


_PLAIN = {"tree": _plain_tree, "commit": _plain_commit, "scored": _plain_scored, "evict": _plain_evict}


def run(state):
    return _run_own(state) if own else _PLAIN[state["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    hq, hkv, d = _HEADS[case["heads"]]
    e, b, s = _BYTES[case["type"]], case["batch"], case["context"]
    row = d // 2 + d // case["group"] * e  # a K or V row of one head
    tokens = sum(_lengths(case))
    if case["op"] == "tree":
        n = case["nodes"]
        masks = (b if case["own_tree"] else 1) * n * n
        return {"bytes": 2 * hkv * row * (tokens + b * n) + 2 * b * hq * n * d * e + masks + 4 * b,
                "flops": 4 * hq * n * d * (tokens + b * n)}
    if case["op"] == "commit":
        most = (case["nodes"] + 1) // 2
        rows = sum(most - i % (most + 1) for i in range(b))
        return {"bytes": 2 * 2 * hkv * row * rows + 4 * rows + 12 * b, "flops": 0}
    if case["op"] == "scored":
        n = case["queries"]
        return {"bytes": 2 * hkv * row * tokens + 2 * b * hq * n * d * e + 8 * hkv * tokens,
                "flops": 4 * hq * n * d * tokens}
    # every score once, the kept rows in and out, and their indices
    return {"bytes": b * hkv * (4 * s + case["keep"] * (2 * 2 * row + 4 + 4)), "flops": 0}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_values(packed, scales, group):
    low, high = (packed % 16).double() - 8, torch.div(packed, 16, rounding_mode="floor").double() - 8
    codes = torch.empty(*packed.shape[:-1], 2 * packed.shape[-1], dtype=torch.float64, device=packed.device)
    codes[..., 0::2], codes[..., 1::2] = low, high
    return codes * scales.double().repeat_interleave(group, dim=-1)


def _exact_softmax(q, k, seen):
    """Weights of the rows of q [n, d] over k [S, d] where seen [n, S]; zeros where a row sees nothing."""
    x = (q.double() @ k.T) / math.sqrt(q.shape[-1])
    x[~seen] = -math.inf
    return torch.nan_to_num(torch.softmax(x, -1), nan=0.0)


def exact(case, seed):
    st = prepare(case, seed)
    op, group = st["op"], st["group"]
    if op == "evict":
        got = _exact_evict(st)
        return {"cache": [None, got[0], None, got[1]], "mass": got[2], "index": None}
    if op == "commit":
        for b, (at, m) in enumerate(zip(st["lens"].tolist(), st["accepted"].tolist())):
            for i, node in enumerate(st["path"][b, :m].tolist()):
                for c, f in zip(st["cache"], st["draft"]):
                    c[b, :, at + i] = f[b, :, node]
        return {"cache": [None, st["cache"][1].double(), None, st["cache"][3].double()], "lens": None}
    q = st["q"]
    r, n = st["hq"] // st["hkv"], q.shape[2]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    mass = st["mass"].double() * st["decay"] if op == "scored" else None
    for b in range(q.shape[0]):
        for h in range(st["hkv"]):
            kp, ks, vp, vs = (t[b, h] for t in st["cache"])
            if op == "tree":
                live = int(st["lens"][b])
                dk, dks, dv, dvs = (t[b, h] for t in st["draft"])
                kp, ks = torch.cat((kp[:live], dk)), torch.cat((ks[:live], dks))
                vp, vs = torch.cat((vp[:live], dv)), torch.cat((vs[:live], dvs))
                seen = torch.ones(n, live + n, dtype=torch.bool, device=q.device)
                seen[:, live:] = st["mask"][b] if st["mask"].dim() == 3 else st["mask"]
            else:
                seen = torch.ones(n, kp.shape[0], dtype=torch.bool, device=q.device).tril(kp.shape[0] - n)
            k, v = _exact_values(kp, ks, group), _exact_values(vp, vs, group)
            p = _exact_softmax(q[b, h * r:(h + 1) * r].reshape(r * n, -1), k, seen.repeat(r, 1))
            out[b, h * r:(h + 1) * r] = (p @ v).reshape(r, n, -1)
            if op == "scored":
                mass[b, h] += p.sum(0)
    return {"out": out, "mass": mass} if op == "scored" else {"out": out}


def _exact_evict(st):
    """Kept scales and scores, by ranking each candidate against the others."""
    mass, s = st["mass"].double(), st["mass"].shape[2]
    room = st["keep"] - st["recent"] - st["sinks"]
    middle = mass[..., st["sinks"]:s - st["recent"]]
    order = torch.argsort(-middle, dim=-1, stable=True)[..., :room] + st["sinks"]
    kept = torch.zeros(mass.shape, dtype=torch.bool, device=mass.device).scatter_(2, order, True)
    kept[..., :st["sinks"]] = True
    kept[..., s - st["recent"]:] = True
    ks, vs = st["cache"][1], st["cache"][3]
    b, h = mass.shape[:2]
    return ks[kept].double().reshape(b, h, -1, ks.shape[-1]), vs[kept].double().reshape(b, h, -1, vs.shape[-1]), mass[kept].reshape(b, h, -1)
