"""Long prompt, cut cache, tree decoding: the INT4 cache's branch and trim operators together.

A random-init Llama (no checkpoint is available offline) reads a prompt into a
``QuantizedKVCache`` that scores its tokens by the last queries; the cache is
cut to ``--keep`` tokens; then decoding goes on twice from the same cut cache:
one token per step, and with a tree of drafted tokens per step verified by
``TreeKVCache``.  The drafter here knows the plain run's tokens and hides them
among random ones (``--hit`` is the chance that a drafted token is the right
one), so that accepted lengths are under control; the tokens of both runs are
compared.

    python kv-cache-triton_b200/benchmarks/speculative_evict.py [--batch 4] [--prompt 4096]
        [--keep 1024] [--steps 64] [--layers 4] [--branch 4] [--depth 4]

Prints one JSON line.
"""

from __future__ import annotations

import argparse
import json
import os
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [os.path.dirname(HERE), HERE]


def draft_tree(branch: int, depth: int) -> list[int]:
    """Parents of a tree: node 0, then ``depth`` levels of ``branch`` nodes that all
    hang on the first node of the level above."""
    parents, top = [-1], 0
    for _ in range(depth):
        first = len(parents)
        parents += [top] * branch
        top = first
    return parents


def run(batch=4, prompt_len=4096, keep=1024, steps=64, layers=4, branch=4, depth=4, hit=0.8, seed=0,
        dtype=torch.bfloat16, config=None):
    from transformers import LlamaForCausalLM

    from llama3_e2e import llama31_8b_config
    from models.llama3.kv_cache import QuantizedKVCache
    from models.llama3.llama3_quant import replace_llama_attention_with_quantized
    from models.llama3.tree_cache import TreeKVCache, accept_greedy, tree_depth, tree_mask

    dev = torch.device("cuda")
    cfg = config or llama31_8b_config(layers)
    torch.manual_seed(seed)
    with torch.device(dev):
        model = LlamaForCausalLM(cfg).to(dtype).eval()
    replace_llama_attention_with_quantized(model)
    gen = torch.Generator(device=dev).manual_seed(seed + 1)
    prompt = torch.randint(0, cfg.vocab_size, (batch, prompt_len), device=dev, generator=gen)

    def forward(tokens, cache, positions):
        return model(input_ids=tokens, past_key_values=cache, use_cache=True, position_ids=positions,
                     cache_position=torch.arange(tokens.shape[1], device=dev)).logits

    def prefilled():
        cache = QuantizedKVCache(track_mass=True)
        where = torch.arange(prompt_len, device=dev).expand(batch, -1)
        logits = model(input_ids=prompt, past_key_values=cache, use_cache=True, position_ids=where,
                       logits_to_keep=1).logits
        kept = cache.evict(keep, recent=min(64, keep // 2), sinks=4 if keep >= 8 else 0)
        return cache, logits[:, -1].argmax(-1), kept

    def timed(fn):
        e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        e[0].record()
        fn()
        e[1].record()
        torch.cuda.synchronize()
        return e[0].elapsed_time(e[1])

    with torch.inference_mode():
        # one token per step
        cache, token, kept = prefilled()
        held = cache.get_seq_length(0)
        plain = [token]

        def plain_run():
            for i in range(steps):
                where = torch.full((batch, 1), prompt_len + i, device=dev)
                plain.append(forward(plain[-1].unsqueeze(1), cache, where)[:, -1].argmax(-1))

        plain_ms = timed(plain_run)
        want = torch.stack(plain, 1)  # [B, steps + 1]

        # a tree per step
        cache, token, _ = prefilled()
        tree = TreeKVCache.from_cache(cache, extra=steps + depth + 2, max_nodes=1 + branch * depth,
                                      tokens_seen=prompt_len)
        parents = torch.tensor(draft_tree(branch, depth), device=dev)
        mask, level = tree_mask(parents), tree_depth(parents)
        got = torch.zeros(batch, steps + depth + 2, dtype=torch.long, device=dev)
        got[:, 0] = token
        done = torch.ones(batch, dtype=torch.long, device=dev)  # tokens decided
        rows = torch.arange(batch, device=dev)
        calls, taken, asked = 0, torch.zeros((), device=dev), torch.zeros((), device=dev)

        def tree_run():
            nonlocal done, calls, token, taken, asked
            while int(done.min()) < steps + 1:
                nodes = torch.randint(0, cfg.vocab_size, (batch, parents.numel()), device=dev, generator=gen)
                nodes[:, 0] = token
                for d in range(depth):  # the first node of a level is often the right one
                    at = (done + d).clamp(max=steps)
                    right = torch.rand(batch, device=dev, generator=gen) < hit
                    nodes[:, 1 + d * branch] = torch.where(right, want[rows, at], nodes[:, 1 + d * branch])
                tree.begin(mask)
                path, accepted, token = accept_greedy(nodes, parents, forward(nodes, tree, tree.positions(level)))
                # sequences that are done stay where they are
                accepted = torch.where(done <= steps, accepted, torch.zeros_like(accepted))
                for j in range(1, depth + 1):
                    take = (j < accepted) & (done + j - 1 <= steps)
                    got[rows, (done + j - 1).clamp(max=got.shape[1] - 1)] = torch.where(
                        take, nodes[rows, path[:, j].long()], got[rows, (done + j - 1).clamp(max=got.shape[1] - 1)])
                last = (done + accepted - 1).clamp(min=0, max=got.shape[1] - 1)
                got[rows, last] = torch.where(accepted > 0, token, got[rows, last])
                tree.commit(path, accepted)
                taken += accepted.sum()
                asked += (accepted > 0).sum()
                done = done + accepted
                calls += 1

        tree_ms = timed(tree_run)
        tree.check()
    same = (got[:, :steps + 1] == want)
    lead = same.int().cumprod(1).sum(1)
    return {
        "workload": f"llama arch random-init {str(dtype)[6:]}, {cfg.num_hidden_layers} layers, batch {batch}, "
                    f"prompt {prompt_len} cut to {held}, {steps} steps, trees of {parents.numel()} nodes",
        "layers_cut": len(kept),
        "plain_ms_per_token": round(plain_ms / steps, 3),
        "tree_ms_per_call": round(tree_ms / calls, 3),
        "tree_calls": calls,
        "tokens_per_sequence_and_call": round(float(taken / asked), 2),
        "leading_tokens_alike": [int(x) for x in lead],
        "tokens_compared": steps + 1,
    }


def main():
    ap = argparse.ArgumentParser()
    for name, value in (("batch", 4), ("prompt", 4096), ("keep", 1024), ("steps", 64), ("layers", 4),
                        ("branch", 4), ("depth", 4), ("seed", 0)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--hit", type=float, default=0.8)
    a = ap.parse_args()
    print(json.dumps(run(a.batch, a.prompt, a.keep, a.steps, a.layers, a.branch, a.depth, a.hit, a.seed)),
          flush=True)


if __name__ == "__main__":
    main()
