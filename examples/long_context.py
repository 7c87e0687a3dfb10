"""A decoder layer's attention over a long context, three ways.

  window    every token attends the newest tokens and the first ones
  search    as window, and the rest of the context through an `Index` over each
            head's keys: the rows that the search returns are attended where they
            lie and joined with the window's part
  budget    the whole cache, cut to a budget by the weight its slots have had

The prompt comes in by window (in parts), then tokens are decoded one by one.  Each
way's rows are compared with attention over everything.  The context is made so
that a new token needs a few tokens of long ago, as text does that refers back;
keys are normed per head, so all have the same length and the largest inner products
are the nearest unit vectors.

    python examples/long_context.py [tokens]
"""
import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import swann_b200 as swann
from swann_b200 import attention as A


def rotation(positions, dims, device, base=10000.0):
    angle = torch.arange(positions, device=device).double()[:, None] * base ** (-torch.arange(0, dims, 2, device=device).double() / dims)
    return angle.cos().float(), angle.sin().float()


def run(tokens=32768, steps=8, q_heads=8, kv_heads=2, d=128, window=1024, sinks=4, k=64, budget=4096, seed=0):
    dev, dt = torch.device("cuda"), torch.float16
    g = torch.Generator(device=dev).manual_seed(seed)
    group, total = q_heads // kv_heads, tokens + steps
    # only a quarter of each head is rotated, so that far keys stay comparable
    cos, sin = rotation(total, d // 4, dev)
    # a learned weight of the queries' norm sets how sharply attention looks
    norm, sharp = torch.ones(d, dtype=dt, device=dev), torch.full((d,), 2.0, dtype=dt, device=dev)
    keys = torch.randn((total, kv_heads, d), generator=g, device=dev)
    values = torch.randn((total, kv_heads, d), generator=g, device=dev)
    queries = torch.randn((total, q_heads, d), generator=g, device=dev)
    # each new token refers back: its queries point at one far key per head, among others
    far = torch.randint(sinks, tokens - window, (steps, kv_heads), generator=g, device=dev)
    heads = torch.arange(kv_heads, device=dev)
    queries[tokens:] += 1.5 * keys[far, heads].repeat_interleave(group, 1)
    queries, keys, values = queries.to(dt), keys.to(dt), values.to(dt)

    cache = swann.KVCache(1, total, kv_heads, d, dtype=dt, track=True)
    for a in range(0, tokens, 8192):
        e = min(tokens, a + 8192)
        starts = torch.tensor([0, e - a], dtype=torch.int32, device=dev)
        q = cache.append(queries[a:e], keys[a:e], values[a:e], cos, sin, starts, q_norm=sharp, k_norm=norm)
        cache.prefill(q, starts, window=window, sinks=sinks)

    # the prompt's rows, head by head: a corpus for each head, and all of them as pages of one row
    def rows(pool):
        return pool[cache.table[0].long()].permute(1, 0, 2, 3).flatten(1, 2)[:, :tokens].contiguous()

    k_rows, v_rows = rows(cache.k), rows(cache.v)
    unit = torch.nn.functional.normalize(k_rows.float(), dim=-1).to(dt)
    index = [swann.Index.build(unit[h], metric="ip", degree=32, candidates=64) for h in range(kv_heads)]
    k_pool, v_pool = (x.view(kv_heads * tokens, 1, 1, d) for x in (k_rows, v_rows))
    found = torch.full((q_heads,), k, dtype=torch.int32, device=dev)

    small = swann.KVCache(1, total, kv_heads, d, dtype=dt, track=True)
    small.k.copy_(cache.k)
    small.v.copy_(cache.v)
    small.lengths, small.seen = cache.lengths.clone(), cache.seen.clone()
    small.positions.copy_(cache.positions)

    off = {"window": 0.0, "search": 0.0, "budget": 0.0}
    hits = 0
    for t in range(steps):
        one = slice(tokens + t, tokens + t + 1)
        q = cache.append(queries[one], keys[one], values[one], cos, sin, q_norm=sharp, k_norm=norm)
        near = A.decode(q, cache.k, cache.v, cache.table, cache.lengths, window=window, sinks=sinks)
        # the search: each query head over its key head's corpus
        uq = torch.nn.functional.normalize(q[0].float(), dim=-1)
        ids = torch.cat([index[h].search_tensors(uq[h * group:(h + 1) * group], k=k, branches=64, queue=k)[0]
                         for h in range(kv_heads)]).to(torch.int32)
        hits += int((ids == far[t].repeat_interleave(group)[:, None]).any(1).sum())
        # what the window and the first tokens cover already is not attended twice
        inside = (ids < sinks) | (ids > tokens + t - window)
        page = (ids + (torch.arange(q_heads, device=dev, dtype=torch.int32) // group * tokens)[:, None]).masked_fill(inside | (ids < 0), -1)
        joined, _ = A.decode(q.view(q_heads, 1, d), k_pool, v_pool, page, found,
                             prior=(near[0].view(q_heads, 1, d), near[1].view(q_heads, 1)))
        full, _ = cache.attend(q)
        qs = small.append(queries[one], keys[one], values[one], cos, sin, q_norm=sharp, k_norm=norm)
        cut, _ = small.attend(qs)
        small.evict(budget, sinks=sinks, recent=window)
        for name, got in (("window", near[0]), ("search", joined.view(1, q_heads, d)), ("budget", cut)):
            off[name] += float((got.float() - full.float()).norm() / full.float().norm()) / steps
    return {**off, "found": hits / (steps * q_heads), "held": int(small.lengths[0])}


if __name__ == "__main__":
    got = run(int(sys.argv[1]) if len(sys.argv) > 1 else 32768)
    print("distance from attention over everything (2-norm, relative):")
    for name in ("window", "search", "budget"):
        print(f"  {name:8s} {got[name]:.4f}")
    print(f"the searches found the far token in {100 * got['found']:.0f}% of the heads' queries; "
          f"the budgeted cache holds {got['held']} slots")
