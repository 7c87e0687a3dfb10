"""The cache as a program uses it: prompts in, tokens decoded, slots evicted; and
the example that joins it with a search."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

import swann_b200 as swann

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROOT = Path(__file__).resolve().parent.parent


def softmax_rows(q, k, v, seen, scale):
    """[heads, d] in 64 bits over the rows that are seen; q [heads, d], k and v [kv_heads, n, d]."""
    G = q.shape[0] // k.shape[0]
    x = (q.double().view(k.shape[0], G, -1) @ k.double().transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    return (torch.softmax(x, -1) @ v.double()).flatten(0, 1), torch.logsumexp(x, -1).flatten()


def turned(x, cos, sin):
    """Rotated by halves, 64 bits; x [tokens, heads, d], cos and sin [tokens, d / 2]."""
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def test_prompts_then_tokens_then_eviction():
    """Two sequences of different lengths against plain attention over everything they were given, then over what
    eviction left: bounds of one 16-bit rounding of keys and queries (2^-11 each, logits up to about 10) and of the
    weights and rows."""
    g = torch.Generator(device=DEV).manual_seed(3)
    hq, hkv, d, dt = 6, 2, 64, torch.float16
    cache = swann.KVCache(2, 400, hkv, d, page_size=16, dtype=dt, track=True)
    angle = torch.rand((500, d // 2), generator=g, device=DEV) * 6.28
    cos, sin = angle.cos(), angle.sin()
    held = [[], []]

    def tokens(n):
        return [torch.randn((n, h, d), generator=g, device=DEV).to(dt) for h in (hq, hkv, hkv)]

    def close(out, lse, want):
        assert (out.double() - want[0]).abs().max() < 0.02 and (lse.double() - want[1]).abs().max() < 0.02

    def check(out, lse, qr, b, seen=None):
        k = torch.stack([x[0] for x in held[b]], 1)
        v = torch.stack([x[1] for x in held[b]], 1).double()
        seen = torch.ones((hkv, 1, k.shape[1]), dtype=torch.bool, device=DEV) if seen is None else seen
        close(out, lse, softmax_rows(qr, k, v, seen, d ** -0.5))

    # two prompts, in two parts each, one part empty
    for counts in ((150, 37), (90, 0)):
        starts = torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32, device=DEV)
        q, k, v = tokens(sum(counts))
        at = torch.cat([torch.arange(len(held[b]), len(held[b]) + n) for b, n in enumerate(counts)]).to(DEV)
        kr, qr = turned(k, cos[at], sin[at]), turned(q, cos[at], sin[at])
        qo = cache.append(q, k, v, cos, sin, starts)
        out, lse = cache.prefill(qo, starts, window=70, sinks=3)
        t = 0
        for b, n in enumerate(counts):
            for i in range(n):
                held[b].append((kr[t], v[t]))
                pos = len(held[b]) - 1
                j = torch.arange(pos + 1, device=DEV)
                if i % 29 == 0 or i == n - 1:
                    check(out[t], lse[t], qr[t], b, ((j > pos - 70) | (j < 3)).expand(hkv, 1, -1))
                t += 1
    assert cache.lengths.tolist() == [240, 37] == cache.seen.tolist()
    # tokens, attending everything
    for _ in range(3):
        q, k, v = tokens(2)
        at = cache.seen.long()
        kr, qr = turned(k, cos[at], sin[at]), turned(q, cos[at], sin[at])
        out, lse = cache.attend(cache.append(q, k, v, cos, sin))
        for b in range(2):
            held[b].append((kr[b], v[b]))
            check(out[b], lse[b], qr[b], b)
    # each attended token had a weight of 1 for every query head
    assert torch.allclose(cache.weights.sum(-1), torch.full((2, hkv), 3.0 * hq / hkv, device=DEV), rtol=1e-4)
    assert (cache.positions[0, :, :243] == torch.arange(243, device=DEV)).all() and (cache.positions[0, :, 243:] == -1).all()
    cache.evict(100, sinks=2, recent=20)
    assert cache.lengths.tolist() == [100, 40] and cache.seen.tolist() == [243, 40]
    for h in range(hkv):
        kept = set(cache.positions[0, h, :100].tolist())
        assert len(kept) == 100 and {0, 1, *range(223, 243)} <= kept
    # what comes after is attended with what was kept, at its own positions
    for _ in range(2):
        q, k, v = tokens(2)
        at = cache.seen.long()
        kr, qr = turned(k, cos[at], sin[at]), turned(q, cos[at], sin[at])
        out, lse = cache.attend(cache.append(q, k, v, cos, sin))
        for b in range(2):
            held[b].append((kr[b], v[b]))
            seen = torch.zeros((hkv, 1, len(held[b])), dtype=torch.bool, device=DEV)
            for h in range(hkv):
                seen[h, 0, cache.positions[b, h, :int(cache.lengths[b])].long()] = True
            check(out[b], lse[b], qr[b], b, seen)
    with pytest.raises(ValueError, match="no window"):
        cache.attend(q, window=8)
    with pytest.raises(ValueError, match="order"):
        cache.prefill(q, cache._each)


def test_cache_refusals():
    with pytest.raises(ValueError, match="power of two"):
        swann.KVCache(1, 10, 1, 64, page_size=3)
    with pytest.raises(ValueError, match="head_dim"):
        swann.KVCache(1, 10, 1, 80)
    with pytest.raises(ValueError, match="float16"):
        swann.KVCache(1, 10, 1, 64, dtype=torch.float32)
    with pytest.raises(ValueError, match="track"):
        swann.KVCache(1, 10, 1, 64).evict(4)


def test_decode_step_in_a_graph():
    """append, attend and the counts of a step captured once and replayed: nothing waits for the device."""
    cache = swann.KVCache(3, 64, 2, 64, dtype=torch.float16)
    other = swann.KVCache(3, 64, 2, 64, dtype=torch.float16)
    cos = torch.rand((64, 32), device=DEV)
    x = torch.randn((3, 8, 64), device=DEV).half()

    def step(c):
        return c.attend(c.append(x[:, :4], x[:, 4:6], x[:, 6:], cos, cos))

    lengths, seen = cache.lengths, cache.seen
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = step(cache)
            lengths.copy_(cache.lengths)
            seen.copy_(cache.seen)
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(5):
        x.copy_(torch.randn((3, 8, 64), device=DEV))
        graph.replay()
        want = step(other)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_long_context_example():
    spec = importlib.util.spec_from_file_location("long_context", ROOT / "examples" / "long_context.py")
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    got = ex.run(tokens=6000, steps=4, window=512, budget=2048)
    assert got["found"] > 0.8 and got["held"] == 2048
    assert got["search"] < 0.5 * got["window"]
