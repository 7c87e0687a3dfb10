"""KVCache at the edges of what a program may do with it."""
import pytest
import torch

import swann_b200 as swann

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def qkv(n, seed=0):
    """A projection's queries, keys and values of 4 and 2 heads of 64."""
    x = torch.randn((n, 8, 64), generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).half()
    return x[:, :4], x[:, 4:6], x[:, 6:]


def turns(n):
    angle = torch.arange(n, device=DEV)[:, None] * 10000.0 ** (-torch.arange(32, device=DEV) / 32)
    return angle.cos(), angle.sin()


@pytest.mark.parametrize("seqs,tokens", [(1, 5), (3, 2), (2, 0), (4, 5)])
@pytest.mark.parametrize("evicted", [False, True])
def test_append_without_starts_wants_a_token_for_each(seqs, tokens, evicted):
    cache = swann.KVCache(seqs, 64, 2, 64, track=True)
    if evicted:
        cache.evict(8)
    with pytest.raises(ValueError, match="one token for each"):
        cache.append(*qkv(tokens), *turns(64))
    assert cache.lengths.tolist() == cache.seen.tolist() == [0] * seqs and (cache.positions == -1).all()


@pytest.mark.parametrize("evicted", [False, True])
def test_append_of_a_padded_batch(evicted):
    """Tokens beyond starts[-1] are nobody's; after an eviction positions come from `seen`, padded or not."""
    cos, sin = turns(64)
    caches = [swann.KVCache(3, 48, 2, 64, page_size=16, track=True) for _ in range(2)]
    for c in caches:
        c.append(*qkv(3 + 9 + 6), cos, sin, ints(0, 3, 12, 18))
        if evicted:
            c.evict(4, sinks=1, recent=2)
    starts = ints(0, 2, 2, 7)
    x = qkv(12, 1)
    padded = caches[0].append(*x, cos, sin, starts)
    plain = caches[1].append(*(t[:7] for t in x), cos, sin, starts)
    assert torch.equal(padded[:7], plain)
    for name in ("k", "v", "lengths", "seen", "positions"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
    assert caches[0].seen.tolist() == [5, 9, 11]
    held = [3, 4, 4] if evicted else [3, 9, 6]
    assert caches[0].lengths.tolist() == [held[0] + 2, held[1], held[2] + 5]
    assert (caches[0].positions[2, :, held[2]:held[2] + 5] == ints(6, 7, 8, 9, 10)).all()
    assert (caches[0].positions[0, :, held[0]:held[0] + 2] == ints(3, 4)).all()
    assert (caches[0].positions[2, :, held[2] + 5:] == -1).all()


@pytest.mark.parametrize("budget", [None, 8])
@pytest.mark.parametrize("prompt", [1, 20])
def test_a_captured_step_goes_on_by_itself(budget, prompt):
    """append, attend and evict captured before the first eviction and replayed: as the same calls one by one."""
    cos, sin = turns(128)
    caches = [swann.KVCache(3, 96, 2, 64, page_size=16, track=True) for _ in range(2)]
    starts = ints(0, prompt, prompt + 1, 2 * prompt + 1)
    q, k, v = qkv(3 + 2 * prompt + 1)
    x = torch.empty((3, 8, 64), device=DEV).half()
    for c in caches:
        c.append(q[:2 * prompt + 1], k[:2 * prompt + 1], v[:2 * prompt + 1], cos, sin, starts)

    def step(c):
        got = c.attend(c.append(x[:, :4], x[:, 4:6], x[:, 6:], cos, sin))
        if budget:
            c.evict(budget, sinks=1, recent=2)
        return got

    held = {name: getattr(caches[0], name) for name in ("lengths", "seen", "weights", "positions", "k", "v", "table")}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    assert all(getattr(caches[0], name) is t for name, t in held.items())
    for i in range(12):
        x.copy_(torch.randn((3, 8, 64), generator=torch.Generator(device=DEV).manual_seed(i), device=DEV))
        graph.replay()
        want = step(caches[1])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
        for name in held:
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), (i, name)
    assert caches[0].seen.tolist() == [prompt + 12, 13, prompt + 12]
    if budget:
        assert caches[0].lengths.tolist() == [8] * 3


def test_a_captured_prompt_after_an_eviction():
    """Several tokens a sequence, captured before the cache is evicted: their positions come from `seen`."""
    cos, sin = turns(128)
    caches = [swann.KVCache(2, 96, 2, 64, page_size=16, track=True) for _ in range(2)]
    starts = ints(0, 5, 7)
    x = qkv(7)
    for c in caches:
        c.append(*x, cos, sin, starts)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = caches[0].append(*x, cos, sin, starts)
    for _ in range(3):
        for c in caches:
            c.evict(4, recent=2)
        graph.replay()
        want = caches[1].append(*x, cos, sin, starts)
        assert torch.equal(got, want)
        for name in ("lengths", "seen", "positions", "k", "v"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
