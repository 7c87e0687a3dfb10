"""The attention operators against their definitions in 64 bits.

Bounds.  u is the unit roundoff of the 16-bit type: half the spacing at 1, 2^-8
for bf16 (8 significant bits) and 2^-11 for fp16 (11).  A logit's error in 32-bit sums of exact products
is at most e = (d + 8) 2^-23 scale sum |q_i k_i|; it moves the lse by at most
max e and each weight by a factor within exp(2 e).  The weights are rounded to
16 bits once before the second product, and so is the result: out is within
  u |out| + (u + 2 e + 2^-18) sum_j p_j |v_j|
and lse within e + 2^-19 (1 + |lse|).  (2^-18 and 2^-19 cover the base-2
exponentials, the rescaling of the running sums and their additions.)  A prior
part adds its own |rows| to the sum.  Half a unit of fp16's smallest steps (2^-25)
is added where values come near zero.
"""
import math

import numpy as np
import pytest
import torch

from swann_b200 import attention as A

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make_cache(lengths, hkv, d, page, dtype, seed, max_pages=None, layout="head", garbage=True):
    """Pools with more pages than are used, pages in any order, and what no call may read set to NaN and infinities."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    per = [-(-n // page) for n in lengths]
    max_pages = max_pages or max(per + [1])
    pages = sum(per) + 3
    shape = (pages, hkv, page, d) if layout == "head" else (pages, page, hkv, d)
    pools = [torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2)]
    if layout != "head":
        pools = [p.transpose(1, 2) for p in pools]
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lengths), max_pages), -1, dtype=torch.int32, device=DEV)
    at, used = 0, torch.zeros((pages, page), dtype=torch.bool, device=DEV)
    for b, n in enumerate(lengths):
        table[b, :per[b]] = order[at:at + per[b]]
        at += per[b]
        for i in range(per[b]):
            used[table[b, i].item(), :min(page, n - i * page)] = True
    if garbage:
        for p, bad in zip(pools, (math.nan, math.inf)):
            p.masked_fill_(~used[:, None, :, None], bad)
    return pools[0], pools[1], table, torch.tensor(lengths, dtype=torch.int32, device=DEV)


def rows(pool, table, b, g, slots):
    """float64 rows of a sequence's slots; -1 pages as zeros, and which are there."""
    page = pool.shape[2]
    p = table[b].cpu().numpy()[slots // page]
    there = (p >= 0) & (p < pool.shape[0])
    x = pool[torch.from_numpy(np.where(there, p, 0)).long().to(DEV), g, torch.from_numpy(slots % page).to(DEV)].double()
    x[~torch.from_numpy(there).to(DEV)] = 0
    return x, torch.from_numpy(there).to(DEV)


def attend(q, k, v, table, b, g, pos, scale, window, sinks, length):
    """One query row at slot `pos`: logits' slots, (lse, out, sum p|v|, weights, e) in 64 bits."""
    cap = table.shape[1] * k.shape[2]
    j = np.arange(max(0, min(pos + 1, cap)))
    if window:
        j = j[(j > pos - window) | (j < sinks)]
    kr, there = rows(k, table, b, g, j)
    vr, _ = rows(v, table, b, g, j)
    qd = q.double()
    x = (kr @ qd * scale).masked_fill(~there, -math.inf)
    d = q.shape[0]
    e = 0.0
    if there.any():
        e = (d + 8) * 2.0 ** -23 * abs(scale) * float((kr[there].abs() @ qd.abs()).max())
    if not there.any():
        return j, -math.inf, torch.zeros(d, dtype=torch.float64, device=DEV), torch.zeros(d, dtype=torch.float64, device=DEV), torch.zeros(len(j), dtype=torch.float64, device=DEV), 0.0
    lse = float(torch.logsumexp(x, 0))
    p = torch.exp(x - lse)
    return j, lse, p @ vr, p @ vr.abs(), p, e


def check_row(out, lse, want, u, prior=None):
    _, wl, wo, wa, _, e = want
    if prior is not None:
        po, pl = prior[0].double(), float(prior[1])
        if pl != -math.inf:
            both = np.logaddexp(wl, pl)
            a, c = math.exp(wl - both) if wl != -math.inf else 0.0, math.exp(pl - both)
            wo, wa, wl = a * wo + c * po, a * wa + c * po.abs(), both
    if wl == -math.inf:
        assert float(lse) == -math.inf and (out == 0).all()
        return wl
    assert abs(float(lse) - wl) <= e + 2.0 ** -19 * (1 + abs(wl)), (float(lse), wl, e)
    bound = u * wo.abs() + (u + 2 * e + 2.0 ** -18) * wa + 2.0 ** -25
    over = ((out.double() - wo).abs() / bound).max()
    assert over <= 1, float(over)
    return wl


DECODE = [
    # lengths, q heads, kv heads, d, page, dtype, window, sinks, layout
    ([1], 1, 1, 64, 1, torch.float16, 0, 0, "head"),
    ([0, 1, 2, 15, 16, 17], 8, 2, 128, 16, torch.bfloat16, 0, 0, "head"),
    ([63, 64, 65, 129, 1000], 14, 2, 64, 64, torch.float16, 0, 0, "row"),
    ([5000], 32, 8, 128, 64, torch.bfloat16, 0, 0, "head"),
    ([5000, 0, 77], 6, 2, 128, 32, torch.float16, 0, 0, "row"),
    ([777, 100, 40, 3, 0], 8, 1, 128, 16, torch.bfloat16, 50, 4, "head"),
    ([3000, 51], 12, 4, 64, 1, torch.float16, 1000, 17, "head"),
    ([300], 20, 1, 64, 8, torch.bfloat16, 0, 0, "head"),
    ([300], 16, 1, 128, 128, torch.float16, 299, 1, "head"),
    ([70], 8, 8, 128, 16, torch.float16, 1, 0, "row"),
    ([4096] * 40, 4, 4, 64, 16, torch.bfloat16, 0, 0, "head"),
]


@pytest.mark.parametrize("lengths,hq,hkv,d,page,dtype,window,sinks,layout", DECODE)
@pytest.mark.parametrize("extra", ["plain", "weights", "prior"])
def test_decode(lengths, hq, hkv, d, page, dtype, window, sinks, layout, extra):
    k, v, table, L = make_cache(lengths, hkv, d, page, dtype, 3, layout=layout)
    g = torch.Generator(device=DEV).manual_seed(4)
    B = len(lengths)
    # queries as a view into a projection that holds more
    q = (torch.randn((B, 3 * hq, d), generator=g, device=DEV) * 1.5).to(dtype)[:, hq:2 * hq]
    prior = weights = None
    if extra == "prior":
        po = torch.randn((B, hq, d), generator=g, device=DEV).to(dtype)
        pl = torch.randn((B, hq), generator=g, device=DEV) * 3 + 3
        pl[::2, ::3] = -math.inf      # a part that saw nothing: its rows must not matter
        po[::2, ::3] = math.nan
        prior = (po, pl)
    if extra == "weights":
        weights = torch.full((B, hkv, table.shape[1] * page + 5), math.nan, device=DEV)
    out, lse = A.decode(q, k, v, table, L, window=window, sinks=sinks, prior=prior, weights=weights)
    assert out.shape == (B, hq, d) and out.dtype == dtype and lse.dtype == torch.float32
    G, scale = hq // hkv, d ** -0.5
    for b in sorted({0, B - 1, *range(min(B, 6))}):
        for grp in range(hkv):
            share = torch.zeros(weights.shape[2], dtype=torch.float64, device=DEV) if weights is not None else None
            e = 0.0
            for h in range(grp * G, (grp + 1) * G):
                want = attend(q[b, h], k, v, table, b, grp, lengths[b] - 1, scale, window, sinks, lengths[b])
                check_row(out[b, h], lse[b, h], want, U[dtype], (po[b, h], pl[b, h]) if prior else None)
                if share is not None:
                    share[torch.from_numpy(want[0]).to(DEV)] += want[4]
                    e = max(e, want[5])
            if share is not None:
                got = weights[b, grp].double()
                assert ((got - share).abs() <= (2 * e + 2.0 ** -18) * share + 1e-30).all()


def test_decode_accumulates_the_joined_shares():
    k, v, table, L = make_cache([200, 31], 2, 64, 16, torch.float16, 5)
    q = torch.randn((2, 4, 64), device=DEV).half()
    prior = (torch.zeros((2, 4, 64), device=DEV).half(), torch.full((2, 4), 1e4, device=DEV))
    w = torch.rand((2, 2, 208), device=DEV)
    w0 = w.clone()
    A.decode(q, k, v, table, L, weights=w, accumulate=True)
    once = torch.zeros_like(w)
    A.decode(q, k, v, table, L, weights=once)
    assert torch.allclose(w, w0 + once, rtol=2.0 ** -22, atol=0)
    assert torch.allclose(once.sum((1, 2)), torch.full((2,), 4.0, device=DEV), rtol=1e-5)
    # beside a part that has all of the weight, nothing is left for the cache's slots
    A.decode(q, k, v, table, L, prior=prior, weights=once)
    assert (once == 0).all()


def test_decode_over_search_results():
    """Pages of one row: a table of row ids, -1 anywhere among them, ids outside the pool ignored."""
    X = torch.randn((500, 1, 1, 128), device=DEV).half()
    V = torch.randn((500, 1, 1, 128), device=DEV).half()
    ids = torch.randint(0, 500, (9, 33), device=DEV, dtype=torch.int32)
    ids[0] = -1
    ids[1, ::2] = -1
    ids[2, 5:] = -1
    ids[3, 0] = 500
    ids[4, 7] = -2 ** 31
    q = torch.randn((9, 1, 128), device=DEV).half()
    n = torch.full((9,), 33, dtype=torch.int32, device=DEV)
    out, lse = A.decode(q, X, V, ids, n)
    for b in range(9):
        check_row(out[b, 0], lse[b, 0], attend(q[b, 0], X, V, ids, b, 0, 32, 128 ** -0.5, 0, 0, 33), U[torch.float16])
    assert (out[0] == 0).all() and lse[0, 0] == -math.inf


@pytest.mark.parametrize("B,hq,hkv,d,page,dtype", [
    (700, 1, 1, 128, 1, torch.float16), (650, 1, 1, 64, 1, torch.bfloat16), (300, 3, 3, 128, 16, torch.bfloat16),
    (700, 4, 1, 128, 1, torch.float16), (620, 7, 1, 64, 8, torch.bfloat16), (600, 12, 1, 128, 1, torch.bfloat16),
    (600, 20, 1, 64, 1, torch.float16)])
@pytest.mark.parametrize("window,sinks,extra", [(0, 0, "prior"), (0, 0, "weights"), (21, 3, "plain")])
def test_decode_of_very_many_short_sequences(B, hq, hkv, d, page, dtype, window, sinks, extra):
    """Short tables and hundreds of sequences: lengths of 0 to 90, -1 at the end of the table and inside it."""
    lengths = [(37 * b) % 91 for b in range(B)]
    k, v, table, L = make_cache(lengths, hkv, d, page, dtype, 51, max_pages=96 // page)
    table[::5, 1::3] = -1
    table[7, :] = -1
    q = (torch.randn((B, hq, d), device=DEV) * 1.5).to(dtype)
    prior = weights = None
    if extra == "prior":
        po, pl = torch.randn((B, hq, d), device=DEV).to(dtype), torch.randn((B, hq), device=DEV) * 3 + 3
        pl[::3], po[::3] = -math.inf, math.nan
        prior = (po, pl)
    if extra == "weights":
        weights = torch.full((B, hkv, 96), math.nan, device=DEV)
    out, lse = A.decode(q, k, v, table, L, window=window, sinks=sinks, prior=prior, weights=weights)
    G = hq // hkv
    for b in [*range(12), 35, B // 2, B - 2, B - 1]:
        for g in range(hkv):
            share, e = torch.zeros(96, dtype=torch.float64, device=DEV), 0.0
            for h in range(g * G, (g + 1) * G):
                want = attend(q[b, h], k, v, table, b, g, lengths[b] - 1, d ** -0.5, window, sinks, lengths[b])
                check_row(out[b, h], lse[b, h], want, U[dtype], (po[b, h], pl[b, h]) if prior else None)
                share[torch.from_numpy(want[0]).to(DEV)] += want[4]
                e = max(e, want[5])
            if weights is not None:
                assert ((weights[b, g].double() - share).abs() <= (2 * e + 2.0 ** -18) * share + 1e-30).all()


def test_decode_lengths_beyond_the_table_are_cut():
    k, v, table, L = make_cache([64], 1, 64, 16, torch.float16, 6)
    q = torch.randn((1, 2, 64), device=DEV).half()
    a = A.decode(q, k, v, table, L)
    L[0] = 2 ** 31 - 1
    b = A.decode(q, k, v, table, L)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    L[0] = -5
    out, lse = A.decode(q, k, v, table, L)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_decode_offsets_past_32_bits():
    """Rows beyond 2^32 elements of the pool."""
    page, d = 16, 64
    pages = (2 ** 32) // (page * d) + 8
    if torch.cuda.mem_get_info()[0] < 3 * pages * page * d * 2:
        pytest.skip("not enough memory")
    k = torch.empty((pages, 1, page, d), dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    far = torch.tensor([[pages - 1, 2, pages - 5]], dtype=torch.int32, device=DEV)
    for p in far[0].tolist():
        k[p], v[p] = torch.randn((1, page, d), device=DEV).half(), torch.randn((1, page, d), device=DEV).half()
    q = torch.randn((1, 2, d), device=DEV).half()
    L = torch.tensor([40], dtype=torch.int32, device=DEV)
    out, lse = A.decode(q, k, v, far, L)
    for h in range(2):
        check_row(out[0, h], lse[0, h], attend(q[0, h], k, v, far, 0, 0, 39, d ** -0.5, 0, 0, 40), U[torch.float16])


def test_decode_large_logits_and_signs():
    """Logits of thousands: the running maximum moves by far more than the exponential's range."""
    k, v, table, L = make_cache([600], 1, 128, 16, torch.bfloat16, 7)
    q = (torch.randn((1, 4, 128), device=DEV) * 300).bfloat16()
    for scale in (1.0, -1.0, 0.0):
        out, lse = A.decode(q, k, v, table, L, scale=scale)
        for h in range(4):
            want = attend(q[0, h], k, v, table, 0, 0, 599, scale, 0, 0, 600)
            check_row(out[0, h], lse[0, h], want, U[torch.bfloat16])


def test_decode_on_another_stream_and_in_a_graph():
    k, v, table, L = make_cache([3000, 5], 2, 128, 16, torch.float16, 8)
    q = torch.randn((2, 8, 128), device=DEV).half()
    want = A.decode(q, k, v, table, L)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = A.decode(q, k, v, table, L)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = A.decode(q, k, v, table, L)
    q.copy_(torch.randn_like(q))
    L.copy_(torch.tensor([2999, 4], dtype=torch.int32))
    graph.replay()
    want = A.decode(q, k, v, table, L)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


PREFILL = [
    # new tokens, held before, q heads, kv heads, d, page, dtype, window, sinks, layout
    ([1], [0], 1, 1, 64, 1, torch.float16, 0, 0, "head"),
    ([1, 0, 2, 127, 128, 129], [0, 5, 3, 0, 0, 1], 4, 2, 128, 16, torch.bfloat16, 0, 0, "head"),
    ([300, 7], [0, 500], 14, 2, 64, 64, torch.float16, 0, 0, "row"),
    ([513], [0], 8, 1, 128, 64, torch.bfloat16, 0, 0, "head"),
    ([400, 90, 1], [0, 300, 1000], 6, 2, 128, 16, torch.float16, 33, 4, "head"),
    ([700], [0], 4, 4, 64, 8, torch.bfloat16, 256, 17, "row"),
    ([260], [130], 20, 1, 64, 32, torch.float16, 128, 0, "head"),
    ([257], [0], 3, 1, 128, 128, torch.float16, 1, 300, "head"),
    ([65, 64, 63], [64, 64, 64], 2, 2, 128, 1, torch.bfloat16, 0, 0, "head"),
]


@pytest.mark.parametrize("new,held,hq,hkv,d,page,dtype,window,sinks,layout", PREFILL)
def test_prefill(new, held, hq, hkv, d, page, dtype, window, sinks, layout):
    lengths = [a + c for a, c in zip(new, held)]
    k, v, table, L = make_cache(lengths, hkv, d, page, dtype, 11, layout=layout)
    g = torch.Generator(device=DEV).manual_seed(12)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = (torch.randn((sum(new), 2 * hq, d), generator=g, device=DEV) * 1.5).to(dtype)[:, hq:]
    out, lse = A.prefill(q, k, v, table, torch.tensor(starts, dtype=torch.int32, device=DEV), L, window=window, sinks=sinks)
    G, scale = hq // hkv, d ** -0.5
    for b, n in enumerate(new):
        for t in sorted({0, 1, n // 2, n - 2, n - 1, *range(5, n, 41)} & set(range(n))):
            for h in {0, hq // 2, hq - 1}:
                want = attend(q[starts[b] + t, h], k, v, table, b, h // G, held[b] + t, scale, window, sinks, lengths[b])
                check_row(out[starts[b] + t, h], lse[starts[b] + t, h], want, U[dtype])
    assert torch.isfinite(out).all()


def test_prefill_of_many_sequences():
    """More sequences than a warp's lanes, more tiles than the GPU has SMs, some sequences without a new token."""
    new = [(37 * b) % 90 for b in range(70)]
    held = [(53 * b) % 200 for b in range(70)]
    lengths = [a + c for a, c in zip(new, held)]
    k, v, table, L = make_cache(lengths, 4, 64, 16, torch.float16, 61)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = torch.randn((sum(new), 4, 64), device=DEV).half()
    for window, sinks in ((0, 0), (64, 2)):
        out, lse = A.prefill(q, k, v, table, torch.tensor(starts, dtype=torch.int32, device=DEV), L, window=window, sinks=sinks)
        for b in (0, 1, 2, 31, 32, 33, 63, 64, 69):
            for t in sorted({0, new[b] // 2, new[b] - 1} & set(range(new[b]))):
                for h in range(4):
                    want = attend(q[starts[b] + t, h], k, v, table, b, h, held[b] + t, 0.125, window, sinks, lengths[b])
                    check_row(out[starts[b] + t, h], lse[starts[b] + t, h], want, U[torch.float16])
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()


def test_prefill_pages_that_hold_nothing():
    """Whole pages missing, among them all that the first tokens see."""
    k, v, table, L = make_cache([200], 2, 64, 16, torch.float16, 13)
    table[0, 0] = -1
    table[0, 5:8] = -1
    table[0, 9] = 10 ** 6
    q = torch.randn((200, 4, 64), device=DEV).half()
    starts = torch.tensor([0, 200], dtype=torch.int32, device=DEV)
    out, lse = A.prefill(q, k, v, table, starts, L)
    assert (out[:16] == 0).all() and (lse[:16] == -math.inf).all()
    for t in (0, 15, 16, 17, 79, 80, 127, 128, 143, 160, 199):
        for h in range(4):
            check_row(out[t, h], lse[t, h], attend(q[t, h], k, v, table, 0, h // 2, t, 0.125, 0, 0, 200), U[torch.float16])


def test_prefill_large_logits():
    k, v, table, L = make_cache([300], 1, 128, 16, torch.bfloat16, 14)
    q = (torch.randn((300, 2, 128), device=DEV) * 300).bfloat16()
    starts = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    for scale in (1.0, -1.0, 0.0):
        out, lse = A.prefill(q, k, v, table, starts, L, scale=scale)
        for t in (0, 1, 100, 255, 299):
            check_row(out[t, 1], lse[t, 1], attend(q[t, 1], k, v, table, 0, 0, t, scale, 0, 0, 300), U[torch.bfloat16])


def test_prefill_of_one_token_is_decode():
    k, v, table, L = make_cache([900, 33], 2, 128, 16, torch.float16, 15)
    q = torch.randn((2, 8, 128), device=DEV).half()
    a = A.decode(q, k, v, table, L, window=100, sinks=3)
    b = A.prefill(q, k, v, table, torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), L, window=100, sinks=3)
    assert torch.allclose(a[1], b[1], rtol=0, atol=1e-5)
    assert torch.allclose(a[0].float(), b[0].float(), rtol=2.0 ** -9, atol=2.0 ** -10)


def test_prefill_starts_outside_the_batch_stay_inside():
    k, v, table, L = make_cache([50, 50], 1, 64, 16, torch.float16, 16)
    q = torch.randn((40, 2, 64), device=DEV).half()
    good = A.prefill(q, k, v, table, torch.tensor([0, 20, 40], dtype=torch.int32, device=DEV), L)
    A.prefill(q, k, v, table, torch.tensor([-7, 20, 10 ** 6], dtype=torch.int32, device=DEV), L)
    again = A.prefill(q, k, v, table, torch.tensor([0, 20, 40], dtype=torch.int32, device=DEV), L)
    assert torch.equal(good[0], again[0])


APPEND = [
    # new tokens, held, q heads, kv heads, d, page, dtype, rotated, interleaved, norm, layout
    ([1], [0], 1, 1, 64, 1, torch.float16, 64, False, True, "head"),
    ([1, 1, 1], [5, 0, 63], 8, 2, 128, 16, torch.bfloat16, 128, False, True, "head"),
    ([37, 0, 130], [0, 7, 33], 6, 3, 128, 64, torch.float16, 64, False, True, "row"),
    ([100], [28], 5, 5, 64, 16, torch.bfloat16, 32, True, False, "head"),
    ([65], [0], 7, 1, 64, 32, torch.float16, 48, False, True, "head"),
    ([9], [3], 4, 2, 128, 8, torch.bfloat16, 128, True, True, "row"),
    ([12], [0], 4, 2, 128, 8, torch.float16, 0, False, True, "row"),
]


@pytest.mark.parametrize("new,held,hq,hkv,d,page,dtype,rot,interleaved,norm,layout", APPEND)
@pytest.mark.parametrize("moved", [False, True])
def test_append(new, held, hq, hkv, d, page, dtype, rot, interleaved, norm, layout, moved):
    """Within one rounding of the definition: |error| <= u |y| + 2^-19 (|a| + |b|) of the rotated pair."""
    lengths = [a + c for a, c in zip(new, held)]
    k, v, table, L = make_cache(lengths, hkv, d, page, dtype, 21, layout=layout, garbage=False)
    g = torch.Generator(device=DEV).manual_seed(22)
    T = sum(new)
    qkv = (torch.randn((T, (hq + 2 * hkv) * d), generator=g, device=DEV) * 2).to(dtype)
    q, kn, vn = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
    w = [(1 + 0.3 * torch.randn(d, generator=g, device=DEV)).to(dtype) if norm else None for _ in range(2)]
    angle = torch.rand((300, rot // 2), generator=g, device=DEV) * 6.28
    cos, sin = angle.cos(), angle.sin()
    pos = torch.randint(0, 300, (T,), generator=g, device=DEV, dtype=torch.int32) if moved else None
    starts = np.concatenate([[0], np.cumsum(new)])
    k0, v0 = k.clone(), v.clone()
    sp = torch.full((len(new), hkv, table.shape[1] * page), -7, dtype=torch.int32, device=DEV)
    out = A.rope_append(q, kn, vn, cos, sin, k, v, table, torch.tensor(starts, dtype=torch.int32, device=DEV), L,
                        q_norm=w[0], k_norm=w[1], positions=pos, interleaved=interleaved, slot_positions=sp)
    first = np.arange(0, rot, 2) if interleaved else np.arange(rot // 2)
    second = first + (1 if interleaved else rot // 2)

    def want(x, weight, p):
        y = x.double()
        if weight is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.double()
        c, s = cos[p].double(), sin[p].double()
        z, a = y.clone(), y.abs()
        z[:, first], z[:, second] = y[:, first] * c - y[:, second] * s, y[:, second] * c + y[:, first] * s
        m = a.clone()
        m[:, first] = m[:, second] = a[:, first] + a[:, second]
        return z, m

    def close(got, pair):
        z, m = pair
        assert ((got.double() - z).abs() <= U[dtype] * z.abs() + 2.0 ** -19 * m + 2.0 ** -25).all()

    for b, n in enumerate(new):
        for i in range(n):
            t, slot = starts[b] + i, held[b] + i
            p = slot if pos is None else int(pos[t])
            pg, r = int(table[b, slot // page]), slot % page
            close(out[t], want(q[t], w[0], p))
            close(k[pg, :, r], want(kn[t], w[1], p))
            assert torch.equal(v[pg, :, r], vn[t])
            assert (sp[b, :, slot] == p).all()
            k0[pg, :, r], v0[pg, :, r] = k[pg, :, r], v[pg, :, r]
            sp[b, :, slot] = -7
    assert torch.equal(k, k0) and torch.equal(v, v0) and (sp == -7).all()   # nothing else was touched


def test_append_where_there_is_no_page():
    """Tokens past the table, or on a page of -1: their queries come out, nothing is written."""
    k, v, table, L = make_cache([64], 1, 64, 16, torch.float16, 23, garbage=False)
    table[0, 1] = -1
    table[0, 2] = 10 ** 6
    L[0] = 70
    x = torch.randn((70, 4, 64), device=DEV).half()
    cos = torch.ones((60, 32), device=DEV)
    k0 = k.clone()
    out = A.rope_append(x[:, :2], x[:, 2:3], x[:, 3:], cos, cos * 0, k, v, table,
                        torch.tensor([0, 70], dtype=torch.int32, device=DEV), L)
    assert torch.equal(out[:60], x[:60, :2])
    assert torch.isnan(out[60:]).all()          # positions past the tables
    for p, first in ((0, 0), (3, 48)):
        n = min(64, 60) - first if p == 3 else 16
        k0[table[0, p], 0, :n] = x[first:first + n, 2]
        k0[table[0, p], 0, n:] = k[table[0, p], 0, n:]
    assert torch.equal(k.nan_to_num(), k0.nan_to_num())


def plain_evict(k, v, table, L, w, pos, budget, seen, sinks, recent):
    k, v, nw, npos, nl = k.clone(), v.clone(), w.clone(), pos.clone(), L.clone()
    page = k.shape[2]
    for b in range(w.shape[0]):
        n = int(L[b])
        nl[b] = min(n, budget)
        for h in range(w.shape[1]):
            nw[b, h, min(n, budget):] = 0
            npos[b, h, min(n, budget):] = -1
            if n <= budget:
                continue
            p, x = pos[b, h, :n].tolist(), w[b, h, :n].double().tolist()
            key = [(2, 0.0) if 0 <= p[j] < sinks or p[j] >= int(seen[b]) - recent else
                   (0, 0.0) if math.isnan(x[j]) else (1, x[j] + 0.0) for j in range(n)]
            keep = sorted(sorted(range(n), key=lambda j: (tuple(-c for c in key[j]), j))[:budget])
            late = [j for j in keep if j >= budget]
            free = sorted(set(range(budget)) - set(keep))
            for a, z in zip(late, free):
                nw[b, h, z], npos[b, h, z] = w[b, h, a], pos[b, h, a]
                pa, pz = int(table[b, a // page]), int(table[b, z // page])
                if pa >= 0 and pz >= 0:
                    k[pz, h, z % page], v[pz, h, z % page] = k[pa, h, a % page].clone(), v[pa, h, a % page].clone()
    return nl, nw, npos, k, v


EVICT = [
    # lengths, kv heads, d, page, budget, sinks, recent, kind, layout
    ([1], 1, 64, 1, 1, 0, 0, "random", "head"),
    ([0, 1, 7, 8, 9, 300], 2, 128, 8, 8, 1, 3, "random", "head"),
    ([513, 1000], 3, 64, 16, 512, 4, 100, "random", "row"),
    ([700, 33], 2, 128, 64, 100, 0, 0, "ties", "head"),
    ([700, 33], 2, 128, 32, 100, 4, 96, "ties", "head"),
    ([2000], 2, 64, 16, 1, 1, 0, "random", "head"),
    ([400], 1, 64, 16, 50, 0, 7, "odd", "row"),
    ([5000, 4097], 1, 64, 16, 4096, 4, 256, "random", "head"),
    ([90000], 1, 64, 128, 777, 4, 256, "ties", "head"),
]


@pytest.mark.parametrize("lengths,hkv,d,page,budget,sinks,recent,kind,layout", EVICT)
def test_evict(lengths, hkv, d, page, budget, sinks, recent, kind, layout):
    k, v, table, L = make_cache(lengths, hkv, d, page, torch.float16, 31, layout=layout, garbage=False)
    W = table.shape[1] * page + 3
    g = torch.Generator(device=DEV).manual_seed(32)
    w = torch.rand((len(lengths), hkv, W), generator=g, device=DEV)
    if kind == "ties":
        w = (w * 4).floor()
        w[..., ::7] = -0.0
    if kind == "odd":
        w = w - 0.5
        w[..., 3::11] = math.nan
        w[..., 4::11] = math.inf
        w[..., 5::11] = -math.inf
    pos = torch.stack([torch.randperm(2 * W, generator=g, device=DEV)[:W] for _ in range(len(lengths) * hkv)])
    pos = pos.view(len(lengths), hkv, W).to(torch.int32)
    seen = torch.full((len(lengths),), 2 * W, dtype=torch.int32, device=DEV)
    want = plain_evict(k, v, table, L, w, pos, budget, seen, sinks, recent)
    before = w.clone(), pos.clone(), L.clone()
    for _ in range(2):    # the inputs are not touched, and rows already moved move again to the same place
        got = (*A.evict(k, v, table, L, w, pos, budget, seen=seen, sinks=sinks, recent=recent), k, v)
        for a, c in zip(got, want):
            assert torch.equal(a.nan_to_num(nan=9.0), c.nan_to_num(nan=9.0)) if a.is_floating_point() else torch.equal(a, c)
    assert all(torch.equal(a.nan_to_num(nan=9.0), c.nan_to_num(nan=9.0)) for a, c in zip(before[:1], (w,)))
    assert torch.equal(before[1], pos) and torch.equal(before[2], L)


def test_refusals():
    k, v, table, L = make_cache([40, 8], 2, 64, 16, torch.float16, 41, garbage=False)
    q = torch.randn((2, 4, 64), device=DEV).half()
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    w, pos = torch.zeros((2, 2, 48), device=DEV), torch.zeros((2, 2, 48), dtype=torch.int32, device=DEV)
    cos = torch.ones((64, 32), device=DEV)
    no = pytest.raises
    with no(ValueError, match="float16 or bfloat16"):
        A.decode(q.float(), k.float(), v.float(), table, L)
    with no(ValueError, match="same strides"):
        A.decode(q, k, v[:, :1], table, L)
    with no(ValueError, match="head_dim"):
        A.decode(q[..., :48], k[..., :48], v[..., :48], table, L)
    with no(ValueError, match="power of two"):
        A.decode(q, k[:, :, :12], v[:, :, :12], table, L)
    with no(ValueError, match="int32"):
        A.decode(q, k, v, table.long(), L)
    with no(ValueError, match="lengths"):
        A.decode(q, k, v, table, L.long())
    with no(ValueError, match="one token"):
        A.decode(q[:1], k, v, table, L)
    with no(ValueError, match="multiple"):
        A.decode(q[:, :3], k, v, table, L)
    with no(ValueError, match="16-byte"):
        A.decode(torch.randn((2, 4 * 64 + 4), device=DEV).half()[:, 4:].unflatten(1, (4, 64)), k, v, table, L)
    with no(ValueError, match="rows of q"):
        A.decode(torch.randn((2, 64, 4), device=DEV).half().transpose(1, 2), k, v, table, L)
    with no(ValueError, match="negative"):
        A.decode(q, k, v, table, L, window=-1)
    with no(ValueError, match="negative"):
        A.prefill(q, k, v, table, starts, L, window=1 << 31)
    with no(ValueError, match="no backward pass"):
        A.decode(q.clone().requires_grad_(), k, v, table, L)
    with torch.no_grad():
        A.decode(q.clone().requires_grad_(), k, v, table, L)
    with no(ValueError, match="narrower"):
        A.decode(q, k, v, table, L, weights=w[..., :40].contiguous())
    with no(ValueError, match="prior"):
        A.decode(q, k, v, table, L, prior=(q, torch.zeros((2, 3), device=DEV)))
    with no(ValueError, match="starts"):
        A.prefill(q, k, v, table, starts[:2], L)
    with no(ValueError, match="cos and sin"):
        A.rope_append(q, q[:, :2], q[:, :2], cos, cos.half(), k, v, table, starts, L)
    with no(ValueError, match="multiple of 16"):
        A.rope_append(q, q[:, :2], q[:, :2], cos[:, :12].contiguous(), cos[:, :12].contiguous(), k, v, table, starts, L)
    with no(ValueError, match="same tokens"):
        A.rope_append(q, q[:1, :2], q[:, :2], cos, cos, k, v, table, starts, L)
    with no(ValueError, match="q_norm"):
        A.rope_append(q, q[:, :2], q[:, :2], cos, cos, k, v, table, starts, L, q_norm=cos[0])
    with no(ValueError, match="budget"):
        A.evict(k, v, table, L, w, pos, 8, seen=L, sinks=4, recent=5)
    with no(ValueError, match="positions"):
        A.evict(k, v, table, L, w, pos[..., :40], 8, seen=L)
    with no(ValueError, match="on the GPU"):
        A.decode(q.cpu(), k.cpu(), v.cpu(), table.cpu(), L.cpu())


def test_a_pool_without_pages_holds_nothing():
    k = torch.empty((0, 2, 16, 64), dtype=torch.float16, device=DEV)
    table, L = torch.zeros((1, 3), dtype=torch.int32, device=DEV), torch.full((1,), 40, dtype=torch.int32, device=DEV)
    q = torch.randn((40, 4, 64), device=DEV).half()
    for out, lse in (A.decode(q[:1], k, k, table, L),
                     A.prefill(q, k, k, table, torch.tensor([0, 40], dtype=torch.int32, device=DEV), L)):
        assert (out == 0).all() and (lse == -math.inf).all()


def test_empty_batches():
    k, v, table, L = make_cache([8], 2, 64, 16, torch.float16, 42)
    none = torch.empty((0, 4, 64), dtype=torch.float16, device=DEV)
    out, lse = A.decode(none, k, v, table[:0], L[:0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    starts = torch.zeros(2, dtype=torch.int32, device=DEV)
    out, lse = A.prefill(none, k, v, table, starts, L)
    assert out.shape == (0, 4, 64)
    cos = torch.ones((4, 32), device=DEV)
    assert A.rope_append(none, none[:, :2], none[:, :2], cos, cos, k, v, table, starts, L).shape == (0, 4, 64)


def test_decode_shares_of_many_heads_to_a_key_head():
    """70 heads share a key head, more than one CTA's table of sums holds, in pairs cut among runs."""
    test_decode([2000, 0, 65], 140, 2, 64, 16, torch.float16, 0, 0, "head", "weights")


@pytest.mark.parametrize("lengths", [[5000], [1, 3000, 64, 0], [40] * 9])
def test_decode_shares_beside_a_prior_part(lengths):
    """One head to a key head: a prior part scales its slots' shares by exp(lse alone - lse of both).

    The two lse are fp32 of magnitude below 16 and each within 2^-19 (1 + |lse|), so the
    factor is within 2 * 17 * 2^-19 < 2^-13."""
    k, v, table, L = make_cache(lengths, 4, 64, 16, torch.float16, 8)
    g = torch.Generator(device=DEV).manual_seed(9)
    B = len(lengths)
    q = torch.randn((B, 4, 64), generator=g, device=DEV).half()
    prior = (torch.randn((B, 4, 64), generator=g, device=DEV).half(), torch.randn((B, 4), generator=g, device=DEV) * 3 + 6)
    prior[1][:, 1] = -math.inf
    alone, both = (torch.full((B, 4, table.shape[1] * 16), math.nan, device=DEV) for _ in range(2))
    _, l0 = A.decode(q, k, v, table, L, weights=alone)
    _, l1 = A.decode(q, k, v, table, L, weights=both, prior=prior)
    assert float(l1[l1 > -math.inf].abs().max()) < 16
    f = torch.where(l0 == -math.inf, 0.0, (l0.double() - l1.double()).exp())
    assert torch.allclose(both.double(), alone.double() * f.unsqueeze(-1), rtol=2.0 ** -13, atol=1e-30)
