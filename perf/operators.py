"""The attention operators' cases: what is timed, on which inputs, and what the answers are.

Four operators over one paged key-value cache (pools [pages, kv_heads, page_size, head_dim], a page table per
sequence, the number of slots each sequence holds):

  append   norms of queries and keys per head and the position rotation, keys and values written to the cache
  decode   attention of one new token per sequence, joined with a prior partial result, weights per slot
  prefill  attention of a ragged batch of new tokens, causal, with a sliding window and first tokens
  evict    the cache cut to a budget by accumulated attention weight

`run` is the plain torch form of each, or with `own` the calls of swann_b200.attention; `exact` is the definition in
64 bits.  Head counts and sizes are generic ones of decoders with grouped key heads; 100 rows a query is the k of this
repository's largest search configuration.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# -- cases ----------------------------------------------------------------------------------------------------------

def _append(name, seqs, tokens, held, hq, hkv, d, page, dtype, rot, interleaved=False, norm=True, moved=False):
    """`tokens`: of the longest sequence's addition, `held`: slots before it, `moved`: positions that are not the slots."""
    return {"name": name, "op": "append", "seqs": seqs, "tokens": tokens, "held": held, "hq": hq, "hkv": hkv, "d": d,
            "page": page, "dtype": dtype, "rot": rot, "interleaved": interleaved, "norm": norm, "moved": moved}


def _decode(name, seqs, longest, ragged, hq, hkv, d, page, dtype, window=0, sinks=0, weights=False, prior=False, rows=0):
    """`rows`: the pool is a corpus of that many rows with a page a row, and the table lists rows (some of them -1)."""
    return {"name": name, "op": "decode", "seqs": seqs, "longest": longest, "ragged": ragged, "hq": hq, "hkv": hkv,
            "d": d, "page": page, "dtype": dtype, "window": window, "sinks": sinks, "weights": weights, "prior": prior,
            "rows": rows}


def _prefill(name, seqs, tokens, ragged, held, hq, hkv, d, page, dtype, window=0, sinks=0):
    return {"name": name, "op": "prefill", "seqs": seqs, "tokens": tokens, "ragged": ragged, "held": held, "hq": hq,
            "hkv": hkv, "d": d, "page": page, "dtype": dtype, "window": window, "sinks": sinks}


def _evict(name, seqs, longest, ragged, hkv, d, page, dtype, budget, sinks, recent):
    return {"name": name, "op": "evict", "seqs": seqs, "longest": longest, "ragged": ragged, "hkv": hkv, "d": d,
            "page": page, "dtype": dtype, "budget": budget, "sinks": sinks, "recent": recent}


def listed():
    return [
        # one conversation's next token, in a cache that eviction has shortened: latency
        _append("append-token", 1, 1, 4095, 32, 8, 128, 64, "bf16", 128, moved=True),
        # several prompts brought in together
        _append("append-prompts", 5, 4711, 0, 32, 8, 128, 16, "bf16", 128),
        # one conversation's next token: latency
        _decode("decode-one", 1, 1027, False, 32, 8, 128, 16, "bf16"),
        # a server's batch of conversations of every length
        _decode("decode-batch", 48, 8191, True, 32, 8, 128, 16, "bf16"),
        # one very long document, with the weights by which its cache is trimmed afterwards
        _decode("decode-long", 1, 131071, False, 32, 4, 128, 64, "fp16", weights=True),
        # the always-attended part of long conversations: the newest tokens and the first ones
        _decode("decode-window", 64, 8192, True, 32, 8, 128, 64, "fp16", window=1024, sinks=4),
        # the rows that a search of each head's keys returned, joined with what the head attended elsewhere
        _decode("decode-retrieved", 4096, 100, True, 1, 1, 128, 1, "fp16", prior=True, rows=1_000_000),
        # a document's next part, after what earlier parts left in the cache
        _prefill("prefill-chunk", 1, 2049, False, 6144, 32, 8, 128, 64, "bf16"),
        # a long document brought in by window and first tokens, the rest left to the index
        _prefill("prefill-window", 1, 8192, False, 0, 32, 8, 128, 64, "bf16", window=1024, sinks=4),
        # a server's batch of ordinary prompts, every head with keys of its own
        _prefill("prefill-prompts", 23, 1500, True, 0, 16, 16, 64, 16, "fp16"),
        # a cache at its budget takes one more token and drops one
        _evict("evict-one", 1, 4097, False, 8, 128, 64, "bf16", 4096, 4, 256),
        # several prompts cut to their budget after they came in
        _evict("evict-prompts", 8, 16384, True, 8, 128, 64, "bf16", 2048, 4, 512),
    ]


def _log(rng, lo, hi):
    """A whole number, spread over the logarithm of lo..hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill", "prefill", "evict"])
    d, dtype = rng.choice([64, 128]), rng.choice(["fp16", "bf16"])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 7, 8])
    page = rng.choice([1, 8, 16, 32, 64, 128])
    window, sinks = rng.choice([(0, 0), (_log(rng, 16, 4096), rng.choice([0, 1, 4, 17]))])
    if op == "append":
        seqs = _log(rng, 1, 512)
        rot = rng.choice([d, d, d // 2])
        return _drawn(_append("", seqs, _log(rng, 1, max(1, 20000 // seqs)), _log(rng, 1, 2048) - 1, hq, hkv, d, page, dtype, rot,
                              rng.random() < 0.3, rng.random() < 0.8, rng.random() < 0.3))
    if op == "decode":
        if rng.random() < 0.25:
            return _drawn(_decode("", _log(rng, 1, 4096), _log(rng, 1, 200), True, 1, 1, d, 1, dtype,
                                  prior=rng.random() < 0.5, rows=_log(rng, 1000, 1_000_000)))
        seqs = _log(rng, 1, 256)
        longest = _log(rng, 1, max(16, min(131072, 3_000_000 // (seqs * hkv))))
        return _drawn(_decode("", seqs, longest, rng.random() < 0.7, hq, hkv, d, page, dtype, window, sinks,
                              rng.random() < 0.3, rng.random() < 0.3))
    if op == "prefill":
        seqs = _log(rng, 1, 32)
        tokens = _log(rng, 1, max(1, min(8192, int(8192 / math.sqrt(seqs * hq / 32 + 1)))))
        held = rng.choice([0, _log(rng, 1, 4096)])
        held = min(held, max(0, 1_500_000_000 // (tokens * seqs * hq) - tokens))
        return _drawn(_prefill("", seqs, tokens, rng.random() < 0.7, held, hq, hkv, d, page, dtype, window, sinks))
    seqs = _log(rng, 1, 32)
    longest = _log(rng, 2, max(64, min(65536, 1_000_000 // (seqs * hkv))))
    budget = max(1, min(longest, _log(rng, 1, longest)))
    sinks = min(rng.choice([0, 1, 4, 17]), budget)
    return _drawn(_evict("", seqs, longest, rng.random() < 0.7, hkv, d, page, dtype, budget, sinks,
                         rng.randint(0, budget - sinks)))


def _drawn(case):
    del case["name"]
    return case


# -- inputs ---------------------------------------------------------------------------------------------------------

def _spread(n, longest, ragged):
    """n lengths up to `longest`, the first the longest; a ragged batch's over the logarithm of 1/16..1 of it."""
    return [max(1, int(longest * 16.0 ** -((i * 0.6180339887) % 1.0))) if ragged else longest for i in range(n)]


def _counts(case):
    """(new tokens, slots held with them) of each sequence."""
    if case["op"] == "append":
        new = _spread(case["seqs"], case["tokens"], True)
        return new, [n + case["held"] for n in new]
    if case["op"] == "prefill":
        new = _spread(case["seqs"], case["tokens"], case["ragged"])
        return new, [n + case["held"] for n in new]
    held = _spread(case["seqs"], case["longest"], case["ragged"])
    return [1] * case["seqs"], held


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(case, held, g):
    """The pools, all sequences' pages in any order, and the table."""
    page, hkv, d, dt = case["page"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    per = [-(-n // page) for n in held]
    pages = sum(per)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(held), max(per)), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(max(per), device="cuda")[None, :] < torch.tensor(per, device="cuda")[:, None]
    table[at] = order
    k = torch.randn((pages, hkv, page, d), generator=g, device="cuda", dtype=dt)
    v = torch.randn((pages, hkv, page, d), generator=g, device="cuda", dtype=dt)
    return k, v, table


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, d, dt, seqs = case["op"], case["d"], DTYPES[case["dtype"]], case["seqs"]
    new, held = _counts(case)
    s = {"case": case, "op": op, "lengths": _ints(held)}

    def randn(*shape, dtype=dt, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    if op == "decode" and case["rows"]:
        rows, k = case["rows"], case["longest"]
        s["k"], s["v"] = randn(rows, 1, 1, d), randn(rows, 1, 1, d)
        s["table"] = torch.randint(0, rows, (seqs, k), generator=g, device="cuda", dtype=torch.int32)
        # a search returns -1 for what it did not find: here from each query's own count of rows on
        s["table"].masked_fill_(torch.arange(k, device="cuda")[None, :] >= s["lengths"][:, None], -1)
        s["lengths"] = _ints([k] * seqs)
    else:
        s["k"], s["v"], s["table"] = _cache(case, held, g)
    if op == "append":
        T, hq, hkv, r = sum(new), case["hq"], case["hkv"], case["rot"]
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s["starts"] = _ints(starts)
        # one projection's output: queries, keys and values of a token side by side
        qkv = randn(T, (hq + 2 * hkv) * d, scale=1.5)
        s["q"], s["kn"], s["vn"] = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
        s["qw"] = (1 + 0.2 * randn(d, dtype=torch.float32)).to(dt) if case["norm"] else None
        s["kw"] = (1 + 0.2 * randn(d, dtype=torch.float32)).to(dt) if case["norm"] else None
        most = max(held) + (20000 if case["moved"] else 0)
        angle = torch.arange(most, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(0, r, 2, device="cuda").double() / r)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["positions"] = torch.randint(0, most, (T,), generator=g, device="cuda", dtype=torch.int32) if case["moved"] else None
    elif op == "decode":
        s["q"] = randn(seqs, case["hq"], d, scale=1.5)
        s["prior"] = None
        if case["prior"]:
            s["prior"] = (randn(seqs, case["hq"], d, scale=0.2), 5.0 + randn(seqs, case["hq"], dtype=torch.float32))
        if case["weights"]:
            s["width"] = s["table"].shape[1] * case["page"]
    elif op == "prefill":
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s["starts"] = _ints(starts)
        s["most"] = max(new)
        s["q"] = randn(sum(new), case["hq"], d, scale=1.5)
    else:
        hkv, W = case["hkv"], s["table"].shape[1] * case["page"]
        # a few slots have most of the weight, many hardly any, some none at all
        w = torch.exp(2.0 * torch.randn((seqs, hkv, W), generator=g, device="cuda"))
        s["weights"] = w * (torch.rand((seqs, hkv, W), generator=g, device="cuda") > 0.02)
        s["seen"] = s["lengths"] * 2
        # an earlier eviction has left the slots in any order, and the later half of the positions
        far = torch.arange(W, device="cuda")[None, None, :] >= s["lengths"][:, None, None]
        order = torch.rand((seqs, hkv, W), generator=g, device="cuda").masked_fill_(far, 2.0).argsort(-1)
        place = (order + s["lengths"][:, None, None]).to(torch.int32)
        place = torch.where((order < case["sinks"]) & ~far, order.to(torch.int32), place)
        s["positions"] = place.masked_fill_(far, -1)
        s["weights"].masked_fill_(far, 0.0)
    return s


# -- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        return _OWN[s["op"]](s, case)
    return _PLAIN[s["op"]](s, case)


def _own_append(s, case):
    from swann_b200 import attention as A
    q = A.rope_append(s["q"], s["kn"], s["vn"], s["cos"], s["sin"], s["k"], s["v"], s["table"], s["starts"], s["lengths"],
                      q_norm=s["qw"], k_norm=s["kw"], eps=EPS, positions=s["positions"], interleaved=case["interleaved"])
    return {"q": q, "k": s["k"], "v": s["v"]}


def _own_decode(s, case):
    from swann_b200 import attention as A
    w = None
    if case["weights"]:
        w = torch.empty((case["seqs"], case["hkv"], s["width"]), dtype=torch.float32, device="cuda")
    out, lse = A.decode(s["q"], s["k"], s["v"], s["table"], s["lengths"], window=case["window"], sinks=case["sinks"],
                        prior=s["prior"], weights=w)
    return {"out": out, "lse": lse, **({"weights": w} if w is not None else {})}


def _own_prefill(s, case):
    from swann_b200 import attention as A
    out, lse = A.prefill(s["q"], s["k"], s["v"], s["table"], s["starts"], s["lengths"], window=case["window"],
                         sinks=case["sinks"])
    return {"out": out, "lse": lse}


def _own_evict(s, case):
    from swann_b200 import attention as A
    lengths, weights, positions = A.evict(s["k"], s["v"], s["table"], s["lengths"], s["weights"], s["positions"],
                                          case["budget"], seen=s["seen"], sinks=case["sinks"], recent=case["recent"])
    return {"lengths": lengths, "weights": weights, "positions": positions, "k": s["k"], "v": s["v"]}


_OWN = {"append": _own_append, "decode": _own_decode, "prefill": _own_prefill, "evict": _own_evict}


def _token_places(s, T):
    """Each token's sequence and slot."""
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"], t, right=True) - 1
    slot = s["lengths"][seq] - (s["starts"][seq + 1] - t)
    return seq, slot


def _normed(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _rotated(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., r:]], -1)


def _plain_append(s, case):
    q, page = s["q"], case["page"]
    seq, slot = _token_places(s, q.shape[0])
    at = slot if s["positions"] is None else s["positions"]
    cos, sin = s["cos"][at], s["sin"][at]
    out = _rotated(_normed(q, s["qw"]), cos, sin, case["interleaved"]).to(q.dtype)
    kn = _rotated(_normed(s["kn"], s["kw"]), cos, sin, case["interleaved"]).to(q.dtype)
    pages, row = s["table"][seq, slot // page], slot % page
    s["k"][pages, :, row] = kn
    s["v"][pages, :, row] = s["vn"]
    return {"q": out, "k": s["k"], "v": s["v"]}


def _dense(pool, table):
    """[sequences, kv_heads, slots, head_dim] in 32 bits."""
    x = pool[table.clamp(min=0)]
    return x.transpose(1, 2).flatten(2, 3).float()


def _plain_decode(s, case):
    q, page, hkv = s["q"], case["page"], case["hkv"]
    B, hq, d = q.shape
    kd, vd = _dense(s["k"], s["table"]), _dense(s["v"], s["table"])
    slot = torch.arange(kd.shape[2], device="cuda")[None, :]
    L = s["lengths"][:, None]
    seen = (slot < L) & (s["table"] >= 0).repeat_interleave(page, 1)
    if case["window"]:
        seen &= (slot >= L - case["window"]) | (slot < case["sinks"])
    seen = seen[:, None, None, :]
    logit = (q.float().view(B, hkv, hq // hkv, d) @ kd.transpose(2, 3)) * d ** -0.5
    logit = logit.masked_fill(~seen, -math.inf)
    top = logit.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(logit - top)
    total = e.sum(-1, keepdim=True)
    lse = (torch.log(total) + top).view(B, hq)
    out = ((e @ vd) / total.clamp(min=1e-30)).view(B, hq, d)
    if s["prior"] is not None:
        po, pl = s["prior"]
        both = torch.logaddexp(lse, pl)
        out = torch.exp(lse - both)[..., None] * out + torch.exp(pl - both)[..., None] * po.float()
        lse = both
    got = {"out": out.to(q.dtype), "lse": lse}
    if case["weights"]:
        got["weights"] = torch.exp(logit - lse.view(B, hkv, -1, 1)).sum(2)
    return got


def _plain_prefill(s, case):
    q, hkv, page = s["q"], case["hkv"], case["page"]
    T, hq, d = q.shape
    seq, slot = _token_places(s, T)
    B, N = s["lengths"].shape[0], s["most"]
    at = torch.arange(T, device="cuda") - s["starts"][seq]
    qd = torch.zeros((B, N, hq, d), dtype=torch.float32, device="cuda")
    qd[seq, at] = q.float()
    place = torch.full((B, N), -1, dtype=torch.int32, device="cuda")
    place[seq, at] = slot
    kd, vd = _dense(s["k"], s["table"]), _dense(s["v"], s["table"])
    key = torch.arange(kd.shape[2], device="cuda")[None, None, :]
    mine = place[:, :, None]
    seen = (key <= mine) & (s["table"] >= 0).repeat_interleave(page, 1)[:, None, :]
    if case["window"]:
        seen &= (key > mine - case["window"]) | (key < case["sinks"])
    seen = seen[:, None, None, :, :]
    logit = qd.view(B, N, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4) @ kd[:, :, None].transpose(3, 4)
    logit = (logit * d ** -0.5).masked_fill_(~seen, -math.inf)
    top = logit.amax(-1, keepdim=True).clamp(min=-3e38)
    e = logit.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    lse = (torch.log(total) + top).squeeze(-1).flatten(1, 2)
    out = ((e @ vd[:, :, None]) / total.clamp(min=1e-30)).flatten(1, 2)
    return {"out": out[seq, :, at].to(q.dtype), "lse": lse[seq, :, at]}


def _plain_evict(s, case):
    m, page, W = case["budget"], case["page"], s["weights"].shape[2]
    L = s["lengths"]
    slot = torch.arange(W, device="cuda")
    inside = slot < L[:, None, None]
    pos = s["positions"]
    fixed = (pos < case["sinks"]) | (pos >= (s["seen"] - case["recent"])[:, None, None])
    key = torch.where(fixed, math.inf, s["weights"]).masked_fill(~inside, -math.inf)
    # equal weights: the lower slot first, which a stable sort keeps
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order))
    kept = (rank < m) & inside
    # the i-th kept slot from the budget on goes to the i-th free one below it
    free = ~kept & (slot < torch.clamp(L, max=m)[:, None, None])
    late = kept & (slot >= m)
    b, h, to = free.nonzero(as_tuple=True)
    source = late.nonzero(as_tuple=True)[2]
    weights = s["weights"].masked_fill(~kept | (slot >= m), 0.0)
    positions = pos.masked_fill(~kept | (slot >= m), -1)
    weights[b, h, to] = s["weights"][b, h, source]
    positions[b, h, to] = pos[b, h, source]
    table = s["table"]
    to_page, to_row = table[b, to // page], to % page
    from_page, from_row = table[b, source // page], source % page
    s["k"][to_page, h, to_row] = s["k"][from_page, h, from_row]
    s["v"][to_page, h, to_row] = s["v"][from_page, h, from_row]
    return {"lengths": L.clamp(max=m), "weights": weights, "positions": positions, "k": s["k"], "v": s["v"]}


_PLAIN = {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill, "evict": _plain_evict}


# -- what a pass cannot do without ----------------------------------------------------------------------------------

def _visible(length, case):
    """How many of `length` slots the token after them sees."""
    if not case["window"] or length <= case["window"]:
        return length
    return case["window"] + min(case["sinks"], length - case["window"])


def work(case):
    d, op = case["d"], case["op"]
    new, held = _counts(case)
    if op == "append":
        T, n = sum(new), case["hq"] + 2 * case["hkv"]
        return {"bytes": T * (4 * n * d + 4 * case["rot"]), "flops": T * (case["hq"] + case["hkv"]) * d * 7}
    hkv = case["hkv"]
    if op == "decode":
        seen = sum(_visible(n, case) for n in held)
        small = case["seqs"] * case["hq"] * (4 * d + 4) * (2 if case["prior"] else 1)
        width = -(-max(held) // case["page"]) * case["page"]
        rows = 4 * hkv * d * seen + 4 * (seen if case["rows"] else -(-seen // case["page"]))
        return {"bytes": rows + small + (4 * hkv * width * case["seqs"] if case["weights"] else 0),
                "flops": 4 * d * case["hq"] * seen}
    if op == "prefill":
        pairs, rows, w = 0, 0, case["window"]
        for n, L in zip(new, held):
            first = L - n
            pairs += _pairs(L, w, case["sinks"]) - _pairs(first, w, case["sinks"])
            rows += L if not w else min(L, n + w - 1 + case["sinks"])
        return {"bytes": 4 * hkv * d * rows + sum(new) * case["hq"] * (4 * d + 4), "flops": 4 * d * case["hq"] * pairs}
    m, width = case["budget"], -(-max(held) // case["page"]) * case["page"]
    moved = sum((m - min(n, case["sinks"] + case["recent"])) * (n - m) / n for n in held if n > m)
    return {"bytes": int(hkv * (sum(held) * 8 + width * 8 * len(held) + moved * 8 * d)), "flops": 2 * hkv * sum(held)}


def _pairs(length, window, sinks):
    """Visible pairs of the tokens at slots 0..length-1."""
    if not window or length <= window:
        return length * (length + 1) // 2
    far = length - window
    ends = sum(min(sinks, i) for i in range(1, min(far, sinks) + 1)) + max(0, far - sinks) * sinks
    return window * (window + 1) // 2 + far * window + ends


# -- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "prefill": _exact_prefill, "evict": _exact_evict}[case["op"]](s, case)


def _exact_append(s, case):
    new, held = _counts(case)
    r, page = case["rot"], case["page"]
    first, second = (torch.arange(0, r, 2), torch.arange(1, r, 2)) if case["interleaved"] else (torch.arange(r // 2), torch.arange(r // 2, r))

    def turned(x, w, c, n):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / case["d"] + EPS) * w.double()
        z = y.clone()
        z[:, :, first] = y[:, :, first] * c[:, None] - y[:, :, second] * n[:, None]
        z[:, :, second] = y[:, :, first] * n[:, None] + y[:, :, second] * c[:, None]
        return z

    k, v, q, t = s["k"].double(), s["v"].double(), [], 0
    for b, (n, L) in enumerate(zip(new, held)):
        slots = torch.arange(L - n, L, device="cuda")
        at = slots if s["positions"] is None else s["positions"][t:t + n].long()
        c, sn = s["cos"].double()[at], s["sin"].double()[at]
        q.append(turned(s["q"][t:t + n], s["qw"], c, sn))
        pages = s["table"][b].long()[torch.div(slots, page, rounding_mode="floor")]
        kr = turned(s["kn"][t:t + n], s["kw"], c, sn)
        for h in range(case["hkv"]):
            k[pages, h, slots % page] = kr[:, h]
            v[pages, h, slots % page] = s["vn"][t:t + n, h].double()
        t += n
    return {"q": torch.cat(q), "k": k, "v": v}


def _rows_of(pool, table, page, b, h, slots):
    return pool[table[b].long()[torch.div(slots, page, rounding_mode="floor")], h, slots % page].double()


def _exact_decode(s, case):
    if case["seqs"] * case["hkv"] > 8192:
        return None
    q, (B, hq, d) = s["q"].double(), s["q"].shape
    G, page, L = hq // case["hkv"], case["page"], s["lengths"].tolist()
    out, lse = torch.zeros(B, hq, d, dtype=torch.float64, device="cuda"), torch.zeros(B, hq, dtype=torch.float64, device="cuda")
    weights = torch.zeros(B, case["hkv"], s["width"], dtype=torch.float64, device="cuda") if case["weights"] else None
    for b in range(B):
        slots = torch.arange(L[b], device="cuda")
        if case["window"]:
            slots = torch.cat([slots[:max(0, L[b] - case["window"])][:case["sinks"]], slots[max(0, L[b] - case["window"]):]])
        if case["rows"]:
            slots = slots[s["table"][b][:L[b]] >= 0]
        for h in range(case["hkv"]):
            mine = slice(h * G, (h + 1) * G)
            x = q[b, mine] @ _rows_of(s["k"], s["table"], page, b, h, slots).T / math.sqrt(d)
            part, o = torch.logsumexp(x, -1), torch.softmax(x, -1) @ _rows_of(s["v"], s["table"], page, b, h, slots)
            if s["prior"] is not None:
                share = torch.sigmoid(s["prior"][1][b, mine].double() - part)[:, None]
                o = (1 - share) * o + share * s["prior"][0][b, mine].double()
                part = torch.logaddexp(part, s["prior"][1][b, mine].double())
            out[b, mine], lse[b, mine] = o, part
            if weights is not None:
                weights[b, h, slots] = torch.exp(x - part[:, None]).sum(0)
    return {"out": out, "lse": lse, **({"weights": weights} if weights is not None else {})}


def _exact_prefill(s, case):
    new, held = _counts(case)
    q, (T, hq, d) = s["q"], s["q"].shape
    G, page, t = hq // case["hkv"], case["page"], 0
    out, lse = torch.zeros(T, hq, d, dtype=torch.float64, device="cuda"), torch.zeros(T, hq, dtype=torch.float64, device="cuda")
    for b, (n, L) in enumerate(zip(new, held)):
        slots = torch.arange(L, device="cuda")
        for h in range(case["hkv"]):
            kr, vr = (_rows_of(s[x], s["table"], page, b, h, slots) for x in ("k", "v"))
            for a in range(0, n, 2048):
                e = min(n, a + 2048)
                me = torch.arange(L - n + a, L - n + e, device="cuda")[:, None]
                hidden = slots[None] > me
                if case["window"]:
                    hidden |= (me - slots[None] >= case["window"]) & (slots[None] >= case["sinks"])
                x = q[t + a:t + e, h * G:(h + 1) * G].double().transpose(0, 1) @ kr.T / math.sqrt(d)
                x[:, hidden] = -math.inf
                lse[t + a:t + e, h * G:(h + 1) * G] = torch.logsumexp(x, -1).T
                out[t + a:t + e, h * G:(h + 1) * G] = (torch.softmax(x, -1) @ vr).transpose(0, 1)
        t += n
    return {"out": out, "lse": lse}


def _exact_evict(s, case):
    """Nothing here is computed in floating point: the kept weights are copies, checked in the same way."""
    m, page, L = case["budget"], case["page"], s["lengths"].tolist()
    weights, positions = s["weights"].double(), s["positions"].cpu()
    k, v = s["k"].double(), s["v"].double()
    w, seen = s["weights"].cpu(), s["seen"].tolist()
    for b, n in enumerate(L):
        if n <= m:
            continue
        for h in range(case["hkv"]):
            p = positions[b, h, :n]
            fixed = (p < case["sinks"]) | (p >= seen[b] - case["recent"])
            key = torch.where(fixed, torch.full((n,), math.inf, dtype=torch.float64), w[b, h, :n].double())
            best = torch.sort(-key, stable=True).indices[:m].sort().values
            late = best[best >= m]
            held = torch.zeros(m, dtype=torch.bool)
            held[best[best < m]] = True
            free = (~held).nonzero()[:, 0]
            weights[b, h, m:] = 0
            weights[b, h, free.cuda()] = w[b, h, late].double().cuda()
            at, to = late.cuda(), free.cuda()
            pages = s["table"][b].long()
            for pool in (k, v):
                pool[pages[torch.div(to, page, rounding_mode="floor")], h, to % page] = \
                    pool[pages[torch.div(at, page, rounding_mode="floor")], h, at % page]
    return {"lengths": None, "weights": weights, "positions": None, "k": k, "v": v}
