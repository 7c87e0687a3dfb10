"""Attention of a language model over a key-value cache that the index can search.

A decoder's cached keys are a corpus: a token's logit is an inner product, and
`Index` finds the rows with the largest ones.  These are the operators around
that search, all on one paged cache:

    rope_append   new tokens in: norms per head, position rotation, keys and
                  values written to their slots
    prefill       attention of many new tokens, causal, with a sliding window
                  and first tokens that stay visible
    decode        attention of one new token per sequence, over the whole cache
                  or the window and first tokens; joined with the attention over
                  other keys (`prior`); the weight of every slot if wanted
    evict         the cache cut to a budget by accumulated weight

The cache is two pools [pages, kv_heads, page_size, head_dim] (fp16 or bf16,
any strides with contiguous rows), a page table [seqs, max_pages] int32 and
the number of slots each sequence holds, [seqs] int32.  Slot j of a sequence is
row j % page_size of page table[seq, j // page_size]; a page of -1 holds
nothing.  With pages of one row the table lists rows: the ids that
`Index.search_tensors` returns (-1 where there are fewer) are a table, and
`decode` over the searched vectors attends exactly what the search found.

`KVCache` keeps the pieces together for the ordinary case.  Nothing here reads
a device value on the host: the calls queue on the current stream and can be
captured in a CUDA graph.  There is no backward pass: the package serves
models, it does not train them.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import _lib as N

_DTYPES = {torch.float16: N.F16, torch.bfloat16: N.BF16}
HEAD_DIMS = (64, 128)


def _fail(what, why):
    raise ValueError(f"{what}: {why}")


def _on(t):
    """Kernels launch on the tensors' device."""
    if t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _ints(what, name, t, shape, device):
    if t.dtype != torch.int32 or t.device != device or tuple(t.shape) != shape or not t.is_contiguous():
        _fail(what, f"{name} must be contiguous int32 {list(shape)} on {device}")


def _cache_arg(what, k, v, table, lengths):
    if k.device.type != "cuda":
        _fail(what, "the cache must be on the GPU")
    if k.dtype not in _DTYPES or v.dtype != k.dtype:
        _fail(what, "the cache must be float16 or bfloat16")
    if k.dim() != 4 or v.shape != k.shape or v.stride() != k.stride() or v.device != k.device:
        _fail(what, "k and v must be [pages, kv_heads, page_size, head_dim] with the same strides")
    pages, heads, page, d = k.shape
    ps, hs, rs, es = k.stride()
    if d not in HEAD_DIMS:
        _fail(what, f"head_dim must be one of {HEAD_DIMS}")
    if es != 1:
        _fail(what, "the rows of the cache must be contiguous")
    if page < 1 or page & (page - 1):
        _fail(what, "page_size must be a power of two")
    if table.dim() != 2 or table.dtype != torch.int32 or table.device != k.device or \
            (table.shape[1] > 1 and table.stride(1) != 1):
        _fail(what, f"the page table must be int32 [seqs, max_pages] on {k.device}, rows contiguous")
    _ints(what, "lengths", lengths, (table.shape[0],), k.device)
    return N.KVCacheArg(N.ptr(k), N.ptr(v), ps, hs, rs, N.ptr(table), table.stride(0), N.ptr(lengths), pages,
                        table.shape[1], page, table.shape[0], heads, d, _DTYPES[k.dtype])


def _heads(what, name, t, k, heads=None):
    """[tokens, heads, head_dim] of the cache's type, any strides with contiguous rows."""
    if t.dim() != 3 or t.shape[2] != k.shape[3] or t.dtype != k.dtype or t.device != k.device:
        _fail(what, f"{name} must be [tokens, heads, {k.shape[3]}] {k.dtype} on {k.device}")
    if heads is not None and t.shape[1] != heads:
        _fail(what, f"{name} must have {heads} heads")
    if t.stride(2) != 1:
        _fail(what, f"the rows of {name} must be contiguous")


def _out(what, name, t, like_shape, dtype, device):
    if t is None:
        return torch.empty(like_shape, dtype=dtype, device=device)
    if tuple(t.shape) != tuple(like_shape) or t.dtype != dtype or t.device != device or not t.is_contiguous():
        _fail(what, f"{name} must be contiguous {dtype} {list(like_shape)} on {device}")
    return t


def rope_append(q, k, v, cos, sin, k_cache, v_cache, table, starts, lengths, *, q_norm=None, k_norm=None, eps=1e-6,
                positions=None, interleaved=False, slot_positions=None, out=None):
    """New tokens' queries and keys normed per head and rotated, keys and values written to the cache.

    q [tokens, q_heads, d], k and v [tokens, kv_heads, d]: views into one
    projection are fine.  Tokens starts[b] .. starts[b + 1] - 1 (starts int32
    [seqs + 1]) are sequence b's, and take the last of its lengths[b] slots:
    lengths count them already.  cos, sin float32 [positions, r / 2] rotate the
    first r dimensions, pairs (i, i + r / 2) or, interleaved, (2i, 2i + 1), by
    the token's position: `positions` int32 [tokens], or its slot.  A position
    outside the tables gives NaN.  q_norm, k_norm [d]: weights of the norms,
    None for no norm.  slot_positions int32 [seqs, kv_heads, slots] records the
    positions.  Returns the queries [tokens, q_heads, d]."""
    what = "rope_append"
    arg = _cache_arg(what, k_cache, v_cache, table, lengths)
    T, hq, d = q.shape if q.dim() == 3 else (0, 0, 0)
    hkv = k_cache.shape[1]
    _heads(what, "q", q, k_cache)
    _heads(what, "k", k, k_cache, hkv)
    _heads(what, "v", v, k_cache, hkv)
    if k.shape[0] != T or v.shape[0] != T:
        _fail(what, "q, k and v must have the same tokens")
    if hq < 1 or hq % hkv:
        _fail(what, "query heads must be a multiple of the cache's key heads")
    dev = q.device
    _ints(what, "starts", starts, (table.shape[0] + 1,), dev)
    if cos.dim() != 2 or cos.shape != sin.shape:
        _fail(what, "cos and sin must be [positions, rotated / 2]")
    for t in (cos, sin):
        if t.dtype != torch.float32 or t.device != dev or not t.is_contiguous():
            _fail(what, f"cos and sin must be contiguous float32 on {dev}")
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None and (w.dtype != q.dtype or w.device != dev or tuple(w.shape) != (d,) or not w.is_contiguous()):
            _fail(what, f"{name} must be contiguous {q.dtype} [{d}] on {dev}")
    if positions is not None:
        _ints(what, "positions", positions, (T,), dev)
    width = 0
    if slot_positions is not None:
        width = slot_positions.shape[-1]
        _ints(what, "slot_positions", slot_positions, (table.shape[0], hkv, width), dev)
    out = _out(what, "out", out, (T, hq, d), q.dtype, dev)
    with _on(q):
        rc = N.lib().swb_rope_append(
            N.ptr(q), q.stride(0), q.stride(1), N.ptr(k), k.stride(0), k.stride(1), N.ptr(v), v.stride(0), v.stride(1),
            hq, N.ptr(starts), T, N.ptr(q_norm), N.ptr(k_norm), float(eps), N.ptr(cos), N.ptr(sin), cos.shape[0],
            2 * cos.shape[1], int(bool(interleaved)), N.ptr(positions), C.byref(arg), N.ptr(out),
            N.ptr(slot_positions), width, N.stream_of(q))
    N.check(rc, what)
    return out


def decode(q, k_cache, v_cache, table, lengths, *, scale=None, window=0, sinks=0, prior=None, weights=None,
           accumulate=False, out=None):
    """Attention of each sequence's newest token over its slots.

    q [seqs, q_heads, d] (normed and rotated).  With a window, only the newest
    `window` slots and the first `sinks` are seen.  scale: d ** -0.5 if None.
    prior (out, lse): attention over other keys, joined as if those had been
    in the cache too.  weights float32 [seqs, kv_heads, slots]: each slot's
    share of the (joined) softmax, summed over the query heads of its key head,
    is written there, or added with `accumulate`.  Returns out [seqs, q_heads,
    d] and lse float32 [seqs, q_heads], 0 and -inf where nothing is seen."""
    what = "decode"
    arg = _cache_arg(what, k_cache, v_cache, table, lengths)
    _heads(what, "q", q, k_cache)
    B, hq, d = q.shape
    if B != table.shape[0]:
        _fail(what, f"q must have one token for each of the {table.shape[0]} sequences")
    if hq < 1 or hq % k_cache.shape[1]:
        _fail(what, "query heads must be a multiple of the cache's key heads")
    dev = q.device
    po = pl = None
    if prior is not None:
        po = _out(what, "the prior rows", prior[0], (B, hq, d), q.dtype, dev)
        pl = _out(what, "the prior lse", prior[1], (B, hq), torch.float32, dev)
    width = 0
    if weights is not None:
        width = weights.shape[-1]
        _out(what, "weights", weights, (B, k_cache.shape[1], width), torch.float32, dev)
        if width < table.shape[1] * k_cache.shape[2]:
            _fail(what, "weights are narrower than the page table's slots")
    out = _out(what, "out", out, (B, hq, d), q.dtype, dev)
    lse = torch.empty((B, hq), dtype=torch.float32, device=dev)
    if B == 0:
        return out, lse
    L = N.lib()
    with _on(q):
        need = L.swb_attn_decode_workspace(C.byref(arg), hq, int(weights is not None))
        ws = torch.empty((need if need < 1 << 62 else 0,), dtype=torch.uint8, device=dev)
        rc = L.swb_attn_decode(
            N.ptr(q), q.stride(0), q.stride(1), hq, C.byref(arg), d ** -0.5 if scale is None else float(scale),
            int(window), int(sinks), N.ptr(po), N.ptr(pl), N.ptr(out), N.ptr(lse), N.ptr(weights), width,
            int(bool(accumulate)), N.ptr(ws), ws.numel(), N.stream_of(q))
    N.check(rc, what)
    return out, lse


def prefill(q, k_cache, v_cache, table, starts, lengths, *, scale=None, window=0, sinks=0, out=None):
    """Attention of a ragged batch of new tokens, causal.

    q [tokens, q_heads, d]; starts and lengths as in `rope_append`, which has
    written the tokens' keys: a token at slot i sees the slots j <= i and, with
    a window, of those only j > i - window and j < sinks.  Returns out
    [tokens, q_heads, d] and lse float32 [tokens, q_heads]."""
    what = "prefill"
    arg = _cache_arg(what, k_cache, v_cache, table, lengths)
    _heads(what, "q", q, k_cache)
    T, hq, d = q.shape
    if hq < 1 or hq % k_cache.shape[1]:
        _fail(what, "query heads must be a multiple of the cache's key heads")
    dev = q.device
    _ints(what, "starts", starts, (table.shape[0] + 1,), dev)
    out = _out(what, "out", out, (T, hq, d), q.dtype, dev)
    lse = torch.empty((T, hq), dtype=torch.float32, device=dev)
    if T == 0:
        return out, lse
    with _on(q):
        rc = N.lib().swb_attn_prefill(
            N.ptr(q), q.stride(0), q.stride(1), hq, N.ptr(starts), T, C.byref(arg),
            d ** -0.5 if scale is None else float(scale), int(window), int(sinks), N.ptr(out), N.ptr(lse),
            None, N.stream_of(q))
    N.check(rc, what)
    return out, lse


def evict(k_cache, v_cache, table, lengths, weights, positions, budget, *, seen, sinks=0, recent=0):
    """Every sequence cut to `budget` slots by accumulated weight.

    weights float32 and positions int32 [seqs, kv_heads, slots], seen int32
    [seqs] the positions given out so far.  Per key head the slots stay whose
    position is below `sinks` or among the `recent` newest, then those with the
    largest weight, ties to the lowest slot.  Kept slots below the budget stay
    in place, kept ones beyond it move, in order, to the free slots below it,
    in order: the order of slots is then no longer the order of positions.
    Rows move inside the pools; returns the new (lengths, weights, positions)
    as tensors of their own, 0 and -1 in slots that hold nothing."""
    what = "evict"
    arg = _cache_arg(what, k_cache, v_cache, table, lengths)
    B, hkv, dev = table.shape[0], k_cache.shape[1], k_cache.device
    if weights.dim() != 3:
        _fail(what, "weights must be float32 [seqs, kv_heads, slots]")
    width = weights.shape[2]
    _out(what, "weights", weights, (B, hkv, width), torch.float32, dev)
    _ints(what, "positions", positions, (B, hkv, width), dev)
    _ints(what, "seen", seen, (B,), dev)
    if width < table.shape[1] * k_cache.shape[2]:
        _fail(what, "weights are narrower than the page table's slots")
    if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
        _fail(what, "the budget must be at least 1, and hold sinks and recent")
    nl, nw, np_ = torch.empty_like(lengths), torch.empty_like(weights), torch.empty_like(positions)
    if B == 0:
        return nl, nw, np_
    L = N.lib()
    with _on(k_cache):
        ws = torch.empty((L.swb_kv_evict_workspace(B, hkv, int(budget)),), dtype=torch.uint8, device=dev)
        rc = L.swb_kv_evict(C.byref(arg), N.ptr(seen), N.ptr(weights), N.ptr(positions), width, int(budget), int(sinks),
                            int(recent), N.ptr(nl), N.ptr(nw), N.ptr(np_), N.ptr(ws), ws.numel(), N.stream_of(k_cache))
    N.check(rc, what)
    return nl, nw, np_
