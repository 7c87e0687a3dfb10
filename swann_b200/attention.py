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
captured in a CUDA graph.  `prefill` waits inside its kernel, with a limit of
seconds; should a wait give up, its rows are NaN and the next call here that is
made after that raises SwannError.  There is no backward pass: the package serves
models, it does not train them, and refuses tensors that want a gradient.
"""
from __future__ import annotations

import torch

from . import _lib as N

_DTYPES = {torch.float16: N.F16, torch.bfloat16: N.BF16}
HEAD_DIMS = (64, 128)


_stream = torch._C._cuda_getCurrentRawStream       # of a device index: no Stream object is made


def _fail(what, why):
    raise ValueError(f"{what}: {why}")


def _call(what, fn, t, *args):
    """A native call on the tensors' device and its current stream."""
    dev = t.get_device()
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(dev))
    if rc:
        N.check(rc, what)


def _no_gradient(what, name, t):
    """A gradient would be lost without a word."""
    if t.requires_grad and torch.is_grad_enabled():
        _fail(what, f"{name} requires a gradient, and there is no backward pass: call under torch.no_grad()")


def _ints(what, name, t, shape, dev):
    if t.dtype is not torch.int32 or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        _fail(what, f"{name} must be contiguous int32 {list(shape)} on cuda:{dev}")


def _cache_arg(what, k, v, table, lengths):
    """The cache as the native calls take it, and its device."""
    dev = k.get_device()
    if dev < 0:
        _fail(what, "the cache must be on the GPU")
    kind = _DTYPES.get(k.dtype)
    if kind is None or v.dtype is not k.dtype:
        _fail(what, "the cache must be float16 or bfloat16")
    shape, strides = k.shape, k.stride()
    if len(shape) != 4 or v.shape != shape or v.stride() != strides or v.get_device() != dev:
        _fail(what, "k and v must be [pages, kv_heads, page_size, head_dim] with the same strides")
    _no_gradient(what, "the cache", k)
    _no_gradient(what, "the cache", v)
    pages, heads, page, d = shape
    ps, hs, rs, es = strides
    if heads < 1:
        _fail(what, "the cache must have a key head")
    if d not in HEAD_DIMS:
        _fail(what, f"head_dim must be one of {HEAD_DIMS}")
    if es != 1:
        _fail(what, "the rows of the cache must be contiguous")
    if page < 1 or page & (page - 1):
        _fail(what, "page_size must be a power of two")
    at = table.shape
    if len(at) != 2 or table.dtype is not torch.int32 or table.get_device() != dev or \
            (at[1] > 1 and table.stride(1) != 1):
        _fail(what, f"the page table must be int32 [seqs, max_pages] on cuda:{dev}, rows contiguous")
    seqs, most = at
    if lengths.dtype is not torch.int32 or lengths.get_device() != dev or lengths.shape != (seqs,) or \
            not lengths.is_contiguous():
        _fail(what, f"lengths must be contiguous int32 [{seqs}] on cuda:{dev}")
    return N.KVCacheArg(k.data_ptr(), v.data_ptr(), ps, hs, rs, table.data_ptr(), table.stride(0), lengths.data_ptr(),
                        pages, most, page, seqs, heads, d, kind), dev


def _heads(what, name, t, d, dtype, dev, heads=None):
    """[tokens, heads, head_dim] of the cache's type, any strides with contiguous rows; its shape and strides."""
    shape, strides = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != d or t.dtype is not dtype or t.get_device() != dev:
        _fail(what, f"{name} must be [tokens, heads, {d}] {dtype} on cuda:{dev}")
    if heads is not None and shape[1] != heads:
        _fail(what, f"{name} must have {heads} heads")
    if strides[2] != 1:
        _fail(what, f"the rows of {name} must be contiguous")
    _no_gradient(what, name, t)
    return shape, strides


def _given(what, name, t, shape, dtype, dev):
    if t.shape != shape or t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        _fail(what, f"{name} must be contiguous {dtype} {list(shape)} on cuda:{dev}")
    _no_gradient(what, name, t)
    return t


def _count(what, name, n):
    """A count as the native calls take it."""
    if not 0 <= n < 1 << 31:
        _fail(what, f"{name} must not be negative or beyond 2^31")
    return n


def _group(what, q_heads, kv_heads):
    if q_heads < 1 or q_heads % kv_heads:
        _fail(what, "query heads must be a multiple of the cache's key heads")


def rope_append(q, k, v, cos, sin, k_cache, v_cache, table, starts, lengths, *, q_norm=None, k_norm=None, eps=1e-6,
                positions=None, interleaved=False, slot_positions=None, out=None):
    """New tokens' queries and keys normed per head and rotated, keys and values written to the cache.

    q [tokens, q_heads, d], k and v [tokens, kv_heads, d]: views into one
    projection are fine.  Tokens starts[b] .. starts[b + 1] - 1 (starts int32
    [seqs + 1], ascending) are sequence b's, and take the last of its lengths[b]
    slots: lengths count them already.  A token whose slot the table has no page
    for is not stored, nor is one of no sequence (a batch padded beyond
    starts[seqs]), whose query is rotated only if `positions` has one.  cos, sin float32 [positions, r / 2] rotate the
    first r dimensions, pairs (i, i + r / 2) or, interleaved, (2i, 2i + 1), by
    the token's position: `positions` int32 [tokens], or its slot.  A position
    outside the tables gives NaN.  q_norm, k_norm [d]: weights of the norms,
    None for no norm.  slot_positions int32 [seqs, kv_heads, slots] records the
    positions.  Returns the queries [tokens, q_heads, d]."""
    what = "rope_append"
    arg, dev = _cache_arg(what, k_cache, v_cache, table, lengths)
    hkv, seqs = arg.kv_heads, arg.seqs
    d, dtype = arg.head_dim, k_cache.dtype
    (T, hq, _), qs = _heads(what, "q", q, d, dtype, dev)
    ksh, ks = _heads(what, "k", k, d, dtype, dev, hkv)
    vsh, vs = _heads(what, "v", v, d, dtype, dev, hkv)
    if ksh[0] != T or vsh[0] != T:
        _fail(what, "q, k and v must have the same tokens")
    _group(what, hq, hkv)
    _ints(what, "starts", starts, (seqs + 1,), dev)
    rows = cos.shape
    if len(rows) != 2 or sin.shape != rows:
        _fail(what, "cos and sin must be [positions, rotated / 2]")
    for t in (cos, sin):
        if t.dtype is not torch.float32 or t.get_device() != dev or not t.is_contiguous():
            _fail(what, f"cos and sin must be contiguous float32 on cuda:{dev}")
        _no_gradient(what, "the rotation table", t)
    if q_norm is not None:
        _given(what, "q_norm", q_norm, (d,), q.dtype, dev)
    if k_norm is not None:
        _given(what, "k_norm", k_norm, (d,), q.dtype, dev)
    if positions is not None:
        _ints(what, "positions", positions, (T,), dev)
    width = 0
    if slot_positions is not None:
        width = slot_positions.shape[-1]
        _ints(what, "slot_positions", slot_positions, (seqs, hkv, width), dev)
    out = (torch.empty_like(q) if q.is_contiguous() else q.new_empty((T, hq, d))) if out is None else _given(what, "out", out, (T, hq, d), q.dtype, dev)
    if T:
        _call(what, N.lib().swb_rope_append, q, q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0],
              vs[1], hq, starts.data_ptr(), T, N.ptr(q_norm), N.ptr(k_norm), eps, cos.data_ptr(), sin.data_ptr(), rows[0],
              2 * rows[1], bool(interleaved), N.ptr(positions), arg, out.data_ptr(), N.ptr(slot_positions), width)
    return out


def decode(q, k_cache, v_cache, table, lengths, *, scale=None, window=0, sinks=0, prior=None, weights=None,
           accumulate=False, out=None):
    """Attention of each sequence's newest token over its slots.

    q [seqs, q_heads, d] (normed and rotated).  With a window, only the newest
    `window` slots and the first `sinks` are seen.  scale: d ** -0.5 if None.
    prior (out, lse): attention over other keys, joined as if those had been
    in the cache too.  weights float32 [seqs, kv_heads, slots]: each slot's
    share of the (joined) softmax, summed over the query heads of its key head,
    is written there, or added with `accumulate`.  `out` and prior rows start on
    8-byte boundaries.  Returns out [seqs, q_heads, d] and lse float32 [seqs,
    q_heads], 0 and -inf where nothing is seen."""
    what = "decode"
    arg, dev = _cache_arg(what, k_cache, v_cache, table, lengths)
    d, dtype = arg.head_dim, k_cache.dtype
    (B, hq, _), qs = _heads(what, "q", q, d, dtype, dev)
    if B != arg.seqs:
        _fail(what, f"q must have one token for each of the {arg.seqs} sequences")
    _group(what, hq, arg.kv_heads)
    po = pl = wp = None
    if prior is not None:
        po = _given(what, "the prior rows", prior[0], (B, hq, d), q.dtype, dev).data_ptr()
        pl = _given(what, "the prior lse", prior[1], (B, hq), torch.float32, dev).data_ptr()
    width = 0
    if weights is not None:
        width = weights.shape[-1]
        wp = _given(what, "weights", weights, (B, arg.kv_heads, width), torch.float32, dev).data_ptr()
        if width < arg.max_pages * arg.page_size:
            _fail(what, "weights are narrower than the page table's slots")
    out = (torch.empty_like(q) if q.is_contiguous() else q.new_empty((B, hq, d))) if out is None else _given(what, "out", out, (B, hq, d), q.dtype, dev)
    lse = q.new_empty((B, hq), dtype=torch.float32)
    if B == 0:
        return out, lse
    L = N.lib()
    need = L.swb_attn_decode_workspace(arg, hq, wp is not None)
    # a size that says the call will be refused is left to the call
    ws = q.new_empty(need if need < 1 << 62 else 0, dtype=torch.uint8)
    _call(what, L.swb_attn_decode, q, q.data_ptr(), qs[0], qs[1], hq, arg, d ** -0.5 if scale is None else scale,
          _count(what, "window", window), _count(what, "sinks", sinks), po, pl, out.data_ptr(), lse.data_ptr(), wp, width, bool(accumulate), ws.data_ptr(), need)
    return out, lse


def prefill(q, k_cache, v_cache, table, starts, lengths, *, scale=None, window=0, sinks=0, out=None):
    """Attention of a ragged batch of new tokens, causal.

    q [tokens, q_heads, d]; starts and lengths as in `rope_append`, which has
    written the tokens' keys: a token at slot i sees the slots j <= i and, with
    a window, of those only j > i - window and j < sinks.  Returns out
    [tokens, q_heads, d] and lse float32 [tokens, q_heads], 0 and -inf where
    nothing is seen and for tokens of no sequence.  Rows that no slot holds may be
    anything; an infinity or NaN in the value row of a slot that is held can make
    NaN of tokens of the batch near it which do not see it."""
    what = "prefill"
    arg, dev = _cache_arg(what, k_cache, v_cache, table, lengths)
    d = arg.head_dim
    (T, hq, _), qs = _heads(what, "q", q, d, k_cache.dtype, dev)
    _group(what, hq, arg.kv_heads)
    _ints(what, "starts", starts, (arg.seqs + 1,), dev)
    out = (torch.empty_like(q) if q.is_contiguous() else q.new_empty((T, hq, d))) if out is None else _given(what, "out", out, (T, hq, d), q.dtype, dev)
    lse = q.new_empty((T, hq), dtype=torch.float32)
    if T:
        _call(what, N.lib().swb_attn_prefill, q, q.data_ptr(), qs[0], qs[1], hq, starts.data_ptr(), T, arg,
              d ** -0.5 if scale is None else scale, _count(what, "window", window), _count(what, "sinks", sinks),
              out.data_ptr(), lse.data_ptr(), None)
    return out, lse


def evict(k_cache, v_cache, table, lengths, weights, positions, budget, *, seen, sinks=0, recent=0):
    """Every sequence cut to `budget` slots by accumulated weight.

    weights float32 and positions int32 [seqs, kv_heads, slots], seen int32
    [seqs] the positions given out so far.  Per key head the slots stay whose
    position is below `sinks` or among the `recent` newest, then those with the
    largest weight, ties to the lowest slot.  Kept slots below the budget stay
    in place, kept ones beyond it move, in order, to the free slots below it,
    in order: the order of slots is then no longer the order of positions.
    Rows move inside the pools: every slot that a sequence holds must have a page,
    and no page may be in the table twice (`decode` and `prefill` read pages that
    sequences share; here one's rows would move under the other).  Returns the new (lengths, weights, positions)
    as tensors of their own, 0 and -1 in slots that hold nothing."""
    what = "evict"
    arg, dev = _cache_arg(what, k_cache, v_cache, table, lengths)
    B, hkv = arg.seqs, arg.kv_heads
    width = weights.shape[-1]
    _given(what, "weights", weights, (B, hkv, width), torch.float32, dev)
    _ints(what, "positions", positions, (B, hkv, width), dev)
    _ints(what, "seen", seen, (B,), dev)
    if width < arg.max_pages * arg.page_size:
        _fail(what, "weights are narrower than the page table's slots")
    if not 1 <= budget < 1 << 31 or sinks < 0 or recent < 0 or sinks + recent > budget:
        _fail(what, "the budget must be at least 1, and hold sinks and recent")
    nl, nw, np_ = torch.empty_like(lengths), torch.empty_like(weights), torch.empty_like(positions)
    if B == 0:
        return nl, nw, np_
    L = N.lib()
    need = L.swb_kv_evict_workspace(B, hkv, budget)
    ws = weights.new_empty(need, dtype=torch.uint8)
    _call(what, L.swb_kv_evict, weights, arg, seen.data_ptr(), weights.data_ptr(), positions.data_ptr(), width, budget, sinks,
          recent, nl.data_ptr(), nw.data_ptr(), np_.data_ptr(), ws.data_ptr(), need)
    return nl, nw, np_


class KVCache:
    """One layer's paged cache of `seqs` sequences of up to `slots` slots.

        cache = KVCache(seqs, slots, kv_heads, head_dim)
        q = cache.append(q, k, v, cos, sin, starts)      # a prompt, or starts=None: a token a sequence
        out, lse = cache.prefill(q, starts, window=4096, sinks=4)
        out, lse = cache.attend(q, window=4096, sinks=4)

    `track` keeps what eviction goes by: every slot's position and the weight it
    has had in `attend` so far (int32 and float32 [seqs, kv_heads, slots]).  An
    `attend` that tracks holds its logits meanwhile: float32 for every query head
    and slot of the table, whatever the lengths are.
    The pools and the table are plain tensors (k, v, table, lengths, seen) and may be
    handed to this module's functions; `lengths` and `seen` are on the device,
    and nothing here waits for them: tokens past the last slot are not stored.
    All of them are the same tensors for the cache's life, written in place (clone
    what is to be kept), so a captured step goes on from where the last replay
    ended.  What a captured step cannot know is an eviction outside of it: its
    `window`, which the slots' order then no longer allows, is refused at the
    capture or not at all."""

    def __init__(self, seqs, slots, kv_heads, head_dim, *, page_size=64, dtype=torch.float16, device="cuda",
                 track=False):
        if page_size < 1 or page_size & (page_size - 1):
            _fail("KVCache", "page_size must be a power of two")
        if head_dim not in HEAD_DIMS:
            _fail("KVCache", f"head_dim must be one of {HEAD_DIMS}")
        if dtype not in _DTYPES:
            _fail("KVCache", "the cache must be float16 or bfloat16")
        per = -(-slots // page_size)
        self.k = torch.zeros((seqs * per, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        dev = self.k.device
        self.table = torch.arange(seqs * per, dtype=torch.int32, device=dev).view(seqs, per)
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self.seen = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self.weights = self.positions = None
        if track:
            self.weights = torch.zeros((seqs, kv_heads, per * page_size), dtype=torch.float32, device=dev)
            self.positions = torch.full(self.weights.shape, -1, dtype=torch.int32, device=dev)
        # a token a sequence
        self._each = torch.arange(seqs + 1, dtype=torch.int32, device=dev)
        self._evicted = False

    def append(self, q, k, v, cos, sin, starts=None, *, q_norm=None, k_norm=None, eps=1e-6, interleaved=False):
        """New tokens' keys and values into their slots; returns their queries, normed and rotated.

        starts int32 [seqs + 1], ascending from 0: tokens starts[b] .. starts[b + 1] - 1 are sequence b's, those
        from starts[seqs] on no sequence's (a padded batch) and not stored; None: one token for each."""
        seqs, n = self.table.shape[0], q.shape[0]
        if starts is None:
            if n != seqs:
                _fail("append", f"without starts there must be one token for each of the {seqs} sequences")
            starts = self._each
        _ints("append", "starts", starts, (seqs + 1,), self.k.get_device())
        counts = starts.diff()
        lengths = self.lengths + counts
        positions = None
        if self.weights is not None and n and seqs:     # after an eviction slots are not positions
            if starts is self._each:
                positions = self.seen
            elif self._evicted or torch.cuda.is_current_stream_capturing():
                at = torch.arange(n, dtype=torch.int32, device=starts.device)
                # a token's sequence: whatever starts holds, one that there is
                of = torch.searchsorted(starts[1:], at, right=True).clamp_(max=seqs - 1)
                positions = at + (self.seen - starts[:-1])[of]
        out = rope_append(q, k, v, cos, sin, self.k, self.v, self.table, starts, lengths, q_norm=q_norm, k_norm=k_norm,
                          eps=eps, positions=positions, interleaved=interleaved, slot_positions=self.positions)
        self.lengths.copy_(lengths)
        self.seen.add_(counts)
        return out

    def prefill(self, q, starts, *, scale=None, window=0, sinks=0):
        """Attention of the tokens just appended, causal."""
        if self._evicted:
            _fail("prefill", "after an eviction the slots' order is not the positions': append and attend token by token")
        return prefill(q, self.k, self.v, self.table, starts, self.lengths, scale=scale, window=window, sinks=sinks)

    def attend(self, q, *, scale=None, window=0, sinks=0, prior=None):
        """Attention of the token just appended to each sequence; with `track` its weights are added to the slots'."""
        if self._evicted and window:
            _fail("attend", "after an eviction the slots' order is not the positions': no window")
        return decode(q, self.k, self.v, self.table, self.lengths, scale=scale, window=window, sinks=sinks, prior=prior,
                      weights=self.weights, accumulate=True)

    def evict(self, budget, *, sinks=0, recent=0):
        """Every sequence cut to `budget` slots: its first `sinks` and newest `recent` positions, then by weight.

        Weight comes from `attend` alone.  Slots that no token has attended yet, a prompt's before the first, have
        none, and among equal weights the lowest slots stay: cut a prompt after some tokens have attended it, or
        write weights of your own into `weights`."""
        if self.weights is None:
            _fail("evict", "the cache was made without track=True")
        new = evict(self.k, self.v, self.table, self.lengths, self.weights, self.positions, budget, seen=self.seen,
                    sinks=sinks, recent=recent)
        for mine, its in zip((self.lengths, self.weights, self.positions), new):
            mine.copy_(its)
        self._evicted = True
