"""The attention operators at the edges of what their calls allow, against their definitions in 64 bits."""
import ctypes as C
import math
import subprocess
import sys
from pathlib import Path

import pytest
import test_attention_gpu as base
import torch
from test_attention_gpu import DEV, make_cache

from swann_b200 import _lib as N
from swann_b200 import attention as A

pytestmark = pytest.mark.gpu


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def test_a_pool_without_pages_beside_lengths_on_any_boundary():
    """Copies of nothing take an address from the lengths, which lie on 4-byte boundaries only."""
    k = torch.empty((0, 2, 16, 64), dtype=torch.float16, device=DEV)
    q = torch.randn((700, 4, 64), device=DEV).half()
    for B, slots in ((1, 3), (700, 3), (1, 4000)):       # by runs, a warp a pair, runs of several units
        table = torch.zeros((B, slots // 16 + 1), dtype=torch.int32, device=DEV)
        for at in (1, 2, 3):
            L = torch.full((B + 4,), slots, dtype=torch.int32, device=DEV)[at:at + B]
            parts = [A.decode(q[:B], k, k, table, L), A.decode(q[:B, :2], k, k, table, L)]
            if B == 1:
                parts.append(A.prefill(q[:3], k, k, table, ints(0, 3), L))
            for out, lse in parts:
                assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("starts,own", [((0, 5, 9), (0, 9)), ((2, 2, 9), (2, 9)), ((0, 0, 0), (0, 0)), ((4, 11, 11), (4, 11))])
@pytest.mark.parametrize("moved", [False, True])
def test_append_leaves_tokens_of_no_sequence_out(starts, own, moved):
    """A padded batch: the tables name pages beyond the lengths, and nothing is written there."""
    k, v, table, L = make_cache([20, 9], 1, 64, 16, torch.float16, 23, max_pages=4, garbage=False)
    table[:, 2:] = ints(3, 4)[:, None]
    table[1, 1] = 5
    k0, v0 = k.clone(), v.clone()
    sp = torch.full((2, 1, 64), -7, dtype=torch.int32, device=DEV)
    x = torch.randn((30, 4, 64), device=DEV).half()
    angle = torch.rand((64, 32), device=DEV) * 6.28
    cos, sin = angle.cos(), angle.sin()
    pos = torch.randint(0, 64, (30,), device=DEV, dtype=torch.int32) if moved else None

    def append(x, starts, pos):
        return A.rope_append(x[:, :2], x[:, 2:3], x[:, 3:], cos, sin, k, v, table, starts, L, positions=pos, slot_positions=sp)

    out = append(x, ints(*starts), pos)
    k1, v1, sp1 = k.clone(), v.clone(), sp.clone()
    k.copy_(k0), v.copy_(v0), sp.fill_(-7)
    a, e = own
    want = append(x[a:e], ints(*starts) - a, None if pos is None else pos[a:e])
    assert torch.equal(k1, k) and torch.equal(v1, v) and torch.equal(sp1, sp)
    assert int((v1 != v0).any(-1).sum()) == e - a
    assert torch.equal(out[a:e], want)
    rest = [t for t in range(30) if not a <= t < e]
    if not moved:
        assert torch.equal(out[rest], x[rest, :2])


def test_append_without_sequences():
    k, v, table, L = make_cache([8], 1, 64, 16, torch.float16, 24, garbage=False)
    k0, x = k.clone(), torch.randn((3, 4, 64), device=DEV).half()
    cos = torch.zeros((4, 32), device=DEV)
    out = A.rope_append(x[:, :2], x[:, 2:3], x[:, 3:], cos, cos, k, v, table[:0], ints(0), L[:0])
    assert torch.equal(out, x[:, :2]) and torch.equal(k, k0)


def evict_into(k, v, table, L, w, pos, budget, seen, sinks=0, recent=0):
    """The native call with outputs that hold what no eviction gives; (lengths, weights, positions)."""
    nl, nw, npos = torch.full_like(L, -9), torch.full_like(w, math.nan), torch.full_like(pos, -9)
    arg, _ = A._cache_arg("evict", k, v, table, L)
    need = N.lib().swb_kv_evict_workspace(w.shape[0], w.shape[1], budget)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    N.check(N.lib().swb_kv_evict(arg, seen.data_ptr(), w.data_ptr(), pos.data_ptr(), w.shape[2], budget, sinks, recent,
                                 nl.data_ptr(), nw.data_ptr(), npos.data_ptr(), ws.data_ptr(), need,
                                 torch.cuda.current_stream().cuda_stream))
    return nl, nw, npos


@pytest.mark.parametrize("lengths", [[1000, 64, 65], [2 ** 31 - 1, -3, 0], [63, 64, 100]])
@pytest.mark.parametrize("budget", [10, 63, 64, 65, 150, 199, 200, 5000])
def test_evict_writes_every_slot_whatever_the_lengths(lengths, budget):
    """Lengths beyond the table and below nothing, and weights that are wider than the table."""
    k, v, table, _ = make_cache([64] * 3, 2, 64, 16, torch.float16, 25, garbage=False)
    L, W = ints(*lengths), 200
    w = torch.rand((3, 2, W), device=DEV)
    pos = torch.arange(W, device=DEV, dtype=torch.int32).expand(3, 2, W).contiguous()
    cut = L.clamp(0, 64)
    want = base.plain_evict(k, v, table, cut, w, pos, budget, cut, 0, 0)
    got = (*evict_into(k, v, table, L, w, pos, budget, cut), k, v)
    for a, c in zip(got, want):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prefill_sums_a_long_flat_tail(dtype):
    """A first logit of 18 and 70000 of about 0: weights of 2^-26 that make up 2^-10 of the sum."""
    n, new = 70000, 9
    k, v, table, L = make_cache([n], 1, 64, 64, dtype, 3, garbage=False)
    k.mul_(0.3)
    k[..., 0] = 0
    k[table[0, 0], :, 0, 0] = 2.25
    q = (torch.randn((new, 4, 64), device=DEV) * 0.05).to(dtype)
    q[..., 0] = 8
    _, lse = A.prefill(q, k, v, table, ints(0, new), L, scale=1.0)
    for t in (0, 4, 8):
        for h in range(4):
            _, wl, _, _, _, e = base.attend(q[t, h], k, v, table, 0, 0, n - new + t, 1.0, 0, 0, n)
            assert abs(float(lse[t, h]) - wl) <= e + 2.0 ** -19 * (1 + abs(wl)), (float(lse[t, h]), wl)


# -- one strong key beside a long flat tail ---------------------------------------------
#
# The first slot's logit is 18 above all others', whose weights are then about 2^-26 of
# the largest, and its value is 0: what comes out is the tail's.  fp16's smallest numbers
# are 2^-24 apart, so a weight among them is rounded by up to 2^-25, however small it is
# itself: with weights multiplied by 2^x, by 2^-(25 + x) of the largest weight, x = 7 in
# prefill and 15 in decode.  That, for every visible slot and times the largest |v| of 1.5,
# is added to the bound of a weight's relative rounding.

def peaked(lengths, hq, hkv, d, page, dtype, tokens, seed=3):
    k, v, table, L = make_cache(lengths, hkv, d, page, dtype, seed, garbage=False)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    k.mul_(0.3)
    k[..., 0] = 0
    v.copy_(torch.rand(v.shape, generator=g, device=DEV) + 0.5)
    for b in range(len(lengths)):
        k[table[b, 0], :, 0, 0] = 2.25
        v[table[b, 0], :, 0] = 0
    q = (torch.randn((tokens, hq, d), generator=g, device=DEV) * 0.05).to(dtype)
    q[..., 0] = 8
    return q, k, v, table, L


def check_tail(out, lse, want, u, lost):
    j, wl, wo, wa, _, e = want
    assert abs(float(lse) - wl) <= e + 2.0 ** -19 * (1 + abs(wl))
    bound = u * wo.abs() + (u + 2 * e + 2.0 ** -18) * wa + 2.0 ** -25 + len(j) * 1.5 * lost
    over = ((out.double() - wo).abs() / bound).max()
    assert over <= 1, float(over)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,new,hq,hkv,d,window", [(3000, 200, 2, 2, 64, 0), (3000, 200, 8, 2, 128, 0), (70000, 9, 4, 1, 64, 0),
                                                   (3000, 200, 4, 2, 64, 1500)])
def test_prefill_keeps_a_long_flat_tail(n, new, hq, hkv, d, window, dtype):
    q, k, v, table, L = peaked([n], hq, hkv, d, 64, dtype, new)
    out, lse = A.prefill(q, k, v, table, ints(0, new), L, scale=1.0, window=window, sinks=1 if window else 0)
    for t in (0, new // 2, new - 1):
        for h in {0, hq - 1}:
            want = base.attend(q[t, h], k, v, table, 0, h * hkv // hq, n - new + t, 1.0, window, 1 if window else 0, n)
            check_tail(out[t, h], lse[t, h], want, base.U[dtype], 2.0 ** -32)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,n,hq,hkv,d", [
    (1, 3000, 8, 1, 128),       # runs of one unit
    (40, 3000, 16, 8, 64),      # runs longer than a pair
    (40, 3000, 160, 8, 64),     # and of two products' rows
    (900, 400, 4, 1, 64),       # a warp a pair
    (1000, 100, 1, 1, 128)])    # of one row
def test_decode_keeps_a_long_flat_tail(B, n, hq, hkv, d, dtype):
    q, k, v, table, L = peaked([n] * B, hq, hkv, d, 16, dtype, B)
    prior = (torch.full((B, hq, d), 0.5, device=DEV).to(dtype), torch.full((B, hq), 0.0, device=DEV))
    w = torch.empty((B, hkv, table.shape[1] * 16), device=DEV)
    out, lse = A.decode(q, k, v, table, L, scale=1.0)
    both = A.decode(q, k, v, table, L, scale=1.0, prior=prior, weights=w)
    for b in (0, B - 1):
        for h in {0, hq - 1}:
            j, wl, wo, wa, p, e = want = base.attend(q[b, h], k, v, table, b, h * hkv // hq, n - 1, 1.0, 0, 0, n)
            check_tail(out[b, h], lse[b, h], want, base.U[dtype], 2.0 ** -40)
            # with a part of lse 0 beside it: e^-wl of the sum
            x = math.exp(-wl) / (1 + math.exp(-wl))
            y = (1 - x) * wo + x * 0.5
            check_tail(both[0][b, h], both[1][b, h], (j, math.log(math.exp(wl) + 1), y, y.abs(), p, e), base.U[dtype], 2.0 ** -40)
        tail = w[b, 0, 1:n].double().sum()
        heads = hq // hkv
        want = sum(float(base.attend(q[b, h], k, v, table, b, 0, n - 1, 1.0, 0, 0, n)[4][1:].sum()) for h in range(heads))
        assert abs(float(tail) - want) <= (2 * e + 2.0 ** -18) * want


def every_call():
    """Each call's tensors of numbers by name, and the calls."""
    k, v, table, L = make_cache([40, 8], 2, 64, 16, torch.float16, 41, garbage=False)
    x = torch.randn((2, 8, 64), device=DEV).half()
    starts, seen = ints(0, 1, 2), L.clone()
    half = dict(q=x[:, :4].contiguous(), kn=x[:, 4:6], vn=x[:, 6:], k=k, v=v, q_norm=torch.ones(64, device=DEV).half(),
                k_norm=torch.ones(64, device=DEV).half(), prior=torch.zeros((2, 4, 64), device=DEV).half(),
                out=torch.zeros((2, 4, 64), device=DEV).half())
    full = dict(cos=torch.ones((64, 32), device=DEV), sin=torch.zeros((64, 32), device=DEV), prior_lse=torch.zeros((2, 4), device=DEV),
                weights=torch.zeros((2, 2, 48), device=DEV))
    pos = torch.zeros((2, 2, 48), dtype=torch.int32, device=DEV)
    calls = {
        "rope_append": lambda t: A.rope_append(t["q"], t["kn"], t["vn"], t["cos"], t["sin"], t["k"], t["v"], table, starts, L,
                                               q_norm=t["q_norm"], k_norm=t["k_norm"], out=t["out"]),
        "decode": lambda t: A.decode(t["q"], t["k"], t["v"], table, L, prior=(t["prior"], t["prior_lse"]), weights=t["weights"], out=t["out"]),
        "prefill": lambda t: A.prefill(t["q"], t["k"], t["v"], table, starts, L, out=t["out"]),
        "evict": lambda t: A.evict(t["k"], t["v"], table, L, t["weights"], pos, 8, seen=seen)}
    return {**half, **full}, calls


@pytest.mark.parametrize("call,names", [
    ("rope_append", ["q", "kn", "vn", "cos", "sin", "k", "v", "q_norm", "k_norm", "out"]),
    ("decode", ["q", "k", "v", "prior", "prior_lse", "weights", "out"]), ("prefill", ["q", "k", "v", "out"]), ("evict", ["k", "v", "weights"])])
def test_no_tensor_that_wants_a_gradient_is_taken(call, names):
    tensors, calls = every_call()
    calls[call](tensors)
    for name in names:
        wants = {**tensors, name: tensors[name].detach().clone().requires_grad_()}
        with pytest.raises(ValueError, match="no backward pass"):
            calls[call](wants)
        with torch.no_grad():
            calls[call](wants)


@pytest.mark.parametrize("length", [0, 5, 9, 64, 70, 100, 2 ** 31 - 1, -7, -2 ** 31])
@pytest.mark.parametrize("window,sinks", [(0, 0), (3, 0), (3, 2), (2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31 - 5, 1)])
def test_prefill_of_lengths_that_the_tokens_or_the_table_do_not_fit(length, window, sinks):
    """Fewer slots than new tokens: the first lie before slot 0 and see nothing.  More than the table: no slot there."""
    k, v, table, _ = make_cache([64], 1, 64, 16, torch.float16, 6)
    q = torch.randn((70, 2, 64), device=DEV).half()
    out, lse = A.prefill(q, k, v, table, ints(0, 70), ints(length), window=window, sinks=sinks)
    n = max(0, length)
    for t in (0, 1, 5, 31, 60, 61, 64, 65, 66, 69):
        for h in range(2):
            want = base.attend(q[t, h], k, v, table, 0, 0, n - 70 + t, 0.125, window, sinks, n)
            base.check_row(out[t, h], lse[t, h], want, base.U[torch.float16])


@pytest.mark.parametrize("B,hq", [(1, 4), (700, 4), (700, 1)])
@pytest.mark.parametrize("length", [0, -1, -2 ** 31])
def test_decode_of_lengths_below_nothing(B, hq, length):
    k, v, table, _ = make_cache([64], 1, 64, 16, torch.float16, 6)
    table, L = table.expand(B, 4), torch.full((B,), length, dtype=torch.int32, device=DEV)
    w = torch.full((B, 1, 64), math.nan, device=DEV)
    q = torch.randn((B, hq, 64), device=DEV).half()
    for window in (0, 5, 2 ** 31 - 1):
        out, lse = A.decode(q, k, v, table, L, window=window, sinks=2, weights=w)
        assert (out == 0).all() and (lse == -math.inf).all() and (w == 0).all()


def prefill_into(q, k, v, table, starts, L, dtype):
    """The native call with outputs that hold NaN."""
    T, hq, d = q.shape
    out, lse = torch.full((T, hq, d), math.nan, dtype=dtype, device=DEV), torch.full((T, hq), math.nan, device=DEV)
    arg, _ = A._cache_arg("prefill", k, v, table, L)
    N.check(N.lib().swb_attn_prefill(q.data_ptr(), hq * d, d, hq, starts.data_ptr(), T, arg, d ** -0.5, 0, 0, out.data_ptr(),
                                     lse.data_ptr(), None, torch.cuda.current_stream().cuda_stream))
    return out, lse


@pytest.mark.parametrize("starts", [(0, 20, 30), (3, 20, 30), (7, 7, 7), (0, 0, 0), (40, 40, 40), (0, 40, 40), (2, 5, 1000)])
@pytest.mark.parametrize("T", [40, 1000])
@pytest.mark.parametrize("hq,d", [(2, 64), (40, 128)])
def test_prefill_writes_every_row_of_a_padded_batch(starts, T, hq, d):
    k, v, table, L = make_cache([50, 60], 2, d, 16, torch.float16, 16)
    q = torch.randn((T, hq, d), device=DEV).half()
    out, lse = prefill_into(q, k, v, table, ints(*starts), L, torch.float16)
    a, e = min(T, starts[0]), min(T, starts[2])
    for none in (slice(0, a), slice(e, T)):
        assert (out[none] == 0).all() and (lse[none] == -math.inf).all()
    if e > a:
        want = A.prefill(q[a:e].contiguous(), k, v, table, ints(*(min(T, s) - a for s in starts)), L)
        assert torch.equal(out[a:e], want[0]) and torch.equal(lse[a:e], want[1])


def test_prefill_without_sequences():
    k, v, table, L = make_cache([8], 1, 64, 16, torch.float16, 24)
    out, lse = prefill_into(torch.randn((5, 2, 64), device=DEV).half(), k, v, table[:0], ints(0), L[:0], torch.float16)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("call", ["rope_append", "decode", "prefill", "evict"])
def test_a_wait_that_gave_up_is_reported_by_the_next_call(call):
    """The word that the kernel writes then, written by the host."""
    tensors, calls = every_call()
    calls["prefill"](tensors)
    torch.cuda.synchronize()
    word = C.c_int32.from_address(N.lib().swb_attn_status())
    assert word.value == 0
    word.value = N.ERR_TIMEOUT
    with pytest.raises(N.SwannError, match="gave up") as e:
        calls[call](tensors)
    assert e.value.code == N.ERR_TIMEOUT and word.value == 0
    calls[call](tensors)


def test_a_first_prefill_under_capture():
    """The word is made while a stream is capturing, in a process of its own."""
    code = """
import torch
from swann_b200 import _lib as N, attention as A
k = torch.randn((4, 1, 16, 64), device="cuda").half()
table, L = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), torch.full((1,), 60, dtype=torch.int32, device="cuda")
q, starts = torch.randn((20, 2, 64), device="cuda").half(), torch.tensor([0, 20], dtype=torch.int32, device="cuda")
assert not N.lib().swb_attn_status()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out, lse = A.prefill(q, k, k, table, starts, L)
assert N.lib().swb_attn_status()
graph.replay()
want = A.prefill(q, k, k, table, starts, L)
assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=Path(__file__).resolve().parent.parent, timeout=300)


@pytest.mark.parametrize("B", [1, 2, 700])
def test_decode_with_weights_of_no_slots(B):
    """A table without columns: the native call with weights of width 0."""
    table, L = torch.zeros((B, 0), dtype=torch.int32, device=DEV), torch.full((B,), 3, dtype=torch.int32, device=DEV)
    k = torch.zeros((2, 1, 16, 64), dtype=torch.float16, device=DEV)
    q = torch.ones((B, 4, 64), dtype=torch.float16, device=DEV)
    out, lse, w = torch.full_like(q, 7), torch.zeros((B, 4), device=DEV), torch.full((4,), 7.0, device=DEV)
    arg, _ = A._cache_arg("decode", k, k, table, L)
    need = N.lib().swb_attn_decode_workspace(arg, 4, 1)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    N.check(N.lib().swb_attn_decode(q.data_ptr(), 256, 64, 4, arg, 0.1, 0, 0, None, None, out.data_ptr(), lse.data_ptr(),
                                    w.data_ptr(), 0, 0, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    assert (out == 0).all() and (lse == -math.inf).all() and (w == 7).all()


@pytest.mark.parametrize("call", ["rope_append", "decode", "prefill", "evict"])
def test_a_cache_without_key_heads_is_refused(call):
    tensors, calls = every_call()
    none = {**tensors, "k": tensors["k"][:, :0], "v": tensors["v"][:, :0]}
    with pytest.raises(ValueError, match="key head"):
        calls[call](none)


@pytest.mark.parametrize("lengths,hq,hkv,window,sinks", [
    ([3000, 70, 0], 8, 2, 200, 5), ([3000, 70, 1], 40, 2, 0, 0), ([300] * 5, 36, 1, 64, 0), ([(37 * b) % 91 for b in range(700)], 12, 1, 21, 3),
    ([(37 * b) % 91 for b in range(900)], 1, 1, 21, 3)])
def test_decode_accumulates_beside_a_window_and_many_heads(lengths, hq, hkv, window, sinks):
    """What is added is what a call that writes gives: one fp32 addition, 2^-24 of the sum; unseen slots stay as they are."""
    k, v, table, L = make_cache(lengths, hkv, 64, 16, torch.float16, 5)
    q = torch.randn((len(lengths), hq, 64), device=DEV).half()
    once = torch.full((len(lengths), hkv, table.shape[1] * 16 + 3), math.nan, device=DEV)
    w = torch.rand(once.shape, device=DEV)
    w0 = w.clone()
    a = A.decode(q, k, v, table, L, window=window, sinks=sinks, weights=once)
    b = A.decode(q, k, v, table, L, window=window, sinks=sinks, weights=w, accumulate=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    j, n = torch.arange(once.shape[2], device=DEV), L.long()[:, None]
    seen = (j < n) & ((j >= n - window) | (j < sinks) if window else j >= 0)
    assert (once.masked_select(~seen[:, None]) == 0).all()
    assert torch.equal(w.masked_select(~seen[:, None].expand_as(w)), w0.masked_select(~seen[:, None].expand_as(w)))
    want = w0.double() + once.double()
    assert ((w.double() - want).abs() <= 2.0 ** -24 * want).all()
    total = hq // hkv * (n > 0).double()
    assert torch.allclose(once.double().sum(-1), total.expand(-1, hkv), rtol=1e-4, atol=0)


@pytest.mark.parametrize("hq,hkv,d,dtype,window,sinks", [(130, 1, 64, torch.float16, 0, 0), (129, 1, 128, torch.bfloat16, 40, 2),
                                                         (400, 2, 64, torch.bfloat16, 0, 0), (256, 1, 128, torch.float16, 9, 0)])
def test_prefill_of_more_heads_to_a_key_head_than_a_tile_has_rows(hq, hkv, d, dtype, window, sinks):
    new, held = [3, 0, 70], [0, 9, 130]
    lengths = [a + b for a, b in zip(new, held)]
    k, v, table, L = make_cache(lengths, hkv, d, 16, dtype, 17)
    q = (torch.randn((73, hq, d), device=DEV) * 1.5).to(dtype)
    out, lse = A.prefill(q, k, v, table, ints(0, 3, 3, 73), L, window=window, sinks=sinks)
    G = hq // hkv
    for b, t in ((0, 0), (0, 2), (2, 0), (2, 1), (2, 33), (2, 69)):
        row = t + (3 if b else 0)
        for h in {0, 1, 127, 128, hq - 1, hq // 2}:
            want = base.attend(q[row, h], k, v, table, b, h // G, held[b] + t, d ** -0.5, window, sinks, lengths[b])
            base.check_row(out[row, h], lse[row, h], want, base.U[dtype])
    assert torch.isfinite(out).all()


def test_pages_that_sequences_share_are_read_as_they_are():
    """A common beginning: the first pages of three sequences are the same."""
    k, v, table, L = make_cache([100, 90, 64], 2, 64, 16, torch.float16, 18)
    table[1, :4] = table[2, :4] = table[0, :4]
    q = torch.randn((33, 4, 64), device=DEV).half()
    starts = [0, 10, 30, 33]
    out, lse = A.prefill(q, k, v, table, ints(*starts), L)
    one, one_lse = A.decode(q[:3], k, v, table, L)
    for b, n in enumerate([100, 90, 64]):
        for h in range(4):
            base.check_row(one[b, h], one_lse[b, h], base.attend(q[b, h], k, v, table, b, h // 2, n - 1, 0.125, 0, 0, n), base.U[torch.float16])
            for t in (starts[b], starts[b + 1] - 1):
                want = base.attend(q[t, h], k, v, table, b, h // 2, n - starts[b + 1] + t, 0.125, 0, 0, n)
                base.check_row(out[t, h], lse[t, h], want, base.U[torch.float16])


@pytest.mark.parametrize("B,hq,hkv,d,page,dtype", [(900, 1, 1, 128, 1, torch.float16), (800, 1, 1, 64, 1, torch.bfloat16),
                                                   (450, 2, 2, 64, 8, torch.float16)])
@pytest.mark.parametrize("window,sinks,extra", [(0, 0, "prior"), (0, 0, "weights"), (21, 3, "plain")])
def test_decode_of_enough_one_row_pairs_for_a_warp_each(B, hq, hkv, d, page, dtype, window, sinks, extra):
    base.test_decode_of_very_many_short_sequences(B, hq, hkv, d, page, dtype, window, sinks, extra)


@pytest.mark.parametrize("lengths,hq,hkv", [([5000], 8, 1), ([90] * 300, 8, 2), ([90] * 900, 1, 1)])
@pytest.mark.parametrize("at", [0, 1, 2, 3, 4, 8, 12])
def test_decode_rows_at_any_offset_are_right_or_refused(lengths, hq, hkv, at):
    """Contiguous views that begin `at` elements into a buffer: 8 bytes are 4 of them."""
    k, v, table, L = make_cache(lengths, hkv, 64, 16, torch.float16, 26)
    B = len(lengths)
    q, po = torch.randn((B, hq, 64), device=DEV).half(), torch.randn((B, hq, 64), device=DEV).half()
    lse = torch.randn((B, hq), device=DEV)
    want = A.decode(q, k, v, table, L, prior=(po, lse))

    def moved(t):
        return torch.empty(t.numel() + 16, dtype=t.dtype, device=DEV)[at:at + t.numel()].view(t.shape).copy_(t)

    for kw in (dict(out=moved(q), prior=(po, lse)), dict(prior=(moved(po), moved(lse)))):
        if at % 4:
            with pytest.raises(ValueError, match="8-byte"):
                A.decode(q, k, v, table, L, **kw)
        else:
            got = A.decode(q, k, v, table, L, **kw)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
