"""The attention operators' C ABI without a GPU: the cache's struct as the header
declares it, and refusals, which come before any CUDA call."""
import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from swann_b200 import _lib as N
from swann_b200 import attention as A

ROOT = Path(__file__).resolve().parent.parent
P = 1 << 20      # an aligned address that nothing reads


def cache(**over):
    arg = N.KVCacheArg(P, P, 16 * 64, 16 * 64, 64, P, 4, P, 8, 4, 16, 2, 1, 64, N.F16)
    for name, value in over.items():
        setattr(arg, name, value)
    return arg


def test_struct_matches_the_header():
    text = (ROOT / "include" / "swann_b200.h").read_text()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct swb_kv_cache \{(.*?)\} swb_kv_cache;", text, re.S).group(1), flags=re.S)
    declared = []
    for line in body.split(";"):
        m = re.match(r"\s*(const int32_t\*|void\*|int64_t|int32_t)\s+(.*)", line.strip(), re.S)
        if m:
            kind = C.c_void_p if "*" in m.group(1) else C.c_int64 if m.group(1) == "int64_t" else C.c_int32
            declared += [(name.strip(), C.sizeof(kind)) for name in m.group(2).split(",")]
    assert declared == [(n, C.sizeof(t)) for n, t in N.KVCacheArg._fields_]


def decode(arg, *, q=P, qs=256, hs=64, heads=4, window=0, sinks=0, prior=None, plse=None, out=P, lse=P, weights=None, width=0,
           ws=P, n=1 << 40):
    return N.lib().swb_attn_decode(q, qs, hs, heads, arg, 0.1, window, sinks, prior, plse, out, lse, weights, width, 0, ws, n, None)


@pytest.mark.parametrize("over,why", [
    (dict(head_dim=80), "head_dim"), (dict(dtype=N.F32), "fp16 or bf16"), (dict(page_size=12), "power of two"),
    (dict(page_size=0), "power of two"), (dict(kv_heads=0), "sizes"), (dict(pages=-1), "sizes"), (dict(k=P + 2), "16-byte"),
    (dict(row_stride=65), "16-byte"), (dict(lengths=None), "null table"), (dict(table=None), "null table"),
    (dict(v=None), "null pool"), (dict(max_pages=1 << 28), "2\\^31")])
def test_a_bad_cache_is_refused_by_every_call(over, why):
    arg, L = cache(**over), N.lib()
    calls = [decode(arg),
             L.swb_attn_prefill(P, 256, 64, 4, P, 8, arg, 0.1, 0, 0, P, P, None, None),
             L.swb_rope_append(P, 256, 64, P, 64, 64, P, 64, 64, 4, P, 8, None, None, 1e-6, P, P, 64, 64, 0, None, arg, P, None, 0, None),
             L.swb_kv_evict(arg, P, P, P, 1 << 40, 8, 0, 0, P + 64, P + 64, P + 64, P, 1 << 40, None)]
    assert calls == [N.ERR_ARG] * 4
    assert re.search(why, L.swb_last_error().decode())
    assert L.swb_attn_decode_workspace(arg, 4, 0) == 2 ** 64 - 1


@pytest.mark.parametrize("args,why", [
    (dict(q=None), "null queries"), (dict(heads=0), "multiple"), (dict(q=P + 8), "16-byte"), (dict(hs=60), "16-byte"),
    (dict(out=None), "null output"), (dict(window=-1), "negative"), (dict(sinks=-1), "negative"), (dict(prior=P), "prior"),
    (dict(weights=P, width=63), "narrower"), (dict(ws=None), "workspace"), (dict(n=8), "workspace")])
def test_decode_refuses(args, why):
    assert decode(cache(), **args) == N.ERR_ARG
    assert why in N.lib().swb_last_error().decode()


def test_heads_that_the_key_heads_do_not_divide():
    arg, L = cache(kv_heads=3), N.lib()
    assert decode(arg, heads=4) == N.ERR_ARG and b"multiple" in L.swb_last_error()
    assert L.swb_attn_prefill(P, 256, 64, 4, P, 8, arg, 0.1, 0, 0, P, P, None, None) == N.ERR_ARG


def test_append_and_evict_refuse():
    arg, L = cache(), N.lib()

    def append(rot=64, cos=P, k=P, ks=64):
        return L.swb_rope_append(P, 256, 64, k, ks, 64, P, 64, 64, 4, P, 8, None, None, 1e-6, cos, P, 64, rot, 0, None, arg, P,
                                 None, 0, None)

    for call, why in ((lambda: append(rot=24), "multiple of 16"), (lambda: append(rot=80), "head_dim"), (lambda: append(cos=None), "tables"),
                      (lambda: append(cos=P + 4), "tables"), (lambda: append(k=None), "null"), (lambda: append(ks=66), "16-byte")):
        assert call() == N.ERR_ARG and why in L.swb_last_error().decode()

    def evict(width=64, budget=8, sinks=0, recent=0, nw=P + 64, n=1 << 40):
        return L.swb_kv_evict(arg, P, P, P, width, budget, sinks, recent, P + 64, nw, P + 64, P, n, None)

    for call, why in ((lambda: evict(budget=0), "budget"), (lambda: evict(sinks=5, recent=4), "fit"), (lambda: evict(width=60), "narrower"),
                      (lambda: evict(nw=P), "own"), (lambda: evict(n=4), "workspace")):
        assert call() == N.ERR_ARG and why in L.swb_last_error().decode()


def test_nothing_to_do_needs_no_gpu():
    L = N.lib()
    assert decode(cache(seqs=0)) == N.OK
    assert L.swb_attn_prefill(P, 256, 64, 4, P, 0, cache(), 0.1, 0, 0, P, P, None, None) == N.OK
    assert L.swb_kv_evict(cache(seqs=0), P, P, P, 64, 8, 0, 0, P + 64, P + 64, P + 64, P, 1 << 40, None) == N.OK


def test_tensors_on_the_host_are_refused():
    k = torch.zeros((2, 1, 16, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="on the GPU"):
        A.decode(k[:1, :, 0], k, k, torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
