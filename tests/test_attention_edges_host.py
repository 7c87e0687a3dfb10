"""Refusals of the attention operators' C ABI that come before any CUDA call, and need no GPU."""
import pytest
from test_attention_host import P, cache, decode

from swann_b200 import _lib as N


@pytest.mark.parametrize("args,why", [
    (dict(out=P + 2), "out"), (dict(out=P + 4), "out"), (dict(prior=P + 2, plse=P), "prior"), (dict(prior=P + 4, plse=P), "prior"),
    (dict(ws=P + 4), "workspace"), (dict(ws=P + 8), "workspace")])
def test_decode_refuses_rows_and_workspaces_that_it_cannot_access(args, why):
    assert decode(cache(), **args) == N.ERR_ARG
    assert "boundar" in N.lib().swb_last_error().decode() and why in N.lib().swb_last_error().decode()


@pytest.mark.parametrize("width,budget", [(65536 * 4096, 8), (1 << 40, 8), (1 << 23, 1 << 22)])
def test_evict_refuses_what_its_second_kernel_cannot_take_before_the_first(width, budget):
    arg = cache(max_pages=1 << 19)
    assert N.lib().swb_kv_evict(arg, P, P, P, width, budget, 0, 0, P + 64, P + 64, P + 64, P, 1 << 40, None) == N.ERR_ARG
    assert "wide" in N.lib().swb_last_error().decode()


@pytest.mark.parametrize("heads,slots,pairs,whole", [
    (1, 512, 592, False), (1, 512, 4096, True), (1, 112, 4096, True), (1, 2048, 18944, False), (1, 1024, 9000, True), (1, 16, 500, False),
    (4, 512, 592, False), (4, 512, 1184, True), (4, 1024, 4096, True), (4, 8192, 4096, False), (4, 64, 100, False), (16, 2048, 592, False)])
def test_decode_takes_whole_pairs_where_that_was_measured_to_pay(heads, slots, pairs, whole):
    """Runs need a workspace for the parts of cut pairs, whole pairs need none."""
    arg = cache(seqs=pairs, max_pages=slots // 16)
    assert (N.lib().swb_attn_decode_workspace(arg, heads, 0) == 0) == whole
