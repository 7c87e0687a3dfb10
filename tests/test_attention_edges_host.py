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
