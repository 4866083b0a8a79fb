"""Refusals and registrations of the rotary positions and the paged cache, without a GPU: sizes that
wrap, outputs that overlap what a call reads, gradients and tangents that a traced call would lose, versions of
what a call writes, shapes of fake tensors."""
import pytest

from conftest import import_pkg
from test_paged_index_cpu import _append, _attend, _lib


@pytest.mark.parametrize("kw", [dict(n=1 << 62), dict(n=1 << 60, Hq=16, Hkv=16), dict(n=(1 << 63) - 1), dict(n=(1 << 62) + 1)])
def test_sizes_that_wrap_are_refused(kw):
    assert _append(**kw) == 3 and "pp_kv_append" in _lib().pp_last_error().decode()
    assert _attend(**kw) == 3 and "pp_paged_attention" in _lib().pp_last_error().decode()


@pytest.mark.parametrize("n,seqs,maxp,page,hq,hkv,d", [(1 << 62, 2, 8, 16, 4, 2, 128), (1 << 60, 1, 64, 16, 16, 16, 128),
                                                       (4, 2, 1 << 30, 1 << 30, 4, 2, 128), (4, 2, 8, 16, 4, 3, 128),
                                                       (4, 1 << 30, 8, 16, 4, 2, 64), (4, 2, 8, 16, 1 << 30, 1 << 30, 64)])
def test_workspace_of_sizes_that_are_refused(n, seqs, maxp, page, hq, hkv, d):
    """None: the call itself says what is wrong with them."""
    assert _lib().pp_paged_attention_workspace_bytes(n, seqs, maxp, page, hq, hkv, d) == 0
