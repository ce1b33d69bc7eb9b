"""CPU checks of what the operators around the attention promise beyond their
formulas.  Where a cache is made on the CPU its page check is stood in for."""

import gc
import types
import weakref

import pytest
import torch


def _stub(monkeypatch, check=lambda *a: None):
    import _nsa_lib
    monkeypatch.setattr(_nsa_lib, "torch_side", lambda: types.SimpleNamespace(check_pages=check))


def _cache(**kw):
    import nsa_paged
    return nsa_paged.PagedKVCache(**{**dict(batch=2, n_kv_heads=1, head_dim=16, max_len=40, page_size=16,
                                            dtype=torch.float32, device="cpu"), **kw})


def test_a_dropped_cache_is_freed(monkeypatch):
    """Without the cyclic collector, which the allocator does not start; the
    account goes on serving the caches that are left."""
    _stub(monkeypatch)
    gc.disable()
    try:
        a = _cache()
        b = _cache(like=a)
        a.lens += 3
        b.lens += 3
        seen = [weakref.ref(x) for x in (a, a.k_pages, b, b.k_pages)]
        b.reserve([20, 5])
        del a
        assert seen[0]() is None and seen[1]() is None
        b.release(0)
        assert b.lens.tolist() == [0, 3] and b.free_pages == 5
        del b
        assert seen[2]() is None and seen[3]() is None
    finally:
        gc.enable()


def test_a_refused_cache_leaves_nothing_in_the_account(monkeypatch):
    _stub(monkeypatch)
    a = _cache()

    def refuse(*args):
        raise AssertionError("paged: refused")
    _stub(monkeypatch, refuse)
    with pytest.raises(AssertionError):
        _cache(like=a, head_dim=48)
    assert list(a._account.caches) == [a]
