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


def test_dual_tensors_are_refused():
    """A tangent would be dropped: refused before anything else is looked at, with
    gradients on and off, wherever it sits."""
    import os
    import torch.autograd.forward_ad as fa
    import _nsa_lib
    if not os.path.exists(_nsa_lib.LIB_PATH):
        pytest.skip("libnsa_hip.so not built")
    import nsa_lm
    import nsa_paged
    x, w = torch.zeros(3, 16), torch.ones(16)
    q, row, pages = torch.zeros(1, 1, 16), torch.zeros(1, 1, 16), torch.zeros(2, 1, 16, 16)
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)

    def calls(d):
        yield lambda: nsa_lm.add_rms_norm(d(x), x, w)
        yield lambda: nsa_lm.add_rms_norm(x, d(x), w)
        yield lambda: nsa_lm.add_rms_norm(x, None, d(w))
        yield lambda: nsa_lm.add_rms_norm_q8(x, d(x), w)
        yield lambda: nsa_lm.token_logprobs(d(x))
        yield lambda: nsa_paged.paged_attend(d(q), pages, pages, table, lens)
        yield lambda: nsa_paged.paged_attend(q, pages, d(pages), table, lens)
        yield lambda: nsa_paged.paged_step(q, d(row), row, pages, pages, table, lens)
        yield lambda: nsa_paged.paged_step(q, row, d(row), pages, pages, table, lens)
        yield lambda: nsa_paged.paged_append(d(row)[:, :, None], row[:, :, None], pages, pages, table, lens)
        yield lambda: nsa_paged.paged_append(row[:, :, None], row[:, :, None], pages, d(pages), table, lens)
    with fa.dual_level():
        for call in calls(lambda t: fa.make_dual(t, torch.ones_like(t))):
            with pytest.raises(AssertionError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(AssertionError, match="forward-mode"):
                call()
        for call in calls(lambda t: t):      # (no tangent: refused as CPU tensors)
            with pytest.raises(AssertionError) as e:
                call()
            assert "forward-mode" not in str(e.value)


def test_rotation_tables_of_inference_serve_training():
    """Tables formed under inference_mode are saved for a later backward."""
    from nsa_model import Rotary
    rope = Rotary(16)
    with torch.inference_mode():
        cos, _ = rope.tables(5, "cpu", torch.float32)
    assert rope.tables(5, "cpu", torch.float32)[0] is cos and not cos.is_inference()
    x = torch.ones(5, 8, requires_grad=True)
    (x * cos).sum().backward()
    assert torch.equal(x.grad, cos)
    with torch.inference_mode():
        late = Rotary(16)
        assert torch.equal(late.tables(5, "cpu", torch.float32)[0], cos)


def test_reserving_takes_nothing_where_it_raises(monkeypatch):
    """The account and the table in step, whatever is refused in between."""
    import nsa_paged
    _stub(monkeypatch)
    c = _cache(n_pages=5)
    c.reserve([17, 0])
    staged = nsa_paged._staged
    monkeypatch.setattr(nsa_paged, "_staged", lambda *a: (_ for _ in ()).throw(AssertionError("capture")))
    with pytest.raises(AssertionError):
        c.reserve([17, 40])
    c.reserve([32, 0])                      # (two pages held already: nothing new, nothing staged)
    monkeypatch.setattr(nsa_paged, "_staged", staged)
    assert c.free_pages == 3 and (c.table >= 0).sum(1).tolist() == [2, 0]
    with pytest.raises(RuntimeError):
        c.reserve([40, 40])
    c.reserve([40, 20])
    assert c.free_pages == 0 and sorted(c.table[c.table >= 0].tolist()) == list(range(5))
    c.release(0)
    c.reserve([0, 40])
    held = [t[t >= 0].tolist() for t in c.table]
    assert c.free_pages == 2 and [len(h) for h in held] == [0, 3] and held == c._account.held
    assert c.counts(None) is None and c.counts(3).tolist() == [3, 3] and c.counts([4, 5]).dtype == torch.int32


def test_an_end_before_the_first_position_is_refused():
    import os
    import _nsa_lib
    if not os.path.exists(_nsa_lib.LIB_PATH):
        pytest.skip("libnsa_hip.so not built")
    lib = _nsa_lib.load()
    shape = (1, 4, 2, 64, 16, 3, 5)
    assert lib.nsa_paged_attend_max(*[None] * 11, 0, *shape, -1, 0.1, 1, None) == _nsa_lib.NSA_ERR_SHAPE
    assert lib.nsa_paged_attend_max(*[None] * 11, 0, *shape, 0, 0.1, 1, None) == _nsa_lib.NSA_ERR_ARG
    assert lib.nsa_paged_append_max(*[None] * 8, 1, 2, 4, 64, 16, 3, 5, -1, 1, None) == _nsa_lib.NSA_ERR_SHAPE
    assert lib.nsa_paged_append_max(*[None] * 8, 1, 2, 4, 64, 16, 3, 5, 7, 1, None) == _nsa_lib.NSA_ERR_ARG


def test_a_step_takes_both_rows():
    """A missing row is refused: not read through, and not taken as an attention
    without one."""
    import os
    import _nsa_lib
    if not os.path.exists(_nsa_lib.LIB_PATH):
        pytest.skip("libnsa_hip.so not built")
    import nsa_paged
    q, row, pages = torch.zeros(1, 1, 16), torch.zeros(1, 1, 16), torch.zeros(2, 1, 16, 16)
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for k, v in ((row, None), (None, row), (None, None)):
        with pytest.raises(AssertionError, match="row"):
            nsa_paged.paged_step(q, k, v, pages, pages, table, lens)
    for k, v in ((row, None), (None, row)):
        with pytest.raises(AssertionError, match="row"):
            _nsa_lib.torch_side().paged(q, k, v, pages, pages, table, lens, None, False, None)


def test_a_model_takes_one_cache_a_block():
    """Fewer would leave the blocks behind them out."""
    from nsa_model import NSATransformer
    m = NSATransformer(vocab_size=20, d_model=32, n_layers=2, n_q_heads=2, n_kv_heads=1, max_seq_len=16,
                       attn_type="full")
    for caches in ([object()], [object()] * 3, []):
        with pytest.raises(AssertionError, match="one cache"):
            m.prefill(torch.zeros(1, 4, dtype=torch.long), caches)
        with pytest.raises(AssertionError, match="one cache"):
            m.step(torch.zeros(1, dtype=torch.long), caches)
