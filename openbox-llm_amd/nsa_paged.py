"""Generation over a paged key-value cache on MI355X: one new token of every
sequence against keys and values that lie in pages.

The reference runs whole sequences only (FullAttention.forward,
nsa_model.py:377-419).  A step here computes that function's newest row for
every sequence of a batch.

* ``paged_step`` appends the new tokens' key and value rows and attends;
  ``paged_attend`` attends alone; ``paged_append`` writes a prompt's rows.
* ``PagedKVCache`` holds one layer's pages, the page table and the lengths, and
  hands pages out to sequences as they grow.

Layout: ``k_pages, v_pages [n_pages, Hkv, page, D]`` (float32 or bfloat16,
``page`` a multiple of 16, ``D`` in 16, 32, 64, 128), ``table [B, max_pages]``
int32 (the page that holds positions ``i page ..``) and ``lens [B]`` int32, all
on the device: the host never waits for it in a generation loop, and a step can be
captured into a graph.  Query head h reads KV head ``h // (Hq // Hkv)``.

Table entries outside ``0 .. n_pages-1`` are no pages: keys there are not
attended and rows are not written.  Rows past a length have no influence,
whatever they hold.  A negative length stands for no sequence: its output is zeros, its length stays.
A score of -inf is a key masked out: where every key is, the output is zeros and
the log sum -1e9, as without keys.  NaN or +inf in a score give NaN, and an
infinite value in a visible row NaN or an infinity.

For inference: inputs that need a gradient, or carry a forward-mode one, are refused.
"""

import weakref

import torch

import _nsa_lib as L
import nsa_hip_ops as _ops


def _attend(q, k_new, v_new, k_pages, v_pages, table, lens, scale, return_lse, max_len=None):
    f = L.torch_side().paged
    if _ops._TIMER is None:
        return f(q, k_new, v_new, k_pages, v_pages, table, lens, scale, return_lse, max_len)
    with _ops._span("nsa_paged_attend"):
        return f(q, k_new, v_new, k_pages, v_pages, table, lens, scale, return_lse, max_len)


def paged_attend(q, k_pages, v_pages, table, lens, scale=None, return_lse=False):
    """``softmax(scale q K^T) V`` of one query per sequence, ``q [B, Hq, D]``, over
    the first ``lens[b]`` positions -> ``out [B, Hq, D]`` (zeros where there are
    none).  ``scale`` defaults to ``D ** -0.5``; ``return_lse`` adds
    ``ln sum e^score`` (float32 ``[B, Hq]``, -1e9 without keys)."""
    out, lse, _ = _attend(q, None, None, k_pages, v_pages, table, lens, scale, return_lse)
    return (out, lse) if return_lse else out


def paged_step(q, k_new, v_new, k_pages, v_pages, table, lens, scale=None, max_len=None):
    """One generation step: the new rows ``[B, Hkv, D]`` go to position
    ``lens[b]`` (in place, in the pages), then ``q [B, Hq, D]`` attends the
    ``lens[b] + 1`` positions -> ``(out, new lens)``; the lengths are a new
    tensor.  A sequence whose position has no page, or is at or past ``max_len``
    (default: the table's end), keeps its pages and length and attends what it
    holds.  Pages that are written may not be shared with
    another sequence of the call."""
    assert k_new is not None and v_new is not None, "paged: a step takes new rows (paged_attend takes none)"
    out, _, lens_out = _attend(q, k_new, v_new, k_pages, v_pages, table, lens, scale, False, max_len)
    return out, lens_out


def paged_append(k, v, k_pages, v_pages, table, lens, count=None, max_len=None):
    """Write rows ``k, v [B, Hkv, T, D]`` (the first ``count[b]`` of them: int32
    ``[B]``, default T) to positions ``lens[b] ..`` -> the new lengths.  A
    sequence whose rows do not all have a page, or do not all lie before
    ``max_len`` (default: the table's end), keeps its pages and length."""
    side = L.torch_side()
    side.no_tangent([k, v, k_pages, v_pages], "paged_append")
    side.check_pages(k_pages, v_pages, table, lens)
    n, Hkv, P, D = k_pages.shape
    B, mp = table.shape
    assert k.dim() == 4 and k.shape[:2] == (B, Hkv) and k.shape[3] == D and v.shape == k.shape, \
        "paged: rows must be [B, Hkv, T, D]"
    assert all(t.dtype == k_pages.dtype and t.device == k_pages.device for t in (k, v)), \
        "paged: rows in the pages' dtype and device"
    assert not (torch.is_grad_enabled() and any(t.requires_grad for t in (k, v, k_pages, v_pages))), \
        "paged: rows in pages have no gradient: call it under torch.no_grad()"
    assert Hkv <= 4096 and B <= 65536, "paged: at most 4096 heads and 65536 sequences"
    assert max_len is None or max_len >= 0, "paged: max_len must not be negative"
    end = 2 ** 31 - 1 if max_len is None else min(max_len, 2 ** 31 - 1)
    k, v, table, lens = _ops._contig(k), _ops._contig(v), table.contiguous(), lens.contiguous()
    if count is not None:
        assert count.dtype == torch.int32 and count.shape == (B,) and count.device == lens.device, \
            "paged: count int32 [B] on the pages' device"
        count = count.contiguous()
    lens_out = torch.empty_like(lens)
    if B > 0:
        with _ops.device_of(k_pages):
            _ops._call("nsa_paged_append", _ops._lib().nsa_paged_append_max, L.ptr(k), L.ptr(v), L.ptr(k_pages),
                       L.ptr(v_pages), L.ptr(table), L.ptr(lens), L.ptr(count), L.ptr(lens_out), B, Hkv, k.shape[2], D,
                       P, mp, n, end, L.dtype_code(k_pages), _ops._stream(k_pages))
    return lens_out


def _staged(numbers, dtype, device):
    """Host numbers as a tensor on ``device``, with no wait for the device: the copy is
    made from pinned memory, which torch keeps until it is done."""
    host, device = torch.as_tensor(numbers, dtype=dtype), torch.device(device)
    if device.type != "cuda":
        return host.to(device)
    assert not torch.cuda.is_current_stream_capturing(), \
        "paged: a capture would read the host's numbers on every replay: reserve, or hand over lengths, before it"
    # (memory of its own: a caller's pinned tensor may be changed while the copy waits its turn)
    return torch.empty(host.shape, dtype=dtype, pin_memory=True).copy_(host).to(device, non_blocking=True)


class _PageAccount:
    """The table of a set of caches, and the host's account of who holds which page.
    The caches themselves are held weakly: a dropped cache frees its pages at once."""

    def __init__(self, batch, max_pages, n_pages, device):
        self.table = torch.full((batch, max_pages), -1, device=device, dtype=torch.int32)
        self.free = list(range(n_pages - 1, -1, -1))
        self.held = [[] for _ in range(batch)]
        self.caches = weakref.WeakSet()


class PagedKVCache:
    """Pages, table and lengths of one dense attention layer for ``batch``
    sequences of up to ``max_len`` tokens (``n_kv_heads`` x ``head_dim``).

    ``n_pages`` pages in all (default: enough for every sequence at
    ``max_len``).  Sequences take pages with ``reserve`` and give them back with
    ``release``, on the host's own account of the table (neither reads the
    device or waits for it).  ``step`` needs the new position reserved.  ``like``, another
    layer's cache of the same sizes: both lie under one table, and reserving or
    releasing on either serves both; each has its own pages and lengths."""

    def __init__(self, batch, n_kv_heads, head_dim, max_len, page_size=64, n_pages=None, dtype=torch.bfloat16,
                 device="cuda", like=None):
        assert page_size >= 16 and page_size % 16 == 0, "paged: the page size must be a multiple of 16"
        assert batch >= 1 and max_len >= 1, "paged: a cache of at least one sequence and one token"
        self.page_size, self.max_len = page_size, max_len
        self.max_pages = -(-max_len // page_size)
        n_pages = batch * self.max_pages if n_pages is None else n_pages
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        if like is not None:
            assert (like.batch, like.page_size, like.max_pages, like.k_pages.shape[0]) == \
                (batch, page_size, self.max_pages, n_pages), "paged: caches under one table differ in size"
        self.k_pages = torch.zeros(shape, device=device, dtype=dtype)
        self.v_pages = torch.zeros(shape, device=device, dtype=dtype)
        self.lens = torch.zeros(batch, device=device, dtype=torch.int32)
        self._account = _PageAccount(batch, self.max_pages, n_pages, device) if like is None else like._account
        L.torch_side().check_pages(self.k_pages, self.v_pages, self.table, self.lens)
        self._account.caches.add(self)

    @property
    def table(self):
        return self._account.table

    @property
    def batch(self):
        return len(self._account.held)

    @property
    def capacity(self):
        return self.max_pages * self.page_size

    @property
    def free_pages(self):
        return len(self._account.free)

    def reserve(self, lengths):
        """Pages for ``lengths`` tokens (an int for all sequences, or one per
        sequence); what a sequence holds already stays.  Raises RuntimeError,
        and takes nothing, where the pages do not suffice.  The table is
        written on the current stream, with no wait for the device; inside a
        capture new pages are refused."""
        acc = self._account
        lengths = [lengths] * self.batch if isinstance(lengths, int) else [int(n) for n in lengths]
        assert len(lengths) == self.batch, "paged: one length for each sequence"
        assert 0 <= min(lengths) and max(lengths) <= self.max_len, "paged: lengths of 0 to max_len"
        need = [-(-n // self.page_size) for n in lengths]
        more = [max(0, n - len(h)) for n, h in zip(need, acc.held)]
        if sum(more) > len(acc.free):
            raise RuntimeError(f"paged: {sum(more)} pages needed, {len(acc.free)} free")
        rows = [b for b, m in enumerate(more) for _ in range(m)]
        if not rows:
            return
        cols = [len(h) + i for h, m in zip(acc.held, more) for i in range(m)]
        pages = acc.free[:-len(rows) - 1:-1]
        at = _staged([rows, cols, pages], torch.int64, self.table.device)
        self.table[at[0], at[1]] = at[2].to(torch.int32)
        del acc.free[-len(rows):]
        for b, page in zip(rows, pages):
            acc.held[b].append(page)

    def release(self, seq):
        """Give back sequence ``seq``'s pages; its length becomes 0.  Refused inside a
        capture, whose replays the account would not see."""
        acc = self._account
        assert 0 <= seq < self.batch, "paged: no such sequence"
        assert not (self.lens.is_cuda and torch.cuda.is_current_stream_capturing()), "paged: release inside a capture"
        acc.free.extend(reversed(acc.held[seq]))
        acc.held[seq] = []
        acc.table[seq].fill_(-1)
        for cache in acc.caches:
            cache.lens[seq].zero_()

    def prefill(self, k, v, lens=None):
        """Append a prompt's rows ``[B, Hkv, T, D]``, ``lens`` of them a sequence
        (int32 ``[B]`` on the device, or host ints; default T); the pages must
        be reserved."""
        self.lens.copy_(paged_append(k, v, self.k_pages, self.v_pages, self.table, self.lens, self.counts(lens),
                                     self.max_len))

    def counts(self, lens):
        """``prefill``'s ``lens`` as it is handed to the kernel (int32 on the device, or
        None): converted once for the caches of many layers."""
        if torch.is_tensor(lens) and lens.device == self.lens.device:
            return lens.to(torch.int32)
        return None if lens is None else _staged(lens, torch.int32, self.lens.device).expand(self.batch)

    def step(self, q, k_new, v_new, scale=None):
        """``paged_step`` on this cache -> ``out [B, Hq, D]``.  The lengths are
        updated in place: a captured step advances the cache on every replay.
        A sequence of ``max_len`` tokens, or whose position is not reserved,
        keeps its length and attends what it holds."""
        out, lens = paged_step(q, k_new, v_new, self.k_pages, self.v_pages, self.table, self.lens, scale,
                               self.max_len)
        self.lens.copy_(lens)
        return out

    def attend(self, q, scale=None, return_lse=False):
        """``paged_attend`` on this cache."""
        return paged_attend(q, self.k_pages, self.v_pages, self.table, self.lens, scale, return_lse)
