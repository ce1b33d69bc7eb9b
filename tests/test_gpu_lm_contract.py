"""What the operators around the attention promise beyond their formulas:
defaults, what is held and for how long, and where they end.
"""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
CFG = dict(vocab_size=203, d_model=128, n_layers=2, n_q_heads=8, n_kv_heads=2, max_seq_len=96, norm="rms",
           ffn="swiglu", ffn_hidden=160, tie_embeddings=False, attn_type="full")


def _model(seed=0, dtype=F32, **kw):
    from nsa_model import NSATransformer
    torch.manual_seed(seed)
    return NSATransformer(**{**CFG, **kw}).cuda().to(dtype)


def _tokens(B, T, seed=0):
    return torch.randint(0, CFG["vocab_size"], (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("res", [True, False])
def test_default_eps_is_rms_norms(dtype, res):
    """``eps=None`` on rows whose mean square is far below, near and above the
    candidates for it: torch.nn.RMSNorm's own result, and its formula in 64 bits
    with 2^-23.

    y: a sum of 200 squares over 25 lanes (8 additions and 6 steps, halved by the
    root) and 7 roundings besides: 14 u, u = 2^-24; then half a step of its dtype.
    Two results of dtype within one step of each other, and 8 bits within half
    a step of e4m3 (2^-4, 2^-10 near zero) and the scale's rounding."""
    import nsa_lm
    dev = require_gpu()
    D, U = 200, 2.0 ** -24
    size = torch.tensor([2.0 ** -12, 2.0 ** -11, 2.0 ** -6, 0.02, 2.0 ** -3, 1.0])[:, None]
    x = (torch.randn(6, D, generator=torch.Generator().manual_seed(1)) * size).to(dtype)
    w = (1 + 0.2 * torch.randn(D, generator=torch.Generator().manual_seed(2))).to(dtype)
    xd, wd = x.to(dev), w.to(dev)
    r = torch.zeros_like(xd) if res else None
    y, _ = nsa_lm.add_rms_norm(xd, r, wd)
    h = x.double()
    ref = h / torch.sqrt((h * h).mean(1, keepdim=True) + 2.0 ** -23) * w.double()
    half = torch.finfo(dtype).eps / 2
    assert ((y.cpu().double() - ref).abs() <= ref.abs() * (half + 14 * U) * (1 + 1e-6)).all()
    m = torch.nn.RMSNorm(D).to(dev).to(dtype)
    with torch.no_grad():
        m.weight.copy_(wd)
        t = m(xd)
    assert ((y.double() - t.double()).abs().cpu() <= 2 * ref.abs() * (half + 14 * U) * (1 + 1e-6)).all()
    assert nsa_lm.add_rms_norm(torch.zeros_like(xd), r, wd, eps=0.0)[0].isnan().all()      # 0 / 0, as the formula
    q, s, _ = nsa_lm.add_rms_norm_q8(xd, r, wd)
    v = q.cpu().double() * s.cpu().double()[:, None]
    assert ((v - ref).abs() <= torch.maximum(ref.abs() * 2.0 ** -4, s.cpu().double()[:, None] * 2.0 ** -10) +
            ref.abs() * 40 * U).all()


def test_fused_norms_in_bf16_are_the_plain_models():
    """A bf16 model at its initialisation, where the embedding's rows have a mean
    square of 4e-4: the fused norms' logits against the plain ones'.  Every
    product's output carries 2^-8 of its size, eight of them in a row over the two
    layers; an eps of bf16's step moves these logits by most of their size."""
    require_gpu()
    ref = _model(dtype=BF, pos="rope").eval()
    new = _model(dtype=BF, pos="rope", norm_impl="fused").eval()
    new.load_state_dict(ref.state_dict())
    x = _tokens(2, 60)
    with torch.no_grad():
        a, b = ref(x)[0].double(), new(x)[0].double()
    assert float((a - b).abs().max()) <= 8 * 2.0 ** -8 * float(a.abs().max())


# ---------------------------------------------------------------------------
# forward-mode derivatives
# ---------------------------------------------------------------------------

def test_tangents_of_inputs_and_incoming_gradients_are_refused():
    import torch.autograd.forward_ad as fa
    import nsa_lm
    dev = require_gpu()
    x, w = torch.randn(3, 16, device=dev), torch.ones(16, device=dev, requires_grad=True)
    z = torch.randn(3, 16, device=dev, requires_grad=True)
    with fa.dual_level():
        for t in (x, x.clone().requires_grad_()):
            d = fa.make_dual(t, torch.ones_like(t))
            for call in (lambda: nsa_lm.add_rms_norm(d, None, w), lambda: nsa_lm.token_logprobs(d)):
                with pytest.raises(AssertionError, match="forward-mode"):
                    call()
        y, _ = nsa_lm.add_rms_norm(x, None, w)
        ent = nsa_lm.token_logprobs(z).entropy
        for out, at in ((y, w), (ent, z)):
            g = torch.ones_like(out)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, at, fa.make_dual(g, g), retain_graph=True)
            torch.autograd.grad(out, at, g)


# ---------------------------------------------------------------------------
# the fused loss
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("bad", [-1, -99, -101, CFG["vocab_size"], 1 << 40], ids=str)
def test_a_target_outside_the_vocabulary_makes_the_loss_nan(bad):
    """Not a smaller mean: the loss and every gradient it has."""
    require_gpu()
    m = _model(pos="rope", loss_impl="fused")
    x, y = _tokens(2, 20), _tokens(2, 20, 1)
    y[0, 3] = -100
    logits, loss = m(x, y)
    want = torch.nn.functional.cross_entropy(logits.double().view(-1, CFG["vocab_size"]), y.view(-1))
    # 39 terms below 16 in at most 39 + 8 float32 additions, each term within 32 u of its size
    assert abs(float(loss.detach()) - float(want)) <= (39 + 8 + 32) * 2.0 ** -24 * 16
    y[1, 7] = bad
    loss = m(x, y)[1]
    assert loss.isnan() and loss.dtype == F32
    loss.backward()
    assert m.lm_head.weight.grad.isnan().any(1).all() and m.tok_emb.weight.grad.isnan().any()
    y[:] = -100
    assert m(x, y)[1].isnan()       # no target at all: cross_entropy's 0 / 0


# ---------------------------------------------------------------------------
# rotation tables
# ---------------------------------------------------------------------------

def test_rotation_tables_are_a_streams_own():
    from nsa_model import Rotary
    dev = require_gpu()
    rope = Rotary(32).to(dev)
    cos, sin = rope.tables(50, dev, BF)
    assert rope.tables(50, dev, BF)[0] is cos
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = rope.tables(50, dev, BF)
        assert other[0].data_ptr() != cos.data_ptr() and rope.tables(50, dev, BF)[0] is other[0]
    torch.cuda.synchronize()
    assert torch.equal(other[0], cos) and torch.equal(other[1], sin)
    assert rope.tables(50, dev, BF)[0] is cos
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):      # made in the graph, and not kept
        inside = rope.tables(50, dev, BF)
    assert inside[0].data_ptr() not in (cos.data_ptr(), other[0].data_ptr())
    with torch.cuda.stream(side):
        assert rope.tables(50, dev, BF)[0] is other[0]
    for _ in range(3):
        inside[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(inside[0], cos) and torch.equal(inside[1], sin)


def test_captured_forward_outlives_the_rotation_tables():
    """A forward of the library arm captured behind a warm-up of the same length,
    replayed after ten other lengths have passed and their memory is written over."""
    require_gpu()
    m = _model(dtype=BF, pos="rope", dense_impl="sdpa").eval()
    x = _tokens(2, 48)
    with torch.no_grad():
        want = m(x)[0]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = m(x)[0]
        for T in range(50, 60):
            for stream in (torch.cuda.current_stream(), side):
                with torch.cuda.stream(stream):
                    m(_tokens(2, T))
        torch.cuda.synchronize()
        junk = [torch.full((48, 8), 7.0, device="cuda") for _ in range(300)]
        for seed in range(3):
            x.copy_(_tokens(2, 48, seed))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, m(x)[0]), seed
            if seed == 0:
                assert torch.equal(out, want)
        del junk


def test_training_behind_inference_of_the_same_length():
    require_gpu()
    m = _model(dtype=BF, pos="rope", dense_impl="sdpa")
    x = _tokens(2, 32)
    with torch.inference_mode():
        want = m(x)[0].clone()
    logits, loss = m(x, x)
    loss.backward()
    assert torch.equal(logits, want) and m.blocks[0].attn.q_proj.weight.grad.abs().sum() > 0


# ---------------------------------------------------------------------------
# paged caches
# ---------------------------------------------------------------------------

def test_a_generation_loop_never_waits_for_the_device():
    """Reserving, prefilling with the host's lengths, stepping and releasing all
    return while the device is still busy with what was asked for before them,
    and what they wrote is right although their numbers were staged meanwhile."""
    require_gpu()
    m = _model(pos="rope").eval()
    x = _tokens(2, 40)
    with torch.no_grad():
        want = m(x)[0]
    big = torch.randn(8192, 8192, device="cuda", dtype=BF)

    def loop(busy):
        caches = m.paged_caches(2, 96, page_size=16)
        lens = [20, 7]
        if busy:
            for _ in range(400):            # about 0.4 s of work ahead of the loop
                big @ big
        ahead = torch.cuda.Event()
        ahead.record()
        caches[0].reserve(lens)
        mine = torch.tensor(lens, dtype=torch.int32).pin_memory()
        pre = m.prefill(x[:, :20], caches, mine)
        mine.zero_()                        # (a pinned tensor of the caller's, changed before the device reads it)
        outs = []
        for s in range(12):
            caches[0].reserve([n + s + 1 for n in lens])
            at = torch.stack([x[0, 20 + s], x[1, 7 + s]])
            outs.append(m.step(at, caches))
        caches[1].release(1)
        running = not ahead.query()
        return caches, pre, outs, running
    loop(False)                             # (pinned memory and workspaces are there)
    torch.cuda.synchronize()
    caches, pre, outs, running = loop(True)
    assert running
    for b, n in enumerate([20, 7]):
        assert (pre[b, :n] - want[b, :n]).abs().max() <= 1e-4 * want.abs().max()
        for s, o in enumerate(outs):
            assert (o[b] - want[b, n + s]).abs().max() <= 1e-4 * want.abs().max(), (b, s)
    assert caches[0].lens.tolist() == [32, 0] and (caches[0].table >= 0).sum(1).tolist() == [2, 0]
    torch.cuda.set_sync_debug_mode("error")
    try:
        loop(False)
    finally:
        torch.cuda.set_sync_debug_mode("default")


def test_host_numbers_inside_a_capture_are_refused():
    """A graph would read the staging memory again on every replay."""
    import nsa_paged
    dev = require_gpu()
    c = nsa_paged.PagedKVCache(2, 1, 16, 64, 16, dtype=F32)
    k = torch.randn(2, 1, 20, 16, device=dev)
    on_device = torch.tensor([20, 3], device=dev)
    c.reserve(32)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.reserve(20)                       # nothing new: allowed
        with pytest.raises(AssertionError, match="capture"):
            c.reserve(40)
        with pytest.raises(AssertionError, match="capture"):
            c.prefill(k, k, [20, 3])
        c.prefill(k, k, on_device)
    assert c.free_pages == 4 and c.lens.tolist() == [0, 0]
    for _ in range(3):
        c.lens.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert c.lens.tolist() == [20, 3]


@pytest.mark.parametrize("B,P", [(3, 144), (3, 64), (300, 64)])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_a_cache_ends_at_max_len_inside_a_page(dtype, B, P):
    """max_len 100 over pages of 64 or 144 (equal shares of all keys): position 99 is the last one taken; a step or a
    prompt past it writes nothing, keeps the length, and attends the 100 keys."""
    import nsa_paged
    dev = require_gpu()
    Hq, Hkv, D = 4, 2, 32
    c = nsa_paged.PagedKVCache(B, Hkv, D, 100, P, dtype=dtype)
    c.reserve(100)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(B, Hkv, 98, D, generator=g).to(dtype).to(dev) for _ in range(2))
    start = [98, 97, 50] + [98] * (B - 3)
    c.prefill(k, v, start)
    for s in range(5):
        q, kn, vn = (torch.randn(B, h, D, generator=g).to(dtype).to(dev) for h in (Hq, Hkv, Hkv))
        before = c.k_pages.clone()
        want_lens = [min(100, n + s + 1) for n in start]
        out = c.step(q, kn, vn)
        assert c.lens.tolist() == want_lens
        assert torch.equal(out, c.attend(q))                # (the same keys in the same pieces)
        ids = c.table.cpu()
        for b in range(3):
            if start[b] + s < 100:
                before[int(ids[b, (start[b] + s) // P]), :, (start[b] + s) % P] = kn[b]
        if B > 3 and s < 2:
            at = 98 + s
            before[c.table[3:, at // P].long(), :, at % P] = kn[3:]
        assert torch.equal(c.k_pages, before)
    c.prefill(k[:, :, :1], v[:, :, :1], 1)                  # one row more: only where it fits
    assert c.lens.tolist() == [100, 100, 56] + [100] * (B - 3)
    c.prefill(k, v, 45)                                     # 56 + 45 = 101
    assert c.lens.tolist() == [100, 100, 56] + [100] * (B - 3)
    c.prefill(k, v, 44)
    assert c.lens.tolist() == [100] * B
    with pytest.raises(AssertionError):
        c.reserve(101)
    lens = torch.full((B,), 100, dtype=torch.int32, device=dev)
    args = (q, kn, vn, c.k_pages, c.v_pages, c.table, lens)
    assert nsa_paged.paged_step(*args)[1].tolist() == [101] * B          # the bare pages go to the table's end
    assert nsa_paged.paged_step(*args, max_len=100)[1].tolist() == [100] * B
    assert nsa_paged.paged_step(*args, max_len=0)[1].tolist() == [100] * B
    with pytest.raises(AssertionError):
        nsa_paged.paged_step(*args, max_len=-1)
    with pytest.raises(AssertionError):
        nsa_paged.paged_append(k, v, *args[3:], max_len=-1)


@pytest.mark.parametrize("pos", ["learned", "rope"])
def test_generation_ends_at_the_models_length(pos):
    """max_seq_len 90 over pages of 64: the last position's logits are the
    forward's, and no token is appended behind it."""
    require_gpu()
    m = _model(pos=pos, max_seq_len=90).eval()
    x = _tokens(2, 90)
    with torch.no_grad():
        want = m(x)[0]
    caches = m.paged_caches(2)
    caches[0].reserve(90)
    m.prefill(x[:, :85], caches)
    for s in range(85, 90):
        logits = m.step(x[:, s], caches)
        assert (logits - want[:, s]).abs().max() <= 1e-4 * want.abs().max()
    kept = [c.k_pages.clone() for c in caches]
    m.step(x[:, 0], caches)
    for c, k in zip(caches, kept):
        assert c.lens.tolist() == [90, 90] and torch.equal(c.k_pages, k)


@pytest.mark.parametrize("n", [5, 100, 4000])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_scores_at_the_ends_of_the_range(dtype, n):
    """Rows whose scores are all far below -1e30, scores of -inf among finite ones,
    nothing but -inf, and NaN or +inf; in one piece and joined.

    The scores are powers of two times small whole numbers, so that the weights are
    exactly equal or 0.  An average over m keys: at most n/16 + 40 additions, one
    product with 1 / m, and half a step of the output's dtype; bf16 weights in two
    parts are exact here."""
    import nsa_paged
    dev = require_gpu()
    D, P, U = 16, 48, 2.0 ** -24
    mp = -(-4100 // P)
    g = torch.Generator().manual_seed(n)
    v = torch.randn(1, 1, n, D, generator=g).to(dtype)
    low = torch.zeros(1, 1, n, D)
    low[..., 0] = -(2.0 ** 50) * (1 + torch.arange(n) % 3)          # scores of -1e31 to -3e31
    some = torch.zeros(1, 1, n, D)
    some[..., 0] = torch.where(torch.arange(n) % 3 == 0, 0.0, -float("inf"))
    none = torch.zeros(1, 1, n, D)
    none[..., 0] = -float("inf")
    q = torch.zeros(1, 2, D)
    q[..., 0] = 2.0 ** 55
    c = nsa_paged.PagedKVCache(1, 1, D, mp * P, P, dtype=dtype)
    c.reserve(n)
    keep = torch.arange(n) % 3 == 0
    vk = v[0, 0, keep].double()
    ref = vk.mean(0)
    tol = ref.abs() * torch.finfo(dtype).eps / 2 * (1 + 1e-6) + vk.abs().mean(0) * (n / 16 + 42) * U
    for k, base in ((low, -(2.0 ** 105) / 4), (some, 0.0)):
        c.lens.zero_()
        c.prefill(k.to(dtype).to(dev), v.to(dev))
        out, lse = c.attend(q.to(dtype).to(dev), return_lse=True)
        assert ((out.cpu().double() - ref).abs() <= tol).all()
        want = base + torch.tensor(float(keep.sum())).double().log()
        assert ((lse.cpu().double() - want).abs() <= 8 * U * want.abs() + 8 * U).all()
    c.lens.zero_()
    c.prefill(none.to(dtype).to(dev), v.to(dev))
    out, lse = c.attend(q.to(dtype).to(dev), return_lse=True)
    assert not out.any() and (lse == -1e9).all()
    for bad in (float("nan"), float("inf")):
        k = some.clone()
        k[0, 0, n // 2, 0] = bad
        c.lens.zero_()
        c.prefill(k.to(dtype).to(dev), v.to(dev))
        out, lse = c.attend(q.to(dtype).to(dev), return_lse=True)
        assert out.isnan().all()


def test_releasing_inside_a_capture_is_refused():
    """The account would give the pages to another sequence, and every replay take
    them from it again."""
    import nsa_paged
    dev = require_gpu()
    c = nsa_paged.PagedKVCache(2, 1, 16, 64, 16, dtype=F32)
    c.reserve(32)
    x = torch.zeros(4, device=dev)
    table = c.table.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(AssertionError, match="capture"):
            c.release(0)
    graph.replay()
    torch.cuda.synchronize()
    assert c.free_pages == 4 and torch.equal(c.table, table)
    c.release(0)
    assert c.free_pages == 6 and (c.table[0] == -1).all()


# B, lens, Hq, Hkv, D, P
COUNTS = [(1, [20000], 64, 4, 128, 80), (1, [33000], 16, 1, 64, 256), (5, [1, 127, 128, 129, 5000], 40, 1, 128, 16),
          (7, [3000, 0, 31, 2049, 4095, 4096, 4097], 12, 2, 32, 48), (300, [(7 * i) % 90 for i in range(300)], 8, 8, 16, 112)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("c", COUNTS, ids=lambda c: f"B{c[0]}-n{max(c[1])}-H{c[2]}:{c[3]}")
def test_every_key_counts_once(c, dtype):
    """Equal scores: every weight is exactly 1 before the division and every sum of
    them a whole number below 2^24, so that only 1 / n, its product (2 u) and the
    output's half step round.  A key left out or taken twice shows in the log
    sum (by 1 / n, against its logarithm's and product's 4 u ln n) and, where it
    has a column of its own at an edge of a tile, share or page, in the output by
    all of it."""
    import nsa_paged
    dev = require_gpu()
    B, lens, Hq, Hkv, D, P = c
    U, half = 2.0 ** -24, torch.finfo(dtype).eps / 2
    g = torch.Generator().manual_seed(B + D)
    cache = nsa_paged.PagedKVCache(B, Hkv, D, max(lens), P, dtype=dtype)
    cache.reserve(lens)
    T = max(lens)
    k = torch.randn(B, Hkv, T, D, generator=g).to(dtype)
    whole = torch.randint(-8, 9, (B, Hkv, T, D), generator=g).to(dtype)
    alone = torch.zeros(B, Hkv, T, D, dtype=dtype)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        edges = [e for m in (32, 128, P, 1024) for x in (m, n // m * m) for e in (x - 1, x)]
        edges += [0, n - 1] + torch.randint(0, n, (D,), generator=g).tolist()
        edges = list(dict.fromkeys(e for e in edges if 0 <= e < n))[:D]
        alone[b][:, edges, torch.arange(len(edges))] = 2.0 ** 14
    q = torch.zeros(B, Hq, D, dtype=dtype, device=dev)
    n = torch.tensor(lens)[:, None, None]
    for v in (whole, alone):
        cache.lens.zero_()
        cache.prefill(k.to(dev), v.to(dev), lens)
        out, lse = cache.attend(q, return_lse=True)
        live = torch.arange(T)[None, None, :, None] < n[..., None]
        ref = (torch.where(live, v.double(), 0.0).sum(2) / n.clamp(min=1)).repeat_interleave(Hq // Hkv, 1)
        err = (out.cpu().double() - ref).abs()
        assert (err <= ref.abs() * (half + 2 * U) * (1 + 1e-6)).all(), float(err.max())
        want = torch.where(n[:, :, 0] > 0, n[:, :, 0].double().log(), -1e9)
        assert ((lse.cpu().double() - want).abs() <= torch.where(n[:, :, 0] > 0, 4 * U * want, 0.0)).all()


@pytest.mark.parametrize("rows,D", [(2, 8), (5, 250), (3, 1001), (4, 2049), (3, 4096), (300, 8192)])
def test_norm_within_one_run_a_thread(rows, D):
    """Rows of up to 8192 elements are one run of 8 a thread: 8 additions, 6 steps
    over the wave, 16 waves, halved by the root, and 7 roundings besides."""
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator().manual_seed(D)
    x, r = torch.randn(rows, D, generator=g), torch.randn(rows, D, generator=g)
    w = 1 + 0.2 * torch.randn(D, generator=g)
    y, h = nsa_lm.add_rms_norm(x.to(dev), r.to(dev), w.to(dev), eps=1e-5)
    h64 = (x + r).double()
    ref = h64 / torch.sqrt((h64 * h64).mean(-1, keepdim=True) + 1e-5) * w.double()
    assert ((y.cpu().double() - ref).abs() <= ref.abs() * (15 + 7 + 1) * 2.0 ** -24).all()


def test_the_c_entry_points_without_an_end():
    """nsa_paged_append and nsa_paged_attend, called as from C, are the functions
    over bare pages."""
    import _nsa_lib as L
    import nsa_paged
    dev = require_gpu()
    lib = L.load()
    B, Hq, Hkv, D, P, mp, T = 2, 8, 2, 64, 16, 6, 90
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(B, Hkv, T, D, generator=g).to(BF).to(dev) for _ in range(2))
    q, kn, vn = (torch.randn(B, h, D, generator=g).to(BF).to(dev) for h in (Hq, Hkv, Hkv))
    table = torch.randperm(B * mp, generator=g).view(B, mp).to(torch.int32).to(dev)
    zero, count = torch.zeros(B, dtype=torch.int32, device=dev), torch.tensor([T, 37], dtype=torch.int32, device=dev)
    want = [torch.zeros(B * mp, Hkv, P, D, device=dev, dtype=BF) for _ in range(2)]
    n = nsa_paged.paged_append(k, v, *want, table, zero, count)
    out, n1 = nsa_paged.paged_step(q, kn, vn, *want, table, n)
    pages = [torch.zeros_like(t) for t in want]
    lens, lens1, o = torch.empty_like(zero), torch.empty_like(zero), torch.empty_like(q)
    stream = L.stream_of(q)
    assert lib.nsa_paged_append(L.ptr(k), L.ptr(v), *map(L.ptr, pages), L.ptr(table), L.ptr(zero), L.ptr(count),
                                L.ptr(lens), B, Hkv, T, D, P, mp, B * mp, L.NSA_BF16, stream) == 0
    size = lib.nsa_paged_workspace(B, Hq, Hkv, D, P, mp, L.NSA_BF16, stream)
    ws = torch.empty(max(16, size), dtype=torch.uint8, device=dev)
    assert lib.nsa_paged_attend(L.ptr(q), L.ptr(kn), L.ptr(vn), *map(L.ptr, pages), L.ptr(table), L.ptr(lens),
                                L.ptr(lens1), L.ptr(o), None, L.ptr(ws), ws.numel(), B, Hq, Hkv, D, P, mp, B * mp,
                                D ** -0.5, L.NSA_BF16, stream) == 0
    assert torch.equal(lens, n) and torch.equal(lens1, n1) and torch.equal(o, out)
    assert all(torch.equal(a, b) for a, b in zip(pages, want))
