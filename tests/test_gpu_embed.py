"""nsa_lm.embed against the definition in 64 bits.

Tolerances, u = 2^-24 (half a float32 step, relative): a row is one fused
multiply-add of a scale that float32 holds within u, so within u |scale w| + u |sum|
and half a step of its dtype.  A gradient row is a sum of c rows in at most c
additions and one product: within (c + 2) u of the sum of its terms' magnitudes, and
half a step of its dtype."""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tokens(shape, V, seed, kind="zipf"):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full(shape, min(V - 1, 3))
    if kind == "ascending":
        n = torch.Size(shape).numel()
        return (torch.arange(n) % V).view(shape)
    t = (torch.exp(torch.rand(shape, generator=g) * torch.log(torch.tensor(V + 1.0))) - 1).long().clamp(0, V - 1)
    t = torch.randperm(V, generator=g)[t]
    if kind == "padded":
        t[torch.rand(shape, generator=g) < 0.3] = -1
        t.view(-1)[:3] = torch.tensor([V, -100, 1 << 40])[:t.numel()]
    if kind == "none":
        t.fill_(-1)
    return t


def _check(tokens, V, D, wd, od, scale, pos, pd=None, P=None, seed=0):
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator().manual_seed(seed + 1)
    w = torch.randn(V, D, generator=g).to(wd)
    T = tokens.shape[-1]
    pw = at = None
    if pos != "none":
        P = T if P is None else P
        pw = torch.randn(P, D, generator=g).to(pd or wd)
        if pos == "given":
            at = torch.randint(-1, P + 1, tokens.shape, generator=g)
    dy = torch.randn(*tokens.shape, D, generator=g).to(od)
    ws = w.to(dev).requires_grad_()
    ps = None if pw is None else pw.to(dev).requires_grad_()
    y = nsa_lm.embed(tokens.to(dev), ws, scale, ps, None if at is None else at.to(dev), od)
    got = torch.autograd.grad(y, [t for t in (ws, ps) if t is not None], dy.to(dev))
    t = tokens.reshape(-1)
    real = (t >= 0) & (t < V)
    term = torch.where(real[:, None], w.double()[t.clamp(0, V - 1)] * scale, 0.0)
    ref = term
    where = None
    if pw is not None:
        where = torch.arange(T).expand(tokens.shape).reshape(-1) if at is None else at.reshape(-1)
        ok = (where >= 0) & (where < P)
        ref = ref + torch.where(ok[:, None], pw.double()[where.clamp(0, P - 1)], 0.0)
    assert y.dtype == od and y.shape == (*tokens.shape, D)
    tol = term.abs() * U + ref.abs() * (U + _half(od)) * (1 + 1e-6) + 1e-40
    err = (y.detach().cpu().double().view(-1, D) - ref).abs()
    assert (err <= tol).all(), float((err - tol).max())

    def grad(idx, rows, s, dtype, mine):
        ok = (idx >= 0) & (idx < rows)
        d = dy.double().view(-1, D)[ok]
        zero = torch.zeros(rows, D, dtype=torch.float64)
        want = zero.clone().index_add_(0, idx[ok], d) * s
        mag = zero.index_add_(0, idx[ok], d.abs()) * abs(s)
        c = torch.bincount(idx[ok], minlength=rows)[:, None]
        tol = (mag * (c + 2) * U + want.abs() * _half(dtype)) * (1 + 1e-6)
        assert mine.dtype == dtype
        err = (mine.cpu().double() - want).abs()
        assert (err <= tol).all(), float((err - tol).max())
        assert not mine.cpu()[c.view(-1) == 0].any()
    grad(t, V, scale, wd, got[0])
    if pw is not None:
        grad(where, P, 1.0, pw.dtype, got[1])


SHAPES = [((1,), 1, 1), ((1, 1), 5, 8), ((3, 7), 11, 17), ((2, 31), 3, 33), ((2, 32), 100, 64), ((4, 65), 1000, 130),
          ((1, 1023), 511, 24), ((2, 513), 512, 40), ((5, 410), 8191, 250), ((8, 700), 32000, 96), ((3, 341), 50257, 520),
          ((2, 100), 300, 1001), ((1, 77), 400, 2100), ((2, 9, 40), 700, 48), ((1, 40000), 131071, 8)]


@pytest.mark.parametrize("kind", ["zipf", "one", "padded", "ascending", "none"])
@pytest.mark.parametrize("shape,V,D", SHAPES, ids=str)
def test_tokens_alone(shape, V, D, kind):
    n = torch.Size(shape).numel()
    _check(_tokens(shape, V, n + V, kind), V, D, F32, F32, 1.0, "none", seed=V)


@pytest.mark.parametrize("types", [(BF, BF, BF), (F32, F32, F32), (BF, F32, F32), (F32, BF, BF)], ids=str)
@pytest.mark.parametrize("pos", ["none", "seq", "given"])
@pytest.mark.parametrize("shape,V,D", [((1, 1), 9, 16), ((3, 33), 50, 65), ((8, 300), 2000, 768), ((32, 1), 32000, 96),
                                       ((7, 129), 100, 1030)], ids=str)
def test_types_scales_and_positions(shape, V, D, pos, types):
    wd, pd, od = types
    _check(_tokens(shape, V, 5, "padded"), V, D, wd, od, D ** 0.5, pos, pd, shape[-1] + 9, seed=D)


@pytest.mark.parametrize("B,T", [(1, 5), (2, 64), (33, 70), (100, 3)])
def test_positions_of_many_sequences(B, T):
    _check(_tokens((B, T), 40, 1), 40, 36, F32, F32, 1.0, "seq", P=T + 70, seed=B)


def test_more_pairs_than_one_block_size():
    """More than 256 blocks of the sort: each thread takes more than four pairs."""
    _check(_tokens((1, 300001), 70000, 3, "padded"), 70000, 8, F32, F32, 1.0, "none")


def test_wide_vocabulary():
    """Tokens of 19 bits are sorted in three passes."""
    _check(_tokens((1, 5000), 400000, 3), 400000, 8, BF, F32, 1.0, "none")


def test_pieces_longer_than_32():
    _check(_tokens((1, 140000), 37, 3), 37, 8, F32, F32, 1.0, "none")


def test_integer_types_strides_and_alignment():
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator().manual_seed(0)
    V, D = 300, 40
    w = torch.randn(V, 2 * D, generator=g).to(BF).to(dev)
    t = torch.randint(0, V, (6, 10), generator=g).to(dev)
    want = nsa_lm.embed(t, w[:, :D].contiguous())
    assert torch.equal(nsa_lm.embed(t, w[:, :D]), want)
    for d in (torch.int32, torch.int16):
        assert torch.equal(nsa_lm.embed(t.to(d), w[:, :D]), want)
    assert torch.equal(nsa_lm.embed(t.t(), w[:, :D]), want.transpose(0, 1))
    flat = torch.randn(V * D + 1, generator=g).to(dev)
    off = flat[1:].view(V, D)
    assert torch.equal(nsa_lm.embed(t, off), off[t])
    assert torch.equal(nsa_lm.embed(t[0, 0], off), off[t[0, 0]])          # a single token
    e = torch.empty(0, 4, dtype=torch.long, device=dev)
    ws, ps = off.detach().requires_grad_(), torch.randn(9, D, device=dev, requires_grad=True)
    y = nsa_lm.embed(e, ws, pos_weight=ps)
    y.sum().backward()
    assert y.shape == (0, 4, D) and not ws.grad.any() and not ps.grad.any()
    # one of the tables alone
    both = torch.autograd.grad(nsa_lm.embed(t, ws, 2.0, torch.cat([ps, ps])).sum(), ws)[0]
    lone = torch.autograd.grad(nsa_lm.embed(t, ws, 2.0, torch.cat([ps, ps]).detach()).sum(), ws)[0]
    assert torch.equal(both, lone)
    a = torch.autograd.grad(nsa_lm.embed(t, ws.detach(), 2.0, ps, t % 9).sum(), ps)[0]
    assert torch.equal(a, torch.bincount((t % 9).view(-1), minlength=9).float()[:, None].expand(9, D))


@pytest.mark.parametrize("shape", [(0,), (4, 0), (0, 4)], ids=str)
@pytest.mark.parametrize("pos", ["none", "given", "index"])
def test_no_tokens(shape, pos):
    import nsa_lm
    dev = require_gpu()
    t = torch.empty(shape, dtype=torch.long, device=dev)
    w, p = (torch.randn(n, 12, device=dev, requires_grad=True) for n in (7, 5))
    y = nsa_lm.embed(t, w, 1.0, None if pos == "none" else p, t if pos == "given" else None)
    assert y.shape == (*shape, 12)
    y.sum().backward()
    assert not w.grad.any() and (pos == "none" or not p.grad.any())


def test_nan_rows_stay_where_they_are():
    import nsa_lm
    dev = require_gpu()
    w = torch.randn(50, 24, device=dev)
    w[7] = float("nan")
    w[9, 3] = float("inf")
    t = torch.tensor([[1, 7, 9, -1, 2]], device=dev)
    y = nsa_lm.embed(t, w)
    assert torch.equal(y.isnan().all(-1), torch.tensor([[False, True, False, False, False]], device=dev))
    assert not y[0, 3].any() and y[0, 2, 3] == float("inf")
    ws = w.detach().requires_grad_()
    dy = torch.ones(1, 5, 24, device=dev)
    dy[0, 0] = float("nan")
    dy[0, 3] = float("nan")                          # (a row without a token: nobody's gradient)
    g, = torch.autograd.grad(nsa_lm.embed(t, ws), ws, dy)
    assert g[1].isnan().all() and torch.equal(g[7], torch.ones(24, device=dev)) and int(g.isnan().any(1).sum()) == 1


def test_same_bits_on_every_run_and_stream():
    import nsa_lm
    dev = require_gpu()
    V, D = 5000, 96
    t = _tokens((4, 3000), V, 2).to(dev)
    w, p = torch.randn(V, D, device=dev), torch.randn(3000, D, device=dev)
    dy = torch.randn(4, 3000, D, device=dev)

    def once():
        a = [w.detach().requires_grad_(), p.detach().requires_grad_()]
        y = nsa_lm.embed(t, a[0], 1.5, a[1])
        return (y.detach(), *torch.autograd.grad(y, a, dy))
    first = once()
    torch.cuda.synchronize()
    got = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(once())
    torch.cuda.synchronize()
    for again in got:
        for a, b in zip(first, again):
            assert torch.equal(a, b)


def test_captured_and_replayed():
    import nsa_lm
    dev = require_gpu()
    V, D, shape = 900, 72, (3, 500)
    t = _tokens(shape, V, 0).to(dev)
    w, p = torch.randn(V, D, device=dev, requires_grad=True), torch.randn(500, D, device=dev, requires_grad=True)
    dy = torch.randn(*shape, D, device=dev)

    def once():
        y = nsa_lm.embed(t, w, 1.0, p)
        return (y.detach(), *torch.autograd.grad(y, (w, p), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for k in range(3):
        t.copy_(_tokens(shape, V, 10 + k, ("zipf", "padded", "one")[k]))
        dy.mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, once()):
            assert torch.equal(a, b)


def test_gradient_against_differences():
    """Linear in both tables: differences of the definition in 64 bits are exact but
    for their rounding."""
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator().manual_seed(3)
    V, D = 13, 21
    t = torch.randint(-1, V, (4, 9), generator=g)
    w, p, dy = (torch.randn(*s, generator=g) for s in ((V, D), (9, D), (4, 9, D)))
    a = [w.to(dev).requires_grad_(), p.to(dev).requires_grad_()]
    grads = torch.autograd.grad(nsa_lm.embed(t.to(dev), a[0], 3.0, a[1]), a, dy.to(dev))

    def loss(ww, pp):
        rows = torch.where((t >= 0)[..., None], ww[t.clamp(min=0)] * 3.0, 0.0)
        return float(((rows + pp) * dy.double()).sum())
    w, p = w.double(), p.double()
    for k, grad in enumerate(grads):
        v = torch.randn(grad.shape, generator=g).double()
        hi, lo = [w, p], [w, p]
        hi[k], lo[k] = hi[k] + v, lo[k] - v
        fd = (loss(*hi) - loss(*lo)) / 2
        mag = float(dy.abs().sum()) * 3 * float(v.abs().max())
        assert abs(float((grad.cpu().double() * v).sum()) - fd) <= 40 * U * mag


def test_second_derivatives_and_refusals():
    import nsa_lm
    import torch.autograd.forward_ad as fwAD
    dev = require_gpu()
    w, p = torch.randn(50, 24, device=dev, requires_grad=True), torch.randn(8, 24, device=dev)
    t = torch.randint(0, 50, (2, 8), device=dev)
    y = nsa_lm.embed(t, w)
    g, = torch.autograd.grad((y * y.detach()).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    for args, kw in (((t.cpu(), w), {}), ((t.float(), w), {}), ((t, w.half()), {}), ((t, w[0]), {}),
                     ((t, w.cpu()), {}), ((t, w, 1.0, p[:, :8]), {}), ((t, w, 1.0, p[:7]), {}),
                     ((t, w, 1.0, p, t[:, :4]), {}), ((t, w, 1.0, None, t), {}), ((t, w, 1.0, p.cpu()), {}),
                     ((t, w, 1.0, p, t.float()), {}), ((t, w), dict(out_dtype=torch.float16)),
                     ((t > 3, w), {})):
        with pytest.raises(AssertionError):
            nsa_lm.embed(*args, **kw)
    with fwAD.dual_level(), pytest.raises(AssertionError):
        nsa_lm.embed(t, fwAD.make_dual(w.detach(), torch.ones_like(w)))
