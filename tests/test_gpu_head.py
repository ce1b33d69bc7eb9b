"""nsa_lm.linear_logprobs against the definition in 64 bits.

Tolerances, u = 2^-24 (half a float32 step, relative), Z = max_v sum_d |x_d w_vd| of a
row:
* a logit is a sum of products that float32 or more holds (float32 operands: planes
  whose left-out products are below 2^-26 of the term), in at most D + 16 additions
  each off by at most a step: within DZ = 2 (D + 16) u Z.
* the log sum: every term's exponent is off by DZ and 4 u of its size, its sum has at
  most V / 4 + 200 additions in a row.
* logp: the target's product by another order, and the log sum.
* a probability is off by DP relative, with DP the two errors above, and 4 u.
* dz is rounded to the operand's precision R (2^-8 for bf16 rows, 2^-24 for float32
  rows); dx and dW are sums of V (N) products in as many additions, each within a step,
  and half a step of their dtype.
"""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _data(N, V, D, xd, wd, seed=0, ignored=True):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g) * (2 / D ** 0.5)
    t = torch.randint(0, V, (N,), generator=g)
    x = torch.randn(N, D, generator=g) + torch.rand(N, 1, generator=g) * 2 * w[t]
    if ignored and N > 2:
        t[torch.rand(N, generator=g) < 0.2] = -100
        t[0], t[1] = V, -1
    dlogp, dlse = -torch.rand(N, generator=g), 0.3 * torch.randn(N, generator=g)
    return x.to(xd), w.to(wd), t, dlogp, dlse


def _bounded(got, ref, tol, what):
    err = (got.detach().double() - ref).abs()
    bad = err - tol
    assert (bad <= 0).all(), f"{what}: {float(bad.max())} past {float(tol.flatten()[bad.argmax()])}"


def _check(N, V, D, xd, wd, seed=0, dev=None, uses="both"):
    """One call, forward and backward; the reference on the same device in 64 bits."""
    import nsa_lm
    dev = require_gpu()
    x, w, t, dlogp, dlse = (a.to(dev) for a in _data(N, V, D, xd, wd, seed))
    xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
    got = nsa_lm.linear_logprobs(xs, ws, t)
    outs, seeds = {"both": ((got.logp, got.lse), (dlogp, dlse)), "logp": ((got.logp,), (dlogp,)),
                   "lse": ((got.lse,), (dlse,))}[uses]
    dx, dw = torch.autograd.grad(outs, (xs, ws), seeds)
    assert (dx.dtype, dw.dtype, got.logp.dtype, got.lse.dtype) == (xd, wd, F32, F32)
    wide = xd == F32
    x64 = x.double()
    w64 = (w if wide else w.to(BF)).double()
    z = x64 @ w64.t().contiguous()
    lse = torch.logsumexp(z, 1)
    Z = (x64.abs() @ w64.abs().t().contiguous()).amax(1)
    DZ = 2 * (D + 16) * U * Z
    top = z.abs().amax(1)
    lse_tol = DZ + (V / 4 + 200) * U + 8 * U * (top + lse.abs())
    _bounded(got.lse, lse, lse_tol, "lse")
    ok = (t >= 0) & (t < V)
    logp = torch.where(ok, z.gather(1, t.clamp(0, V - 1)[:, None])[:, 0] - lse, 0.0)
    lp_tol = torch.where(ok, lse_tol + DZ + 4 * U * (top + lse.abs()), 0.0)
    _bounded(got.logp, logp, lp_tol, "logp")
    b = torch.where(ok, dlogp.double(), 0.0) if uses != "lse" else torch.zeros(N, device=dev, dtype=torch.float64)
    a = (dlse.double() if uses != "logp" else 0.0) - b
    p = torch.exp(z - lse[:, None])
    dz = p * a[:, None]
    hit = torch.zeros_like(dz)
    hit.scatter_add_(1, t.clamp(0, V - 1)[:, None], ok.double()[:, None])
    dz += hit * b[:, None]
    DP = lse_tol + lp_tol + DZ + 12 * U * (top + lse.abs()) + 8 * U
    R = 2.0 ** -24 if wide else 2.0 ** -8
    # (the target's element is (a + b) p + b (1 - p): each within DP of its size, or of p's)
    dz_tol = dz.abs() * R + (p * (a.abs() + 2 * b.abs())[:, None] * DP[:, None] + 4 * U * dz.abs()) * (1 + R)
    for got_, left, right, n, dt, what in ((dx, dz, w64, V, xd, "dx"), (dw, dz.t().contiguous(), x64, N, wd, "dw")):
        ref = left @ right
        mag = left.abs() @ right.abs()
        e = (dz_tol if what == "dx" else dz_tol.t().contiguous()) @ right.abs() + 2 * (n + 16) * U * mag
        _bounded(got_, ref, (e + ref.abs() * _half(dt)) * (1 + 1e-5) + e * _half(dt) * 2 + 1e-35, what)


TYPES = [(BF, BF), (F32, F32), (BF, F32), (F32, BF)]
SHAPES = [(1, 1, 1), (1, 128, 64), (2, 7, 8), (31, 129, 63), (32, 1000, 64), (33, 255, 65), (128, 256, 72), (129, 513, 200),
          (257, 4099, 40), (700, 300, 768), (64, 127, 130), (1023, 1000, 96), (5, 3001, 513)]


@pytest.mark.parametrize("types", TYPES, ids=lambda t: f"{str(t[0])[6:]}-{str(t[1])[6:]}")
@pytest.mark.parametrize("N,V,D", SHAPES)
def test_forward_and_backward(N, V, D, types):
    _check(N, V, D, *types, seed=N + V + D)


@pytest.mark.parametrize("uses", ["logp", "lse"])
def test_one_of_the_outputs(uses):
    _check(150, 700, 136, BF, BF, seed=4, uses=uses)
    _check(150, 700, 136, F32, F32, seed=5, uses=uses)


@pytest.mark.parametrize("N,V,D,xd", [(4100, 4100, 72, BF), (4100, 4100, 72, F32), (22100, 600, 768, BF),
                                      (8192, 8192, 256, BF)])
def test_large_tiles(N, V, D, xd):
    _check(N, V, D, xd, xd, seed=N)


@pytest.mark.parametrize("N,V,D,xd", [(32, 140001, 72, BF), (64, 140001, 72, BF), (65, 70001, 136, BF), (128, 70001, 40, F32),
                                      (32, 70001, 64, F32), (64, 70001, 72, F32), (200, 20001, 96, F32), (500, 40001, 72, F32),
                                      (16, 1100001, 32, F32), (16, 1100001, 32, BF)])
def test_few_rows_of_many_tokens(N, V, D, xd):
    """Several tiles of the vocabulary one after another in a workgroup."""
    _check(N, V, D, xd, xd, seed=N)


@pytest.mark.parametrize("N,V,D,xd", [(22100, 13000, 64, BF), (8000, 13001, 40, F32)])
def test_several_pieces_of_the_vocabulary(N, V, D, xd):
    _check(N, V, D, xd, xd, seed=V)


def test_gradient_against_differences():
    """Directional derivatives against central differences of the definition in 64 bits
    (step 1e-5: truncation about 1e-10, rounding 1e-16 |L| / 1e-5)."""
    import nsa_lm
    dev = require_gpu()
    N, V, D = 20, 37, 24
    x, w, t, dlogp, dlse = _data(N, V, D, F32, F32, seed=8)
    xs, ws = x.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    got = nsa_lm.linear_logprobs(xs, ws, t.to(dev))
    grads = torch.autograd.grad((got.logp, got.lse), (xs, ws), (dlogp.to(dev), dlse.to(dev)))
    ok = (t >= 0) & (t < V)

    def loss(xx, ww):
        z = xx @ ww.t()
        s = torch.logsumexp(z, 1)
        lp = torch.where(ok, z.gather(1, t.clamp(0, V - 1)[:, None])[:, 0] - s, 0.0)
        return float((lp * dlogp.double()).sum() + (s * dlse.double()).sum())
    at = [x.double(), w.double()]
    g = torch.Generator().manual_seed(1)
    for k, grad in enumerate(grads):
        v = torch.randn(grad.shape, generator=g).double()
        hi, lo, e = list(at), list(at), 1e-5
        hi[k], lo[k] = at[k] + e * v, at[k] - e * v
        fd = (loss(*hi) - loss(*lo)) / (2 * e)
        # every product of the gradient within 2 (D + V + N + 300) u of the largest terms, summed over all
        mag = float(grad.abs().max()) * float(v.abs().sum()) * (1 + float(at[0].abs().max()))
        assert abs(float((grad.cpu().double() * v).sum()) - fd) <= 2 * (D + V + N + 300) * U * mag + 1e-8


def test_shapes_strides_alignment_and_empty():
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator().manual_seed(0)
    V, D = 300, 64
    x = torch.randn(4, 10, 2 * D, generator=g).to(BF).to(dev)[:, :, 5:5 + D]
    w = torch.randn(D, V, generator=g).to(BF).to(dev).t()
    t = torch.randint(0, V, (4, 10), generator=g).to(dev)
    a = nsa_lm.linear_logprobs(x, w, t.to(torch.int32))
    b = nsa_lm.linear_logprobs(x.reshape(40, D), w.contiguous(), t.view(-1))
    assert a.logp.shape == (4, 10) and torch.equal(a.logp.view(-1), b.logp) and torch.equal(a.lse.view(-1), b.lse)
    flat = torch.empty(V * D + 1, dtype=BF, device=dev)
    off = flat[1:].view(V, D).copy_(w)                   # dense, one element off 16 bytes
    c = nsa_lm.linear_logprobs(x, off, t)
    assert torch.equal(a.lse, c.lse) and torch.equal(a.logp, c.logp)
    xo = torch.empty(40 * D + 1, dtype=BF, device=dev)[1:].view(40, D).copy_(x.reshape(40, D))
    leaves = [[p.detach().requires_grad_() for p in (q, r)] for q, r in ((x.reshape(40, D), w.contiguous()), (xo, off))]
    grads = [torch.autograd.grad(nsa_lm.linear_logprobs(*l, t.view(-1)).logp.sum(), l) for l in leaves]
    assert all(torch.equal(p, q) for p, q in zip(*grads))
    none = nsa_lm.linear_logprobs(x, w)
    assert none.logp is None and torch.equal(none.lse, a.lse)
    one = nsa_lm.linear_logprobs(x[0, 0], w, t[0, 0])
    assert one.lse.shape == () and abs(float(one.lse - a.lse[0, 0])) <= 1e-5
    ws = w.detach().contiguous().requires_grad_()
    e = torch.empty(0, D, dtype=BF, device=dev, requires_grad=True)
    r = nsa_lm.linear_logprobs(e, ws, torch.empty(0, dtype=torch.long, device=dev))
    r.logp.sum().backward()
    assert r.lse.shape == (0,) and not ws.grad.any() and e.grad.shape == (0, D)


def test_one_of_the_gradients():
    import nsa_lm
    dev = require_gpu()
    x, w, t, dlogp, dlse = (a.to(dev) for a in _data(200, 500, 128, BF, BF))
    a = [x.detach().requires_grad_(), w.detach().requires_grad_()]
    r = nsa_lm.linear_logprobs(*a, t)
    both = torch.autograd.grad((r.logp, r.lse), a, (dlogp, dlse))
    for k in range(2):
        a = [x.detach().requires_grad_(k == 0), w.detach().requires_grad_(k == 1)]
        r = nsa_lm.linear_logprobs(*a, t)
        g, = torch.autograd.grad((r.logp, r.lse), a[k], (dlogp, dlse))
        assert torch.equal(g, both[k])


def test_ignored_rows_sure_rows_and_nan():
    import nsa_lm
    dev = require_gpu()
    N, V, D = 40, 200, 32
    x, w, t, _, _ = _data(N, V, D, F32, F32, ignored=False)
    x[0] = w[t[0]] * 40                                   # a row that is all but sure: logp about 0
    x[1] = 0                                              # uniform
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    t[4] = -100
    x, w, t = x.to(dev), w.to(dev), t.to(dev)
    r = nsa_lm.linear_logprobs(x, w, t)
    assert r.logp[2].isnan() and r.lse[2].isnan() and r.lse[3].isnan() and r.logp[4] == 0
    assert abs(float(r.lse[1]) - float(torch.log(torch.tensor(float(V))))) <= 1e-5
    assert int(r.lse.isnan().sum()) == 2
    keep = torch.ones(N, dtype=torch.bool)
    keep[2] = keep[3] = False
    xs, ws = x[keep].requires_grad_(), w.detach().requires_grad_()
    t2 = t[keep]
    r = nsa_lm.linear_logprobs(xs, ws, t2)
    dx, dw = torch.autograd.grad(-r.logp.sum(), (xs, ws))
    assert not dx[2].any()                                # (row 4 of x)
    z = xs.detach().double() @ w.double().t()
    p = torch.softmax(z, 1)
    ok = t2 >= 0
    p[ok, t2[ok]] -= 1
    p[~ok] = 0
    # the sure row's gradient keeps its digits: 1 - p comes from logp itself
    ref = p @ w.double()
    assert torch.allclose(dx.double(), ref, rtol=1e-4, atol=1e-5)
    lp = r.logp.detach().double()[0]
    assert float(dx[0].double().norm()) <= 2 * float(-torch.expm1(lp)) * float(w.double().norm(dim=1).max()) + 1e-12


def test_same_bits_on_every_run_and_stream():
    import nsa_lm
    dev = require_gpu()
    sets = [[a.to(dev) for a in _data(2500, 3000, 256, BF, BF, seed=s)] for s in range(2)]

    def once(x, w, t, dlogp, dlse):
        a = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        r = nsa_lm.linear_logprobs(*a, t)
        return (r.logp.detach(), r.lse.detach(), *torch.autograd.grad((r.logp, r.lse), a, (dlogp, dlse)))
    want = [once(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(once(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            for a, b in zip(o, want[i]):
                assert torch.equal(a, b)


def test_captured_and_replayed():
    import nsa_lm
    dev = require_gpu()
    x, w, t, dlogp, dlse = (a.to(dev) for a in _data(300, 900, 200, BF, BF))
    a = [x.clone().requires_grad_(), w.clone().requires_grad_()]

    def once():
        r = nsa_lm.linear_logprobs(*a, t)
        return (r.logp.detach(), r.lse.detach(), *torch.autograd.grad((r.logp, r.lse), a, (dlogp, dlse)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for k in range(3):
        with torch.no_grad():
            a[0].copy_(x * (1 - 0.2 * k))
            t.copy_(t.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, once()):
            assert torch.equal(p, q)


def test_second_derivatives_and_refusals():
    import nsa_lm
    import torch.autograd.forward_ad as fwAD
    dev = require_gpu()
    x, w, t, _, _ = (a.to(dev) for a in _data(6, 50, 32, F32, F32))
    xs = x.detach().requires_grad_()
    r = nsa_lm.linear_logprobs(xs, w, t)
    g, = torch.autograd.grad(r.lse.sum(), xs, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    for bad in ((x.cpu(), w, t), (x, w.cpu(), t), (x.half(), w, t), (x, w.double(), t), (x[:, :16], w, t),
                (x, w[:, 0], t), (x, w, t[:3]), (x, w, t.float()), (x, w, t.cpu())):
        with pytest.raises(AssertionError):
            nsa_lm.linear_logprobs(*bad)
    with fwAD.dual_level(), pytest.raises(AssertionError):
        nsa_lm.linear_logprobs(fwAD.make_dual(x, torch.ones_like(x)), w, t)
