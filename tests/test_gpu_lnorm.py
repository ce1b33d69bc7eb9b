"""nsa_lm.add_layer_norm against the definition in 64 bits.

Tolerances, u = 2^-24 (half a float32 step, relative), A = mean |h| of a row:
* the mean: at most CHAIN additions, so |error| <= (CHAIN + 1) u A; a centred
  element is off by that and u of itself.
* the variance: the mean's error adds nothing to first order (centred elements sum
  to 0); its sum of squares has at most CHAIN additions of terms within 3 u, so that
  rstd is within (CHAIN / 2 + 6) u of itself.
* n = (h - mean) rstd is then within E = |n| (CHAIN / 2 + 8) u + rstd (CHAIN + 3) u A,
  y within |w| E + 2 u (|n w| + |b|), and half a step of its dtype.
* gradients: dh = dh_out + rstd (g - mean g - n mean(g n)) term by term; dw and db
  are sums of `rows` products, in at most `rows` additions.
"""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def _chain(D):
    runs = max(4, -(-D // 8192)) if D > 2048 else -(-D // 512)
    return 8 * runs + 6 + 16


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(rows, D, xd, rd, wd, seed=0, off=True):
    g = torch.Generator().manual_seed(seed)
    chan = torch.exp(0.5 * torch.randn(D, generator=g))
    chan[:: max(1, D // 3)] *= 20
    res = torch.randn(rows, D, generator=g) * chan
    if off:   # rows far off zero, where a sum of squares would lose the variance
        res += 50 * torch.randn(rows, 1, generator=g)
    x = torch.randn(rows, D, generator=g).to(xd)
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(wd)
    b = torch.randn(D, generator=g).to(wd)
    return x, res.to(rd), w, b


class Ref:
    """The definition in 64 bits, and the bounds of the module's docstring."""

    def __init__(self, h, w, b, eps, yd):
        C = _chain(h.shape[1])
        h, self.w = h.double(), w.double()
        b = torch.zeros_like(self.w) if b is None else b.double()
        d = h - h.mean(1, keepdim=True)
        self.rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
        self.n = d * self.rstd
        self.C = C
        self.E = self.n.abs() * (C / 2 + 8) * U + self.rstd * (C + 3) * U * h.abs().mean(1, keepdim=True)
        nw = self.n * self.w
        self.y = nw + b
        t = self.w.abs() * self.E + 2 * U * (nw.abs() + b.abs())
        self.y_tol = (t + self.y.abs() * _half(yd)) * (1 + 1e-6) + t * _half(yd) + 1e-30

    def grads(self, dy, dh, xd):
        C, n, rstd, E = self.C, self.n, self.rstd, self.E
        dy = dy.double()
        g = dy * self.w
        s1, s2 = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
        m1, m2 = g.abs().mean(1, keepdim=True), (g * n).abs().mean(1, keepdim=True)
        out = rstd * (g - s1 - n * s2)
        t = rstd * (g.abs() * 4 * U + (C + 4) * U * m1 +
                    (n.abs() + E) * ((C + 5) * U * m2 + (g.abs() * E).mean(1, keepdim=True)) + E * s2.abs())
        t = t + (C / 2 + 8) * U * rstd * (g.abs() + m1 + n.abs() * m2)
        if dh is not None:
            out = out + dh.double()
            t = t + 2 * U * (dh.double().abs() + out.abs())
        return out, t, dy


def _close(got, ref, err, dtype):
    bad = (got.detach().cpu().double() - ref).abs() - ((err + ref.abs() * _half(dtype)) * (1 + 1e-6) +
                                                       err * _half(dtype) * 2 + 1e-30)
    assert (bad <= 0).all(), float(bad.max())


TYPES = [(BF, BF, BF, BF), (BF, F32, F32, BF), (F32, F32, F32, F32), (F32, BF, F32, F32), (BF, BF, F32, F32),
         (F32, F32, BF, BF)]
SHAPES = [(1, 1), (3, 7), (5, 8), (2, 64), (1, 511), (300, 512), (257, 768), (9, 1001), (700, 1537), (4, 2048),
          (600, 2049), (3, 4095), (300, 4104), (300, 8192), (2, 8200), (260, 9001), (2, 16384), (260, 20001),
          (2, 32768), (3, 33001), (1003, 64), (517, 128), (301, 250), (5000, 30)]


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x)[6:] for x in t))
@pytest.mark.parametrize("rows,D", SHAPES)
def test_forward_and_backward(rows, D, types):
    import nsa_lm
    dev = require_gpu()
    xd, rd, wd, yd = types
    eps = 1e-5
    x, res, w, b = _inputs(rows, D, xd, rd, wd, seed=rows * 31 + D)
    g = torch.Generator().manual_seed(D)
    dy, dh = torch.randn(rows, D, generator=g).to(yd), torch.randn(rows, D, generator=g).to(rd)
    xs = [t.to(dev).requires_grad_() for t in (x, res, w, b)]
    y, h = nsa_lm.add_layer_norm(*xs, eps=eps, out_dtype=yd)
    dx, dr, dw, db = torch.autograd.grad((y, h), xs, (dy.to(dev), dh.to(dev)))
    assert (y.dtype, h.dtype, dx.dtype, dr.dtype, dw.dtype, db.dtype) == (yd, rd, xd, rd, wd, wd)
    h_ref = (x.float() + res.float()).to(rd)
    assert torch.equal(h.cpu(), h_ref)
    ref = Ref(h_ref, w, b, eps, yd)
    err = (y.detach().cpu().double() - ref.y).abs()
    assert (err <= ref.y_tol).all(), float((err - ref.y_tol).max())
    out, t, dy64 = ref.grads(dy, dh, xd)
    _close(dx, out, t, xd)
    _close(dr, out, t, rd)
    prod = dy64 * ref.n
    _close(dw, prod.sum(0), prod.abs().sum(0) * (rows + 4) * U + (dy64.abs() * ref.E).sum(0), wd)
    _close(db, dy64.sum(0), dy64.abs().sum(0) * (rows + 2) * U, wd)


def test_gradient_against_differences():
    """The kernels' directional derivative against central differences of the
    definition in 64 bits (step 1e-6: truncation about 1e-12, the difference's
    rounding 1e-16 |L| / 1e-6, both far below float32)."""
    import nsa_lm
    dev = require_gpu()
    rows, D, eps = 6, 77, 1e-6
    x, res, w, b = _inputs(rows, D, F32, F32, F32, seed=3, off=False)
    g = torch.Generator().manual_seed(9)
    dy, dh = torch.randn(rows, D, generator=g), torch.randn(rows, D, generator=g)
    xs = [t.to(dev).requires_grad_() for t in (x, res, w, b)]
    y, h = nsa_lm.add_layer_norm(*xs, eps=eps)
    grads = torch.autograd.grad((y, h), xs, (dy.to(dev), dh.to(dev)))
    at = [h.detach().cpu().double(), w.double(), b.double()]

    def loss(hh, ww, bb):
        d = hh - hh.mean(1, keepdim=True)
        yy = d / torch.sqrt((d * d).mean(1, keepdim=True) + eps) * ww + bb
        return float((yy * dy.double()).sum() + (hh * dh.double()).sum())
    for k, grad in enumerate(grads):
        v = torch.randn(grad.shape, generator=g).double()
        e, which = 1e-6, max(0, k - 1)
        hi, lo = list(at), list(at)
        hi[which], lo[which] = at[which] + e * v, at[which] - e * v
        fd = (loss(*hi) - loss(*lo)) / (2 * e)
        got = float((grad.cpu().double() * v).sum())
        ref = Ref(h.detach().cpu(), w, b, eps, F32)
        out, t, dy64 = ref.grads(dy, dh, F32)
        if k < 2:
            err = float(((t + out.abs() * U) * v.abs()).sum())
        else:
            n = ref.n if k == 2 else torch.ones_like(ref.n)
            err = float((((dy64 * n).abs() * (rows + 6) * U + (dy64.abs() * ref.E)).sum(0) * v.abs()).sum())
        scale = float((at[0].abs() * dh.abs()).sum() + (ref.y.abs() * dy.abs()).sum())
        assert abs(got - fd) <= 2 * err + 1e-9 * scale, (k, got, fd)


def test_without_residual_or_bias_and_partial_uses():
    import nsa_lm
    dev = require_gpu()
    x, r, w, b = _inputs(37, 300, F32, F32, F32, seed=1)
    for res in (False, True):
        for bias in (False, True):
            for use_h in (False, True):
                xs = [x.to(dev).requires_grad_(), r.to(dev).requires_grad_() if res else None,
                      w.to(dev).requires_grad_(), b.to(dev).requires_grad_() if bias else None]
                y, h = nsa_lm.add_layer_norm(*xs, eps=1e-5)
                assert res or h is xs[0]
                leaves = [t for t in xs if t is not None]
                g = torch.autograd.grad(y.sum() + (h.sum() if use_h else 0), leaves)
                hr = (x + r if res else x)
                ref = Ref(hr, w, b if bias else None, 1e-5, F32)
                assert ((y.detach().cpu().double() - ref.y).abs() <= ref.y_tol).all()
                out, t, dy = ref.grads(torch.ones(37, 300), torch.ones(37, 300) if use_h else None, F32)
                _close(g[0], out, t + 2 * U * (out.abs() + 1), F32)
                if res:
                    assert torch.equal(g[0], g[1])
                _close(g[1 + res], ref.n.sum(0), ref.n.abs().sum(0) * 50 * U + ref.E.sum(0), F32)
                if bias:
                    assert torch.equal(g[-1].cpu(), torch.full((300,), 37.0))
    a, c, d, e = (t.to(dev).requires_grad_() for t in _inputs(5, 64, BF, F32, F32))
    _, h = nsa_lm.add_layer_norm(a, c, d, e)
    h.sum().backward()
    assert torch.equal(a.grad, torch.ones_like(a)) and torch.equal(c.grad, torch.ones_like(c))
    assert not (d.grad is not None and d.grad.any()) and not (e.grad is not None and e.grad.any())
    # one of the parameters alone
    y, _ = nsa_lm.add_layer_norm(a, c, d, e)
    all4 = torch.autograd.grad(y, (a, c, d, e), torch.ones_like(y))
    for k in range(4):
        ts = [t.detach().requires_grad_(i == k) for i, t in enumerate((a, c, d, e))]
        y, _ = nsa_lm.add_layer_norm(*ts)
        g, = torch.autograd.grad(y, ts[k], torch.ones_like(y))
        assert torch.equal(g, all4[k])


def test_equal_elements_infinities_and_nan():
    import nsa_lm
    dev = require_gpu()
    D = 200
    x = torch.randn(6, D, generator=torch.Generator().manual_seed(0))
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    x[3] = 3.0
    x[4] = torch.linspace(-1, 1, D) * 2.0 ** -70
    x, w, b = x.to(dev), torch.ones(D, device=dev), torch.full((D,), 0.5, device=dev)
    y, _ = nsa_lm.add_layer_norm(x, None, w, b, eps=1e-6)
    # (200 equal elements sum exactly, and 1 / 200 is off by half a step: the mean by one)
    assert torch.equal(y[0], b) and (y[3] - 0.5).abs().max() <= 3 * 2.0 ** -23 * 1e3
    assert y[1].isnan().all() and y[2].isnan().all() and torch.isfinite(y[[0, 3, 4, 5]]).all()
    g = torch.randn(6, D, device=dev)
    xr = x.clone().requires_grad_()
    dx, = torch.autograd.grad(nsa_lm.add_layer_norm(xr, None, w, b, eps=1e-6)[0], xr, g)
    assert torch.isfinite(dx[[0, 3, 4, 5]]).all() and dx[1].isnan().all() and dx[2].isnan().all()


def test_strides_alignment_and_empty():
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator().manual_seed(4)
    base = torch.randn(8, 3, 200, generator=g).to(BF).to(dev)
    w, b = torch.randn(200, generator=g).to(dev)[::2], torch.randn(100, generator=g).to(dev)
    x = base[:, 1, 1:101]                                # strided rows, odd offset
    r = base.transpose(0, 1)[0, :, 100:]
    y, h = nsa_lm.add_layer_norm(x, r, w, b)
    y2, h2 = nsa_lm.add_layer_norm(x.clone(), r.clone(), w.clone(), b)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    flat = torch.randn(100 * 5 + 1, generator=g).to(BF).to(dev)
    off = flat[1:].view(5, 100)                          # dense, one element off any alignment
    assert torch.equal(nsa_lm.add_layer_norm(off, None, w, b)[0], nsa_lm.add_layer_norm(off.clone(), None, w, b)[0])
    xs = [torch.empty(0, 7, 64, device=dev, requires_grad=True), torch.empty(0, 7, 64, device=dev, requires_grad=True),
          torch.ones(64, device=dev, requires_grad=True), torch.ones(64, device=dev, requires_grad=True)]
    y, h = nsa_lm.add_layer_norm(*xs)
    (y.sum() + h.sum()).backward()
    assert y.shape == (0, 7, 64) and not xs[2].grad.any() and not xs[3].grad.any()
    assert xs[0].grad.shape == (0, 7, 64)
    # a gradient that comes expanded (of a sum) and one that comes transposed
    t = [torch.randn(4, 64, device=dev, requires_grad=True), torch.ones(64, device=dev, requires_grad=True)]
    v = torch.randn(64, 4, device=dev)
    a = torch.autograd.grad(nsa_lm.add_layer_norm(t[0], None, t[1])[0], t, v.t())
    c = torch.autograd.grad(nsa_lm.add_layer_norm(t[0], None, t[1])[0], t, v.t().contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_same_bits_on_every_run_and_stream():
    import nsa_lm
    dev = require_gpu()
    x, r, w, b = (t.to(dev) for t in _inputs(5000, 768, BF, F32, F32))
    dy = torch.randn(5000, 768, device=dev).to(BF)

    def once():
        a = [t.detach().requires_grad_() for t in (x, r, w, b)]
        y, h = nsa_lm.add_layer_norm(*a, eps=1e-5, out_dtype=BF)
        return (y, h, *torch.autograd.grad((y, h), a, (dy, r)))
    first = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(once())
    torch.cuda.synchronize()
    for again in got:
        for p, q in zip(first, again):
            assert torch.equal(p, q)


def test_captured_and_replayed():
    import nsa_lm
    dev = require_gpu()
    x, r, w, b = (t.to(dev) for t in _inputs(33, 768, BF, F32, F32))
    dy, dh = torch.randn(33, 768, device=dev).to(BF), torch.randn(33, 768, device=dev)
    a = [t.detach().clone().requires_grad_() for t in (x, r, w, b)]

    def once():
        y, h = nsa_lm.add_layer_norm(*a, eps=1e-5, out_dtype=BF)
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), a, (dy, dh)))
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
            a[0].copy_(x * (k + 1))
            a[1].copy_(r + k)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, once()):
            assert torch.equal(p, q)


def test_more_rows_than_one_launch():
    """2^21 rows go to one launch; the rows around the seam and the last ones."""
    import nsa_lm
    dev = require_gpu()
    rows, D = (1 << 21) + 3, 5
    g = torch.Generator(device=dev).manual_seed(0)
    x, r = (torch.randn(rows, D, generator=g, device=dev) for _ in range(2))
    w = torch.rand(D, generator=g, device=dev) + 0.5
    dy = torch.randn(rows, D, generator=g, device=dev)
    xs = [t.requires_grad_() for t in (x, r, w)]
    y, h = nsa_lm.add_layer_norm(*xs, eps=1e-5)
    dx, = torch.autograd.grad(y, x, dy)
    for at in (slice(0, 4), slice((1 << 21) - 3, rows)):
        hh = (x[at] + r[at]).detach()
        assert torch.equal(h[at], hh)
        ref = Ref(hh.cpu(), w.detach().cpu(), None, 1e-5, F32)
        assert ((y[at].detach().cpu().double() - ref.y).abs() <= ref.y_tol).all()
        out, t, _ = ref.grads(dy[at].cpu(), None, F32)
        _close(dx[at], out, t, F32)


def test_second_derivatives_are_refused():
    import nsa_lm
    dev = require_gpu()
    x = torch.randn(7, 40, device=dev, requires_grad=True)
    w = torch.rand(40, device=dev, requires_grad=True)
    y, h = nsa_lm.add_layer_norm(x, x, w)
    assert torch.equal(h, x + x)
    y, _ = nsa_lm.add_layer_norm(x, None, w)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals():
    import nsa_lm
    import torch.autograd.forward_ad as fwAD
    dev = require_gpu()
    x, r, w, b = (t.to(dev) for t in _inputs(4, 64, BF, F32, F32))
    for bad in [(x.cpu(), r, w, b), (x.half(), r, w, b), (x, r[:, :32], w, b), (x, r, w[:32], b), (x, r[:2], w, b),
                (x, r.double(), w, b), (x, r, w.cpu(), b), (x, r, w, b[:32]), (x, r, w, b.to(BF)), (x, r, w, b.cpu())]:
        with pytest.raises(AssertionError):
            nsa_lm.add_layer_norm(*bad)
    with pytest.raises(AssertionError):
        nsa_lm.add_layer_norm(x, r, w, b, eps=-1.0)
    with pytest.raises(AssertionError):
        nsa_lm.add_layer_norm(x, r, w, b, out_dtype=torch.float16)
    with fwAD.dual_level(), pytest.raises(AssertionError):
        nsa_lm.add_layer_norm(x, r, w, fwAD.make_dual(b, torch.ones_like(b)))
