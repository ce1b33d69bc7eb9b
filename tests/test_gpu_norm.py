"""nsa_lm.add_rms_norm / add_rms_norm_q8 against the definition in 64 bits.

Tolerances, u = 2^-24 (half a float32 step, relative):
* h is one float32 addition rounded to its dtype: equal bits to torch's.
* y: the sum of squares takes at most CHAIN additions of positive terms in a
  row, so its relative error is at most CHAIN u, halved by the root; the mean's
  product, eps, root, division and the two products of y add 7 u.  Then y's
  own rounding, half a step of its dtype.
* gradients: every term of dh = dh_out + rstd (g - n mean(g n)) is formed within
  (2 CHAIN + 12) u of its magnitude; dw is a sum of `rows` products, each within
  (CHAIN + 9) u, in at most `rows` additions.
CHAIN: 8 elements x runs of a thread + 6 steps over the wave + 16 waves.
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


def _inputs(rows, D, xd, rd, wd, seed=0):
    g = torch.Generator().manual_seed(seed)
    chan = torch.exp(0.5 * torch.randn(D, generator=g))
    chan[:: max(1, D // 3)] *= 20
    res = (torch.randn(rows, D, generator=g) * chan).to(rd)
    x = torch.randn(rows, D, generator=g).to(xd)
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(wd)
    return x, res, w


def _norm64(h, w, eps):
    h, w = h.double(), w.double()
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w


def _tol(ref, dtype, rel):
    return ref.abs() * (_half(dtype) + rel) * (1 + 1e-6) + 1e-30


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
    x, res, w = _inputs(rows, D, xd, rd, wd, seed=rows * 31 + D)
    g = torch.Generator().manual_seed(D)
    dy, dh = torch.randn(rows, D, generator=g).to(yd), torch.randn(rows, D, generator=g).to(rd)
    xs = [t.to(dev).requires_grad_() for t in (x, res, w)]
    y, h = nsa_lm.add_rms_norm(*xs, eps=eps, out_dtype=yd)
    dx, dr, dw = torch.autograd.grad((y, h), xs, (dy.to(dev), dh.to(dev)))
    assert (y.dtype, h.dtype, dx.dtype, dr.dtype, dw.dtype) == (yd, rd, xd, rd, wd)
    h_ref = (x.float() + res.float()).to(rd)
    assert torch.equal(h.cpu(), h_ref)
    C = _chain(D)
    y_ref = _norm64(h_ref, w, eps)
    err = (y.cpu().double() - y_ref).abs()
    assert (err <= _tol(y_ref, yd, (C / 2 + 7) * U)).all(), float(err.max())
    # gradients in 64 bits, from the formula
    h64, w64, dy64 = h_ref.double(), w.double(), dy.double()
    rstd = 1 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + eps)
    n, gg = h64 * rstd, dy64 * w64
    ref = dh.double() + rstd * (gg - n * (gg * n).mean(1, keepdim=True))
    mag = dh.double().abs() + rstd * (gg.abs() + n.abs() * (gg * n).abs().mean(1, keepdim=True))
    for got, dt in ((dx, xd), (dr, rd)):
        err = (got.cpu().double() - ref).abs()
        assert (err <= ref.abs() * _half(dt) * (1 + 1e-6) + mag * (2 * C + 12) * U * (1 + _half(dt) * 4)).all(), \
            float(err.max())
    dw_ref = (dy64 * n).sum(0)
    err = (dw.cpu().double() - dw_ref).abs()
    assert (err <= dw_ref.abs() * _half(wd) * (1 + 1e-6) + (dy64 * n).abs().sum(0) * (rows + C + 9) * U *
            (1 + _half(wd) * 4)).all(), float(err.max())


def test_gradient_against_differences():
    """The kernels' directional derivative against central differences of the
    definition in 64 bits (step 1e-6: the truncation is about 1e-12, the
    rounding of the difference 1e-16 |L| / 1e-6, both far below float32)."""
    import nsa_lm
    dev = require_gpu()
    rows, D, eps = 6, 77, 1e-6
    x, res, w = _inputs(rows, D, F32, F32, F32, seed=3)
    g = torch.Generator().manual_seed(9)
    dy, dh = torch.randn(rows, D, generator=g), torch.randn(rows, D, generator=g)
    xs = [t.to(dev).requires_grad_() for t in (x, res, w)]
    y, h = nsa_lm.add_rms_norm(*xs, eps=eps)
    grads = torch.autograd.grad((y, h), xs, (dy.to(dev), dh.to(dev)))
    h0, w0 = h.detach().cpu().double(), w.double()

    def loss(hh, ww):
        return float((_norm64(hh, ww, eps) * dy.double()).sum() + (hh * dh.double()).sum())
    for k, grad in enumerate(grads):
        v = torch.randn(grad.shape, generator=g).double()
        e = 1e-6
        if k < 2:
            fd = (loss(h0 + e * v, w0) - loss(h0 - e * v, w0)) / (2 * e)
        else:
            fd = (loss(h0, w0 + e * v) - loss(h0, w0 - e * v)) / (2 * e)
        got = float((grad.cpu().double() * v).sum())
        # every product of grad and v within the gradients' own bound, and the difference's rounding
        mag = float((grad.cpu().double().abs() * v.abs()).sum())
        scale = float((h0.abs() * dh.abs()).sum() + (_norm64(h0, w0, eps).abs() * dy.abs()).sum())
        assert abs(got - fd) <= mag * 20 * (2 * _chain(D) + 12) * U + 1e-9 * scale


def test_without_residual_and_partial_uses():
    import nsa_lm
    dev = require_gpu()
    x, _, w = _inputs(37, 300, BF, BF, F32, seed=1)
    for use_h in (False, True):
        xs = [x.to(dev).requires_grad_(), w.to(dev).requires_grad_()]
        y, h = nsa_lm.add_rms_norm(xs[0], None, xs[1], eps=1e-5, out_dtype=F32)
        assert h is xs[0]
        r = [t.detach().double().requires_grad_() for t in xs]
        ref = _norm64_grad(r[0], r[1])
        (y.sum() + (h.float().sum() if use_h else 0)).backward()
        (ref.sum() + (r[0].sum() if use_h else 0)).backward()
        for a, b in zip(xs, r):
            # bf16 rounding of the gradient, and of its sum with h's
            assert torch.allclose(a.grad.double(), b.grad, rtol=2 ** -7, atol=float(b.grad.abs().max()) * 2 ** -8)
    # only the sum is used, or only the weight needs a gradient
    a, b, c = (t.to(dev).requires_grad_() for t in _inputs(5, 64, BF, F32, F32))
    _, h = nsa_lm.add_rms_norm(a, b, c)
    h.sum().backward()
    assert torch.equal(a.grad, torch.ones_like(a)) and torch.equal(b.grad, torch.ones_like(b))
    assert c.grad is None or not c.grad.any()
    y, _ = nsa_lm.add_rms_norm(a.detach(), b.detach(), c)
    gw, = torch.autograd.grad(y, c, torch.ones_like(y))
    y2, _ = nsa_lm.add_rms_norm(a, b, c.detach())
    gx, = torch.autograd.grad(y2, a, torch.ones_like(y2))
    y3, _ = nsa_lm.add_rms_norm(a, b, c)
    gx3, gw3 = torch.autograd.grad(y3, (a, c), torch.ones_like(y3))
    assert torch.equal(gw, gw3) and torch.equal(gx, gx3)


def _norm64_grad(h, w):
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5) * w


@pytest.mark.parametrize("rows,D", [(1, 1), (4, 9), (33, 768), (300, 2050), (5, 8192), (2, 30001), (3, 40001)])
@pytest.mark.parametrize("res", [True, False])
def test_rows_in_8_bits(rows, D, res):
    import nsa_lm
    dev = require_gpu()
    x, r, w = _inputs(rows, D, BF, BF, F32, seed=D)
    r = r if res else None
    q, s, h = nsa_lm.add_rms_norm_q8(x.to(dev), None if r is None else r.to(dev), w.to(dev), eps=1e-5)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == F32 and s.shape == (rows,)
    h_ref = x if r is None else (x.float() + r.float()).to(BF)
    assert torch.equal(h.cpu(), h_ref)
    y = _norm64(h_ref, w, 1e-5)
    rel = (_chain(D) / 2 + 7) * U
    s_ref = y.abs().amax(1).clamp(min=2.0 ** -100) / 448
    assert ((s.cpu().double() - s_ref).abs() <= s_ref * (rel + 2 * U)).all()
    # the value that the byte stands for: half a step of e4m3, 2^-4 of the value and
    # 2^-10 below the normal numbers (2^-6); before that y 448 / amax in float32
    v = y / s_ref[:, None]
    err = (q.cpu().float().double() - v).abs()
    assert (err <= torch.maximum(v.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10)) * (1 + 1e-5) +
            v.abs() * (2 * rel + 4 * U)).all(), float(err.max())


def test_rows_of_zeros_infinities_and_nan():
    import nsa_lm
    dev = require_gpu()
    D = 200
    x = torch.randn(6, D, generator=torch.Generator().manual_seed(0))
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    x[3] = torch.finfo(BF).min
    x[4] = 2.0 ** -130
    x = x.to(BF).to(dev)
    r, w = torch.zeros_like(x), torch.ones(D, device=dev)
    y, h = nsa_lm.add_rms_norm(x, r, w, eps=1e-6, out_dtype=F32)
    assert not y[0].any() and not h[0].any()
    assert y[1, 3].isnan() and not y[1, :3].any() and y[2].isnan().all()
    # squares past float32's range: the mean is infinite and the row 0
    assert not y[3].any()
    ref = torch.nn.functional.rms_norm(x.float(), (D,), w, 1e-6)
    assert torch.equal(y.isnan(), ref.isnan())
    q, s, _ = nsa_lm.add_rms_norm_q8(x, r, w, eps=1e-6)
    assert not q[0].float().any() and s[0] == 2.0 ** -100 / 448
    assert s[1].isnan() and s[2].isnan() and torch.isfinite(s[[0, 3, 4, 5]]).all()
    assert torch.isfinite(q[5].float()).all() and q[5].float().abs().max() == 448


def test_strides_alignment_and_empty():
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator().manual_seed(4)
    base = torch.randn(8, 3, 200, generator=g).to(BF).to(dev)
    w = torch.randn(100, generator=g).to(dev)
    x = base[:, 1, 1:101]                                # strided rows, odd offset
    r = base.transpose(0, 1)[0, :, 100:]
    y, h = nsa_lm.add_rms_norm(x, r, w, eps=1e-5)
    y2, h2 = nsa_lm.add_rms_norm(x.clone(), r.clone(), w, eps=1e-5)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    flat = torch.randn(100 * 5 + 1, generator=g).to(BF).to(dev)
    off = flat[1:].view(5, 100)                          # dense, one element off any alignment
    assert torch.equal(nsa_lm.add_rms_norm(off, None, w)[0], nsa_lm.add_rms_norm(off.clone(), None, w)[0])
    xs = [torch.empty(0, 7, 64, device=dev, requires_grad=True), torch.empty(0, 7, 64, device=dev, requires_grad=True),
          torch.ones(64, device=dev, requires_grad=True)]
    y, h = nsa_lm.add_rms_norm(*xs)
    (y.sum() + h.sum()).backward()
    assert y.shape == (0, 7, 64) and not xs[2].grad.any() and xs[0].grad.shape == (0, 7, 64)


def test_same_bits_on_every_run_and_stream():
    import nsa_lm
    dev = require_gpu()
    x, r, w = (t.to(dev) for t in _inputs(5000, 768, BF, F32, F32))
    dy = torch.randn(5000, 768, device=dev).to(BF)

    def once():
        a = [t.detach().requires_grad_() for t in (x, r, w)]
        y, h = nsa_lm.add_rms_norm(*a, eps=1e-5, out_dtype=BF)
        return (y, h, *torch.autograd.grad((y, h), a, (dy, r)))
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_captured_and_replayed():
    import nsa_lm
    dev = require_gpu()
    x, r, w = (t.to(dev) for t in _inputs(33, 768, BF, F32, F32))
    dy, dh = torch.randn(33, 768, device=dev).to(BF), torch.randn(33, 768, device=dev)
    a = [t.detach().clone().requires_grad_() for t in (x, r, w)]

    def once():
        y, h = nsa_lm.add_rms_norm(*a, eps=1e-5, out_dtype=BF)
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), a, (dy, dh)),
                *nsa_lm.add_rms_norm_q8(a[0].detach(), a[1].detach(), a[2].detach(), eps=1e-5)[:2])
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
        want = once()
        for p, q in zip(out, want):
            assert torch.equal(p.float() if p.dtype == torch.float8_e4m3fn else p,
                               q.float() if q.dtype == torch.float8_e4m3fn else q)


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
    y, h = nsa_lm.add_rms_norm(*xs, eps=1e-5)
    q, s, _ = nsa_lm.add_rms_norm_q8(x.detach(), r.detach(), w.detach(), eps=1e-5)
    dx, = torch.autograd.grad(y, x, dy)
    C = _chain(D)
    for at in (slice(0, 4), slice((1 << 21) - 3, rows)):
        hh = (x[at] + r[at]).detach()
        assert torch.equal(h[at], hh)
        ref = _norm64(hh, w.detach(), 1e-5)
        assert ((y[at].double() - ref).abs() <= _tol(ref, F32, (C / 2 + 7) * U)).all()
        assert ((s[at].double() * 448 - ref.abs().amax(1)).abs() <= ref.abs().amax(1) * ((C / 2 + 9) * U)).all()
        h64, g64 = hh.double(), dy[at].double() * w.detach().double()
        rstd = 1 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + 1e-5)
        n = h64 * rstd
        d = rstd * (g64 - n * (g64 * n).mean(1, keepdim=True))
        mag = rstd * (g64.abs() + n.abs() * (g64 * n).abs().mean(1, keepdim=True))
        assert ((dx[at].double() - d).abs() <= mag * (2 * C + 14) * U).all()


def test_one_tensor_twice_and_second_derivatives():
    import nsa_lm
    dev = require_gpu()
    x = torch.randn(7, 40, device=dev, requires_grad=True)
    w = torch.rand(40, device=dev, requires_grad=True)
    y, h = nsa_lm.add_rms_norm(x, x, w, eps=1e-5)
    assert torch.equal(h, x + x)
    gx, = torch.autograd.grad((y, h), x, (torch.ones_like(y), torch.ones_like(h)))
    a, b = x.detach().clone().requires_grad_(), x.detach().clone().requires_grad_()
    y2, h2 = nsa_lm.add_rms_norm(a, b, w.detach(), eps=1e-5)
    ga, gb = torch.autograd.grad((y2, h2), (a, b), (torch.ones_like(y), torch.ones_like(h)))
    assert torch.equal(ga, gb) and torch.equal(gx, ga + gb)
    y, _ = nsa_lm.add_rms_norm(x, None, w, eps=1e-5)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_two_streams_at_once():
    """Calls in flight on two streams share nothing."""
    import nsa_lm
    dev = require_gpu()
    sets = [tuple(t.to(dev) for t in _inputs(4000, 1024, BF, F32, F32, seed=s)) for s in range(2)]
    dy = torch.randn(4000, 1024, device=dev).to(BF)

    def once(x, r, w):
        a = [t.detach().requires_grad_() for t in (x, r, w)]
        y, h = nsa_lm.add_rms_norm(*a, eps=1e-5, out_dtype=BF)
        return (y, h, *torch.autograd.grad((y, h), a, (dy, r)))
    want = [once(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(once(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            for a, b in zip(o, want[i]):
                assert torch.equal(a, b)


def test_refusals():
    import nsa_lm
    dev = require_gpu()
    x, r, w = (t.to(dev) for t in _inputs(4, 64, BF, F32, F32))
    for bad in [(x.cpu(), r, w), (x.half(), r, w), (x, r[:, :32], w), (x, r, w[:32]), (x, r[:2], w),
                (x, r.double(), w), (x, r, w.cpu())]:
        with pytest.raises(AssertionError):
            nsa_lm.add_rms_norm(*bad)
    with pytest.raises(AssertionError):
        nsa_lm.add_rms_norm(x, r, w, eps=-1.0)
    with pytest.raises(AssertionError):
        nsa_lm.add_rms_norm(x, r, w, out_dtype=torch.float16)
    with pytest.raises(AssertionError):
        nsa_lm.add_rms_norm_q8(x, r, w.requires_grad_())
