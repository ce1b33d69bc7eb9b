"""nsa_lm.add_layer_norm of rows far off zero, against the definition in 64 bits.

The mean is a float32 number: its error is half a step of itself and nothing else, u |mean| with u = 2^-24.  So

* rows of equal elements have exactly that mean: y is the bias, whatever eps, and NaN with eps 0;
* n = (h - mean) rstd is off by u |mean| rstd beside the errors of the deviations' squares ((CHAIN / 2 + 8) u
  of n, CHAIN additions) and of the product;
* the backward recomputes n from the same mean; its sums are of at most D (rows) terms.
"""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


@pytest.mark.parametrize("D", [1, 3, 7, 41, 47, 55, 107, 200, 501, 768, 1001, 4100, 9001, 20001, 33001])
def test_rows_of_equal_elements(D):
    import nsa_lm
    dev = require_gpu()
    vals = torch.tensor([0.1, -0.3, 3.0, 1024.0, 16384.0, -1e6, 1e-30, 7e20])
    x = vals[:, None].expand(8, D).contiguous().to(dev)
    w, b = torch.linspace(0.5, 2, D, device=dev), torch.linspace(-1, 1, D, device=dev)
    for eps in (1e-5, 1e-12):
        for r in (None, torch.zeros_like(x)):
            xs = x.clone().requires_grad_()
            y, _ = nsa_lm.add_layer_norm(xs, r, w, b, eps=eps)
            assert torch.equal(y, b.expand(8, D))
            g, = torch.autograd.grad(y.sum(), xs)
            assert torch.isfinite(g).all()
    assert nsa_lm.add_layer_norm(x, None, w, b, eps=0.0)[0].isnan().all()
    xb = vals.to(BF)[:, None].expand(8, D).contiguous().to(dev)
    assert torch.equal(nsa_lm.add_layer_norm(xb, None, w, b, out_dtype=F32)[0], b.expand(8, D))


@pytest.mark.parametrize("rows,D", [(5, 8), (9, 41), (300, 107), (40, 512), (40, 768), (9, 1001), (5, 2049), (5, 8192),
                                    (3, 16385), (2, 33001)])
@pytest.mark.parametrize("far", [1e2, 1e4, 3e5])
def test_rows_far_off_zero(rows, D, far):
    """|mean| / deviation of `far`."""
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator().manual_seed(rows + D)
    x = far * (1 + torch.rand(rows, 1, generator=g)) + torch.randn(rows, D, generator=g)
    w = 1 + 0.2 * torch.randn(D, generator=g)
    dy = torch.randn(rows, D, generator=g)
    eps = 1e-6
    xs, ws = x.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    y, _ = nsa_lm.add_layer_norm(xs, None, ws, eps=eps)
    dx, dw = torch.autograd.grad(y, (xs, ws), dy.to(dev))
    C = 8 * max(4, -(-D // 8192)) + 22
    h, w64, d64 = x.double(), w.double(), dy.double()
    mean = h.mean(1, keepdim=True)
    d = h - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    n = d * rstd
    # the deviations about a mean that is off by m: their squares' mean grows by m^2, to second order
    off = U * mean.abs() * rstd
    E = off * (1 + off * n.abs()) + n.abs() * (C / 2 + 8) * U
    t = w64.abs() * E + 2 * U * (n * w64).abs()
    err = (y.detach().cpu().double() - n * w64).abs() - (t + U * (n * w64).abs() + 1e-30)
    assert (err <= 0).all(), float(err.max())
    gw = d64 * w64
    s1, s2 = gw.mean(1, keepdim=True), (gw * n).mean(1, keepdim=True)
    m1, m2 = gw.abs().mean(1, keepdim=True), (gw * n).abs().mean(1, keepdim=True)
    ref = rstd * (gw - s1 - n * s2)
    e = rstd * (4 * U * gw.abs() + (C + 4) * U * m1 + (n.abs() + E) * ((C + 5) * U * m2 + (gw.abs() * E).mean(1, keepdim=True))
                + E * s2.abs()) + (C / 2 + 8) * U * rstd * (gw.abs() + m1 + n.abs() * m2) + off * off * ref.abs()
    err = (dx.cpu().double() - ref).abs() - (e + U * ref.abs() + 1e-30)
    assert (err <= 0).all(), float(err.max())
    prod = d64 * n
    err = (dw.cpu().double() - prod.sum(0)).abs() - (prod.abs().sum(0) * (rows + 4) * U + (d64.abs() * E).sum(0)) * (1 + 4 * U) - U * prod.sum(0).abs()
    assert (err <= 0).all(), float(err.max())
