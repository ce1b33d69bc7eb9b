"""The gradients of nsa_lm.linear_logprobs beside bf16 rows keep the digits of the targets' own elements, which make up
most of them: against the definition in 64 bits.  u = 2^-24 (half a float32 step, relative).

With dlse = dlogp = b a row's dz is b at its target and 0 elsewhere, so that dx_n = b_n W_{t_n} and dW_v = sum over
t_n = v of b_n x_n:

* b is formed from two terms within 8 u of it, and split into a bf16 and a float32 part without a loss;
* dx adds their two products: within 4 u more, and half a step of its dtype;
* dW's parts are sums of n products in float32 (2 (n + 16) u of the products' sizes); the sum of the float32 parts, each
  2^-8 of its whole at most, is rounded to bf16 once: 2^-16 of the products' sizes.
"""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def _targets(N, V, kind, g):
    if kind == "one":
        t = torch.full((N,), V // 2)
    elif kind == "text":      # a tenth of the rows have one token, the rest fall off
        t = ((V + 1.0) ** torch.rand(N, generator=g) - 1).long().clamp(max=V - 1)
        t = (t * 7919 + 5) % V
    else:
        t = torch.randint(0, V, (N,), generator=g)
    t[torch.rand(N, generator=g) < 0.1] = -100
    t[0] = V - 1
    return t


@pytest.mark.parametrize("wd", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("kind", ["any", "text", "one"])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 130, 64), (7, 40, 33), (40, 1000, 64), (300, 700, 136), (2100, 5300, 72), (4096, 500, 128),
                                   (4097, 9000, 100), (9000, 301, 520), (22100, 13000, 64), (16, 70001, 768), (50, 30, 1300),
                                   (1024, 2000, 1100), (1025, 2000, 1100), (2048, 70, 600), (2049, 70, 600),
                                   (5000, 3000, 2100)])
def test_the_targets_elements(N, V, D, kind, wd):
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator().manual_seed(N + V + D)
    x, w = torch.randn(N, D, generator=g).to(BF).to(dev), (torch.randn(V, D, generator=g) * 2 / D ** 0.5).to(wd).to(dev)
    t = _targets(N, V, kind, g).to(dev)
    ok = t >= 0
    b = torch.where(ok, -torch.rand(N, generator=g).to(dev), 0.0)
    xs, ws = x.requires_grad_(), w.requires_grad_()
    r = nsa_lm.linear_logprobs(xs, ws, t)
    dx, dw = torch.autograd.grad((r.logp, r.lse), (xs, ws), (b, b))
    at, b64 = t.clamp(min=0), b.double()
    ref = b64[:, None] * w.detach().to(BF).double()[at]
    err = (dx.double() - ref).abs() - ref.abs() * (2.0 ** -8 + 14 * U)
    assert (err <= 0).all(), float(err.max())
    prod = b64[:, None] * x.detach().double()
    ref = torch.zeros(V, D, device=dev, dtype=torch.float64).index_add_(0, at, prod)
    mag = torch.zeros(V, D, device=dev, dtype=torch.float64).index_add_(0, at, prod.abs())
    n = torch.bincount(at, minlength=V).double()[:, None]
    e = mag * (2.0 ** -16 + (2 * (n + 16) + 12) * U)
    err = (dw.double() - ref).abs() - (e * 1.01 + ref.abs() * torch.finfo(wd).eps / 2)
    assert (err <= 0).all(), float(err.max())
    # one gradient alone: the same bits
    a, = torch.autograd.grad((nsa_lm.linear_logprobs(xs, w.detach(), t)), (xs,), (b, b))
    c, = torch.autograd.grad((nsa_lm.linear_logprobs(x.detach(), ws, t)), (ws,), (b, b))
    assert torch.equal(a, dx) and torch.equal(c, dw)


@pytest.mark.parametrize("N,V,D", [(3, 59648, 512), (39, 768, 32), (75, 3968, 768), (300, 2000, 200), (2100, 5300, 256), (8000, 1536, 640)])
def test_as_near_as_the_results_rounding(N, V, D):
    """Rows from no idea of their target to sure of it: dx and dW as a whole (root of the sum of squares) are off by
    no more than their own rounding to bf16, e0, and that of the other elements of dz, e1, each at its size;
    a third of slack for what of the two is not independent (with one's rounding of the target's it is 1.3 to 1.6 e0)."""
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator().manual_seed(V)
    w = torch.randn(V, D, generator=g) * 2 / D ** 0.5
    t = torch.randint(0, V, (N,), generator=g)
    x = (torch.randn(N, D, generator=g) + torch.rand(N, 1, generator=g) * 2.5 * w[t]).to(BF).to(dev)
    w, t = w.to(BF).to(dev), t.to(dev)
    dlogp, dlse = -torch.rand(N, generator=g).to(dev), 0.05 * torch.rand(N, generator=g).to(dev)
    xs, ws = x.requires_grad_(), w.requires_grad_()
    r = nsa_lm.linear_logprobs(xs, ws, t)
    dx, dw = torch.autograd.grad((r.logp, r.lse), (xs, ws), (dlogp, dlse))
    x64, w64 = x.detach().double(), w.detach().double()
    dz = torch.softmax(x64 @ w64.t().contiguous(), 1) * (dlse - dlogp).double()[:, None]
    dz.scatter_add_(1, t[:, None], dlogp.double()[:, None])
    other = dz.to(BF).double()
    other.scatter_(1, t[:, None], dz.gather(1, t[:, None]))
    for got, f in ((dx, lambda q: q @ w64), (dw, lambda q: q.t().contiguous() @ x64)):
        ref = f(dz)
        e0, e1 = float((ref.to(BF).double() - ref).norm()), float((f(other) - ref).norm())
        assert float((got.double() - ref).norm()) <= 1.15 * (e0 * e0 + e1 * e1) ** 0.5
