"""nsa_lm.linear_logprobs of rows that are sure of a token, against the definition in 64 bits.

The logits are exact: x[n] is a unit vector, z[n] a column of w.  Eight tokens of a row, anywhere in the
vocabulary, lie 0 to 30 below its largest logit, all others 200 below, so that their weights are 0 in
float32.  u = 2^-24 (half a float32 step, relative):

* a weight's exponent is at most 9 bits above 0 or it weighs little: rounded to 9 u (6.3 u of the weight), the
  exponential 2 u; the sum has at most 8 + 6 additions that are not of 0, and 4 rescalings of 3 u each (the halves of a
  wave, the waves, the shares of a row); the logarithm of it 2 u, and logp's own roundings 2 u of its size:
  within (6.3 + 2 + 14 + 12 + 2) u < 40 u and 4 u |logp|.
* 1 - p of the target, which its gradient is made of, is within the same 40 u.
* the other seven probabilities are formed from lse: within (2 |lse| + 48) u of themselves.
"""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
SHAPES = [(32, 1000), (64, 1000), (128, 3000), (300, 1000), (2100, 5300)]
TOPS = (0.0, 10.0, 37.0, 100.0, 160.0, 1000.0, 3000.0, 5000.0, 1e5, -100.0, -3000.0)


def _data(N, V, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.zeros(V, 128)
    for c in range(64):
        top = TOPS[c % len(TOPS)]
        near = torch.randperm(V, generator=g)[:8]
        w[:, c] = top - 200 - 0.01 * abs(top)
        w[near, c] = top - 30 * torch.rand(8, generator=g)
        w[near[0], c] = top
    w[:, 64:] = torch.randint(0, 2, (V, 64), generator=g) * 2.0 - 1
    w = w.to(dtype)
    x = torch.zeros(N, 128)
    col = torch.arange(N) % 64
    x[torch.arange(N), col] = 1
    z = w.double()[:, col].t().contiguous()
    t = z.argmax(1)
    pick = torch.rand(N, generator=g) < 0.25            # rows whose target is another of the eight, or any
    t[pick] = z.topk(8, 1).indices[:, 5][pick]
    t[torch.rand(N, generator=g) < 0.05] = 7
    return x.to(dtype).to(dev), w.to(dev), t.to(dev), z.to(dev)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("N,V", SHAPES)
def test_sure_rows_keep_their_digits(N, V, dtype):
    import nsa_lm
    dev = require_gpu()
    for seed in range(3):
        x, w, t, z = _data(N, V, dtype, dev, seed)
        xs = x.clone().requires_grad_()
        r = nsa_lm.linear_logprobs(xs, w, t)
        lse = torch.logsumexp(z, 1)
        want = z.gather(1, t[:, None])[:, 0] - lse
        assert (r.logp <= 0).all()
        err = (r.logp.detach().double() - want).abs() - (40 + 4 * want.abs()) * U
        assert (err <= 0).all(), float(err.max())
        err = (r.lse.detach().double() - lse).abs() - (40 + 2 * lse.abs()) * U
        assert (err <= 0).all(), float(err.max())
        if dtype == BF:
            continue
        g, = torch.autograd.grad(r.logp.sum(), xs)
        p = torch.exp(z - lse[:, None])
        dz = -p
        dz.scatter_add_(1, t[:, None], torch.ones_like(dz[:, :1]))
        e = p * ((2 * lse.abs() + 48) * U)[:, None]
        e.scatter_(1, t[:, None], torch.full_like(e[:, :1], 40 * U))
        # (sums of at most 64 elements that are not 0, in any order, and the planes' left-out products)
        tol = e.sum(1) + 80 * U * dz.abs().sum(1)
        err = (g[:, 64:].double() - dz @ w[:, 64:].double()).abs() - tol[:, None]
        assert (err <= 0).all(), float(err.max())
