"""nsa_lm.linear_logprobs of logits of any finite size, against the definition in 64 bits.

The logits are exact: x[n] has one element that is not 0, a power of two, so that z[n, v] =
x[n, 0] w[v, 0] in either type.  u = 2^-24 (half a float32 step, relative):

* a weight e^(z - M) is off by 4 u |z - M| and 4 u of its size (the difference, its product with
  log2 e, the exponential; near zero the maximum so far may lie 28 below M: 28 u);
* their sum has at most 64 additions in a tile, one for each of at most 42 tiles and at most 80 in the joins:
  the log sum is within (256 + 28) u + 4 u sum p |z - M|, and 4 u of its size;
* logp adds half a step of the target's logit and of the log sum;
* a probability is e^(z - lse) with the lse of float32: off by 4 u |lse| beside the above; where the logits lie 64 or
  more apart it is 0 or, at |lse| >= 4096, 1.
"""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
# a few rows of every tile shape: 32, 64 and 128 rows, 128 x 128 and 256 x 256
SHAPES = [(3, 100), (40, 300), (100, 1000), (300, 700), (2100, 5300)]
SIZES = [1.0, 2.0 ** 9, 2.0 ** 11, 2.0 ** 13, 2.0 ** 20, 2.0 ** 31, 8e29, 1e30, 1e35, 2.0 ** 126]


def _data(N, V, size, dtype, kind, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "equal":
        a = torch.ones(V)
    elif kind == "apart":     # 128 different values, neighbours 1 / 128 apart, in any order
        a = (1 + torch.arange(V) % 128 / 128)[torch.randperm(V, generator=g)]
    else:
        a = 1 + torch.rand(V, generator=g)
    w = torch.randn(V, 64, generator=g)
    w[:, 0] = a * size
    x = torch.zeros(N, 64)
    x[:, 0] = torch.tensor([1.0, -1.0, 0.5, -0.25, 0.0])[torch.arange(N) % 5]
    t = torch.randint(0, V, (N,), generator=g)
    return x.to(dtype).to(dev), w.to(dtype).to(dev), t.to(dev)


@pytest.mark.parametrize("kind", ["equal", "apart", "any"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("N,V", SHAPES)
def test_every_finite_logit_counts(N, V, dtype, kind):
    import nsa_lm
    dev = require_gpu()
    for size in SIZES:
        x, w, t = _data(N, V, size, dtype, kind, dev)
        z = x[:, :1].double() * w[:, 0].double()[None]
        lse = torch.logsumexp(z, 1)
        M = z.amax(1, keepdim=True)
        p = torch.exp(z - lse[:, None])
        far = torch.where(p > 0, p * (z - M).abs(), 0.0).sum(1)
        tol = (284 + 4 * far + 4 * lse.abs()) * U
        got = nsa_lm.linear_logprobs(x, w, t)
        err = (got.lse.double() - lse).abs() - tol
        assert (err <= 0).all(), (size, float(err.max()))
        zt = z.gather(1, t[:, None])[:, 0]
        err = (got.logp.double() - (zt - lse)).abs() - (tol + 2 * U * (zt.abs() + lse.abs()))
        assert (err <= 0).all(), (size, float(err.max()))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("N", [3, 40, 100, 300, 2100])
def test_gradients_of_logits_far_apart(N, dtype):
    """Logits 64 or more apart: a row's gradient is a at its largest logit and b at its
    target.  Sums of at most max(N, V) products, each within half a step of the operand."""
    import nsa_lm
    dev = require_gpu()
    V, g = 100, torch.Generator().manual_seed(N)
    R = 2.0 ** -8 if dtype == BF else 2.0 ** -23
    for size in (2.0 ** 15, 2.0 ** 20, 2.0 ** 31, 1e30, 2.0 ** 120):
        x, w, t = _data(N, V, size, dtype, "apart", dev)
        x[:, 0] = torch.tensor([1.0, -1.0, 2.0, -0.5], device=dev)[torch.arange(N, device=dev) % 4].to(dtype)
        dlogp, dlse = torch.rand(N, generator=g).to(dev), torch.rand(N, generator=g).to(dev)
        xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
        r = nsa_lm.linear_logprobs(xs, ws, t)
        dx, dw = torch.autograd.grad((r.logp, r.lse), (xs, ws), (dlogp, dlse))
        z = x[:, :1].double() * w[:, 0].double()[None]
        dz = torch.zeros_like(z)
        dz.scatter_add_(1, z.argmax(1, keepdim=True), (dlse - dlogp).double()[:, None])
        dz.scatter_add_(1, t[:, None], dlogp.double()[:, None])
        size_ = torch.zeros_like(z)
        size_.scatter_add_(1, z.argmax(1, keepdim=True), (dlse + dlogp).double()[:, None])
        size_.scatter_add_(1, t[:, None], dlogp.double()[:, None])
        h = torch.finfo(dtype).eps / 2
        for got, left, mag, right, n in ((dx, dz, size_, w.double(), V), (dw, dz.t().contiguous(), size_.t().contiguous(), x.double(), N)):
            ref, m = left @ right, mag @ right.abs()
            err = (got.double() - ref).abs() - ((R + 2 * (n + 16) * U) * m * (1 + h) + h * ref.abs() + 1e-30)
            assert (err <= 0).all(), (size, float(err.max()))


def test_infinite_logits():
    """Minus infinity (of bf16 weights) has no weight beside a finite logit; a row of nothing
    else is NaN, as a row with plus infinity is."""
    import nsa_lm
    dev = require_gpu()
    for N in (4, 300):
        x, w, t = _data(N, 300, 1.0, BF, "any", dev)
        x[:, 0] = 1
        w[7:200, 0] = float("-inf")
        t[:] = 3
        t[1] = 9
        want = torch.log_softmax(w[:, 0].double(), 0)
        got = nsa_lm.linear_logprobs(x, w, t)
        keep = torch.arange(N, device=dev) != 1
        assert ((got.logp[keep].double() - want[3]).abs() <= 300 * U).all() and got.logp[1] == float("-inf")
        w[:, 0] = float("-inf")
        got = nsa_lm.linear_logprobs(x, w, t)
        assert got.lse.isnan().all() and got.logp.isnan().all()
        w[:, 0] = 1
        w[250, 0] = float("inf")
        got = nsa_lm.linear_logprobs(x, w, t)
        assert got.lse.isnan().all() and got.logp.isnan().all()


@pytest.mark.parametrize("N", [5, 60, 200, 2100])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_ignored_rows_have_no_gradient_whatever_their_logits(N, dtype):
    """Rows whose products pass float32 (x is finite), and rows with NaN: 0 where they are ignored
    or their results' gradients are 0; the other rows' gradients are as without them."""
    import nsa_lm
    dev = require_gpu()
    V, D = 5300 if N > 2000 else 300, 64
    g = torch.Generator().manual_seed(N)
    x, w = torch.randn(N, D, generator=g).to(dtype).to(dev), torch.randn(V, D, generator=g).to(dtype).to(dev)
    t = torch.randint(0, V, (N,), generator=g).to(dev)
    dlogp = -torch.rand(N, generator=g).to(dev)
    bad = torch.zeros(N, dtype=torch.bool, device=dev)
    bad[1::3] = True
    t[bad] = -100
    last = int(bad.nonzero()[-1])
    t[last], dlogp[last] = 7, 0.0                                  # not ignored, of no weight

    def grads(x):
        xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
        r = nsa_lm.linear_logprobs(xs, ws, t)
        return r, torch.autograd.grad(r.logp, (xs, ws), dlogp)
    tame = x.clone()
    tame[bad] = 0
    _, (dx0, dw0) = grads(tame)
    wild = tame.clone()
    wild[bad] = 3e38
    r, (dx, dw) = grads(wild)
    assert not r.lse[bad].isfinite().any() and r.lse[~bad].isfinite().all()
    assert torch.equal(dx, dx0) and torch.equal(dw, dw0)
    wild[bad] = float("nan")
    r, (dx, _) = grads(wild)
    assert r.lse[bad].isnan().all() and torch.equal(dx, dx0)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("N,V", SHAPES)
def test_one_logit_far_from_the_others(N, V, dtype):
    """Logits within 4 of 0 and one, late in the vocabulary, far above or (in rows of x = -1) far below them all: the maximum passes
    from near zero to far off it.  Above, its probability is 1; below it is 0 and the row is as without it, bit for bit
    where the same wave has rows of the other kind."""
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator().manual_seed(V)
    w = torch.randn(V, 64, generator=g)
    w[:, 0] = (torch.randint(-32, 33, (V,), generator=g) / 8.0)
    x = torch.zeros(N, 64)
    x[:, 0] = torch.tensor([1.0, -1.0, -1.0])[torch.arange(N) % 3]
    t = torch.randint(0, V - 8, (N,), generator=g)
    x, t = x.to(dtype).to(dev), t.to(dev)
    up = x[:, 0] > 0
    for size in (300.0, 4095.0, 4100.0, 1e6, 1e30, 2.0 ** 126):
        for at in (V - 3, V // 2):
            w2 = w.to(dtype).to(dev)
            w2[at, 0] = size
            tt = torch.where(up & (torch.arange(N, device=dev) % 2 == 0), at, torch.where(t == at, t + 1, t))
            z = x[:, :1].double() * w2[:, 0].double()[None]
            lse = torch.logsumexp(z, 1)
            want = z.gather(1, tt[:, None])[:, 0] - lse
            xs, ws = x.clone().requires_grad_(), w2.clone().requires_grad_()
            r = nsa_lm.linear_logprobs(xs, ws, tt)
            tol = (284 + 8 * lse.abs()) * U
            assert ((r.lse.double() - lse).abs() <= tol).all(), (size, at)
            assert ((r.logp.double() - want).abs() <= tol + 2 * U * want.abs()).all(), (size, at)
            one = torch.ones(N, device=dev)
            dx, dw = torch.autograd.grad((r.logp, r.lse), (xs, ws), (one, 0.25 * one))
            assert dx[~up].isfinite().all() and dw[:at].isfinite().all()
            # dz of the row above: 1 at its target, -3/4 at the far token; columns of w that x does not see
            other = w2[:, 1:].double()
            ref = other[tt] - 0.75 * other[at]
            err = (dx[:, 1:].double() - ref).abs() - 2.0 ** -7 * (other[tt].abs() + other[at].abs())
            assert (err[up] <= 0).all(), (size, at)
            xi = x.clone()
            xi[up] = 0                                   # the far rows gone: the others' bits stay
            xs = xi.requires_grad_()
            r2 = nsa_lm.linear_logprobs(xs, ws, tt)
            d2, = torch.autograd.grad((r2.logp, r2.lse), xs, (one, 0.25 * one))
            assert torch.equal(r2.lse[~up], r.lse[~up]) and torch.equal(r2.logp[~up], r.logp[~up])
            assert torch.equal(d2[~up], dx[~up]), (size, at)
