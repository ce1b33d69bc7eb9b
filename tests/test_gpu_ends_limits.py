"""The decoder's ends at their limits: 2^24 tokens of a vocabulary (pieces of 2^20), more than 2^24 tokens to embed."""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def test_the_largest_vocabulary():
    """x[n] is a unit vector: exact logits, and dW[v, c] is dz[n, v] of column c's row.  Column c is between -1
    and 0 where v // 8 = c modulo 64, else 200 below.  The log sum is within 284 u and 4 u of its size (64 additions
    in a tile, 128 tiles of a workgroup at most, the joins); a probability within that, 2 u |lse| and 8 u, dz and dW are
    rounded to bf16 (2^-8; dW is dz again).  The weights of the columns 200 below are e^-212: less than
    float32's smallest number, 2^-126, and 0 there."""
    import nsa_lm
    dev = require_gpu()
    V, N, D = 1 << 24, 16, 64
    v = torch.arange(V, device=dev)
    w = torch.full((V, D), -200.0, device=dev, dtype=BF)
    w[v, v // 8 % 64] = (-((v * 37) % 65).float() / 64).to(BF)
    c = torch.arange(N, device=dev) * 4 + 1
    x = torch.zeros(N, D, device=dev, dtype=BF)
    x[torch.arange(N, device=dev), c] = 1
    z = w[:, c].double().t().contiguous()
    lse = torch.logsumexp(z, 1)
    t = torch.randint(0, V, (N,), device=dev, generator=torch.Generator(dev).manual_seed(0))
    t[0], t[1], t[2] = V - 1, V, (1 << 20) - 1
    ok = t < V
    xs, ws = x.requires_grad_(), w.requires_grad_()
    r = nsa_lm.linear_logprobs(xs, ws, t)
    tol = (284 + 4 * lse) * U
    assert ((r.lse.double() - lse).abs() <= tol).all()
    want = torch.where(ok, z.gather(1, t.clamp(max=V - 1)[:, None])[:, 0] - lse, 0.0)
    assert ((r.logp.double() - want).abs() <= tol + 4 * U * want.abs()).all()
    dlse = torch.linspace(1, 2, N, device=dev)
    dw, = torch.autograd.grad((r.logp, r.lse), ws, (torch.full((N,), -0.5, device=dev), dlse))
    dz = torch.exp(z - lse[:, None]) * (dlse.double() + 0.5 * ok)[:, None]
    dz.scatter_add_(1, t.clamp(max=V - 1)[:, None], -0.5 * ok.double()[:, None])
    got = dw[:, c].double().t()
    assert ((got - dz).abs() <= dz.abs() * (2.0 ** -8 + float(tol.max()) + 100 * U) + 40 * U * (dz < 0) + 2.0 ** -126).all()
    rest = torch.ones(D, dtype=torch.bool, device=dev)
    rest[c] = False
    assert not dw[:, rest].any()


@pytest.mark.parametrize("given", [False, True])
def test_more_tokens_than_one_launch(given):
    """2^24 tokens go to one launch of the forward; the gradient's sums are of whole numbers: exact."""
    import nsa_lm
    dev = require_gpu()
    n, V, D, P = (1 << 24) + 77, 1000, 4, 96
    T = next(k for k in (93, 89, 71, 53, 37, 31, 23, 19, 17, 13, 11, 7, 5, 3, 1) if n % k == 0)
    g = torch.Generator(dev).manual_seed(0)
    tok = torch.randint(-3, V + 3, (n // T, T), generator=g, device=dev)
    pos = torch.randint(0, P, (n // T, T), generator=g, device=dev) if given else None
    w = torch.randint(-4, 5, (V, D), generator=g, device=dev).float().requires_grad_()
    p = torch.randint(-4, 5, (P, D), generator=g, device=dev).float().requires_grad_()
    y = nsa_lm.embed(tok, w, 2.0, p, pos)
    ok = (tok >= 0) & (tok < V)
    at = torch.arange(T, device=dev).expand_as(tok) if pos is None else pos
    want = torch.where(ok[..., None], 2 * w.detach()[tok.clamp(0, V - 1)], 0.0) + p.detach()[at]
    assert torch.equal(y, want)
    dy = torch.randint(-1, 2, y.shape, generator=g, device=dev).float()
    dw, dp = torch.autograd.grad(y, (w, p), dy)
    flat = dy.double().view(-1, D)
    ref = torch.zeros(V + 1, D, device=dev, dtype=torch.float64).index_add_(0, torch.where(ok, tok, V).view(-1), flat)[:V] * 2
    assert torch.equal(dw.double(), ref)
    assert torch.equal(dp.double(), torch.zeros(P, D, device=dev, dtype=torch.float64).index_add_(0, at.reshape(-1), flat))
