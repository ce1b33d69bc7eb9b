"""The decoder's ends where elements lie more than 2^32 apart, and in several graphs
and streams at once.  Far rows are compared with the same rows in small tensors."""
import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _rows(n, D, seed):
    """A tensor of n rows whose last 64 are random; the rest repeats one random row."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(1, D, generator=g).to(BF).cuda().expand(n, D).clone()
    tail = torch.randn(64, D, generator=g).to(BF).cuda()
    x[-64:] = tail
    return x, tail


def test_lnorm_far_rows():
    import nsa_lm
    require_gpu()
    n, D = (1 << 20) + 65, 4104
    assert n * D > 1 << 32
    x, tail = _rows(n, D, 0)
    w, b = (torch.randn(D, device="cuda", dtype=BF) for _ in range(2))
    ws = w.clone().requires_grad_()
    y, h = nsa_lm.add_layer_norm(x, x, ws, b)
    yt, ht = nsa_lm.add_layer_norm(tail, tail, w, b)
    assert torch.equal(y[-64:], yt) and torch.equal(h[-64:], ht) and torch.equal(y[5], y[n - 65])
    # gradients from the last row alone: every other row's are zeros, and its own those of a small call
    dy = torch.zeros_like(y)
    dy[-1] = 1
    xs = x.requires_grad_()
    y, h = nsa_lm.add_layer_norm(xs, None, ws, b)
    dx, dw = torch.autograd.grad(y, (xs, ws), dy)
    ts, wt = tail.clone().requires_grad_(), w.clone().requires_grad_()
    ex, ew = torch.autograd.grad(nsa_lm.add_layer_norm(ts, None, wt, b)[0], (ts, wt), dy[-64:])
    assert torch.equal(dx[-64:], ex) and torch.equal(dw, ew) and not dx[:-64].any()


def test_embed_far_rows():
    import nsa_lm
    require_gpu()
    n, V, D = (1 << 20) + 5, 101, 4104
    t = torch.arange(n, device="cuda") % V
    w = torch.randn(V, D, device="cuda").to(BF).requires_grad_()
    y = nsa_lm.embed(t, w)
    assert torch.equal(y[-7:], w[t[-7:]]) and torch.equal(y[1 << 19], w[t[1 << 19]])
    dy = torch.ones_like(y)
    # up to 2^24 ones are counted exactly in float32, and rounded once
    (dw,) = torch.autograd.grad(y, w, dy)
    count = torch.bincount(t, minlength=V).float().to(BF)
    assert torch.equal(dw, count[:, None].expand(V, D))
    del y, dy, dw
    # a table whose last rows lie that far
    big, tail = _rows(n, D, 1)
    idx = torch.tensor([n - 64, n - 1, 0, -1, n, n - 1], device="cuda")
    bs = big.requires_grad_()
    out = nsa_lm.embed(idx, bs)
    assert torch.equal(out[:2], tail[[0, -1]]) and torch.equal(out[5], tail[-1]) and not out[3:5].any()
    (db,) = torch.autograd.grad(out, bs, torch.ones_like(out))
    want = torch.zeros(64, device="cuda", dtype=BF)
    want[0], want[-1] = 1, 2
    assert torch.equal(db[-64:], want[:, None].expand(64, D)) and (db[0] == 1).all() and not db[1:-64].any()


def test_head_far_rows():
    """Rows of x past 2^32 elements: row by row the values of a small call."""
    import nsa_lm
    require_gpu()
    n, V, D = (1 << 21) + 64, 70, 2112
    assert n * D > 1 << 32
    x, tail = _rows(n, D, 2)
    w = (torch.randn(V, D, device="cuda") / D ** 0.5).to(BF).requires_grad_()
    t = torch.full((n,), -100, device="cuda")
    t[-64:] = torch.arange(64, device="cuda")
    xs = x.requires_grad_()
    out = nsa_lm.linear_logprobs(xs, w, t)
    z = tail.float() @ w.detach().float().t()
    lse = torch.logsumexp(z, 1)
    logp = z.gather(1, t[-64:, None])[:, 0] - lse
    # D products of bf16 are exact in float32; their sums, of terms below 32 in all, are off by
    # at most D 2^-24 32 in either order
    tol = 2 * D * 2.0 ** -24 * 32
    assert (out.lse[-64:] - lse).abs().max() < tol and (out.logp[-64:] - logp).abs().max() < tol
    assert not out.logp[:-64].any()
    dx, dw = torch.autograd.grad(out.logp, (xs, w), torch.ones_like(out.logp))
    dz = -torch.exp(z - lse[:, None])
    dz[torch.arange(64, device="cuda"), t[-64:]] += 1
    ex, ew = dz @ w.detach().float(), dz.t() @ tail.float()
    # dz and the result are rounded to bf16 once each: half a step of the terms' sizes and of the sum
    mx, mw = dz.abs() @ w.detach().float().abs(), dz.abs().t() @ tail.float().abs()
    assert ((dx[-64:].float() - ex).abs() <= 2.0 ** -7 * mx + 1e-5).all() and not dx[:-64].any()
    assert ((dw.float() - ew).abs() <= 2.0 ** -7 * mw + 1e-5).all()


def test_head_far_vocabulary():
    """Rows of W past 2^32 elements: few distinct ones, so that the sums are known."""
    import nsa_lm
    require_gpu()
    V, D, N = (1 << 22) + 64, 1088, 5
    assert V * D > 1 << 32
    w, tail = _rows(V, D, 3)
    w.mul_(2.0 ** -5)
    tail = tail * 2.0 ** -5
    g = torch.Generator().manual_seed(4)
    x = torch.randn(N, D, generator=g).to(BF).cuda()
    t = torch.tensor([V - 1, V - 64, 0, V, -1], device="cuda")
    ws, xs = w.requires_grad_(), x.requires_grad_()
    out = nsa_lm.linear_logprobs(xs, ws, t)
    one = w.detach()[:1]
    z = x.detach().double() @ torch.cat([one, tail]).double().t()                  # [N, 1 + 64]
    n0 = V - 64
    lse = torch.logsumexp(torch.cat([z[:, :1] + torch.log(torch.tensor(float(n0), dtype=torch.float64)), z[:, 1:]], 1), 1)
    where = torch.tensor([64, 1, 0], device="cuda")
    logp = z[:3].gather(1, where[:, None])[:, 0] - lse[:3]
    # sums of D terms (tol of float32 sums as above) and of V float32 terms in a tree of lanes,
    # registers and parts: fewer than 2^12 in a row at any level, 2^-12 relative to the sum
    tol = D * 2.0 ** -24 * 32 + 2.0 ** -11
    assert (out.lse.double() - lse).abs().max() < tol and (out.logp[:3].double() - logp).abs().max() < tol
    assert not out.logp[3:].any()
    dlp = torch.zeros(N, device="cuda")
    dlp[0] = 1.0
    dx, dw = torch.autograd.grad(out.logp, (xs, ws), dlp)
    p = torch.exp(z[0] - lse[0])
    want = -p.clone()
    want[64] += 1
    got = dw[-64:].double()
    xd = x.detach()[0].double()
    # dz and dW are rounded once each, and e^(z - lse) is off by the sums above
    rel = 2.0 ** -7 + 2 * tol
    assert ((got - want[1:, None] * xd).abs() <= rel * (want[1:, None] * xd).abs() + 1e-30).all()
    far = dw[n0 - 1].double()
    assert ((far - want[0] * xd).abs() <= rel * (want[0] * xd).abs() + 1e-30).all()
    ex = want[1:] @ tail.double() - n0 * p[0] * one[0].double()
    mag = want[1:].abs() @ tail.double().abs() + n0 * p[0] * one[0].double().abs()
    assert ((dx[0].double() - ex).abs() <= rel * mag).all() and not dx[1:].any()


def test_two_graphs_on_two_streams():
    """Two captured passes with workspaces of their own, replayed side by side."""
    import nsa_lm
    require_gpu()
    torch.manual_seed(5)
    work = []
    for k, (n, V, D) in enumerate([(300, 1000, 96), (513, 2000, 128)]):
        t = torch.randint(0, V, (1, n), device="cuda")
        w, p = (torch.randn(m, D, device="cuda").to(BF).requires_grad_() for m in (V, n))
        g = torch.ones(D, device="cuda", dtype=BF).requires_grad_()

        def run(t=t, w=w, p=p, g=g):
            y, _ = nsa_lm.add_layer_norm(nsa_lm.embed(t, w, 1.0, p), None, g)
            out = nsa_lm.linear_logprobs(y, w, t.roll(1, 1))
            return [out.logp.detach(), *torch.autograd.grad(out.logp.sum(), (w, p, g))]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        work.append((graph, side, t, V, run, got))
    for _ in range(3):
        for graph, side, t, V, run, got in work:
            t.copy_(torch.randint(0, V, t.shape))
            side.wait_stream(torch.cuda.current_stream())
        for graph, side, *_ in work:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for graph, side, t, V, run, got in work:
            for a, b in zip(got, run()):
                assert torch.equal(a, b)
        torch.cuda.synchronize()
