"""nsa_lm.token_logprobs against the definition in 64 bits.

Tolerances, u = 2^-24: a weight e^(z-m) is formed within 4 u (1 + |z-m|) of
itself (the difference, its product with log2 e, the exponential); the sum l
of a row takes at most CHAIN additions of positive terms, so that l is within
(CHAIN + 6) u (the weights' own errors, weighted: e^-x x <= 0.37).  Then
  logp = (z_t - m) - ln l:          that, and 2 u of either term;
  H = ln l - s / l:                 that, with s within (CHAIN + 8) u of sum e |z-m|;
  dz = -p (dl + dH (ln p + H)):      p within (CHAIN + 10 + 4 |ln p|) u, H's error, half a step.
CHAIN: V / 256 elements of a lane (32 for one wave's rows) + 6 + 4 + 64 parts + 32;
a wave that takes a row of up to 8192 by itself has V / 64 + 6, no more than that.
"""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
INF = float("inf")


def _chain(V):
    return (V / 256 if V > 2048 else 32) + 32 + 6 + 4 + 64


def _rows(rows, V, dtype, seed=0, banned=True):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, V, generator=g) * (0.5 + 3 * torch.rand(rows, 1, generator=g))
    if banned and V > 3:
        z[:, torch.randint(0, V, (max(1, V // 50),), generator=g)] = -INF
    t = torch.randint(0, V, (rows,), generator=g)
    return z.to(dtype), t


def _ref(z, t):
    # against the maximum first: beside the lowest float32 value even 64 bits lose ln l
    # (a row of -inf alone: log probabilities of -inf, entropy 0)
    z = z.double()
    m = z.amax(1, keepdim=True)
    d = z - m.masked_fill(m == -INF, 0)
    lp = d - torch.log(torch.exp(d).sum(1, keepdim=True).masked_fill(m == -INF, 1))
    lp0 = lp.masked_fill(lp == -INF, 0)
    p = lp.exp()
    H = -(p * lp0).sum(1)
    ok = (t >= 0) & (t < z.shape[1])
    logp = torch.where(ok, lp.gather(1, t.clamp(0, z.shape[1] - 1)[:, None])[:, 0], torch.zeros(()).double())
    return lp, lp0, p, H, logp, ok


def _check(z, t, top, dev, grad=True):
    import nsa_lm
    rows, V = z.shape
    zd = z.to(dev).requires_grad_(grad)
    got = nsa_lm.token_logprobs(zd, t.to(dev), top)
    lp, lp0, p, H, logp, ok = _ref(z, t)
    C = _chain(V)
    m = z.double().amax(1)
    m = m.masked_fill(m == -INF, 0)
    logl = torch.logsumexp(z.double() - m[:, None], 1).clamp(min=0)   # (0: a row of -inf alone)
    S = (p * (z.double() - m[:, None]).abs().masked_fill(z.double() == -INF, 0)).sum(1)
    zt = z.double().gather(1, t.clamp(0, V - 1)[:, None])[:, 0]
    tl = (C + 6) * U
    dt = torch.where(zt == -INF, 0.0, (zt - m).abs())
    tol = tl + 2 * U * (dt + logl)
    a = got.logp.detach().cpu().double()
    fin = ok & (zt != -INF)
    assert ((a - logp).abs() <= tol)[fin].all()
    assert (a[~ok] == 0).all() and (a[ok & (zt == -INF)] == -INF).all()
    tH = tl + (2 * C + 20) * U * S + 3 * U * (logl + S)
    assert ((got.entropy.detach().cpu().double() - H).abs() <= tH).all()
    if top:
        order = torch.sort(z.double() + 0.0, dim=1, descending=True, stable=True)
        assert torch.equal(got.top_idx.cpu(), order.indices[:, :top])
        v = lp.gather(1, order.indices[:, :top])
        e = (got.top_logp.cpu().double() - v).abs()
        d = (m[:, None] - order.values[:, :top])
        okv = v != -INF
        assert (e <= tl + 2 * U * (d + logl[:, None]))[okv].all()
        assert (got.top_logp.cpu()[~okv] == -INF).all()
    if not grad:
        return
    g = torch.Generator().manual_seed(V)
    dl, dH = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    for use_l, use_h in ((1, 1), (1, 0), (0, 1)):
        outs = ([got.logp] if use_l else []) + ([got.entropy] if use_h else [])
        gos = ([dl.to(dev)] if use_l else []) + ([dH.to(dev)] if use_h else [])
        dz, = torch.autograd.grad(outs, zd, gos, retain_graph=True)
        assert dz.dtype == z.dtype and dz.shape == z.shape
        L = torch.where(ok, dl.double() * use_l, 0.0)[:, None]
        h = dH.double()[:, None] * use_h
        ref = -p * (L + h * (lp0 + H[:, None]))
        ref = ref.scatter_add(1, t.clamp(0, V - 1)[:, None], L)
        mag = p * (L.abs() + h.abs() * (lp0.abs() + H[:, None].abs())) * ((C + 12 + 4 * lp0.abs()) * U) + \
            p * h.abs() * (tH[:, None] + tl)
        mag = mag.scatter_add(1, t.clamp(0, V - 1)[:, None], 2 * U * L.abs())
        half = torch.finfo(z.dtype).eps / 2
        tiny = 2.0 ** -126      # below the normal numbers a weight may be flushed to 0
        e = (dz.cpu().double() - ref).abs()
        assert (e <= ref.abs() * half * (1 + 1e-6) + mag * (1 + 4 * half) + tiny * (L.abs() + h.abs() * 100 + 1)).all(), \
            float((e - ref.abs() * half - mag).max())


SHAPES = [(1, 1, 1), (1, 2, 2), (5, 7, 3), (3, 64, 64), (9, 100, 20), (4, 511, 64), (6, 513, 5), (7, 2048, 64),
          (3, 2049, 1), (2, 4097, 64), (1, 8191, 20), (5, 8193, 33), (1, 50257, 20), (33, 32000, 5), (1, 131072, 64),
          (2, 200001, 7), (1100, 4100, 3), (1030, 20011, 10),
          (9, 1000, 7), (2001, 129, 2), (4099, 2300, 24), (4096, 8191, 5)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,V,top", SHAPES)
def test_forward_and_backward(rows, V, top, dtype):
    dev = require_gpu()
    z, t = _rows(rows, V, dtype, seed=rows + V)
    if rows > 2:
        t[1], t[2] = -100, V
    _check(z, t, top, dev, grad=rows * V < 1 << 23)


@pytest.mark.parametrize("V", [1000, 3000, 40000])
def test_rows_that_overfill_the_candidate_list(V):
    """Ties and rising rows: the alternatives come from the exact selection."""
    dev = require_gpu()
    up = torch.arange(V).float() / V
    few = torch.zeros(V)
    few[V // 2:] = 1.0
    lanes = torch.zeros(V)
    lanes[torch.arange(V) % 2048 < 8] = torch.rand(V, generator=torch.Generator().manual_seed(1))[torch.arange(V) % 2048 < 8] + 1
    steps = (torch.arange(V) // 97).float()
    z = torch.stack([torch.zeros(V), up, up.flip(0), few, lanes, steps, -steps, torch.full((V,), torch.finfo(F32).min)])
    t = torch.arange(8) * 31
    for top in (1, 5, 64):
        _check(z, t, top, dev, grad=False)
    _check(z[:7].to(BF), t[:7], 64, dev, grad=False)
    _check(z[:2], t[:2], 64, dev, grad=False)


@pytest.mark.parametrize("rows,V,top", [(4, 700, 5), (3, 9000, 24), (33, 32000, 20), (2, 140000, 40), (4200, 4096, 8)])
def test_masked_vocabularies(rows, V, top):
    """All but a few tokens masked, with -inf or the type's lowest value: fewer left than alternatives
    asked for (the masked ones follow by index), as many, and more."""
    dev = require_gpu()
    for dtype in (BF, F32):
        for mask in (-INF, torch.finfo(dtype).min):
            z, t = _rows(rows, V, dtype, seed=V, banned=False)
            g = torch.Generator().manual_seed(rows)
            order = torch.rand(rows, V, generator=g).argsort(1) if rows < 100 else \
                (torch.arange(V)[None] * 7919 + torch.randint(0, V, (rows, 1), generator=g)) % V
            left = torch.tensor([0, 1, top - 1, top, top + 1, 100]).repeat(rows // 6 + 1)[:rows]
            keep = torch.zeros(rows, V, dtype=torch.bool).scatter_(1, order, torch.arange(V)[None] < left[:, None])
            z = z.masked_fill(~keep, mask)
            _check(z, t, top, dev, grad=False)


def test_many_rows_of_one_wave_that_overfill_the_list():
    dev = require_gpu()
    V = 3000
    r = torch.arange(V).float()
    z = torch.stack([torch.zeros(V), r / V, -(r / 97).floor(), (r >= V // 2).float()]).repeat(1025, 1)
    _check(z, torch.arange(4100) % V, 20, dev, grad=False)


def test_signed_zeros_tie():
    import nsa_lm
    dev = require_gpu()
    z = torch.full((2, 300), -1.0)
    z[0, [5, 9, 200]] = torch.tensor([-0.0, 0.0, -0.0])
    z[1, [5, 9, 200]] = torch.tensor([0.0, -0.0, 0.0])
    got = nsa_lm.token_logprobs(z.to(dev), None, 4)
    assert got.logp is None and got.top_idx.cpu().tolist() == [[5, 9, 200, 0]] * 2


@pytest.mark.parametrize("V", [40, 5000])
def test_masked_infinite_and_nan_rows(V):
    import nsa_lm
    dev = require_gpu()
    z = torch.randn(7, V, generator=torch.Generator().manual_seed(0))
    z[0] = -INF                                    # nothing left
    z[1] = -INF
    z[1, 17] = 3.0                                 # one token left
    z[2] = torch.finfo(F32).min                    # masked with the lowest value: uniform
    z[3, 5] = INF
    z[4, 6] = float("nan")
    z[5, 1:] = torch.finfo(F32).min
    z[6, :20] = -INF
    t = torch.tensor([3, 17, 2, 5, 6, 0, 4])
    zd = z.to(dev).requires_grad_()
    got = nsa_lm.token_logprobs(zd, t.to(dev), 3)
    dz, = torch.autograd.grad((got.logp, got.entropy), zd, (torch.ones(7, device=dev), torch.ones(7, device=dev)))
    lp, H, dz = got.logp.detach().cpu(), got.entropy.detach().cpu(), dz.cpu()
    assert lp[0] == -INF and H[0] == 0 and not dz[0].any()
    assert got.top_idx[0].tolist() == [0, 1, 2] and (got.top_logp[0] == -INF).all()
    assert lp[1] == 0 and H[1] == 0 and not dz[1].any() and got.top_idx[1].tolist() == [17, 0, 1]
    lnv = torch.tensor(float(V)).log()
    assert abs(lp[2] + lnv) < 1e-5 and abs(H[2] - lnv) < 1e-5 and got.top_idx[2].tolist() == [0, 1, 2]
    assert abs(float(dz[2].sum())) < 1e-5 and torch.isfinite(dz[2]).all()
    assert lp[3].isnan() and H[3].isnan() and got.top_idx[3, 0] == 5
    assert lp[4].isnan() and H[4].isnan() and got.top_idx[4, 0] == 6 and dz[4].isnan().all()
    assert lp[5] == 0 and H[5] == 0 and got.top_idx[5, 0] == 0
    assert lp[6] == -INF and torch.isfinite(H[6]) and torch.isfinite(dz[6]).all()
    assert ((got.top_idx >= 0) & (got.top_idx < V)).all()


def test_gradient_against_differences():
    """Central differences of the definition in 64 bits, step 1e-6."""
    import nsa_lm
    dev = require_gpu()
    z, t = _rows(5, 60, F32, seed=2, banned=False)
    g = torch.Generator().manual_seed(5)
    dl, dH = torch.randn(5, generator=g), torch.randn(5, generator=g)
    zd = z.to(dev).requires_grad_()
    got = nsa_lm.token_logprobs(zd, t.to(dev))
    dz, = torch.autograd.grad((got.logp, got.entropy), zd, (dl.to(dev), dH.to(dev)))

    def loss(zz):
        _, _, _, H, logp, _ = _ref(zz, t)
        return float((logp * dl.double()).sum() + (H * dH.double()).sum())
    for s in range(3):
        v = torch.randn(z.shape, generator=g).double()
        e = 1e-6
        fd = (loss(z.double() + e * v) - loss(z.double() - e * v)) / (2 * e)
        a = dz.cpu().double()
        # the gradient's elements within 300 u of terms of at most |dl| + |dH| (|ln p| + H), p-weighted: under 10 a row
        assert abs(float((a * v).sum()) - fd) <= 300 * U * 10 * 5 * float(v.abs().max()) + 1e-8


def test_shapes_strides_and_types():
    import nsa_lm
    dev = require_gpu()
    z, t = _rows(24, 333, BF, seed=1)
    zd, td = z.to(dev), t.to(dev)
    ref = nsa_lm.token_logprobs(zd, td, 4)
    got = nsa_lm.token_logprobs(zd.view(2, 3, 4, 333), td.view(2, 3, 4).to(torch.int32), 4)
    assert got.logp.shape == (2, 3, 4) and got.top_idx.shape == (2, 3, 4, 4)
    wide = torch.zeros(24, 400, dtype=BF, device=dev)
    wide[:, 3:336] = zd
    off = torch.zeros(24 * 333 + 1, dtype=BF, device=dev)
    off[1:] = zd.flatten()
    for other in (wide[:, 3:336], off[1:].view(24, 333), zd.t().contiguous().t()):
        o = nsa_lm.token_logprobs(other, td, 4)
        # the lanes' runs follow the addresses, and the order of a row's sum with them: each result is within
        # (CHAIN + 6) u (logp, top_logp; 2 u of its terms, below 20, besides) and (2 CHAIN + 20) u 20 (entropy, S
        # below 20) of the value, so two of them are within twice that
        assert torch.equal(o.top_idx, ref.top_idx)
        C = _chain(333)
        for a, b, tol in ((o.logp, ref.logp, C + 46), (o.top_logp, ref.top_logp, C + 46),
                          (o.entropy, ref.entropy, C + 46 + (2 * C + 20) * 20)):
            fin = torch.isfinite(b)
            assert torch.equal(fin, torch.isfinite(a)) and float((a - b)[fin].abs().max()) <= 2 * tol * U
    for a, b in zip(got, ref):
        assert torch.equal(a.flatten(), b.flatten())
    one = nsa_lm.token_logprobs(zd[0], td[0], 2)
    assert one.logp.shape == () and one.top_idx.shape == (2,) and torch.equal(one.logp, ref.logp[0])
    # a padded tail of the rows' gradient: expanded and strided gradients of the results
    zz = zd.float().requires_grad_()
    nsa_lm.token_logprobs(zz, td).logp.sum().backward()
    z2 = zd.float().requires_grad_()
    torch.autograd.backward(nsa_lm.token_logprobs(z2, td).logp, torch.ones(24, 2, device=dev)[:, 0])
    assert torch.equal(zz.grad, z2.grad)
    empty = nsa_lm.token_logprobs(torch.zeros(0, 50, device=dev), torch.zeros(0, device=dev, dtype=torch.long), 3)
    assert empty.logp.shape == (0,) and empty.top_idx.shape == (0, 3)


def test_same_bits_captured_and_replayed():
    import nsa_lm
    dev = require_gpu()
    for rows, V, top in ((3, 50257, 20), (2000, 3000, 5)):
        z, t = _rows(rows, V, BF, seed=7)
        zd, td = z.to(dev).requires_grad_(), t.to(dev)
        dl, dH = torch.randn(rows, device=dev), torch.randn(rows, device=dev)

        def once():
            got = nsa_lm.token_logprobs(zd, td, top)
            dz, = torch.autograd.grad((got.logp, got.entropy), zd, (dl, dH))
            return (*(x.detach() for x in got), dz)
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
                zd.copy_((z.to(dev).float() * (1 - 0.2 * k)).to(BF))
                td.copy_((t.to(dev) + k) % V)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, once()):
                assert torch.equal(a, b)


def test_more_rows_than_one_launch():
    """2^21 rows go to one launch; the rows around the seam and the last ones."""
    dev = require_gpu()
    import nsa_lm
    rows, V = (1 << 21) + 5, 7
    g = torch.Generator(device=dev).manual_seed(0)
    z = torch.randn(rows, V, generator=g, device=dev).requires_grad_()
    t = torch.randint(0, V, (rows,), generator=g, device=dev)
    dl, dH = torch.randn(rows, generator=g, device=dev), torch.randn(rows, generator=g, device=dev)
    got = nsa_lm.token_logprobs(z, t, 2)
    dz, = torch.autograd.grad((got.logp, got.entropy), z, (dl, dH))
    C = _chain(V)
    for at in (slice(0, 4), slice((1 << 21) - 3, rows)):
        lp, lp0, p, H, logp, _ = _ref(z[at].detach(), t[at])
        # 7 elements: all terms below 8 in magnitude
        assert ((got.logp[at].double() - logp).abs() <= (C + 6 + 2 * 16) * U).all()
        assert ((got.entropy[at].double() - H).abs() <= (C + 6 + (2 * C + 20) * 8) * U).all()
        assert torch.equal(got.top_idx[at], torch.sort(z[at].detach(), dim=1, descending=True, stable=True).indices[:, :2])
        L, h = dl[at].double()[:, None], dH[at].double()[:, None]
        ref = (-p * (L + h * (lp0 + H[:, None]))).scatter_add(1, t[at][:, None], L)
        tol = (p * (L.abs() + 16 * h.abs()) * (C + 12 + 4 * 16) + 2 * L.abs() + p * h.abs() * (2 * C + 20) * 8) * U
        assert ((dz[at].double() - ref).abs() <= tol + ref.abs() * U).all()


def test_second_derivatives_are_refused():
    import nsa_lm
    dev = require_gpu()
    z = torch.randn(4, 30, device=dev, requires_grad=True)
    got = nsa_lm.token_logprobs(z, torch.zeros(4, device=dev, dtype=torch.long))
    g, = torch.autograd.grad(got.logp.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        g.square().sum().backward()


def test_refusals():
    import nsa_lm
    dev = require_gpu()
    z, t = torch.zeros(4, 50, device=dev), torch.zeros(4, dtype=torch.long, device=dev)
    for bad in [(z.cpu(), t, 0), (z.half(), t, 0), (z, t[:2], 0), (z, t.float(), 0), (z, t.cpu(), 0), (z, t, 51),
                (z, t, -1), (z, t, 2.0), (z[:, :0], t, 0), (torch.zeros(4, 100, device=dev), t, 65)]:
        with pytest.raises(AssertionError):
            nsa_lm.token_logprobs(*bad)
