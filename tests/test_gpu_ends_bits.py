"""A training step of this framework's own kernels alone (embedding, layer norms, log probabilities without logits):
captured and replayed, it has the eager step's bits in every output."""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("B,T,V,D,rows,table", [(2, 96, 203, 128, BF, BF), (3, 333, 1009, 200, BF, F32), (2, 33, 101, 72, F32, F32),
                                                (8, 700, 2500, 256, BF, F32)])
def test_captured_steps_have_the_eager_bits(B, T, V, D, rows, table):
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator(dev).manual_seed(D)

    def rnd(*s):
        return torch.randn(*s, generator=g, device=dev)
    ps = [rnd(V, D).to(table), (0.2 * rnd(T, D)).to(table), (1 + 0.2 * rnd(D)).to(table), rnd(D).to(table),
          (1 + 0.2 * rnd(D)).to(table)]
    ps = [p.requires_grad_() for p in ps]
    tok = torch.empty(B, T, dtype=torch.long, device=dev)
    tgt = torch.empty_like(tok)

    def fill(seed):
        g = torch.Generator(dev).manual_seed(seed)
        tok.copy_(torch.randint(0, V, (B, T), generator=g, device=dev) % (1 + seed * 31 % V))   # (long and short runs of a token)
        tgt.copy_(torch.randint(0, V, (B, T), generator=g, device=dev))
        tgt[torch.rand(B, T, generator=g, device=dev) < 0.1] = -100
        tok[0, :seed % 5] = -1

    def step():
        x = nsa_lm.embed(tok, ps[0], 0.5, ps[1], out_dtype=F32)
        y, h = nsa_lm.add_layer_norm(x.to(rows), x, ps[2], ps[3], out_dtype=rows)
        z, _ = nsa_lm.add_layer_norm(y, h, ps[4], None, out_dtype=rows)
        r = nsa_lm.linear_logprobs(z, ps[0], tgt)
        grads = torch.autograd.grad((r.logp, r.lse), ps, (-torch.ones_like(r.logp), 0.01 * torch.ones_like(r.lse)))
        return [r.logp.detach(), r.lse.detach(), h.detach(), *grads]
    fill(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(2, 6):
        fill(k * 7)
        graph.replay()
        torch.cuda.synchronize()
        got_now = [a.clone() for a in got]
        want = step()
        for i, (a, b) in enumerate(zip(got_now, want)):
            assert torch.equal(a, b), (k, i)
            assert bool(a.isfinite().all()) and bool(a.any()), (k, i)
        torch.cuda.synchronize()


@pytest.mark.parametrize("N,V,D,rows,table", [(5, 300, 64, BF, BF), (300, 1009, 200, BF, F32), (1500, 2500, 256, BF, BF), (40, 500, 72, F32, F32),
                                              (700, 3000, 96, F32, F32), (9000, 200000, 64, BF, BF)])
def test_nothing_is_read_that_was_not_written(N, V, D, rows, table):
    """Workspaces and outputs that start as 0xff bytes and NaN: the same bits."""
    import nsa_lm
    dev = require_gpu()
    g = torch.Generator(dev).manual_seed(N)
    w = torch.randn(V, D, generator=g, device=dev).to(table).requires_grad_()
    p = torch.randn(N, D, generator=g, device=dev).to(table).requires_grad_()
    a = (1 + 0.1 * torch.randn(D, generator=g, device=dev)).to(table).requires_grad_()
    tok = torch.randint(-2, V // 3, (1, N), generator=g, device=dev)
    tgt = torch.randint(-5, V, (1, N), generator=g, device=dev)

    def step():
        x = nsa_lm.embed(tok, w, 1.0, p, out_dtype=rows)
        y, h = nsa_lm.add_layer_norm(x, x, a, a, out_dtype=rows)
        r = nsa_lm.linear_logprobs(y, w, tgt)
        return [x.detach(), y.detach(), h.detach(), r.logp.detach(), r.lse.detach(),
                *torch.autograd.grad((r.logp, r.lse), (w, p, a), (torch.ones_like(r.logp), 0.5 * torch.ones_like(r.lse)))]
    want = step()
    was = torch.are_deterministic_algorithms_enabled(), torch.is_deterministic_algorithms_warn_only_enabled()
    fill = torch.utils.deterministic.fill_uninitialized_memory
    try:
        torch.use_deterministic_algorithms(True, warn_only=True)
        torch.utils.deterministic.fill_uninitialized_memory = True
        assert torch.empty(4, device=dev).isnan().all()
        got = step()
    finally:
        torch.utils.deterministic.fill_uninitialized_memory = fill
        torch.use_deterministic_algorithms(was[0], warn_only=was[1])
    for i, (b, c) in enumerate(zip(want, got)):
        assert torch.equal(b, c), i
