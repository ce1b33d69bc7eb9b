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
