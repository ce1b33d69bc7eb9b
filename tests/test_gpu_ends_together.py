"""The decoder's ends as the decoder uses them: training steps with the embedding, the
layer norms and the loss on the kernels, and generation.

Tolerances as in test_gpu_lm_together.py: float32 models of two layers, 1e-4 of the
largest value; in bf16 8 * 2^-8 of it (gradients: twice that)."""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
CFG = dict(vocab_size=203, d_model=128, n_layers=2, n_q_heads=8, n_kv_heads=2, max_seq_len=96)
ENDS = dict(norm_impl="joined", embed_impl="fused", loss_impl="pieces")


def _model(seed=0, dtype=F32, **kw):
    from nsa_model import NSATransformer
    torch.manual_seed(seed)
    m = NSATransformer(**{**CFG, **kw})
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "ln" in n:
                p.add_(0.2 * torch.randn(p.shape))
            elif p.dim() == 2:
                p.mul_(4.0)               # scores and logits of order one
    return m.cuda().to(dtype)


def _tokens(B, T, seed=0):
    return torch.randint(0, CFG["vocab_size"], (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


def _near(a, b, rel):
    a, b = a.double(), b.double()
    assert float((a - b).abs().max()) <= rel * max(1e-3, float(b.abs().max())), float((a - b).abs().max())


ARMS = [dict(attn_type="full"), dict(attn_type="nsa", attn_impl="fused", block_size=16),
        dict(attn_type="full", tie_embeddings=False, pos="rope", norm="rms"), dict(attn_type="full", pos="rope")]


@pytest.mark.parametrize("arm", ARMS, ids=["full", "nsa", "rms-rope-untied", "rope"])
@pytest.mark.parametrize("ckpt", [False, True], ids=["plain", "ckpt"])
def test_training_step(arm, ckpt):
    """Tied weights gather the embedding's gradient and the head's."""
    require_gpu()
    ref, new = _model(**arm), _model(**arm, **ENDS)
    new.load_state_dict(ref.state_dict())
    x, y = _tokens(2, 96), _tokens(2, 96, 1)
    y[0, 5:9] = -100
    out = []
    for m in (ref, new):
        m.train()
        m.grad_checkpoint = ckpt
        logits, loss = m(x, y)
        assert (logits is None) == (m is new)
        loss.backward()
        out.append((loss.detach(), {n: p.grad for n, p in m.named_parameters()}))
    _near(out[1][0], out[0][0], 1e-4)
    for n, g in out[0][1].items():
        assert (g is None) == (out[1][1][n] is None), n
        if g is not None:
            _near(out[1][1][n], g, 1e-4)
    with torch.no_grad():
        _near(new(x)[0], ref(x)[0], 1e-4)
        got, want = new.logprobs(x, y), ref.score(x, y)
        _near(got.logp, want.logp, 1e-4)
        assert got.logp.shape == got.lse.shape == y.shape


def test_training_step_autocast():
    """Mixed precision: float32 stream and parameters, bf16 branches and rows; the
    parameters' gradients come in float32."""
    require_gpu()
    arm = dict(attn_type="full", dense_impl="sdpa")
    ref, new = _model(**arm), _model(**arm, **ENDS)
    x, y = _tokens(2, 96), _tokens(2, 96, 1)
    res = []
    for m in (ref, new):
        with torch.autocast("cuda", dtype=BF):
            _, loss = m(x, y)
        loss.backward()
        res.append((loss.detach(), [p.grad for p in m.parameters()]))
    assert res[1][0].dtype == F32
    _near(res[1][0], res[0][0], 8 * 2.0 ** -8)
    for a, b in zip(res[1][1], res[0][1]):
        assert a.dtype == b.dtype == F32
        _near(a, b, 16 * 2.0 ** -8)


def test_captured_training_steps():
    """A step of the whole model in one graph, replayed over changing tokens and with
    eager work between; equal to the eager step's bits."""
    require_gpu()
    m = _model(attn_type="full", dense_impl="sdpa", dtype=BF, **ENDS)
    x, y = _tokens(2, 96), _tokens(2, 96, 1)
    params = list(m.parameters())

    def one():
        loss = m(x, y)[1]
        return [loss.detach(), *torch.autograd.grad(loss, params)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = one()
    names = ["loss", *(n for n, _ in m.named_parameters())]
    for k in range(3):
        x.copy_(_tokens(2, 96, 10 + k))
        y.copy_(_tokens(2, 96, 20 + k))
        graph.replay()
        torch.cuda.synchronize()
        for n, a, b in zip(names, got, one()):
            # (the library's attention and products keep their bits from run to run or not;
            # what follows from this framework's ends is compared where nothing else comes before)
            _near(a, b, 8 * 2.0 ** -8)
        torch.cuda.synchronize()


@pytest.mark.parametrize("kw,dtype", [(dict(), F32), (dict(), BF), (dict(pos="rope", norm="rms"), F32)], ids=str)
def test_generation_is_the_forward(kw, dtype):
    require_gpu()
    m = _model(attn_type="full", dtype=dtype, **ENDS, **kw).eval()
    B, T = 3, 60
    x = _tokens(B, T, 4)
    with torch.no_grad():
        want = m(x)[0]
    lens = [30, 17, 1]
    caches = m.paged_caches(B, 96, page_size=16)
    caches[0].reserve([n + 20 for n in lens])
    tol = 1e-4 if dtype == F32 else 8 * 2.0 ** -8
    pre = m.prefill(x[:, :30], caches, lens)
    for b, n in enumerate(lens):
        _near(pre[b, :n], want[b, :n], tol)
    pos = torch.tensor(lens).cuda()
    for s in range(20):
        logits = m.step(x.gather(1, pos[:, None])[:, 0], caches)
        for b in range(B):
            _near(logits[b], want[b, lens[b] + s], tol)
        pos += 1


def test_a_target_outside_the_vocabulary_makes_the_loss_nan():
    require_gpu()
    m = _model(attn_type="full", **ENDS)
    x, y = _tokens(2, 16), _tokens(2, 16, 1)
    y[1, 3] = CFG["vocab_size"]
    loss = m(x, y)[1]
    loss.backward()
    assert loss.isnan() and m.lm_head.weight.grad.isnan().any()
    y[:] = -100
    assert m(x, y)[1].isnan()              # nothing to average, as F.cross_entropy's


def test_options():
    from nsa_model import NSATransformer
    for bad in (dict(norm_impl="fused"), dict(norm_impl="fast"), dict(loss_impl="fast"), dict(embed_impl="fast")):
        with pytest.raises(AssertionError):
            NSATransformer(**CFG, **bad)
