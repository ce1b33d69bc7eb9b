"""The operators around the attention as a decoder uses them: training steps
with the fused norms and loss, and generation over paged caches.

Tolerances: float32 models of two layers; the two forms of a norm or a loss
differ by a few dozen float32 roundings (2^-24 each) of values of order one,
and each layer's products pass them on with weights of norm about one: 1e-4
relative to the largest value leaves a factor of ten over the sum of them.  In
bf16 every matrix product's output carries 2^-8 of its size; eight of them in a
row over two layers: 8 * 2^-8 of the largest value.
"""

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
CFG = dict(vocab_size=203, d_model=128, n_layers=2, n_q_heads=8, n_kv_heads=2, max_seq_len=96, norm="rms",
           ffn="swiglu", ffn_hidden=160, tie_embeddings=False)


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


@pytest.mark.parametrize("arm", [dict(attn_type="full"), dict(attn_type="nsa", attn_impl="fused", block_size=16)],
                         ids=["full", "nsa"])
@pytest.mark.parametrize("ckpt", [False, True], ids=["plain", "ckpt"])
def test_training_step(arm, ckpt):
    require_gpu()
    ref = _model(pos="rope", **arm)
    new = _model(pos="rope", norm_impl="fused", loss_impl="fused", **arm)
    new.load_state_dict(ref.state_dict())
    x, y = _tokens(2, 96), _tokens(2, 96, 1)
    y[0, 5:9] = -100
    out = []
    for m in (ref, new):
        m.train()
        m.grad_checkpoint = ckpt
        logits, loss = m(x, y)
        loss.backward()
        out.append((logits.detach(), loss.detach(), {n: p.grad for n, p in m.named_parameters()}))
    _near(out[1][0], out[0][0], 1e-4)
    _near(out[1][1], out[0][1], 1e-4)
    for n, g in out[0][2].items():
        assert (g is None) == (out[1][2][n] is None), n
        if g is not None:
            _near(out[1][2][n], g, 1e-4)


def test_training_step_autocast():
    """Mixed precision: float32 stream and parameters, bf16 branches."""
    require_gpu()
    m = _model(attn_type="full", dense_impl="sdpa", pos="rope", norm_impl="fused", loss_impl="fused")
    ref = _model(attn_type="full", dense_impl="sdpa", pos="rope")
    x, y = _tokens(2, 96), _tokens(2, 96, 1)
    res = []
    for mm in (ref, m):
        with torch.autocast("cuda", dtype=BF):
            logits, loss = mm(x, y)
        loss.backward()
        res.append((loss.detach(), [p.grad for p in mm.parameters()]))
    assert res[1][0].dtype == F32
    _near(res[1][0], res[0][0], 8 * 2.0 ** -8)
    for a, b in zip(res[1][1], res[0][1]):
        assert a.dtype == b.dtype == F32
        _near(a, b, 16 * 2.0 ** -8)


KINDS = [dict(pos="rope"), dict(pos="learned"), dict(pos="rope", norm_impl="fused"), dict(pos="rope", norm="layer")]


# (the library's attention kernels take 16-bit inputs only)
@pytest.mark.parametrize("kw,dtype", [(k, d) for k in KINDS for d in (F32, BF)] +
                         [(dict(pos="rope", dense_impl="sdpa", norm_impl="fused"), BF)], ids=str)
def test_generation_is_the_forward(kw, dtype):
    """Prefill and steps over paged caches give the forward's logits row by row,
    with sequences of unlike lengths and pages taken as they grow."""
    require_gpu()
    m = _model(attn_type="full", dtype=dtype, **kw).eval()
    B, T = 3, 80
    x = _tokens(B, T, 4)
    with torch.no_grad():
        want = m(x)[0]
    lens = [40, 17, 1]
    caches = m.paged_caches(B, 96, page_size=16)
    caches[0].reserve(lens)
    tol = 1e-4 if dtype == F32 else 8 * 2.0 ** -8
    pre = m.prefill(x[:, :40], caches, lens)
    for b, n in enumerate(lens):
        _near(pre[b, :n], want[b, :n], tol)
    pos = torch.tensor(lens).cuda()
    for s in range(40):
        caches[0].reserve([n + s + 1 for n in lens])
        logits = m.step(x.gather(1, pos[:, None])[:, 0], caches)
        for b in range(B):
            _near(logits[b], want[b, lens[b] + s], tol)
        pos += 1
    for c in caches:
        assert c.lens.tolist() == [n + 40 for n in lens]


def test_captured_generation_with_log_probabilities():
    """Greedy generation in one graph a token: step, then the chosen token with
    its log probability and entropy; equal to the eager loop's bits."""
    import nsa_lm
    require_gpu()
    m = _model(attn_type="full", dtype=BF, pos="rope", norm_impl="fused").eval()
    x = _tokens(2, 20, 9)

    def start():
        caches = m.paged_caches(2, 64, page_size=16)
        caches[0].reserve(64)
        logits = m.prefill(x, caches)[:, -1]
        return caches, nsa_lm.token_logprobs(logits, None, 1).top_idx[:, 0].clone()

    def one(tok, caches):
        got = nsa_lm.token_logprobs(m.step(tok, caches), None, 3)
        return got.top_idx, got.top_logp, got.entropy
    caches, tok = start()
    eager = []
    for _ in range(12):
        eager.append(one(tok, caches))
        tok = eager[-1][0][:, 0].clone()
    caches, tok = start()
    lens0 = [c.lens.clone() for c in caches]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(tok, caches)
    torch.cuda.current_stream().wait_stream(side)
    for c, n in zip(caches, lens0):
        c.lens = n
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one(tok, caches)
        tok.copy_(out[0][:, 0])
        for c, n in zip(caches, lens0):
            n.copy_(c.lens)
    for s in range(12):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager[s]):
            assert torch.equal(a, b), s


def test_eager_steps_beside_a_capture_that_has_not_run():
    """A step's rotation does not come from memory that a capture has only
    recorded the writing of."""
    require_gpu()
    m = _model(attn_type="full", pos="rope").eval()
    x = _tokens(2, 30, 5)
    with torch.no_grad():
        want = m(x)[0]

    def start(max_len, n):
        caches = m.paged_caches(2, max_len, page_size=16)
        caches[0].reserve(max_len)
        m.prefill(x[:, :n], caches)
        return caches
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(x[:, 20], start(64, 20))
    torch.cuda.current_stream().wait_stream(side)
    caches = start(96, 25)
    tok = x[:, 25].contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step(tok, caches)
    eager = start(96, 10)
    for s in range(10, 30):
        _near(m.step(x[:, s], eager), want[:, s], 1e-4)
    for s in range(25, 30):       # every replay is a step further
        tok.copy_(x[:, s])
        graph.replay()
        torch.cuda.synchronize()
        _near(out, want[:, s], 1e-4)
    assert all(c.lens.tolist() == [30, 30] for c in caches + eager)


def test_layers_steps_under_gradients():
    """A layer's step has no gradient; its prefill has the forward's."""
    require_gpu()
    m = _model(attn_type="full", pos="rope")
    at = m.blocks[0].attn
    x = torch.randn(2, 20, CFG["d_model"], generator=torch.Generator().manual_seed(0)).cuda().requires_grad_()
    cache = at.paged_cache(2, 32, page_size=16)
    cache.reserve(21)
    y = at.prefill(x, cache)
    want = at(x)
    _near(y.detach(), want.detach(), 1e-5)
    g = torch.ones_like(y)
    _near(torch.autograd.grad(y, x, g)[0], torch.autograd.grad(want, x, g)[0], 1e-5)
    assert not at.step(x[:, 0], cache).requires_grad


def test_score():
    require_gpu()
    m = _model(attn_type="full", pos="rope").eval()
    x, y = _tokens(2, 30), _tokens(2, 30, 3)
    y[1, 4] = -100
    got = m.score(x, y, top=2)
    with torch.no_grad():
        logits, loss = m(x, y)
    lp = torch.log_softmax(logits.double(), -1)
    keep = y != -100
    _near(got.logp[keep], lp.gather(2, y.clamp(min=0)[..., None])[..., 0][keep], 1e-5)
    assert got.logp[1, 4] == 0 and abs(float(-got.logp.sum() / keep.sum()) - float(loss)) < 1e-5
    assert torch.equal(got.top_idx[..., 0], logits.argmax(-1)) and got.entropy.shape == (2, 30)


def test_8_bit_rows_in_a_product():
    """q and its scales are what an 8-bit product takes: q's own values times the
    scales give y within half a step of e4m3 (2^-4 a value)."""
    import nsa_lm
    require_gpu()
    g = torch.Generator().manual_seed(0)
    x, r = (torch.randn(64, 256, generator=g).to(BF).cuda() for _ in range(2))
    w = torch.ones(256, device="cuda", dtype=BF)
    q, s, h = nsa_lm.add_rms_norm_q8(x, r, w, eps=1e-5)
    y, h2 = nsa_lm.add_rms_norm(x, r, w, eps=1e-5, out_dtype=F32)
    assert torch.equal(h, h2)
    m = torch.randn(256, 32, generator=g).cuda()
    got = (q.float() @ m) * s[:, None]
    # each of the 256 terms within 2^-4 |y m| (and 2^-10 s |m| near zero)
    tol = (y.abs() @ m.abs()) * 2.0 ** -4 + s[:, None] * 2.0 ** -10 * m.abs().sum(0)
    assert ((got - y @ m).abs() <= tol * 1.001).all()


def test_refusals():
    from nsa_model import NSATransformer
    require_gpu()
    with pytest.raises(AssertionError):
        NSATransformer(**{**CFG, "norm": "layer"}, norm_impl="fused")
    with pytest.raises(AssertionError):
        NSATransformer(**CFG, norm_impl="fast")
    with pytest.raises(AssertionError):
        NSATransformer(**CFG, loss_impl="fast")
    m = _model(attn_type="nsa", attn_impl="ref", block_size=16)
    with pytest.raises(AssertionError):
        m.paged_caches(2)
    with pytest.raises(AssertionError):
        _model(attn_type="full").paged_caches(2, 97)
