"""The decoder's options that take a module's parameters in its place (``norm_impl``, ``embed_impl``,
``loss_impl='pieces'``) leave modules that are not plain ones alone.  On the CPU: such a
module is called, so that no kernel runs."""

import pytest
import torch
import torch.nn as nn

CFG = dict(vocab_size=31, d_model=32, n_layers=2, n_q_heads=4, n_kv_heads=2, max_seq_len=16, attn_type="full")


def _pair(**kw):
    from nsa_model import NSATransformer
    torch.manual_seed(0)
    ref = NSATransformer(**CFG)
    new = NSATransformer(**CFG, **kw)
    new.load_state_dict(ref.state_dict())
    return ref, new


def _tokens(seed=0):
    return torch.randint(0, CFG["vocab_size"], (2, 12), generator=torch.Generator().manual_seed(seed))


def _hooked(name):
    def change(m):
        getattr(m, name).register_forward_hook(lambda mod, args, out: out * 1.5)
    return change


def _replaced(name, kind, **kw):
    def change(m):
        old = getattr(m, name)
        new = kind(old.num_embeddings, old.embedding_dim, **kw)
        new.weight = old.weight
        setattr(m, name, new)
    return change


class Louder(nn.Embedding):
    def forward(self, x):
        return 2 * super().forward(x)


def _own_forward(m):
    table = m.tok_emb
    table.forward = lambda t: 3 * nn.functional.embedding(t, table.weight)


@pytest.mark.parametrize("change", [_hooked("tok_emb"), _hooked("pos_emb"), _replaced("tok_emb", Louder),
                                    _replaced("tok_emb", nn.Embedding, padding_idx=3),
                                    _replaced("tok_emb", nn.Embedding, scale_grad_by_freq=True),
                                    _replaced("pos_emb", nn.Embedding, max_norm=0.01), _own_forward],
                         ids=["hook", "hook-positions", "subclass", "padding", "freq", "max_norm", "forward"])
def test_embeddings(change):
    ref, new = _pair(embed_impl="fused")
    out = []
    for m in (ref, new):
        change(m)
        logits, loss = m(_tokens(), _tokens(1))
        loss.backward()
        out.append((logits, loss, *(p.grad for p in m.parameters())))
    for a, b in zip(*out):
        assert torch.equal(a, b)


class Shifted(nn.LayerNorm):
    def forward(self, x):
        return super().forward(x) + 1


@pytest.mark.parametrize("kind", ["hook", "pre-hook", "subclass", "parametrized"])
def test_norms(kind):
    ref, new = _pair(norm_impl="joined")
    x, y = _tokens(), _tokens(1)
    out = []
    for m in (ref, new):
        for blk in (*m.blocks, m):
            for name in ("ln1", "ln2", "ln_f"):
                ln = getattr(blk, name, None)
                if ln is None:
                    continue
                if kind == "hook":
                    ln.register_forward_hook(lambda mod, args, o: o * 0.5)
                elif kind == "pre-hook":
                    ln.register_forward_pre_hook(lambda mod, args: (args[0] * 2 + 1,))
                elif kind == "parametrized":
                    nn.utils.parametrize.register_parametrization(ln, "weight", nn.Softplus())
                else:
                    s = Shifted(CFG["d_model"])
                    s.load_state_dict(ln.state_dict())
                    setattr(blk, name, s)
        loss = m(x, y)[1]
        loss.backward()
        out.append((loss, *(p.grad for p in m.parameters())))
    for a, b in zip(*out):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-7)      # (additions in another place: the same rounding of them)


def _bias(m):
    m.lm_head.bias = nn.Parameter(torch.ones(CFG["vocab_size"]))


class Adapter(nn.Module):
    def __init__(self, base):
        super().__init__()
        self.base, self.weight = base, base.weight

    def forward(self, x):
        return self.base(x) + 1


@pytest.mark.parametrize("change", [_bias, _hooked("lm_head"), lambda m: setattr(m, "lm_head", Adapter(m.lm_head)),
                                    lambda m: nn.utils.parametrize.register_parametrization(m.lm_head, "weight", nn.Tanh())],
                         ids=["bias", "hook", "adapter", "parametrized"])
def test_heads_are_refused(change):
    _, new = _pair(loss_impl="pieces")
    change(new)
    with pytest.raises(AssertionError, match="lm_head"):
        new(_tokens(), _tokens(1))
    with pytest.raises(AssertionError, match="lm_head"):
        new.logprobs(_tokens(), _tokens(1))
    assert new(_tokens())[0].shape == (2, 12, CFG["vocab_size"])      # its logits: called as ever


def test_plain_modules_take_the_kernels():
    """... which refuse CPU tensors."""
    for kw in (dict(embed_impl="fused"), dict(norm_impl="joined"), dict(loss_impl="pieces")):
        _, new = _pair(**kw)
        with pytest.raises(AssertionError, match="GPU"):
            new(_tokens(), _tokens(1))
