"""CPU checks of the decoder's ends (layer norm, embedding, log probabilities from the
rows): what the C entry points refuse before any launch, and what the Python ones do
of CPU tensors."""

import os

import pytest
import torch

SHAPE, DTYPE, ARG, WORKSPACE = -1, -2, -3, -5


def _lib():
    import _nsa_lib
    if not os.path.exists(_nsa_lib.LIB_PATH):
        pytest.skip("libnsa_hip.so not built")
    return _nsa_lib.load()


def test_lnorm_refusals():
    lib = _lib()
    no = [None] * 7
    assert lib.nsa_lnorm_fwd(*no, 0, 64, 1e-5, 0, 0, 0, 0, None) == 0            # no rows: nothing to do
    for rows, D in ((4, 0), (-1, 64), (4, (1 << 24) + 1), (1 << 31, 8)):
        assert lib.nsa_lnorm_fwd(*no, rows, D, 1e-5, 0, 0, 0, 0, None) == SHAPE
        assert lib.nsa_lnorm_bwd_workspace(rows, D, None) == 0
        assert lib.nsa_lnorm_bwd(*[None] * 10, 0, rows, D, 0, 0, 0, 0, None) == SHAPE
    for types in ((2, 0, 0, 0), (0, 5, 0, 0), (0, 0, 3, 0), (0, 0, 0, 3), (1, 0, 0, 0)):   # last: no residual, two types
        assert lib.nsa_lnorm_fwd(*no, 4, 64, 1e-5, *types, None) == DTYPE
    assert lib.nsa_lnorm_fwd(*no, 4, 64, 1e-5, 0, 0, 0, 0, None) == ARG
    assert lib.nsa_lnorm_bwd(*[None] * 10, 0, 4, 64, 0, 0, 0, 0, None) == ARG
    assert lib.nsa_lnorm_bwd(*[None] * 10, 0, 4, 64, 0, 0, 0, 3, None) == DTYPE
    assert lib.nsa_lnorm_bwd_workspace(1000, 768, None) >= 2 * 768 * 4


def test_embed_refusals():
    lib = _lib()

    def fwd(n=4, T=2, V=10, P=3, D=8, w=0, pw=0, out=0, pos=None):
        return lib.nsa_embed_fwd(None, None, None, pos, None, n, T, V, P, D, 1.0, w, pw, out, None)
    assert fwd(n=0) == 0 and fwd() == ARG
    for bad in (dict(n=-1), dict(n=1 << 31), dict(V=0), dict(V=1 << 31), dict(D=0), dict(D=(1 << 20) + 1)):
        assert fwd(**bad) == SHAPE, bad
    for bad in (dict(w=2), dict(out=3), dict(pw=2, pos=16)):
        assert fwd(**bad) == DTYPE, bad
    assert fwd(P=0, pos=16) == SHAPE and fwd(T=0, pos=16) == SHAPE and fwd(P=0) == ARG

    def bwd(index=16, n=4, T=2, V=10, D=8, dy=0, w=0, at=None):
        return lib.nsa_embed_bwd(index, at, at, None, 0, n, T, V, D, 1.0, dy, w, None)
    for bad in (dict(n=0), dict(V=0), dict(D=0), dict(index=None, T=3), dict(index=None, T=0),
                dict(index=None, T=4, V=3)):
        assert bwd(**bad) == SHAPE, bad
    assert bwd(dy=2) == DTYPE and bwd(w=3) == DTYPE and bwd() == ARG and bwd(at=16) == WORKSPACE
    size = lib.nsa_embed_bwd_workspace
    assert size(-1, 8, 1) == 0 and size(4, 0, 1) == 0 and size(0, 8, 1) == 16
    assert size(1000, 64, 1) > size(1000, 64, 0) >= 2 * 64 * 4


def test_embed_of_no_tokens():
    lib = _lib()
    for T in (0, 4):   # [.., 0] and [0, 4], by position
        assert lib.nsa_embed_fwd(None, None, None, 16, None, 0, T, 10, 3, 8, 1.0, 0, 0, 0, None) == 0


def test_head_refusals():
    lib = _lib()

    def fwd(N=4, V=10, D=8, xt=1, wt=1, target=None, logp=None, x=None):
        return lib.nsa_head_fwd(x, x, target, logp, x, None, 0, N, V, D, xt, wt, None)

    def bwd(N=4, V=10, D=8, xt=1, wt=1, x=None, dlogp=None, dx=16):
        return lib.nsa_head_bwd(x, x, None, None, x, dlogp, None, dx, None, None, 0, N, V, D, xt, wt, None)
    assert fwd(N=0) == 0 and bwd(N=0) == SHAPE
    for bad in (dict(N=-1), dict(N=(1 << 22) + 1), dict(V=0), dict(V=(1 << 24) + 1), dict(D=0), dict(D=65537)):
        assert fwd(**bad) == SHAPE and bwd(**bad) == SHAPE, bad
        full = {**dict(N=4, V=10, D=8), **bad}
        assert lib.nsa_head_fwd_workspace(*full.values(), 1, 1, 1, None) == 0
        assert lib.nsa_head_bwd_workspace(*full.values(), 1, 1, 1, None) == 0
    for bad in (dict(xt=2), dict(wt=3)):
        assert fwd(**bad) == DTYPE and bwd(**bad) == DTYPE, bad
    assert fwd() == ARG and fwd(x=16, target=16) == ARG and fwd(x=16, logp=16) == ARG and fwd(x=16) == WORKSPACE
    assert bwd() == ARG and bwd(x=16, dx=None) == ARG and bwd(x=16, dlogp=16) == ARG and bwd(x=16) == WORKSPACE


def test_workspaces_off_16_bytes_are_refused():
    lib = _lib()
    big = 1 << 40
    assert lib.nsa_head_fwd(16, 16, None, None, 16, 24, big, 4, 10, 8, 1, 1, None) == ARG
    assert lib.nsa_head_bwd(16, 16, None, None, 16, None, 16, 16, None, 24, big, 4, 10, 8, 1, 1, None) == ARG
    assert lib.nsa_embed_bwd(16, 16, 16, 24, big, 4, 2, 10, 8, 1.0, 0, 0, None) == ARG


def test_the_backward_never_holds_the_logits():
    """What the backward takes beside its results stays near 1 GB of dz, however large
    the vocabulary: dz of 32768 rows x 131072 tokens would be 8.6 GB in bf16."""
    lib = _lib()
    D = 512
    for N, V in ((32768, 32000), (32768, 131072), (131072, 131072)):
        size = lib.nsa_head_bwd_workspace(N, V, D, 1, 1, 1, None)
        assert 0 < size <= (1 << 30) + N * D * 4 + (512 << 20), (N, V, size)


def test_cpu_tensors_are_refused():
    import nsa_lm
    x, w, t = torch.zeros(3, 8), torch.ones(8), torch.zeros(3, dtype=torch.long)
    for call in (lambda: nsa_lm.add_layer_norm(x, x, w), lambda: nsa_lm.embed(t, x), lambda: nsa_lm.linear_logprobs(x, x, t)):
        with pytest.raises(AssertionError):
            call()
