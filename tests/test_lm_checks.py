"""CPU checks of the operators around the attention: what the C entry points
refuse before any launch, the Python refusals of CPU tensors, and the page
addressing (run on the host)."""

import os
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "openbox-llm_amd")
HIPCC = "/opt/rocm/bin/hipcc"
SHAPE, DTYPE, ARG, WORKSPACE = -1, -2, -3, -5


def _lib():
    import _nsa_lib
    if not os.path.exists(_nsa_lib.LIB_PATH):
        pytest.skip("libnsa_hip.so not built")
    return _nsa_lib.load()


def test_norm_refusals():
    lib = _lib()
    no = [None] * 7
    assert lib.nsa_norm_fwd(*no, 0, 64, 1e-5, 0, 0, 0, 0, None) == 0            # no rows: nothing to do
    assert lib.nsa_norm_fwd(*no, 4, 0, 1e-5, 0, 0, 0, 0, None) == SHAPE
    assert lib.nsa_norm_fwd(*no, -1, 64, 1e-5, 0, 0, 0, 0, None) == SHAPE
    assert lib.nsa_norm_fwd(*no, 4, (1 << 24) + 1, 1e-5, 0, 0, 0, 0, None) == SHAPE
    for types in ((2, 0, 0, 0), (0, 5, 0, 0), (0, 0, 3, 0), (0, 0, 0, 2), (1, 0, 0, 0)):   # last: no residual, two types
        assert lib.nsa_norm_fwd(*no, 4, 64, 1e-5, *types, None) == DTYPE
    assert lib.nsa_norm_fwd(*no, 4, 64, 1e-5, 0, 0, 0, 0, None) == ARG
    assert lib.nsa_norm_bwd(*[None] * 9, 0, 4, 64, 0, 0, 0, 0, None) == ARG
    assert lib.nsa_norm_bwd(*[None] * 9, 0, 0, 64, 0, 0, 0, 0, None) == SHAPE
    assert lib.nsa_norm_bwd(*[None] * 9, 0, 4, 64, 0, 0, 0, 3, None) == DTYPE
    assert lib.nsa_norm_bwd_workspace(4, 0, None) == 0 and lib.nsa_norm_bwd_workspace(-1, 8, None) == 0
    assert lib.nsa_norm_bwd_workspace(1000, 768, None) >= 768 * 4


def test_logprob_refusals():
    lib = _lib()
    no = [None] * 8
    assert lib.nsa_logprob_fwd(*no, 0, 0, 100, 0, 0, None) == 0
    for rows, V, k in ((1, 0, 0), (-1, 10, 0), (1, 10, 11), (1, 100, 65), (1, 100, -1), (1, (1 << 28) + 1, 0),
                       ((1 << 25) + 1, 10, 0)):
        assert lib.nsa_logprob_fwd(*no, 0, rows, V, k, 0, None) == SHAPE
        assert lib.nsa_logprob_workspace(rows, V, k, None) == 0
    assert lib.nsa_logprob_fwd(*no, 0, 1, 100, 0, 2, None) == DTYPE
    assert lib.nsa_logprob_fwd(*no, 0, 1, 100, 0, 0, None) == ARG
    assert lib.nsa_logprob_bwd(*[None] * 7, 1, 100, 3, None) == DTYPE
    assert lib.nsa_logprob_bwd(*[None] * 7, 1, 100, 0, None) == ARG
    assert lib.nsa_logprob_workspace(1, 100000, 64, None) > lib.nsa_logprob_workspace(1, 100000, 0, None) > 16


def test_paged_refusals():
    lib = _lib()
    no = [None] * 11

    def attend(B=1, Hq=4, Hkv=2, D=64, P=16, mp=3, n=5, dt=1):
        return lib.nsa_paged_attend(*no, 0, B, Hq, Hkv, D, P, mp, n, 0.1, dt, None)
    assert attend(B=0) == 0
    for bad in (dict(B=-1), dict(Hq=3), dict(Hkv=0), dict(D=48), dict(P=24), dict(P=0), dict(mp=0), dict(n=0),
                dict(P=1 << 20, mp=1 << 20), dict(Hq=8192), dict(B=70000)):
        assert attend(**bad) == SHAPE, bad
        assert "n" in bad or "B" in bad and bad["B"] < 0 or \
            lib.nsa_paged_workspace(*{**dict(B=1, Hq=4, Hkv=2, D=64, P=16, mp=3), **bad}.values(), 1, None) == 0
    assert attend(dt=2) == DTYPE
    assert attend() == ARG
    no = [None] * 8

    def append(B=1, Hkv=2, T=4, D=64, P=16, mp=3, n=5, dt=1):
        return lib.nsa_paged_append(*no, B, Hkv, T, D, P, mp, n, dt, None)
    assert append(B=0) == 0 and append(T=-1) == SHAPE and append(D=40) == SHAPE and append(dt=2) == DTYPE
    assert append() == ARG


def test_cpu_tensors_are_refused():
    import nsa_lm
    import nsa_paged
    x, w = torch.zeros(3, 8), torch.ones(8)
    for call in (lambda: nsa_lm.add_rms_norm(x, x, w), lambda: nsa_lm.add_rms_norm_q8(x, x, w),
                 lambda: nsa_lm.token_logprobs(x),
                 lambda: nsa_paged.PagedKVCache(1, 1, 16, 20, 16, device="cpu"),
                 lambda: nsa_paged.paged_attend(torch.zeros(1, 1, 16), torch.zeros(2, 1, 16, 16),
                                                torch.zeros(2, 1, 16, 16), torch.zeros(1, 1, dtype=torch.int32),
                                                torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(AssertionError):
            call()


@pytest.mark.skipif(not (os.path.exists(HIPCC) or shutil.which("hipcc")), reason="needs hipcc")
def test_page_addressing_on_the_host(tmp_path):
    """Rows of good, bad and missing pages: every offset inside the pages
    (tests/host/check_paged_runs.hip)."""
    exe = tmp_path / "check_paged_runs"
    subprocess.run([HIPCC, "-std=c++17", "-O1", "--offload-arch=gfx950", f"-I{ROOT}/include", f"-I{PKG}/csrc",
                    os.path.join(ROOT, "tests", "host", "check_paged_runs.hip"), "-o", str(exe)],
                   check=True, capture_output=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    print(r.stdout)
    assert r.returncode == 0, r.stdout
