"""Every token of the vocabulary counts once in nsa_lm.linear_logprobs' log sums, and unlike types in
the large tiles.

Column c of w is between -1 and 0 (multiples of 1 / 64) where v // 8 = c modulo 64 and -200 elsewhere: a weight of 0
in float32.  x[n] is a unit vector, so that the logits are exact in either type and a row's sum is
that of every 64th run of eight tokens: a run that is missed or counted twice moves the log sum by at least
e^-1 8 / (V / 64).  u = 2^-24: a weight is within 6 u (its exponent, the exponential), the sum has at most 64
additions in a tile, one for each of a workgroup's tiles (42 at most here) and 80 in the joins, the logarithm
4 u of its size: within 256 u + 4 u lse, a tenth of that at V = 2^20 and less below.
"""

import pytest
import torch

from nsa_testlib import require_gpu
from test_gpu_head import _check

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


@pytest.mark.parametrize("N,V,dtype", [(32, 140001, BF), (64, 140001, BF), (128, 70001, BF), (300, 20001, BF), (2100, 13001, BF),
                                       (16, 1048577, BF), (32, 140001, F32), (64, 70001, F32), (128, 70001, F32),
                                       (500, 40001, F32), (2100, 13001, F32), (16, 1048577, F32)])
def test_every_token_counts_once(N, V, dtype):
    import nsa_lm
    dev = require_gpu()
    v = torch.arange(V, device=dev)
    w = torch.full((V, 64), -200.0, device=dev)
    w[v, v // 8 % 64] = -((v * 37) % 65).float() / 64
    col = w.double()
    lse_of = torch.logsumexp(col, 0)
    w = w.to(dtype)
    for first in range(0, 64, N):                          # (all columns, whatever N)
        c = (first + torch.arange(N, device=dev)) % 64
        x = torch.zeros(N, 64, device=dev, dtype=dtype)
        x[torch.arange(N, device=dev), c] = 1
        t = torch.randint(0, V, (N,), device=dev, generator=torch.Generator(dev).manual_seed(N))
        got = nsa_lm.linear_logprobs(x, w, t)
        tol = (256 + 4 * lse_of[c].abs()) * U
        assert float((tol * (V / 64) / 8 * 2.72).max()) < 0.2   # (a run of eight is seen)
        err = (got.lse.double() - lse_of[c]).abs() - tol
        assert (err <= 0).all(), float(err.max())
        want = col[t, c] - lse_of[c]
        assert ((got.logp.double() - want).abs() <= tol + 4 * U * want.abs()).all()


@pytest.mark.parametrize("N,V,D,xd,wd", [(2100, 5300, 72, BF, F32), (2100, 5300, 72, F32, BF), (2050, 6000, 128, BF, F32),
                                         (22100, 13000, 64, BF, F32), (8000, 13001, 40, F32, BF)])
def test_unlike_types_in_large_tiles(N, V, D, xd, wd):
    _check(N, V, D, xd, wd, seed=N + V)
