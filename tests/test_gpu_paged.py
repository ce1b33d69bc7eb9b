"""nsa_paged against attention in 64 bits over the same keys.

Tolerance of an output element, u = 2^-24, E = sum_j p_j |v_j|: a score is within
ds = ((D + 8) sum |q k| scale + 4 |s|) u (its products are exact in float32 for
bf16 and one rounding each for float32, D additions, the scalings); a weight is
within 2 ds + 4 u of itself, the sums over n keys in at most n + 16 additions;
the bf16 path holds a weight in two bf16 parts, 2^-17 of it.  Then half a
step of the output's own dtype.
"""

import math

import pytest
import torch

from nsa_testlib import require_gpu

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
IDS = {BF: "bf16", F32: "f32"}


def _setup(B, lens, Hq, Hkv, D, P, mp, dtype, seed=0, extra=3, fill=float("nan")):
    """Random pages in random places; unwritten rows hold ``fill``."""
    g = torch.Generator().manual_seed(seed)
    n_pages = B * mp + extra
    kp = torch.full((n_pages, Hkv, P, D), fill, dtype=dtype)
    vp = torch.full((n_pages, Hkv, P, D), fill, dtype=dtype)
    perm = torch.randperm(n_pages, generator=g)
    table = torch.full((B, mp), -1, dtype=torch.int32)
    ks, vs, at = [], [], 0
    for b in range(B):
        n = max(0, lens[b])
        k = torch.randn(Hkv, n, D, generator=g).to(dtype)
        v = torch.randn(Hkv, n, D, generator=g).to(dtype)
        held = min(mp, n // P + 1)
        for i in range(held):
            pg = int(perm[at])
            at += 1
            table[b, i] = pg
            m = min(P, n - i * P)
            if m > 0:
                kp[pg, :, :m] = k[:, i * P:i * P + m]
                vp[pg, :, :m] = v[:, i * P:i * P + m]
        ks.append(k)
        vs.append(v)
    q = (torch.randn(B, Hq, D, generator=g) * 1.5).to(dtype)
    kn, vn = torch.randn(B, Hkv, D, generator=g).to(dtype), torch.randn(B, Hkv, D, generator=g).to(dtype)
    return q, kn, vn, kp, vp, table, torch.tensor(lens, dtype=torch.int32), ks, vs


def _compare(out, q, ks, vs, scale=None, lse=None):
    """out [B, Hq, D] against the keys and values of each sequence."""
    out = out.cpu()
    B, Hq, D = q.shape
    for b in range(B):
        k, v = ks[b].double(), vs[b].double()
        Hkv, n = k.shape[0], k.shape[1]
        if n == 0:
            assert not out[b].any(), b
            if lse is not None:
                assert (lse[b] == -1e9).all()
            continue
        sc = D ** -0.5 if scale is None else scale
        qq = q[b].double().view(Hkv, Hq // Hkv, D)
        s = torch.einsum("hgd,hnd->hgn", qq, k) * sc
        p = torch.softmax(s, -1)
        ref = torch.einsum("hgn,hnd->hgd", p, v).reshape(Hq, D)
        E = torch.einsum("hgn,hnd->hgd", p, v.abs()).reshape(Hq, D)
        ds = ((D + 8) * torch.einsum("hgd,hnd->hgn", qq.abs(), k.abs()) * abs(sc) + 4 * s.abs()).amax(-1) * U
        rel = (2 * (2 * ds + 4 * U) + (2 * n + 32) * U + (2.0 ** -17 if q.dtype == BF else 0)).reshape(Hq, 1)
        half = torch.finfo(q.dtype).eps / 2
        err = (out[b].double() - ref).abs()
        tol = ref.abs() * half * (1 + 1e-6) + E * rel * (1 + 4 * half) + 1e-30
        assert (err <= tol).all(), (b, float((err / tol).max()))
        if lse is not None:
            l = torch.logsumexp(s, -1).reshape(Hq)
            assert ((lse[b].cpu().double() - l).abs() <= rel[:, 0] + 4 * U * l.abs() + 4 * U).all()


# B, lens, Hq, Hkv, D, P, max_pages
CASES = [
    (1, [0], 1, 1, 16, 16, 1),
    (1, [15], 4, 2, 32, 16, 1),
    (3, [0, 16, 5], 8, 8, 64, 16, 3),
    (4, [31, 32, 33, 0], 6, 2, 64, 32, 4),
    (2, [127, 128], 16, 1, 128, 64, 5),
    (5, [1, 47, 48, 200, 95], 12, 3, 64, 48, 6),
    (2, [300, 511], 40, 1, 128, 128, 4),
    (2, [1000, 63], 34, 2, 32, 256, 5),
    (3, [700, 0, 1536], 64, 4, 128, 64, 40),
    (1, [5000], 16, 16, 16, 16, 313),
    (70, [(37 * i) % 400 for i in range(70)], 8, 2, 64, 16, 26),
    (1, [20000], 64, 4, 128, 80, 300),
    (300, [(7 * i) % 90 for i in range(300)], 20, 4, 32, 112, 1),
]


@pytest.mark.parametrize("dtype", [BF, F32], ids=IDS.get)
@pytest.mark.parametrize("c", CASES, ids=lambda c: f"B{c[0]}-n{max(c[1])}-H{c[2]}:{c[3]}-D{c[4]}-P{c[5]}")
def test_step_and_attend(c, dtype):
    import nsa_paged
    dev = require_gpu()
    B, lens, Hq, Hkv, D, P, mp = c
    q, kn, vn, kp, vp, table, L, ks, vs = _setup(B, lens, Hq, Hkv, D, P, mp, dtype, seed=B + D + P)
    dkp, dvp, dt, dl = kp.to(dev), vp.to(dev), table.to(dev), L.to(dev)
    out, lse = nsa_paged.paged_attend(q.to(dev), dkp, dvp, dt, dl, return_lse=True)
    _compare(out, q, ks, vs, lse=lse)
    out, new = nsa_paged.paged_step(q.to(dev), kn.to(dev), vn.to(dev), dkp, dvp, dt, dl)
    assert torch.equal(dl.cpu(), L)
    ks2, vs2, want = [], [], []
    for b in range(B):
        fits = lens[b] < mp * P
        want.append(lens[b] + int(fits))
        ks2.append(torch.cat([ks[b], kn[b][:, None]], 1) if fits else ks[b])
        vs2.append(torch.cat([vs[b], vn[b][:, None]], 1) if fits else vs[b])
        if fits:
            pg, r = int(table[b, lens[b] // P]), lens[b] % P
            kp[pg, :, r], vp[pg, :, r] = kn[b], vn[b]
    assert new.cpu().tolist() == want
    _compare(out, q, ks2, vs2)
    for a, b in ((dkp, kp), (dvp, vp)):      # the new rows and nothing else
        a = a.cpu()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    # the step's attention is the attention over what it left
    assert torch.equal(out, nsa_paged.paged_attend(q.to(dev), dkp, dvp, dt, new))


@pytest.mark.parametrize("dtype", [BF, F32], ids=IDS.get)
def test_bad_pages_lengths_and_full_sequences(dtype):
    import nsa_paged
    dev = require_gpu()
    Hq, Hkv, D, P, mp = 8, 2, 64, 32, 6
    lens = [100, -1, 192, 150, 64, 500, -2 ** 31, 2 ** 31 - 1, 90]
    B = len(lens)
    real = [min(max(n, 0), mp * P) for n in lens]
    q, kn, vn, kp, vp, table, L, ks, vs = _setup(B, real, Hq, Hkv, D, P, mp, dtype, seed=5)
    n_pages = kp.shape[0]
    L = torch.tensor(lens, dtype=torch.int32)
    # entries outside the pages: in the middle (keys not attended), at the step's position (no append), behind
    table[0, 1], table[3, 0], table[3, 4], table[4, 2], table[8, 5] = -1, n_pages, -7, 2 ** 31 - 1, n_pages + 9
    table[0, 5], table[2, 0] = -2 ** 31, -1
    gone = {0: [1], 2: [0], 3: [0, 4]}
    before = kp.clone()
    dkp, dvp, dt, dl = kp.to(dev), vp.to(dev), table.to(dev), L.to(dev)
    out, new = nsa_paged.paged_step(q.to(dev), kn.to(dev), vn.to(dev), dkp, dvp, dt, dl)
    fits = [True, False, False, False, False, False, False, False, True]
    assert new.cpu().tolist() == [n + int(f) for n, f in zip(lens, fits)]
    ks2, vs2 = [], []
    for b in range(B):
        keep = torch.tensor([j // P not in gone.get(b, []) for j in range(real[b])], dtype=torch.bool)
        k, v = ks[b][:, keep], vs[b][:, keep]
        if fits[b]:
            k, v = torch.cat([k, kn[b][:, None]], 1), torch.cat([v, vn[b][:, None]], 1)
            before[int(table[b, lens[b] // P]), :, lens[b] % P] = kn[b]
        ks2.append(k)
        vs2.append(v)
    _compare(out, q, ks2, vs2)
    assert torch.equal(dkp.cpu().nan_to_num(7.0), before.nan_to_num(7.0))


def test_page_offsets_past_32_bits():
    """Pages whose elements and bytes lie past 2^31 and 2^32 in the pool."""
    import nsa_paged
    dev = require_gpu()
    Hkv, D, P, dtype = 1, 128, 256, BF
    n_pages = (1 << 31) // (Hkv * P * D) + 40          # 2^31 elements, 2^32 bytes, and some more
    kp = torch.empty(n_pages, Hkv, P, D, device=dev, dtype=dtype)
    vp = torch.empty_like(kp)
    far = [n_pages - 1, n_pages - 7, (1 << 30) // (P * D) + 3, n_pages - 20]
    n = 3 * P + 100
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(Hkv, n, D, generator=g).to(dtype), torch.randn(Hkv, n, D, generator=g).to(dtype)
    table = torch.tensor([far], dtype=torch.int32, device=dev)
    lens = nsa_paged.paged_append(k[None].to(dev), v[None].to(dev), kp, vp, table,
                                  torch.zeros(1, dtype=torch.int32, device=dev))
    assert lens.tolist() == [n]
    for i, pg in enumerate(far):
        m = min(P, n - i * P)
        assert torch.equal(kp[pg, :, :m].cpu(), k[:, i * P:i * P + m])
    q, kn, vn = (torch.randn(1, h, D, generator=g).to(dtype) for h in (16, 1, 1))
    out, new = nsa_paged.paged_step(q.to(dev), kn.to(dev), vn.to(dev), kp, vp, table, lens)
    _compare(out, q, [torch.cat([k, kn[0][:, None]], 1)], [torch.cat([v, vn[0][:, None]], 1)])
    assert torch.equal(kp[far[3], :, 100].cpu(), kn[0]) and new.tolist() == [n + 1]


@pytest.mark.parametrize("dtype", [BF, F32], ids=IDS.get)
@pytest.mark.parametrize("D,P", [(16, 16), (64, 48), (128, 64)])
def test_append_of_prompts(D, P, dtype):
    import nsa_paged
    dev = require_gpu()
    Hkv, mp, T = 3, 6, 3 * P + 5
    lens = [0, 7, 2 * P, 6 * P - 10, -3, P, 0]
    count = [T, 5, 2 * P + 1, 11, 4, 0, T + 50]
    B = len(lens)
    g = torch.Generator().manual_seed(D)
    k, v = (torch.randn(B, Hkv, T, D, generator=g).to(dtype) for _ in range(2))
    table = torch.randperm(B * mp + 2, generator=g)[:B * mp].view(B, mp).to(torch.int32)
    kp = torch.randn(B * mp + 2, Hkv, P, D, generator=g).to(dtype)
    vp = kp.flip(0).clone()
    table[1, 3] = -1                                    # not reached
    table[2, 4] = B * mp + 2                            # reached by the last row: nothing is written
    dkp, dvp = kp.to(dev), vp.to(dev)
    new = nsa_paged.paged_append(k.to(dev), v.to(dev), dkp, dvp, table.to(dev),
                                 torch.tensor(lens, dtype=torch.int32, device=dev),
                                 torch.tensor(count, dtype=torch.int32, device=dev))
    want = []
    for b in range(B):
        n = min(count[b], T)
        ok = lens[b] >= 0 and lens[b] + n <= mp * P and b != 2
        want.append(lens[b] + n if ok else lens[b])
        for t in range(n if ok else 0):
            pg, r = int(table[b, (lens[b] + t) // P]), (lens[b] + t) % P
            kp[pg, :, r], vp[pg, :, r] = k[b, :, t], v[b, :, t]
    assert new.cpu().tolist() == want
    assert torch.equal(dkp.cpu(), kp) and torch.equal(dvp.cpu(), vp)


def test_shared_prefix_scale_and_peaked_rows():
    """Two sequences over one page, a scale of the caller's, scores of thousands."""
    import nsa_paged
    dev = require_gpu()
    q, kn, vn, kp, vp, table, L, ks, vs = _setup(2, [64, 80], 8, 2, 64, 64, 3, F32, seed=2)
    table[1, 0] = table[0, 0]
    ks[1] = torch.cat([ks[0], ks[1][:, 64:]], 1)
    vs[1] = torch.cat([vs[0], vs[1][:, 64:]], 1)
    for scale in (1.0, -0.3, 0.0, 40.0):
        out, lse = nsa_paged.paged_attend(q.to(dev), kp.to(dev), vp.to(dev), table.to(dev), L.to(dev), scale, True)
        _compare(out, q, ks, vs, scale, lse)


def test_captured_steps_share_nothing():
    """A graph of steps replayed among eager steps of other caches, and a second graph."""
    import nsa_paged
    dev = require_gpu()

    def make(seed, n):
        c = nsa_paged.PagedKVCache(3, 2, 64, 700, 32)
        c.reserve(700)
        g = torch.Generator().manual_seed(seed)
        k = torch.randn(3, 2, n, 64, generator=g).to(BF).to(dev)
        c.prefill(k, k.flip(2), lens=[n, n // 2, 1])
        return c
    rows = [[torch.randn(3, h, 64, generator=torch.Generator().manual_seed(10 * s + h)).to(BF).to(dev)
             for h in (8, 2, 2)] for s in range(5)]
    ref = []
    for n in (300, 500):
        c = make(n, n)
        ref.append([c.step(*r) for r in rows])
        ref[-1].append(c.lens)
    graphs = []
    for n in (300, 500):
        c = make(n, n)
        static = [torch.zeros_like(t) for t in rows[0]]
        lens0 = c.lens.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            c.step(*static)
        torch.cuda.current_stream().wait_stream(side)
        c.lens = lens = lens0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c.step(*static)
            lens.copy_(c.lens)
        graphs.append((graph, static, out, lens, c))
    for s in range(5):
        for i, (graph, static, out, lens, _) in enumerate(graphs):
            for a, b in zip(static, rows[s]):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            make(7, 100).step(*rows[s])
            torch.cuda.synchronize()
            assert torch.equal(out, ref[i][s]), (i, s)
    for i, g in enumerate(graphs):
        assert torch.equal(g[3], ref[i][5])


def test_other_stream_and_same_bits():
    import nsa_paged
    dev = require_gpu()
    q, kn, vn, kp, vp, table, L, _, _ = (t.to(dev) if torch.is_tensor(t) else t
                                         for t in _setup(4, [900, 3000, 0, 17], 64, 4, 128, 64, 50, BF, fill=0.0))
    first = nsa_paged.paged_step(q, kn, vn, kp.clone(), vp.clone(), table, L)
    side = torch.cuda.Stream()
    kp2, vp2 = kp.clone(), vp.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = nsa_paged.paged_step(q, kn, vn, kp2, vp2, table, L)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_two_streams_at_once():
    """Steps in flight on two streams, over caches of their own, share nothing."""
    import nsa_paged
    dev = require_gpu()
    sets = [[t.to(dev) if torch.is_tensor(t) else t
             for t in _setup(5, [900 + 300 * s, 3000, 0, 17, 400], 64, 4, 128, 64, 50, BF, seed=s, fill=0.0)]
            for s in range(2)]
    want = [nsa_paged.paged_step(*[t.clone() for t in s[:7]]) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(nsa_paged.paged_step(*sets[i][:7]))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lens in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lens, want[i][1])


def test_many_sequences_and_shares():
    """More sequences than threads count at once, shares of many rows and rows of many shares."""
    import nsa_paged
    dev = require_gpu()
    lens = [(i * 7919) % 60 for i in range(700)]
    lens[350] = 3000
    q, kn, vn, kp, vp, table, L, ks, vs = _setup(700, lens, 4, 1, 32, 16, 200, BF, seed=1, extra=1)
    kp, vp = kp[:1 + int(table.max())], vp[:1 + int(table.max())]
    # a capacity past 1 MiB a row: shares, not a row to a workgroup
    table = torch.nn.functional.pad(table, (0, 400), value=-1)
    out, new = nsa_paged.paged_step(*(t.to(dev) for t in (q, kn, vn, kp, vp, table, L)))
    _compare(out, q, [torch.cat([k, n[:, None]], 1) for k, n in zip(ks, kn)],
             [torch.cat([v, n[:, None]], 1) for v, n in zip(vs, vn)])
    assert new.tolist() == [n + 1 for n in lens]


def test_cache_pages():
    import nsa_paged
    dev = require_gpu()
    c = nsa_paged.PagedKVCache(2, 1, 16, 100, 16, n_pages=8, dtype=F32)
    two = nsa_paged.PagedKVCache(2, 1, 16, 100, 16, n_pages=8, dtype=F32, like=c)
    c.reserve([33, 16])
    assert c.free_pages == 4 and two.table is c.table and (c.table.cpu() >= 0).sum(1).tolist() == [3, 1]
    with pytest.raises(RuntimeError):
        c.reserve([33, 100])
    for bad in (101, -1, [5]):
        with pytest.raises(AssertionError):
            c.reserve(bad)
    assert c.free_pages == 4
    two.reserve([40, 80])                 # 3 held already, 4 more for the second
    ids = c.table.cpu()
    assert c.free_pages == 0 and len(set(ids[ids >= 0].tolist())) == 8
    k = torch.randn(2, 1, 20, 16, device=dev)
    for x in (c, two):
        x.prefill(k, k, lens=[20, 3])
        assert x.lens.tolist() == [20, 3]
    two.release(0)
    assert c.free_pages == 3 and c.lens.tolist() == [0, 3] and two.lens.tolist() == [0, 3]
    assert (c.table[0] == -1).all() and not c.attend(torch.randn(2, 4, 16, device=dev))[0].any()


def test_refusals():
    import nsa_paged
    dev = require_gpu()
    q, kn, vn, kp, vp, table, L, _, _ = (t.to(dev) if torch.is_tensor(t) else t
                                         for t in _setup(2, [5, 20], 4, 2, 64, 16, 3, BF))
    ok = dict(q=q, k_pages=kp, v_pages=vp, table=table, lens=L)
    bad = [dict(q=q[:1]), dict(q=q[:, :3]), dict(q=q.float()), dict(q=q[..., :32]), dict(v_pages=vp[:-1]),
           dict(v_pages=vp.float()), dict(table=table.long()), dict(table=table[:1]), dict(lens=L.long()),
           dict(k_pages=kp[:, :, :, :48], v_pages=vp[:, :, :, :48]), dict(k_pages=kp.transpose(0, 1)),
           dict(k_pages=kp[:, :, :8], v_pages=vp[:, :, :8]), dict(k_pages=kp.half(), v_pages=vp.half()),
           dict(table=table.cpu()), dict(q=q.cpu())]
    nsa_paged.paged_attend(**ok)
    for b in bad:
        with pytest.raises(AssertionError):
            nsa_paged.paged_attend(**{**ok, **b})
    for rows in [(kn[:, :1], vn), (kn, vn.float()), (kn[..., :32], vn)]:
        with pytest.raises(AssertionError):
            nsa_paged.paged_step(q, *rows, kp, vp, table, L)
    with pytest.raises(AssertionError):
        nsa_paged.paged_append(kn, vn, kp, vp, table, L)
    with pytest.raises(AssertionError):
        nsa_paged.paged_append(kn[:, :, None], vn[:, :, None], kp, vp, table, L, count=L.long())
    with pytest.raises(AssertionError):
        nsa_paged.PagedKVCache(2, 1, 64, 100, page_size=24)
    with pytest.raises(AssertionError):
        nsa_paged.PagedKVCache(2, 1, 48, 100)
    assert math.isfinite(float(nsa_paged.paged_attend(**ok).float().sum()))


def test_gradients_are_refused():
    import nsa_paged
    dev = require_gpu()
    q, kn, vn, kp, vp, table, L, _, _ = (t.to(dev) if torch.is_tensor(t) else t
                                         for t in _setup(2, [5, 20], 4, 2, 64, 16, 3, F32))
    leaf = q.detach().clone().requires_grad_()
    row = kn.detach().clone().requires_grad_()
    with pytest.raises(AssertionError):
        nsa_paged.paged_attend(leaf, kp, vp, table, L)
    with pytest.raises(AssertionError):
        nsa_paged.paged_step(q, row, vn, kp, vp, table, L)
    with pytest.raises(AssertionError):
        nsa_paged.paged_append(row[:, :, None], vn[:, :, None], kp, vp, table, L)
    with torch.no_grad():
        assert torch.equal(nsa_paged.paged_attend(leaf, kp, vp, table, L), nsa_paged.paged_attend(q, kp, vp, table, L))
