"""The operators around the attention, and how their speed and outputs are followed.

Three operators, each with its plain form (elementary torch operations in float32) and its call:

* ``norm``: the residual's addition with the root-mean-square norm of the sum (``nsa_lm.add_rms_norm``); ``out`` is the
  normalised rows' type, ``e4m3`` for rows in 8 bits with one scale each (``nsa_lm.add_rms_norm_q8``); ``grad`` adds the
  backward pass;
* ``logp``: log probabilities of given tokens with the entropy and the ``top`` best alternatives of every row
  (``nsa_lm.token_logprobs``); ``grad`` returns the logits' gradient of a loss in both;
* ``paged``: one new token of every sequence over a paged key-value cache: its key and value rows appended, then its
  query's attention (``nsa_paged.paged_step``).
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
Q8_MAX = 448.0            # the largest e4m3 value
Q8_FLOOR = 2.0 ** -100    # smallest row maximum that a scale is formed from


def listed():
    return [
        # a generation step of 32 sequences through one norm of a wide model: latency alone counts
        dict(name="norm_step_32x8192", kind="norm", rows=32, D=8192, x="bf16", r="bf16", w="bf16", out="bf16",
             grad=False),
        # one norm of the 12-layer d768 decoder in mixed-precision training: float32 stream, bf16 branch
        dict(name="norm_train_32768x768", kind="norm", rows=32768, D=768, x="bf16", r="f32", w="f32", out="bf16",
             grad=True),
        # a prompt of no round length on its way into 8-bit products
        dict(name="norm_q8_8191x8192", kind="norm", rows=8191, D=8192, x="bf16", r="bf16", w="bf16", out="e4m3",
             grad=False),
        # a small float32 experiment with a width of no whole vectors
        dict(name="norm_f32_1021x1001", kind="norm", rows=1021, D=1001, x="f32", r="f32", w="f32", out="f32",
             grad=True),
        # the tokens a batch has just chosen, with the 20 best alternatives a server reports
        dict(name="logp_step_32x32000", kind="logp", rows=32, V=32000, dtype="bf16", top=20, ignored=False,
             grad=False),
        # scoring a document: an odd vocabulary, so that rows start at any 2-byte address
        dict(name="logp_score_2047x50257", kind="logp", rows=2047, V=50257, dtype="bf16", top=5, ignored=False,
             grad=False),
        # the loss of the 12-layer d768 decoder's training step, 8 x 4096 tokens
        dict(name="logp_train_32768x32000", kind="logp", rows=32768, V=32000, dtype="bf16", top=0, ignored=True,
             grad=True),
        # the loss of a small model in float32, its padding ignored
        dict(name="logp_train_f32_1023x8191", kind="logp", rows=1023, V=8191, dtype="f32", top=1, ignored=True,
             grad=True),
        # one conversation being generated at 32K tokens
        dict(name="paged_1x32k", kind="paged", B=1, T=32768, Hq=64, Hkv=4, D=128, page=64, dtype="bf16",
             ragged=False),
        # a server's batch, its sequences of unlike lengths up to 32K
        dict(name="paged_32x32k", kind="paged", B=32, T=32768, Hq=64, Hkv=4, D=128, page=64, dtype="bf16",
             ragged=True),
        # many short chats over small pages, groups of six heads
        dict(name="paged_200x900", kind="paged", B=200, T=900, Hq=12, Hkv=2, D=64, page=16, dtype="bf16",
             ragged=True),
        # a numerics check in float32: every head with its own keys
        dict(name="paged_f32_3x1021", kind="paged", B=3, T=1021, Hq=8, Hkv=8, D=64, page=32, dtype="f32",
             ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "logp", "paged"])
    if kind == "norm":
        D = _log_int(rng, 64, 16384)
        if rng.random() < 0.6:
            D = max(64, D // 64 * 64)
        rows = _log_int(rng, 1, min(32768, (1 << 26) // D))
        x, r, w = rng.choice([("bf16", "bf16", "bf16"), ("bf16", "f32", "f32"), ("f32", "f32", "f32"),
                              ("bf16", "bf16", "f32")])
        out = rng.choice(["bf16", "e4m3"] if x == "bf16" else ["f32", "bf16"])
        return dict(kind=kind, rows=rows, D=D, x=x, r=r, w=w, out=out, grad=out != "e4m3" and rng.random() < 0.6)
    if kind == "logp":
        V = _log_int(rng, 100, 200000)
        if rng.random() < 0.5:
            V = max(128, V // 128 * 128)
        grad = rng.random() < 0.5
        rows = _log_int(rng, 1, min(32768, (1 << 30 if grad else 1 << 27) // V))
        top = rng.choice([0, 0, 1]) if grad else rng.choice([0, 1, 5, 20, 32])
        if top:
            rows = min(rows, (1 << 27) // V)
        return dict(kind=kind, rows=rows, V=V, dtype=rng.choice(["bf16", "bf16", "f32"]), top=top,
                    ignored=grad and rng.random() < 0.5, grad=grad)
    Hq, Hkv, D = rng.choice([(64, 4, 128), (32, 2, 128), (16, 1, 128), (16, 16, 128), (16, 1, 64), (16, 4, 64),
                             (12, 2, 64), (8, 8, 64), (8, 2, 32), (40, 1, 128)])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    T = _log_int(rng, 1, 131072)
    B = _log_int(rng, 1, max(1, min(256, (1 << 28) // (T * Hkv * D))))
    return dict(kind=kind, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, page=rng.choice([16, 32, 48, 64, 128, 256]), dtype=dtype,
                ragged=rng.random() < 0.6)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lens(c):
    """The sequences' lengths before the step, in some order: all the capacity but one place, or spread from an
    eighth of that up to it, the shortest empty where there are several."""
    B, full = c["B"], c["T"] - 1
    if not c["ragged"] or B == 1:
        return [full] * B
    return [0] + [full // 8 + (full - full // 8) * b // (B - 1) for b in range(1, B)]


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)

    def rnd(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype)

    if c["kind"] == "norm":
        rows, D = c["rows"], c["D"]
        # a residual stream: unlike channels, a few of them far larger, rows of unlike size
        chan = torch.exp(0.5 * rnd(D))
        chan[torch.randint(0, D, (max(1, D // 256),), generator=g, device=DEV)] *= 20.0
        size = torch.exp(0.3 * rnd(rows, 1))
        c["res"] = (rnd(rows, D) * chan * size).to(DTYPES[c["r"]])
        c["branch"] = rnd(rows, D, dtype=DTYPES[c["x"]])
        c["weight"] = (1.0 + 0.2 * rnd(D)).to(DTYPES[c["w"]])
        if c["grad"]:
            c["dy"] = rnd(rows, D, dtype=DTYPES[c["out"]])
            c["dh"] = rnd(rows, D, dtype=DTYPES[c["r"]])
    elif c["kind"] == "logp":
        rows, V = c["rows"], c["V"]
        # rows from flat to peaked, a few tokens of each banned (minus infinity)
        z = rnd(rows, V)
        z *= 0.5 + 3.0 * torch.rand(rows, 1, generator=g, device=DEV)
        z[:, torch.randint(0, V, (max(1, V // 1000),), generator=g, device=DEV)] = -math.inf
        c["logits"] = z.to(DTYPES[c["dtype"]])
        # targets from the better half of 64 candidates: likely tokens, none of them banned
        cand = torch.randint(0, V, (rows, 64), generator=g, device=DEV)
        c["targets"] = cand.gather(1, c["logits"].float().gather(1, cand).argmax(1, keepdim=True)).squeeze(1)
        if c["ignored"]:
            c["targets"][torch.rand(rows, generator=g, device=DEV) < 0.1] = -100
        if c["grad"]:
            c["dlogp"] = -torch.rand(rows, generator=g, device=DEV)
            c["dent"] = 0.1 * rnd(rows)
    else:
        B, P, Hkv, D, dt = c["B"], c["page"], c["Hkv"], c["D"], DTYPES[c["dtype"]]
        lens = torch.tensor(_lens(c), device=DEV)[torch.randperm(B, generator=g, device=DEV)]
        mp = -(-c["T"] // P)
        need = lens // P + 1                                        # pages that hold the new token too
        used = torch.arange(mp, device=DEV)[None, :] < need[:, None]
        n_pages = B * mp + 3
        c["table"] = torch.where(used, torch.randperm(n_pages, generator=g, device=DEV)[:B * mp].view(B, mp),
                                 -1).to(torch.int32)
        c["k_pages"] = torch.randn(n_pages, Hkv, P, D, generator=g, device=DEV, dtype=dt)
        c["v_pages"] = torch.randn(n_pages, Hkv, P, D, generator=g, device=DEV, dtype=dt)
        c["lens"] = lens.to(torch.int32)
        c["q"] = (rnd(B, c["Hq"], D) * (0.5 + torch.rand(1, c["Hq"], 1, generator=g, device=DEV))).to(dt)
        c["k_new"], c["v_new"] = rnd(B, Hkv, D, dtype=dt), rnd(B, Hkv, D, dtype=dt)
    return c


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    c = state
    if own:
        return _own(c)
    return {"norm": _plain_norm, "logp": _plain_logp, "paged": _plain_paged}[c["kind"]](c)


def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "openbox-llm_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


def _own(c):
    if "nsa_lm" not in sys.modules:
        _package()
    if c["kind"] == "paged":
        import nsa_paged
        out, lens = nsa_paged.paged_step(c["q"], c["k_new"], c["v_new"], c["k_pages"], c["v_pages"], c["table"],
                                         c["lens"])
        return dict(out=out, lens=lens, k_pages=c["k_pages"], v_pages=c["v_pages"])
    import nsa_lm
    if c["kind"] == "norm":
        x, r, w = c["branch"], c["res"], c["weight"]
        if c["out"] == "e4m3":
            q, scale, h = nsa_lm.add_rms_norm_q8(x, r, w, eps=EPS)
            return dict(q=q, scale=scale, h=h)
        if not c["grad"]:
            y, h = nsa_lm.add_rms_norm(x, r, w, eps=EPS, out_dtype=DTYPES[c["out"]])
            return dict(y=y, h=h)
        x, r, w = (t.detach().requires_grad_() for t in (x, r, w))
        y, h = nsa_lm.add_rms_norm(x, r, w, eps=EPS, out_dtype=DTYPES[c["out"]])
        dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (c["dy"], c["dh"]))
        return dict(y=y, h=h, dx=dx, dr=dr, dw=dw)
    z = c["logits"].detach().requires_grad_(c["grad"])
    got = nsa_lm.token_logprobs(z, c["targets"], top=c["top"])
    res = dict(logp=got.logp, entropy=got.entropy)
    if c["top"]:
        res.update(top_logp=got.top_logp, top_idx=got.top_idx)
    if c["grad"]:
        res["dz"], = torch.autograd.grad((got.logp, got.entropy), (z,), (c["dlogp"], c["dent"]))
    return res


def _plain_norm(c):
    h = (c["branch"].float() + c["res"].float()).to(c["res"].dtype)
    h32, w = h.float(), c["weight"].float()
    rstd = torch.rsqrt(h32.square().mean(1, keepdim=True) + EPS)
    n = h32 * rstd
    if c["out"] == "e4m3":
        y = n * w
        amax = y.abs().amax(1).clamp(min=Q8_FLOOR)
        return dict(q=(y * (Q8_MAX / amax)[:, None]).to(torch.float8_e4m3fn), scale=amax / Q8_MAX, h=h)
    res = dict(y=(n * w).to(DTYPES[c["out"]]), h=h)
    if c["grad"]:
        dy = c["dy"].float()
        g = dy * w
        dh = c["dh"].float() + rstd * (g - n * (g * n).mean(1, keepdim=True))
        res.update(dx=dh.to(c["branch"].dtype), dr=dh.to(c["res"].dtype), dw=(dy * n).sum(0).to(c["weight"].dtype))
    return res


def _plain_logp(c):
    z, t = c["logits"].float(), c["targets"]
    m = z.amax(1, keepdim=True)
    d = z - m
    e = torch.exp(d)
    tot = e.sum(1)
    logl = torch.log(tot)
    s = torch.where(e > 0, d, 0.0)
    ent = logl - (e * s).sum(1) / tot
    keep = (t >= 0) & (t < z.shape[1])
    at = t.clamp(0, z.shape[1] - 1)[:, None]
    logp = torch.where(keep, d.gather(1, at).squeeze(1) - logl, 0.0)
    res = dict(logp=logp, entropy=ent)
    if c["top"]:
        val, idx = torch.sort(z, dim=1, descending=True, stable=True)
        res.update(top_logp=val[:, :c["top"]] - (m + logl[:, None]), top_idx=idx[:, :c["top"]].contiguous())
    if c["grad"]:
        p = e / tot[:, None]
        dl = torch.where(keep, c["dlogp"], 0.0)[:, None]
        dz = -p * (dl + c["dent"][:, None] * (s - logl[:, None] + ent[:, None]))
        dz.scatter_add_(1, at, dl)
        res["dz"] = dz.to(c["logits"].dtype)
    return res


def _plain_paged(c):
    kp, vp, table, lens = c["k_pages"], c["v_pages"], c["table"].long(), c["lens"].long()
    (B, Hq, D), (_, Hkv, P, _) = c["q"].shape, kp.shape
    at = table.gather(1, (lens // P)[:, None]).squeeze(1)
    kp[at, :, lens % P] = c["k_new"]
    vp[at, :, lens % P] = c["v_new"]
    n = lens + 1
    span = c["T"]
    tab = table.clamp(min=0)
    k = kp[tab].transpose(1, 2).reshape(B, Hkv, -1, D)[:, :, :span].float()
    v = vp[tab].transpose(1, 2).reshape(B, Hkv, -1, D)[:, :, :span].float()
    qt = c["q"].float().view(B, Hkv, Hq // Hkv, D).transpose(2, 3).contiguous()
    s = torch.matmul(k, qt) * D ** -0.5                             # [B, Hkv, span, G]
    dead = torch.arange(span, device=DEV)[None, :] >= n[:, None]
    s = s.masked_fill(dead[:, None, :, None], -math.inf)
    e = torch.exp(s - s.amax(2, keepdim=True))
    p = (e / e.sum(2, keepdim=True)).transpose(2, 3).contiguous()
    out = torch.matmul(p, v).view(B, Hq, D).to(c["q"].dtype)
    return dict(out=out, lens=n.to(torch.int32), k_pages=kp, v_pages=vp)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its outputs in 64 bits
# ---------------------------------------------------------------------------

def _size(name):
    return {"bf16": 2, "f32": 4, "e4m3": 1}[name]


def work(case):
    c = case
    if c["kind"] == "norm":
        n, D = c["rows"] * c["D"], c["D"]
        b = n * (_size(c["x"]) + 2 * _size(c["r"]) + _size(c["out"])) + D * _size(c["w"])
        if c["out"] == "e4m3":
            b += 4 * c["rows"]
        f = 6 * n
        if c["grad"]:      # dy, dh and h again in; dx, dr, dw out (one of dx and dr where their types agree)
            b += n * (_size(c["out"]) + 2 * _size(c["r"])) + 2 * D * _size(c["w"])
            b += n * (_size(c["r"]) + (_size(c["x"]) if c["x"] != c["r"] else 0))
            f += 12 * n
        return dict(bytes=b, flops=f)
    if c["kind"] == "logp":
        n = c["rows"] * c["V"]
        b = n * _size(c["dtype"]) + c["rows"] * (16 + 12 * c["top"])
        f = 6 * n
        if c["grad"]:
            b += 2 * n * _size(c["dtype"]) + 8 * c["rows"]
            f += 7 * n
        return dict(bytes=b, flops=f)
    keys = sum(t + 1 for t in _lens(c))
    row = c["D"] * _size(c["dtype"])
    b = 2 * (keys + c["B"]) * c["Hkv"] * row + 2 * c["B"] * c["Hq"] * row + 4 * keys // c["page"] + 8 * c["B"]
    return dict(bytes=b, flops=4 * keys * c["Hq"] * c["D"])


def exact(case, seed):
    c = prepare(case, seed)
    if c["kind"] == "norm":
        h = c["branch"].double() + c["res"].double()
        hr = h.to(c["res"].dtype).double().requires_grad_()         # the norm is taken of the stored sum
        w = c["weight"].double().requires_grad_()
        y = w * hr / torch.sqrt((hr * hr).sum(1, keepdim=True) / c["D"] + EPS)
        if c["out"] == "e4m3":
            y = y.detach()
            s = y.abs().max(dim=1).values.clamp(min=Q8_FLOOR) / Q8_MAX
            return dict(q=y / s[:, None], scale=s, h=h)
        res = dict(y=y.detach(), h=h)
        if c["grad"]:
            gh, gw = torch.autograd.grad((y, hr), (hr, w), (c["dy"].double(), c["dh"].double()))
            res.update(dx=gh, dr=gh, dw=gw)
        return res
    if c["kind"] == "logp":
        V, t = c["V"], c["targets"]
        step = max(1, (1 << 27) // V)
        outs = []
        for a in range(0, c["rows"], step):
            z, tt = c["logits"][a:a + step].double().requires_grad_(c["grad"]), t[a:a + step]
            lp = z - torch.logsumexp(z, 1, keepdim=True)
            safe = lp.masked_fill(lp == -math.inf, 0.0)
            ent = -(torch.exp(lp) * safe).sum(1)
            ok = (tt >= 0) & (tt < V)
            logp = torch.where(ok, lp.gather(1, tt.clamp(0, V - 1)[:, None])[:, 0], 0.0)
            o = dict(logp=logp.detach(), entropy=ent.detach())
            if c["top"]:
                o["top_logp"] = lp.detach().topk(c["top"], dim=1).values
            if c["grad"]:
                o["dz"], = torch.autograd.grad((logp, ent), (z,), (c["dlogp"][a:a + step].double(),
                                                                   c["dent"][a:a + step].double()))
            outs.append(o)
        res = {k: torch.cat([o[k] for o in outs]) for k in outs[0]}
        if c["top"]:
            res["top_idx"] = None
        return res
    B, Hq, D = c["q"].shape
    Hkv, P = c["Hkv"], c["page"]
    out = torch.empty(B, Hq, D, device=DEV, dtype=torch.float64)
    for b in range(B):
        n = int(c["lens"][b])
        ids = c["table"][b, :-(-n // P)].long()
        k, v = (torch.cat([p[ids].permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :n], r[b][:, None]], 1).double()
                for p, r in ((c["k_pages"], c["k_new"]), (c["v_pages"], c["v_new"])))
        s = (c["q"][b].double().view(Hkv, Hq // Hkv, 1, D) * k[:, None]).sum(-1) / math.sqrt(D) if n < 4096 else \
            torch.matmul(k, c["q"][b].double().view(Hkv, Hq // Hkv, D).mT.contiguous()).mT / math.sqrt(D)
        out[b] = torch.matmul(torch.softmax(s, -1).contiguous(), v).view(Hq, D)
    return dict(out=out, lens=None, k_pages=None, v_pages=None)
