"""Timed cases of the token-attention operators (turtlevsr_amd/token_ops.py): rotary positions over several
axes, the per-head norm of queries and keys with that rotation, token attention with its masks and
gradients, and attention over a paged history cache.

``run`` computes a case with elementary torch operations in fp32 (``own`` false) or with the
framework's operators (``own`` true); ``exact`` gives the same outputs from the definitions in fp64.
"""
import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
BASE = 10000.0
EPS = 1e-6


# -------------------------------------------------------------------------------------------------
# cases
# -------------------------------------------------------------------------------------------------

def _rope(name, op, dtype, train, B, grid, Hq, Hk, axes, D, t0=0):
    return {"name": name, "op": op, "dtype": dtype, "train": train, "B": B, "t": grid[0], "h": grid[1], "w": grid[2],
            "Hq": Hq, "Hk": Hk, "a_t": axes[0], "a_h": axes[1], "a_w": axes[2], "D": D, "t0": t0}


def _attn(name, dtype, train, B, Sq, Sk, Hq, Hk, D, causal=False, prefix=0, docs=0, softcap=0.0, bias=False):
    return {"name": name, "op": "attention", "dtype": dtype, "train": train, "B": B, "Sq": Sq, "Sk": Sk, "Hq": Hq, "Hk": Hk,
            "D": D, "causal": causal, "prefix": prefix, "docs": docs, "softcap": softcap, "bias": bias}


def _paged(name, dtype, B, Sq, most, page, Hq, Hk, D, causal=True, softcap=0.0, bias=False):
    return {"name": name, "op": "paged", "dtype": dtype, "train": False, "B": B, "Sq": Sq, "most": most, "page": page, "Hq": Hq,
            "Hk": Hk, "D": D, "causal": causal, "softcap": softcap, "bias": bias}


def listed():
    return [
        # the latent tokens of one 64 x 64 frame: a call that is all latency
        _rope("rope_frame_64", "rope", "bf16", False, 1, (1, 8, 8), 2, 0, (16, 24, 24), 64),
        # rotation alone in an fp32 training step of 5-frame clips, late in a long video
        _rope("rope_clip_train_fp32", "rope", "fp32", True, 2, (5, 16, 16), 8, 0, (16, 24, 24), 64, t0=100003),
        # queries and keys of one 1920 x 1080 frame at the latent level (136 x 240 tokens, width 512)
        _rope("qk_frame_1080p", "qk", "bf16", False, 1, (1, 136, 240), 8, 8, (16, 24, 24), 64),
        # the training clip: 8 clips of 5 frames of 256 x 256, latent level
        _rope("qk_clip_train", "qk", "bf16", True, 8, (5, 32, 32), 8, 8, (16, 24, 24), 64),
        # odd sizes: ragged crop, shared key heads, a width that is no power of two with an unrotated rest
        _rope("qk_odd_train_fp16", "qk", "fp16", True, 3, (3, 13, 21), 6, 2, (8, 16, 12), 40, t0=977),
        # 8 x 8 windows of a 1920 x 1088 frame's latent map with a distance bias, inference
        _attn("attn_windows", "bf16", False, 510, 64, 64, 4, 4, 64, bias=True),
        # training on clips: the frames of the past as prefix, the rest causal
        _attn("attn_clip_train", "bf16", True, 2, 5120, 5120, 8, 8, 64, causal=True, prefix=2048),
        # training on ragged clips packed into one row of tokens, shared key heads, capped scores
        _attn("attn_docs_train", "bf16", True, 1, 8192, 8192, 16, 4, 128, docs=7, softcap=30.0),
        # fp32 gradients at odd sizes: a crop's tokens against a longer history
        _attn("attn_odd_train_fp32", "fp32", True, 2, 333, 517, 6, 3, 48, causal=True, bias=True),
        # all tokens of one 1920 x 1080 frame at the latent level against each other
        _attn("attn_frame_1080p", "bf16", False, 1, 32640, 32640, 8, 8, 64),
        # one new token for each of 16 streams over long histories
        _paged("paged_token", "bf16", 16, 1, 16384, 64, 16, 4, 128),
        # a new frame's tokens (ragged crops) for 4 streams, one page for each frame of history
        _paged("paged_frame", "fp16", 4, 256, 5040, 240, 8, 8, 64, causal=False, softcap=20.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("flops", "bytes")}
    while True:
        op = rng.choice(["rope", "qk", "attention", "attention", "paged"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        train = op != "paged" and rng.random() < 0.5
        if op in ("rope", "qk"):
            D = rng.choice([32, 40, 64, 96, 128])
            a = 2 * rng.randrange(2, D // 6 + 1)
            rest = (D - a) // 2 // 2 * 2
            Hk = rng.choice([1, 2, 3, 8])
            c = _rope("", op, dtype, train, rng.randint(1, 8), (rng.randint(1, 6), _log(rng, 4, 136), _log(rng, 4, 240)),
                      Hk * rng.choice([1, 2, 3]), Hk if op == "qk" else 0, (a, rest, D - a - rest if rng.random() < 0.7 else 2), D,
                      t0=rng.choice([0, rng.randrange(1000), rng.randrange(1000000)]))
        else:
            D = rng.choice([32, 48, 64, 64, 128])
            Hk = rng.choice([1, 2, 4, 8])
            Hq = Hk * rng.choice([1, 1, 2, 4])
            cap, bias = rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.3
            if op == "attention":
                Sq = _log(rng, 1, 12000)
                kind = rng.choice(["full", "causal", "prefix", "docs"])
                Sk = Sq if kind == "docs" or rng.random() < 0.6 else _log(rng, max(1, Sq // 8), Sq * 4)
                if train:       # a row of one key has no gradient but dv: keep more than such rows
                    Sq, Sk = max(Sq, 4), max(Sk, 4)
                B = max(1, _log(rng, 1, 64) if Sq <= 1024 else rng.randint(1, 3))
                c = _attn("", dtype, train, B, Sq, Sk, Hq, Hk, D, causal=kind in ("causal", "prefix") or (kind == "docs" and cap > 0),
                          prefix=max(1, Sk // rng.randint(2, 5)) if kind == "prefix" else 0,
                          docs=rng.randint(1, 9) if kind == "docs" else 0, softcap=cap, bias=bias)
            else:
                page = rng.choice([16, 64, 100, 240, 256])
                c = _paged("", dtype, rng.randint(1, 24), rng.choice([1, 1, 1, _log(rng, 2, 300)]), _log(rng, 300, 16384), page, Hq, Hk, D,
                           causal=rng.random() < 0.7, softcap=cap, bias=bias)
        c.pop("name")
        w = work(c)
        # fp32 products run at a sixteenth of the bf16 rate and more
        if w["flops"] * (16 if dtype == "fp32" else 1) <= most["flops"] and w["bytes"] <= most["bytes"]:
            return c


def _ragged(case, n, total):
    """n document lengths that fill about 15/16 of total tokens, fixed by the case's sizes."""
    r = random.Random("%d %d %d" % (case["B"], n, total))
    use = total - total // 16
    cut = sorted(r.randint(0, use) for _ in range(n - 1))
    return [b - a for a, b in zip([0] + cut, cut + [use])]


def _lens(case):
    """(kv_lens, q_lens) of a paged case, fixed by its sizes: histories between a third and all of ``most``,
    chunks between half and all of Sq, the chunk included in the history."""
    r = random.Random("%d %d %d" % (case["B"], case["Sq"], case["most"]))
    ql = [r.randint((case["Sq"] + 1) // 2, case["Sq"]) for _ in range(case["B"])]
    ql[0] = case["Sq"]
    kl = [max(q, r.randint(case["most"] // 3, case["most"])) for q in ql]
    kl[-1] = max(case["most"], ql[-1])
    return kl, ql


def _pairs(case):
    """visible (query, key) pairs of all sequences, for one head."""
    if case["op"] == "paged":
        kl, ql = _lens(case)
        return sum(sum(k - q + i + 1 for i in range(q)) if case["causal"] else q * k for k, q in zip(kl, ql))
    Sq, Sk, B = case["Sq"], case["Sk"], case["B"]
    if case["docs"]:
        return B * sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _ragged(case, case["docs"], Sq))
    if not case["causal"]:
        return B * Sq * Sk
    return B * sum(min(Sk, max(i + Sk - Sq + 1, case["prefix"])) for i in range(Sq))


def work(case):
    e, D, H = SIZE[case["dtype"]], case["D"], case["Hq"] + case["Hk"]
    if case["op"] in ("rope", "qk"):
        n = case["t"] * case["h"] * case["w"]
        x = case["B"] * n * H * D
        # forward: read x, write y; backward: dy and (for the norm) x again, write dx
        passes = 2 if not case["train"] else (4 if case["op"] == "rope" else 5)
        return {"bytes": passes * e * x + 12 * n, "flops": x * ((3 if case["op"] == "rope" else 8) * (3 if case["train"] else 1))}
    flops = 4 * D * case["Hq"] * _pairs(case)
    if case["op"] == "paged":
        kl, ql = _lens(case)
        rows = 2 * case["Hk"] * sum(kl) + 2 * case["Hq"] * case["Sq"] * case["B"]
        return {"bytes": e * D * rows, "flops": flops}
    q, k = case["B"] * case["Sq"] * case["Hq"] * D, case["B"] * case["Sk"] * case["Hk"] * D
    if not case["train"]:
        return {"bytes": e * (2 * q + 2 * k), "flops": flops}
    # q, k, v, do in; o, dq, dk, dv out; two products forward, five backward
    return {"bytes": e * (4 * q + 4 * k), "flops": flops * 7 // 2}


# -------------------------------------------------------------------------------------------------
# inputs
# -------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    st = {"case": case}
    B, D, Hq, Hk = case["B"], case["D"], case["Hq"], case["Hk"]
    if case["op"] in ("rope", "qk"):
        t, h, w = case["t"], case["h"], case["w"]
        S = t * h * w
        pos = torch.stack(torch.meshgrid(torch.arange(t) + case["t0"], torch.arange(h), torch.arange(w), indexing="ij"), -1)
        st["pos"] = pos.reshape(S, 3).to(device="cuda", dtype=torch.int32)
        st["axes"] = (case["a_t"], case["a_h"], case["a_w"])
        # queries, keys and values of a token side by side, as a 1x1 projection writes them
        qkv = randn(B, S, Hq + 2 * Hk, D).mul_(1.5).to(dt)
        st["q"] = qkv[:, :, :Hq].detach()
        if case["op"] == "qk":
            st["k"] = qkv[:, :, Hq:Hq + Hk].detach()
            st["wq"], st["wk"] = 1 + 0.1 * randn(D), 1 + 0.1 * randn(D)
        if case["train"]:
            st["dq"] = randn(B, S, Hq, D).to(dt)
            if case["op"] == "qk":
                st["dk"] = randn(B, S, Hk, D).to(dt)
    elif case["op"] == "attention":
        Sq, Sk = case["Sq"], case["Sk"]
        # normed and rotated queries and keys are dense; the values are still a slice of the projection
        st["q"], st["k"] = randn(B, Sq, Hq, D).to(dt), randn(B, Sk, Hk, D).to(dt)
        st["v"] = randn(B, Sk, 2 * Hk, D).to(dt)[:, :, Hk:].detach()
        if case["train"]:
            st["do"] = randn(B, Sq, Hq, D).to(dt)
        if case["prefix"]:
            st["prefix"] = torch.full((B,), case["prefix"], dtype=torch.int32, device="cuda")
        if case["docs"]:
            ids = []
            for i, n in enumerate(_ragged(case, case["docs"], Sq)):
                ids += [i] * n
            ids += [-1] * (Sq - len(ids))
            st["doc"] = torch.tensor(ids, dtype=torch.int32, device="cuda").repeat(B, 1)
    else:
        kl, ql = _lens(case)
        M = -(-max(kl) // case["page"])
        n = B * M
        st["lens"] = (kl, ql)
        st["q"] = randn(B, case["Sq"], Hq, D).to(dt)
        st["kp"], st["vp"] = randn(n, case["page"], Hk, D).to(dt), randn(n, case["page"], Hk, D).to(dt)
        st["table"] = torch.randperm(n, device="cuda", generator=g).to(torch.int32).reshape(B, M)
        st["kv_lens"] = torch.tensor(kl, dtype=torch.int32, device="cuda")
        st["q_lens"] = torch.tensor(ql, dtype=torch.int32, device="cuda")
    if case.get("bias"):
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / Hq) for i in range(Hq)], device="cuda")
    if own and case["train"]:
        for n in ("q", "k", "v", "wq", "wk"):
            if n in st:
                st[n] = st[n].requires_grad_(True)
    return st


# -------------------------------------------------------------------------------------------------
# one pass
# -------------------------------------------------------------------------------------------------

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    from turtlevsr_amd import token_ops

    c = st["case"]
    if c["op"] == "rope":
        y = token_ops.axial_rope(st["q"], st["pos"], st["axes"], base=BASE)
        if not c["train"]:
            return y
        (dx,) = torch.autograd.grad(y, st["q"], st["dq"])
        return y, dx
    if c["op"] == "qk":
        q, k = token_ops.qk_norm_rope(st["q"], st["k"], st["pos"], st["wq"], st["wk"], st["axes"], base=BASE, eps=EPS)
        if not c["train"]:
            return q, k
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), (st["q"], st["k"], st["wq"], st["wk"]), (st["dq"], st["dk"]))
        return q, k, dq, dk, dwq, dwk
    if c["op"] == "attention":
        o = token_ops.attention(st["q"], st["k"], st["v"], softcap=c["softcap"], slopes=st.get("slopes"), causal=c["causal"],
                                prefix=st.get("prefix"), q_doc=st.get("doc"))
        if not c["train"]:
            return o
        dq, dk, dv = torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"])
        return o, dq, dk, dv
    return token_ops.paged_attention(st["q"], st["kp"], st["vp"], st["table"], st["kv_lens"], q_lens=st["q_lens"],
                                     softcap=c["softcap"], slopes=st.get("slopes"), causal=c["causal"])


def _angles(st):
    """cos and sin [S, D] of every channel's pair (angle 0 for channels that are not rotated); the angles of
    far positions in fp64."""
    c, pos = st["case"], st["pos"].double()
    parts = []
    for a, d in enumerate(st["axes"]):
        f = BASE ** (-torch.arange(0, d, 2, device=pos.device, dtype=torch.float64) / d)
        parts.append((pos[:, a:a + 1] * f).repeat_interleave(2, dim=1))
    parts.append(torch.zeros(pos.shape[0], c["D"] - sum(st["axes"]), device=pos.device, dtype=torch.float64))
    th = torch.cat(parts, 1)
    return th.cos().float()[:, None], th.sin().float()[:, None]


def _swap(x):
    """(x0, x1) -> (-x1, x0) of every channel pair."""
    return torch.stack((-x[..., 1::2], x[..., 0::2]), -1).flatten(-2)


def _plain_norm_rope(x, w, dy, cos, sin):
    """(y, dx, dw) of the per-head norm (when w is given) and the rotation; dx, dw None without dy."""
    xf = x.float()
    if w is not None:
        r = (xf.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        xn = xf * r
        z = xn * w
    else:
        z = xf
    y = (z * cos + _swap(z) * sin).to(x.dtype)
    if dy is None:
        return y, None, None
    g = dy.float()
    dz = g * cos - _swap(g) * sin
    if w is None:
        return y, dz.to(x.dtype), None
    dw = (dz * xn).sum((0, 1, 2), dtype=torch.float64).float()
    dn = dz * w
    dx = r * (dn - xn * (dn * xn).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), dw


def _visible(i, j, off, causal, prefix, qd, kd):
    """bool [b, rows, keys] for query numbers i and key numbers j of sequences with these (optional) masks."""
    vis = torch.ones(1, i.numel(), j.numel(), dtype=torch.bool, device=i.device)
    if causal:
        vis = (j[None, :] <= i[:, None] + off)[None]
        if prefix is not None:
            vis = vis | (j[None, None, :] < prefix[:, None, None])
    if qd is not None:
        vis = vis & (qd[:, :, None] == kd[:, None, :]) & (qd[:, :, None] >= 0)
    return vis


def _scores(q, k, case, slopes, dist):
    """(scores before the mask, derivative of the cap or None): q [b, Hk, G, rows, D], k [b, Hk, keys, D]."""
    b, Hk, G, R, D = q.shape
    z = torch.matmul(q.reshape(b * Hk, G * R, D), k.reshape(b * Hk, -1, D).transpose(1, 2)).mul_(1 / math.sqrt(D))
    z = z.view(b, Hk, G, R, -1)
    dcap = None
    if case["softcap"]:
        t = torch.tanh(z / case["softcap"])
        z, dcap = case["softcap"] * t, 1 - t * t
    if slopes is not None:
        z = z - slopes.view(1, Hk, G, 1, 1) * dist
    return z, dcap


def _softmax(s, vis):
    s = s.masked_fill(~vis[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    return p / torch.where(l == 0, 1.0, l)


def _heads_first(x, Hk):
    B, S, H, D = x.shape
    return x.float().view(B, S, Hk, H // Hk, D).permute(0, 2, 3, 1, 4)


def _plain_attention(st):
    c = st["case"]
    B, Sq, Sk, Hq, Hk, D = c["B"], c["Sq"], c["Sk"], c["Hq"], c["Hk"], c["D"]
    G, dev, dt = Hq // Hk, st["q"].device, st["q"].dtype
    q = _heads_first(st["q"], Hk)
    k, v = (st[n].float().transpose(1, 2).contiguous() for n in ("k", "v"))
    o = torch.empty_like(q)
    if c["train"]:
        do = _heads_first(st["do"], Hk)
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    j = torch.arange(Sk, device=dev)
    # rows and sequences in pieces of at most 2^28 scores
    rows = max(1, min(Sq, (1 << 28) // (Hq * Sk)))
    nb = max(1, min(B, (1 << 28) // (Hq * Sk * rows)))
    for b in range(0, B, nb):
        bs = slice(b, b + nb)
        kb, vb = k[bs], v[bs]
        n = kb.shape[0]
        for r in range(0, Sq, rows):
            i = torch.arange(r, min(Sq, r + rows), device=dev)
            rs = slice(r, r + i.numel())
            pre, doc = st.get("prefix"), st.get("doc")
            vis = _visible(i, j, Sk - Sq, c["causal"], None if pre is None else pre[bs], None if doc is None else doc[bs, rs],
                           None if doc is None else doc[bs])
            dist = (i[:, None] + (Sk - Sq) - j[None, :]).abs().float() if c["bias"] else None
            s, dcap = _scores(q[bs, :, :, rs], kb, c, st.get("slopes"), dist)
            p = _softmax(s, vis)
            flat = p.reshape(n * Hk, -1, Sk)
            o[bs, :, :, rs] = torch.matmul(flat, vb.reshape(n * Hk, Sk, D)).view(n, Hk, G, -1, D)
            if not c["train"]:
                continue
            g = do[bs, :, :, rs].reshape(n * Hk, -1, D)
            dp = torch.matmul(g, vb.reshape(n * Hk, Sk, D).transpose(1, 2))
            delta = (g * o[bs, :, :, rs].reshape(n * Hk, -1, D)).sum(-1, keepdim=True)
            ds = flat * (dp - delta)
            if dcap is not None:
                ds = ds * dcap.reshape(n * Hk, -1, Sk)
            ds = ds / math.sqrt(D)
            dv[bs] += torch.matmul(flat.transpose(1, 2), g).view(n, Hk, Sk, D)
            dk[bs] += torch.matmul(ds.transpose(1, 2), q[bs, :, :, rs].reshape(n * Hk, -1, D)).view(n, Hk, Sk, D)
            dq[bs, :, :, rs] = torch.matmul(ds, kb.reshape(n * Hk, Sk, D)).view(n, Hk, G, -1, D)
    back = lambda x: x.permute(0, 3, 1, 2, 4).reshape(B, Sq, Hq, D).to(dt)
    if not c["train"]:
        return back(o)
    return back(o), back(dq), dk.transpose(1, 2).to(dt).contiguous(), dv.transpose(1, 2).to(dt).contiguous()


def _plain_paged(st):
    c = st["case"]
    B, Sq, Hq, Hk, D = c["B"], c["Sq"], c["Hq"], c["Hk"], c["D"]
    dt, dev = st["q"].dtype, st["q"].device
    table = st["table"].long()
    n = table.shape[1] * c["page"]
    k, v = (st[x][table].float().view(B, n, Hk, D).transpose(1, 2) for x in ("kp", "vp"))
    i, j = torch.arange(Sq, device=dev), torch.arange(n, device=dev)
    kl, ql = st["kv_lens"].long(), st["q_lens"].long()
    at = i[None, :] + (kl - ql)[:, None]                                   # the place of every query
    vis = (j[None, None] < kl[:, None, None]) & (i[None, :, None] < ql[:, None, None])
    if c["causal"]:
        vis = vis & (j[None, None] <= at[:, :, None])
    dist = (at[:, :, None] - j).abs().float()[:, None, None] if c["bias"] else None
    s, _ = _scores(_heads_first(st["q"], Hk), k, c, st.get("slopes"), dist)
    p = _softmax(s, vis).reshape(B * Hk, -1, n)
    o = torch.matmul(p, v.reshape(B * Hk, n, D)).view(B, Hk, Hq // Hk, Sq, D)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Sq, Hq, D).to(dt)


def _run_plain(st):
    c = st["case"]
    if c["op"] in ("rope", "qk"):
        cos, sin = _angles(st)
        y, dx, dw = _plain_norm_rope(st["q"], st.get("wq"), st.get("dq"), cos, sin)
        if c["op"] == "rope":
            return (y, dx) if c["train"] else y
        yk, dk, dwk = _plain_norm_rope(st["k"], st["wk"], st.get("dk"), cos, sin)
        return (y, yk, dx, dk, dw, dwk) if c["train"] else (y, yk)
    return _plain_attention(st) if c["op"] == "attention" else _plain_paged(st)


# -------------------------------------------------------------------------------------------------
# the definitions in fp64
# -------------------------------------------------------------------------------------------------

def _turn(z, pos, axes):
    """The pairs of z [..., S, H, D] as complex numbers, turned by their positions' angles."""
    n = sum(axes)
    th = torch.cat([pos[:, a:a + 1].double() / BASE ** (torch.arange(d // 2, device=z.device).double() * 2 / d)
                    for a, d in enumerate(axes)], 1)
    c = torch.view_as_complex(z[..., :n].reshape(*z.shape[:-1], n // 2, 2)) * torch.polar(torch.ones_like(th), th)[:, None]
    return torch.cat((torch.view_as_real(c).flatten(-2), z[..., n:]), -1)


def _attend(q, k, v, scale, cap, penalty, vis):
    """One head: q [n, D], k, v [m, D], penalty [n, m] or None, vis [n, m]."""
    z = q @ k.t() * scale
    if cap:
        z = cap * torch.tanh(z / cap)
    if penalty is not None:
        z = z - penalty
    some = vis.any(1, keepdim=True)
    a = torch.softmax(torch.where(vis, z, torch.where(some, -math.inf, 0.0)), dim=1)
    return torch.where(some, a, torch.zeros((), dtype=a.dtype, device=a.device)) @ v


def exact(case, seed):
    st = prepare(case, seed)
    f64 = lambda x: x.detach().double()
    if case["op"] in ("rope", "qk"):
        out, grads, wgrads = [], [], []
        for x, w, dy in (("q", "wq", "dq"), ("k", "wk", "dk")):
            if x not in st:
                continue
            xs = f64(st[x]).requires_grad_(case["train"])
            ws = f64(st[w]).requires_grad_(case["train"]) if w in st else None
            z = xs if ws is None else xs / torch.sqrt((xs * xs).sum(-1, keepdim=True) / case["D"] + EPS) * ws
            y = _turn(z, st["pos"], st["axes"])
            out.append(y.detach())
            if case["train"]:
                g = torch.autograd.grad(y, [xs] if ws is None else [xs, ws], f64(st[dy]))
                grads.append(g[0])
                wgrads += g[1:]
        res = out + grads + wgrads
        return res[0] if len(res) == 1 else tuple(res)
    scale, cap = case["D"] ** -0.5, case["softcap"]
    B, Hq, G, dev = case["B"], case["Hq"], case["Hq"] // case["Hk"], st["q"].device
    q = f64(st["q"])
    o = torch.zeros_like(q)
    if case["op"] == "paged":
        kl, ql = st["lens"]
        for b in range(B):
            n, m = ql[b], kl[b]
            at = torch.arange(m - n, m, device=dev)[:, None] - torch.arange(m, device=dev)[None]
            vis = at >= 0 if case["causal"] else torch.ones_like(at, dtype=torch.bool)
            rows = st["table"][b, :-(-m // case["page"])].long()
            k, v = (f64(st[x][rows].flatten(0, 1)[:m]) for x in ("kp", "vp"))
            for h in range(Hq):
                pen = float(st["slopes"][h]) * at.abs().double() if case["bias"] else None
                o[b, :n, h] = _attend(q[b, :n, h], k[:, h // G], v[:, h // G], scale, cap, pen, vis)
        return o
    Sq, Sk = case["Sq"], case["Sk"]
    k, v = f64(st["k"]), f64(st["v"])
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    # the pairs of one head at a time, in pieces of rows when there are very many
    step = max(1, min(Sq, (1 << 27) // Sk))
    for b in range(B):
        for r in range(0, Sq, step):
            at = torch.arange(r, min(Sq, r + step), device=dev)[:, None] + (Sk - Sq) - torch.arange(Sk, device=dev)[None]
            rs = slice(r, r + at.shape[0])
            vis = at >= 0 if case["causal"] else torch.ones_like(at, dtype=torch.bool)
            if case["prefix"]:
                vis = vis | (torch.arange(Sk, device=dev)[None] < st["prefix"][b])
            if case["docs"]:
                d = st["doc"][b]
                vis = vis & (d[rs, None] == d[None]) & (d[rs, None] >= 0)
            for h in range(Hq):
                pen = float(st["slopes"][h]) * at.abs().double() if case["bias"] else None
                leaves = [q[b, rs, h], k[b, :, h // G], v[b, :, h // G]]
                if case["train"]:
                    leaves = [x.clone().requires_grad_(True) for x in leaves]
                y = _attend(*leaves, scale, cap, pen, vis)
                o[b, rs, h] = y.detach()
                if case["train"]:
                    g = torch.autograd.grad(y, leaves, f64(st["do"][b, rs, h]))
                    dq[b, rs, h] = g[0]
                    dk[b, :, h // G] += g[1]
                    dv[b, :, h // G] += g[2]
    return (o, dq, dk, dv) if case["train"] else o
