"""Token attention operators (turtlevsr_amd/token_ops.py): axial_rope, qk_norm_rope, attention, paged_attention
against their definitions in fp64, gradients included, at the sizes and masks where such kernels go wrong.

Tolerances are error bounds of the algorithm, element by element. u = eps / 2 of the type is one rounding. Scores are
fp32 sums of D products: their error E is at most (D / 2 + 8) 2^-23 of the largest sum of |q k|, and p's relative error
is E. With A = p |v|: |o - ref| <= (2 u + E) A (p rounded once, o rounded once). Likewise dv over p^T |do|; dq and dk add
the absolute errors of dP and delta times p, through |k| and |q|: both are fp32 sums of D products, and delta = do . o takes
the o that the rounded p gave (u A, before o's own rounding, whose remainder the kernel keeps: 2 u^2), so its error is
(u + 2 u^2 + E) |do| . A besides.
"""
import math
import os
import re

import pytest
import torch

from turtlevsr_amd import _lib, token_ops as T

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def unit(dt):
    return torch.finfo(dt).eps / 2


def randn(*shape, dtype=torch.float32, seed=0, dev=DEV):
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + sum(shape))
    return torch.randn(*shape, device=dev, generator=g).to(dtype)


def within(got, ref, tol, what):
    got = got.detach().double()
    assert got.shape == ref.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bad = (got - ref).abs() > tol
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        t = tol.expand_as(ref)[i]
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {i}: {got[i]} for {ref[i]} (+- {t})")


# -------------------------------------------------------------------------------------------------
# definitions in fp64
# -------------------------------------------------------------------------------------------------

def rope_ref(x, pos, axes, base=10000.0, inverse=False):
    B, S, H, D = x.shape
    p = pos.double().expand(B, S, len(axes))
    y = x.clone()
    c = 0
    for a, d in enumerate(axes):
        for i in range(d // 2):
            th = p[:, :, a] * base ** (-2.0 * i / d) * (-1 if inverse else 1)
            co, si = th.cos()[:, :, None], th.sin()[:, :, None]
            x0, x1 = x[..., c], x[..., c + 1]
            y[..., c], y[..., c + 1] = x0 * co - x1 * si, x0 * si + x1 * co
            c += 2
    return y


def visible_ref(B, Sq, Sk, causal=False, prefix=None, q_doc=None, k_doc=None, dev=DEV):
    i, j = torch.arange(Sq, device=dev)[:, None] + (Sk - Sq), torch.arange(Sk, device=dev)[None]
    vis = torch.ones(B, Sq, Sk, dtype=torch.bool, device=dev)
    if causal:
        vis &= (j <= i)[None]
        if prefix is not None:
            pre = torch.as_tensor(prefix, device=dev).expand(B)
            vis |= j[None] < pre[:, None, None]
    if q_doc is not None:
        k_doc = q_doc if k_doc is None else k_doc
        vis &= (q_doc[:, :, None] == k_doc[:, None, :]) & (q_doc[:, :, None] >= 0)
    return vis


def attn_ref(q, k, v, vis, scale=None, softcap=0.0, slopes=None, do=None, dist=None):
    """Results and their error bounds from fp64 matrices: {"o": (ref, tol), "dq": ...}."""
    dt = q.dtype
    B, Sq, Hq, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    G = Hq // Hk
    u = unit(dt)
    scale = D ** -0.5 if scale is None else scale
    # what no query may see is not part of the definition
    seen = vis.any(1)[:, :, None, None]
    rows = vis.any(2)[:, None, :, None]
    f = lambda t: t.detach().double().permute(0, 2, 1, 3)
    Q = torch.where(rows, f(q), 0.0)
    K, V = (torch.where(seen.permute(0, 2, 1, 3), f(t), 0.0).repeat_interleave(G, 1) for t in (k, v))
    raw = Q @ K.transpose(2, 3) * scale
    mag = (Q.abs() @ K.abs().transpose(2, 3)).max() * abs(scale)
    E = (D / 2 + 8) * 2.0 ** -23 * float(mag) + 2.0 ** -20
    s = softcap * torch.tanh(raw / softcap) if softcap else raw
    if softcap:
        E += softcap * 2.0 ** -22
    if slopes is not None:
        if dist is None:
            dist = (torch.arange(Sq, device=q.device)[:, None] + (Sk - Sq) - torch.arange(Sk, device=q.device)[None]).abs().double()[None, None]
        pen = slopes.double().view(1, Hq, 1, 1) * dist
        s = s - pen
        E += float(torch.where(vis[:, None], pen, 0.0).max()) * 2.0 ** -22
    m = vis[:, None]
    s = s.masked_fill(~m, -math.inf)
    p = torch.softmax(torch.where(rows, s, 0.0), -1) * rows * m
    o = p @ V
    out = {"o": (o, (2 * u + E) * (p @ V.abs()) + 1e-30)}
    if do is not None:
        g = torch.where(rows, f(do), 0.0)
        dp = g @ V.transpose(2, 3)
        delta = (g * o).sum(-1, keepdim=True)
        dcap = 1 - torch.tanh(raw / softcap) ** 2 if softcap else 1.0
        pd = p * (dp - delta)
        ds = pd * dcap * scale
        e32 = (D / 2 + 8) * 2.0 ** -23
        edp = e32 * (g.abs() @ V.abs().transpose(2, 3))
        edl = (e32 + u + 2 * u * u + 2 * E) * (g.abs() * (p @ V.abs())).sum(-1, keepdim=True)
        eds = ((u + E + 2.0 ** -20) * pd.abs() + p * (edp + edl) + (2.0 ** -24 if dt == torch.float16 else 0.0) * m * rows) * abs(scale)
        dq, dqt = ds @ K, eds @ K.abs() * (1 + 2 * u)
        sums = lambda t: t.view(B, Hk, G, Sk, D).sum(2)
        dk, dkt = sums(ds.transpose(2, 3) @ Q), sums(eds.transpose(2, 3) @ Q.abs()) * (1 + 2 * u)
        dv, dvt = sums(p.transpose(2, 3) @ g), (2 * u + E) * sums(p.transpose(2, 3) @ g.abs())
        floor = 2.0 ** -24 if dt == torch.float16 else 1e-30
        out.update(dq=(dq, dqt + u * dq.abs() + floor), dk=(dk, dkt + u * dk.abs() + floor), dv=(dv, dvt + floor))
    return {n: (a.permute(0, 2, 1, 3), b.permute(0, 2, 1, 3)) for n, (a, b) in out.items()}


def check_attention(q, k, v, do=None, **kw):
    vis = visible_ref(q.shape[0], q.shape[1], k.shape[1], kw.get("causal", False), kw.get("prefix"), kw.get("q_doc"), kw.get("k_doc"))
    ref = attn_ref(q, k, v, vis, kw.get("scale"), kw.get("softcap", 0.0), kw.get("slopes"), do)
    if do is None:
        within(T.attention(q, k, v, **kw), *ref["o"], "o")
        return
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = T.attention(q, k, v, **kw)
    within(o, *ref["o"], "o")
    for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)):
        within(g, *ref[n], n)


# -------------------------------------------------------------------------------------------------
# refusals and the C surface (no GPU)
# -------------------------------------------------------------------------------------------------

def test_token_exports_match_header():
    hdr = open(os.path.join(REPO, "include", "turtle_token.h")).read()
    declared = set(re.findall(r"\b(turtle_token_[a-z0-9_]+)\s*\(", hdr))
    assert len(declared) == 9
    L = _lib.lib()
    for s in declared:
        assert hasattr(L, s), s
    T.lib()


def test_c_entries_refuse_bad_arguments():
    """Every entry returns an error for missing pointers and sizes out of range; none launches anything."""
    L = T.lib()
    s, ax = bytes(T._SIDE.size), T._axes_table((8, 8, 8), 1e4)
    assert L.turtle_token_rope(s, None, ax, None, 0, 0, 1, 1, 64, 0, 1, None) == -1
    assert L.turtle_token_norm_rope_fwd(s, s, ax, None, 0, 0, 1, 1, 64, 1e-6, 1, None) == -1
    assert L.turtle_token_norm_rope_bwd(s, s, ax, None, 0, 0, 1, 1, 64, 1e-6, None, None, 0, 1, None) == -1
    assert L.turtle_token_norm_rope_workspace(0, 64) == 0

    def args(B, Sq, Sk, Hq, Hk, D):
        a = [0] * (len(T._ATTN.unpack(bytes(T._ATTN.size))))
        a[12:18] = B, Sq, Sk, Hq, Hk, D
        return T._ATTN.pack(*a)
    none = args(0, 0, 0, 0, 0, 0)
    assert L.turtle_token_attn_fwd(none, 1, None) == -1 and L.turtle_token_attn_bwd(none + bytes(T._GRADS.size), 1, None) == -1
    assert L.turtle_token_attn_fwd(None, 1, None) == -1 and L.turtle_token_attn_bwd(None, 1, None) == -1
    assert L.turtle_token_attn_workspace(none, 1) == 0 and L.turtle_token_attn_workspace(None, 1) == 0
    assert L.turtle_token_attn_fwd(args(1, 1, 100, 4, 3, 64), 1, None) == -1           # heads not a multiple
    assert L.turtle_token_attn_fwd(args(1, 1, 100, 4, 1, 60), 1, None) == -1           # channels
    assert L.turtle_token_attn_fwd(args(1, 1, 100, 4, 1, 64), 1, None) == -1           # no tensors
    big = args(1, 1 << 29, 100, 4, 1, 64)                                              # 2^31 rows
    assert L.turtle_token_attn_workspace(big, 1) == 0 and L.turtle_token_attn_fwd(big, 1, None) == -1


def _cpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_rope_refusals():
    x, pos = _cpu(2, 5, 3, 64), torch.zeros(5, 3, dtype=torch.int32)
    ok = (16, 24, 24)
    with pytest.raises(RuntimeError, match="ROCm device"):
        T.axial_rope(x, pos, ok)
    with pytest.raises(ValueError, match="S, heads, D"):
        T.axial_rope(x[0], pos, ok)
    with pytest.raises(TypeError):
        T.axial_rope(x.double(), pos, ok)
    with pytest.raises(ValueError, match="multiple of 8"):
        T.axial_rope(x[..., :60], pos, (8, 8, 8))
    with pytest.raises(ValueError, match="multiple of 8"):
        T.axial_rope(_cpu(2, 5, 3, 136), pos, (8, 8, 8))
    for axes in [(16, 24, 26), (15, 8, 8), (), (8,) * 5, (-2, 8, 8)]:
        with pytest.raises(ValueError, match="axes"):
            T.axial_rope(x, pos, axes)
    with pytest.raises(ValueError, match="base"):
        T.axial_rope(x, pos, ok, base=0.5)
    with pytest.raises(TypeError, match="pos"):
        T.axial_rope(x, pos.float(), ok)
    for shape in [(5, 2), (4, 3), (3, 5, 3)]:
        with pytest.raises(ValueError, match="pos"):
            T.axial_rope(x, torch.zeros(*shape, dtype=torch.int64), ok)
    k = _cpu(2, 5, 1, 64)
    with pytest.raises(RuntimeError, match="ROCm device"):
        T.qk_norm_rope(x, k, pos, None, None, ok)
    with pytest.raises(ValueError, match="does not match"):
        T.qk_norm_rope(x, k[:, :4], pos, None, None, ok)
    with pytest.raises(TypeError, match="k is"):
        T.qk_norm_rope(x, k.float(), pos, None, None, ok)
    with pytest.raises(ValueError, match="q_weight"):
        T.qk_norm_rope(x, k, pos, torch.zeros(32), None, ok)
    with pytest.raises(TypeError, match="k_weight"):
        T.qk_norm_rope(x, k, pos, None, torch.zeros(64, dtype=torch.int32), ok)
    with pytest.raises(ValueError, match="eps"):
        T.qk_norm_rope(x, k, pos, None, None, ok, eps=-1.0)


def test_attention_refusals():
    q, k = _cpu(2, 5, 4, 64), _cpu(2, 7, 2, 64)
    with pytest.raises(RuntimeError, match="ROCm device"):
        T.attention(q, k, k)
    with pytest.raises(ValueError, match="not a multiple"):
        T.attention(q, _cpu(2, 7, 3, 64), _cpu(2, 7, 3, 64))
    with pytest.raises(ValueError, match="one shape"):
        T.attention(q, k, k[:, :6])
    with pytest.raises(ValueError, match="sequences"):
        T.attention(q, k[:1], k[:1])
    with pytest.raises(TypeError):
        T.attention(q, k, k.float())
    with pytest.raises(ValueError, match="prefix"):
        T.attention(q, k, k, prefix=3)
    with pytest.raises(ValueError, match="prefix"):
        T.attention(q, k, k, causal=True, prefix=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(TypeError, match="prefix"):
        T.attention(q, k, k, causal=True, prefix=torch.zeros(2))
    with pytest.raises(ValueError, match="k_doc"):
        T.attention(q, k, k, q_doc=torch.zeros(2, 5, dtype=torch.int32))
    with pytest.raises(ValueError, match="k_doc"):
        T.attention(q, k, k, k_doc=torch.zeros(2, 7, dtype=torch.int32))
    with pytest.raises(TypeError, match="q_doc"):
        T.attention(q, k, k, q_doc=torch.zeros(2, 5), k_doc=torch.zeros(2, 7))
    for c in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="softcap"):
            T.attention(q, k, k, softcap=c)
    with pytest.raises(ValueError, match="scale"):
        T.attention(q, k, k, scale=float("inf"))
    with pytest.raises(ValueError, match="slopes"):
        T.attention(q, k, k, slopes=torch.zeros(2))
    with pytest.raises(TypeError, match="slopes"):
        T.attention(q, k, k, slopes=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="no gradient"):
        T.attention(q, k, k, slopes=torch.zeros(4, requires_grad=True))


def test_paged_refusals():
    q, pool = _cpu(2, 1, 4, 64), _cpu(6, 16, 2, 64)
    tab, kl = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm device"):
        T.paged_attention(q, pool, pool, tab, kl)
    with pytest.raises(ValueError, match="block_table"):
        T.paged_attention(q, pool, pool, tab[0], kl)
    with pytest.raises(TypeError, match="block_table"):
        T.paged_attention(q, pool, pool, tab.long(), kl)
    with pytest.raises(TypeError, match="kv_lens"):
        T.paged_attention(q, pool, pool, tab, kl.long())
    with pytest.raises(ValueError, match="kv_lens"):
        T.paged_attention(q, pool, pool, tab, kl[:1])
    with pytest.raises(ValueError, match="q_lens"):
        T.paged_attention(q, pool, pool, tab, kl, q_lens=kl[:1])
    with pytest.raises(ValueError, match="one shape"):
        T.paged_attention(q, pool, pool[:5], tab, kl)
    with pytest.raises(RuntimeError, match="no gradient"):
        T.paged_attention(q.requires_grad_(True), pool, pool, tab, kl)


# -------------------------------------------------------------------------------------------------
# rotation and norm
# -------------------------------------------------------------------------------------------------

def _grid(S, naxis, t0=0):
    g = torch.Generator().manual_seed(S)
    p = torch.randint(0, 50, (S, naxis), generator=g)
    p[:, 0] += t0
    return p.to(DEV)


ROPES = [(1, 1, 1, (8,), 8, 0), (2, 7, 3, (2, 4, 2), 8, 5), (1, 33, 2, (16, 24, 24), 64, 100003), (3, 19, 5, (8, 16, 12), 40, -70000),
         (2, 130, 9, (32, 48, 48), 128, 2000000000), (1, 5, 17, (0, 10, 0, 14), 24, 3), (1, 300, 1, (20,), 96, 1 << 20)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,S,H,axes,D,t0", ROPES)
def test_axial_rope_matches_definition(dt, B, S, H, axes, D, t0):
    """|y - ref| <= u |ref| + the angle's and functions' error (2^-20 in 16-bit types, 2^-22 in fp32) of the pair."""
    x, dy = randn(B, S, H, D, dtype=dt, seed=1), randn(B, S, H, D, dtype=dt, seed=2)
    err = 2.0 ** -22 if dt == torch.float32 else 2.0 ** -18
    for pos in (_grid(S, len(axes), t0).to(torch.int32), torch.stack([_grid(S, len(axes), t0 + b) for b in range(B)]).long()):
        leaf = x.detach().requires_grad_(True)
        y = T.axial_rope(leaf, pos, axes)
        (dx,) = torch.autograd.grad(y, leaf, dy)
        for got, src, inv in ((y, x, False), (dx, dy, True)):
            ref = rope_ref(src.double(), pos, axes, inverse=inv)
            pair = src.double().abs()
            pair = pair + pair.view(B, S, H, D // 2, 2).flip(-1).reshape(B, S, H, D)
            within(got, ref, unit(dt) * ref.abs() + (err + unit(dt) * 2.0 ** -8) * pair, "dx" if inv else "y")
        n = sum(axes)
        assert torch.equal(y.detach()[..., n:], x[..., n:])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,S,Hq,Hk,axes,D", [(1, 1, 1, 1, (8,), 8), (2, 65, 4, 2, (16, 24, 24), 64), (3, 41, 6, 2, (8, 16, 12), 40),
                                               (1, 700, 9, 3, (32, 48, 48), 128), (2, 257, 16, 16, (2, 2, 2), 16)])
def test_qk_norm_rope_matches_definition(dt, B, S, Hq, Hk, axes, D):
    """fp32 arithmetic, results rounded once: |y - ref| <= u |ref| + 2^-18 (16-bit) or 2^-20 of the pair's magnitude;
    dx in terms of the magnitudes that cancel in it; dw is a sum of N terms in fp32: 2^-20 of the sum of |terms|
    (blocked partial sums: under 64 roundings a path)."""
    eps = 1e-6
    err = 2.0 ** -20 if dt == torch.float32 else 2.0 ** -18
    pos = _grid(S, len(axes), 1234)
    qkv = randn(B, S, Hq + 2 * Hk, D, dtype=dt, seed=3)
    wq, wk = 1 + 0.2 * randn(D, seed=4), 1 + 0.2 * randn(D, seed=5)
    g = [randn(B, S, h, D, dtype=dt, seed=6 + h) for h in (Hq, Hk)]
    q, k = qkv[:, :, :Hq].detach().requires_grad_(True), qkv[:, :, Hq:Hq + Hk].detach().requires_grad_(True)
    lw = [w.clone().requires_grad_(True) for w in (wq, wk)]
    out = T.qk_norm_rope(q, k, pos, *lw, axes, eps=eps)
    grads = torch.autograd.grad(out, (q, k, *lw), g)
    for n, x, w, y, dy, dx, dw in (("q", q, wq, out[0], g[0], grads[0], grads[2]), ("k", k, wk, out[1], g[1], grads[1], grads[3])):
        X, W, H = x.detach().double(), w.double(), x.shape[2]
        r = 1 / (X.pow(2).mean(-1, keepdim=True) + eps).sqrt()
        swap = lambda t: t.abs() + t.abs().view(B, S, H, D // 2, 2).flip(-1).reshape(B, S, H, D)
        ref = rope_ref(X * r * W, pos, axes)
        within(y, ref, unit(dt) * ref.abs() + err * swap(X * r * W), n)
        dz = rope_ref(dy.double(), pos, axes, inverse=True)
        gw = dz * W
        m = (gw * X * r).mean(-1, keepdim=True)
        ref = r * (gw - X * r * m)
        mag = r * (swap(dy.double()) * W.abs() + (X * r).abs() * (swap(dy.double()) * (W * X * r).abs()).mean(-1, keepdim=True))
        within(dx, ref, unit(dt) * ref.abs() + err * mag, "d" + n)
        terms = dz * X * r
        within(dw, terms.sum((0, 1, 2)), err * (swap(dy.double()) * (X * r).abs()).sum((0, 1, 2)), "dw " + n)
    assert torch.equal(T.qk_norm_rope(q, k, pos, wq, wk, axes)[0], out[0])


@pytest.mark.gpu
def test_qk_norm_rope_partial_gains_and_repeat():
    """None for a gain is a gain of one; a gain in bf16 gets a bf16 gradient; repeats are bit-identical."""
    q, k = randn(2, 100, 4, 64, dtype=torch.bfloat16, seed=1), randn(2, 100, 2, 64, dtype=torch.bfloat16, seed=2)
    pos = _grid(100, 3)
    one = torch.ones(64, device=DEV)
    a = T.qk_norm_rope(q, k, pos, None, one, (16, 24, 24))
    b = T.qk_norm_rope(q, k, pos, one, None, (16, 24, 24))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    w = one.bfloat16().requires_grad_(True)
    ql = q.detach().requires_grad_(True)
    runs = []
    for _ in range(3):
        y = T.qk_norm_rope(ql, k, pos, w, None, (16, 24, 24))
        runs.append(torch.autograd.grad(y[0], (ql, w), a[0]))
    assert runs[0][1].dtype == torch.bfloat16
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))


@pytest.mark.gpu
def test_rope_empty_and_unaligned():
    pos = _grid(6, 3)
    for shape in [(0, 6, 2, 64), (2, 0, 2, 64)]:
        x = torch.zeros(*shape, device=DEV, requires_grad=True)
        y = T.axial_rope(x, pos[:shape[1]], (16, 24, 24))
        assert y.shape == x.shape
        q, k = T.qk_norm_rope(x, x, pos[:shape[1]], torch.ones(64, device=DEV, requires_grad=True), None, (16, 24, 24))
        (q.sum() + k.sum()).backward()
        assert x.grad.shape == x.shape
    # rows that do not start at 16 bytes, heads before tokens, a transposed channel axis: same values
    x = randn(2, 6, 2, 64, dtype=torch.bfloat16)
    want = T.axial_rope(x, pos, (16, 24, 24))
    odd = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x)
    swapped = x.transpose(1, 2).contiguous().transpose(1, 2)
    chan = x.transpose(2, 3).contiguous().transpose(2, 3)
    for y in (odd, swapped, chan):
        assert torch.equal(T.axial_rope(y, pos, (16, 24, 24)), want)


# -------------------------------------------------------------------------------------------------
# attention
# -------------------------------------------------------------------------------------------------

SIZES = [(1, 1, 1, 1, 1, 8), (2, 1, 5, 2, 1, 64), (1, 2, 64, 4, 4, 64), (1, 33, 65, 2, 2, 40), (2, 64, 64, 4, 2, 64), (1, 129, 127, 3, 1, 128),
         (1, 31, 200, 8, 1, 16), (2, 200, 31, 2, 2, 96), (1, 257, 511, 2, 1, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,Sq,Sk,Hq,Hk,D", SIZES)
@pytest.mark.parametrize("kind", ["full", "causal", "prefix", "bias_cap"])
def test_attention_and_gradients(dt, B, Sq, Sk, Hq, Hk, D, kind):
    q, k, v = (randn(B, s, h, D, dtype=dt, seed=i) for i, (s, h) in enumerate(((Sq, Hq), (Sk, Hk), (Sk, Hk))))
    do = randn(B, Sq, Hq, D, dtype=dt, seed=9)
    kw = {"full": {}, "causal": dict(causal=True), "prefix": dict(causal=True, prefix=torch.tensor([Sk // 3 + b for b in range(B)], device=DEV)),
          "bias_cap": dict(softcap=2.0, slopes=torch.linspace(0.01, 0.5, Hq, device=DEV))}[kind]
    check_attention(q, k, v, do, **kw)


def _docs(B, S, seed, pad):
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(1, max(2, S // 4), (B, S), generator=g)
    d = torch.zeros(B, S, dtype=torch.int64)
    for b in range(B):
        ids = torch.repeat_interleave(torch.arange(S), n[b])[:S - pad]
        d[b, :S - pad] = ids
        d[b, S - pad:] = -1
    return d.to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,S,Hq,Hk,D,pad,causal", [(1, 1, 1, 1, 64, 0, False), (2, 70, 4, 2, 64, 9, False), (1, 300, 2, 1, 128, 70, True),
                                                     (1, 700, 2, 2, 64, 0, False), (3, 20, 2, 1, 32, 20, True), (1, 1100, 1, 1, 48, 130, True)])
def test_attention_documents_hide_padding_that_holds_nan(dt, B, S, Hq, Hk, D, pad, causal):
    q, k, v = (randn(B, S, h, D, dtype=dt, seed=i) for i, h in enumerate((Hq, Hk, Hk)))
    do = randn(B, S, Hq, D, dtype=dt, seed=9)
    doc = _docs(B, S, S, pad)
    for t in (q, k, v, do):
        t[doc < 0] = float("nan")
    if pad:
        q[:, -1], v[:, -1] = float("inf"), float("-inf")
    check_attention(q, k, v, do, q_doc=doc, causal=causal, softcap=0.0 if S == 70 else 3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_attention_documents_out_of_order_and_cross(dt):
    """Numbers in any order, query numbers that no key has, keys against another clip's queries."""
    q, k, v = randn(2, 150, 4, 64, dtype=dt, seed=1), randn(2, 333, 2, 64, dtype=dt, seed=2), randn(2, 333, 2, 64, dtype=dt, seed=3)
    g = torch.Generator().manual_seed(4)
    qd = torch.randint(-1, 5, (2, 150), generator=g).to(DEV)
    kd = torch.randint(-1, 4, (2, 333), generator=g).to(DEV, torch.int32)
    check_attention(q, k, v, randn(2, 150, 4, 64, dtype=dt, seed=5), q_doc=qd, k_doc=kd)
    qd[0], kd[1] = 7, 9                        # nothing matches at all
    check_attention(q, k, v, randn(2, 150, 4, 64, dtype=dt, seed=5), q_doc=qd, k_doc=kd)
    # few rows over many tiles of documents
    q1, qd1 = q[:, :3].contiguous(), torch.tensor([[2, 0, 3], [1, 1, 6]], device=DEV)
    kd2 = torch.arange(333, device=DEV).div(60, rounding_mode="floor").expand(2, 333)
    check_attention(q1, k, v, randn(2, 3, 4, 64, dtype=dt, seed=6), q_doc=qd1, k_doc=kd2)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,Sk", [(1, 9000), (5, 3001), (40, 5000), (700, 2100)])
@pytest.mark.parametrize("dt", DTYPES)
def test_attention_few_rows_over_many_keys(dt, Sq, Sk):
    """The keys split over blocks and joined."""
    q, k, v = randn(1, Sq, 4, 64, dtype=dt, seed=1), randn(1, Sk, 2, 64, dtype=dt, seed=2), randn(1, Sk, 2, 64, dtype=dt, seed=3)
    do = randn(1, Sq, 4, 64, dtype=dt, seed=4)
    check_attention(q, k, v, do)
    check_attention(q, k, v, do, causal=True, slopes=torch.tensor([0.3, 0.02, 0.001, 0.0], device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_attention_large_scores_and_scales(dt):
    """Scores in the hundreds (a one-hot softmax), a negative scale, a scale of zero, one key far above the rest late."""
    q, k, v = randn(1, 100, 2, 64, dtype=dt, seed=1), randn(1, 300, 2, 64, dtype=dt, seed=2), randn(1, 300, 2, 64, dtype=dt, seed=3)
    do = randn(1, 100, 2, 64, dtype=dt, seed=4)
    for scale in (3.0, -0.125, 0.0):
        check_attention(q, k, v, do, scale=scale)
    k2 = k.clone()
    k2[:, 290] *= 16
    check_attention(q, k2, v, do)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_attention_strides_and_broadcast(dt):
    """Slices of a channels-last projection, heads-first layouts, a key shared by expand (its gradient is the sum), a
    gradient that arrives expanded."""
    B, H, W, heads, D = 2, 6, 7, 2, 64
    S = H * W
    qkv = randn(B, 3 * heads * D, H, W, dtype=dt, seed=1).to(memory_format=torch.channels_last)
    q, k, v = qkv.permute(0, 2, 3, 1).reshape(B, S, 3, heads, D).unbind(2)
    assert q.data_ptr() == qkv.data_ptr()
    do = randn(B, S, heads, D, dtype=dt, seed=2)
    check_attention(q, k, v, do)
    hf = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    check_attention(hf(q), hf(k), hf(v), hf(do))
    k1 = randn(1, S, heads, D, dtype=dt, seed=3).requires_grad_(True)
    o = T.attention(q, k1.expand(B, -1, -1, -1), v)
    (gk,) = torch.autograd.grad(o, k1, do)
    kf = k1.detach().expand(B, -1, -1, -1).contiguous().requires_grad_(True)
    (gf,) = torch.autograd.grad(T.attention(q, kf, v), kf, do)
    assert torch.equal(gk, gf.sum(0, keepdim=True))
    ql = q.detach().requires_grad_(True)
    (a,) = torch.autograd.grad(T.attention(ql, k, v).sum(), ql)
    (b,) = torch.autograd.grad(T.attention(ql, k, v), ql, torch.ones_like(do))
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_attention_rows_past_32_bit_offsets():
    """Token strides that put the last keys 5 GB behind the first."""
    S, D, stride = 40001, 64, 65536
    big = torch.empty(S * stride, dtype=torch.bfloat16, device=DEV)
    k = big.as_strided((1, S, 1, D), (0, stride, D, 1))
    v = big.as_strided((1, S, 1, D), (0, stride, D, 1), D)
    k.copy_(randn(1, S, 1, D, dtype=torch.bfloat16, seed=1))
    v.copy_(randn(1, S, 1, D, dtype=torch.bfloat16, seed=2))
    q = randn(1, 3, 2, D, dtype=torch.bfloat16, seed=3)
    do = randn(1, 3, 2, D, dtype=torch.bfloat16, seed=4)
    check_attention(q, k, v, do)


@pytest.mark.gpu
def test_attention_no_tokens():
    for Sq, Sk in ((0, 5), (5, 0), (0, 0)):
        q, k = torch.zeros(2, Sq, 2, 64, device=DEV, requires_grad=True), torch.ones(2, Sk, 2, 64, device=DEV, requires_grad=True)
        o = T.attention(q, k, k)
        assert o.shape == q.shape and not o.any()
        o.sum().backward()
        assert q.grad.shape == q.shape and k.grad.shape == k.shape and not q.grad.any() and not k.grad.any()


@pytest.mark.gpu
def test_attention_gradient_against_differences():
    """fp32: the directional derivative of sum(do o) along random directions, by central differences in fp64 of the
    definition and from the kernel's gradients."""
    B, Sq, Sk, Hq, Hk, D = 1, 9, 14, 2, 1, 16
    q, k, v = (randn(B, s, h, D, seed=i) for i, (s, h) in enumerate(((Sq, Hq), (Sk, Hk), (Sk, Hk))))
    do, kw = randn(B, Sq, Hq, D, seed=5), dict(causal=True, softcap=1.5)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(T.attention(*leaves, **kw), leaves, do)

    def value(ts):
        qd, kd, vd = (t.double().transpose(1, 2) for t in ts)
        z = qd @ kd.repeat_interleave(Hq // Hk, 1).transpose(2, 3) * D ** -0.5
        z = 1.5 * torch.tanh(z / 1.5)
        z = z.masked_fill(~visible_ref(B, Sq, Sk, True)[:, None], -math.inf)
        return float((torch.softmax(z, -1) @ vd.repeat_interleave(Hq // Hk, 1) * do.double().transpose(1, 2)).sum())

    for i in range(3):
        d = randn(*leaves[i].shape, seed=20 + i).double()
        h = 1e-5
        at = lambda s: [t.detach().double() + (s * h * d if j == i else 0) for j, t in enumerate(leaves)]
        diff = (value(at(1)) - value(at(-1))) / (2 * h)
        got = float((grads[i].double() * d).sum())
        assert abs(got - diff) <= 1e-5 * float((grads[i].double() * d).abs().sum()) + 1e-7


@pytest.mark.gpu
def test_attention_repeats_bit_for_bit_and_only_wanted_gradients():
    q, k, v = (randn(2, 500, h, 64, dtype=torch.bfloat16, seed=h) for h in (4, 2, 2))
    do = randn(2, 500, 4, 64, dtype=torch.bfloat16, seed=9)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    first = torch.autograd.grad(T.attention(*leaves, causal=True), leaves, do)
    for _ in range(3):
        again = torch.autograd.grad(T.attention(*leaves, causal=True), leaves, do)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    (dq,) = torch.autograd.grad(T.attention(q, k.detach(), v.detach(), causal=True), q, do)
    (dv,) = torch.autograd.grad(T.attention(q.detach(), k.detach(), v, causal=True), v, do)
    assert torch.equal(dq, first[0]) and torch.equal(dv, first[2])


# -------------------------------------------------------------------------------------------------
# pages
# -------------------------------------------------------------------------------------------------

def _pages(B, lens, page, Hk, D, dt, spare=2, seed=0):
    """(k_pages, v_pages, table, dense k, dense v): random page order; everything past a length is NaN."""
    M = max(1, max(-(-n // page) for n in lens))
    n = B * M + spare
    kp, vp = (torch.full((n, page, Hk, D), float("nan"), dtype=dt, device=DEV) for _ in range(2))
    table = torch.randperm(n, generator=torch.Generator().manual_seed(seed))[:B * M].reshape(B, M).to(torch.int32)
    k, v = randn(B, max(1, max(lens)), Hk, D, dtype=dt, seed=seed + 1), randn(B, max(1, max(lens)), Hk, D, dtype=dt, seed=seed + 2)
    for b in range(B):
        for j in range(0, lens[b], page):
            e = min(page, lens[b] - j)
            kp[table[b, j // page], :e], vp[table[b, j // page], :e] = k[b, j:j + e], v[b, j:j + e]
        table[b, -(-lens[b] // page):] = -1
    return kp, vp, table.to(DEV), k, v


def check_paged(q, kp, vp, table, kl, k, v, ql=None, hidden=None, **kw):
    """hidden: bool [B, keys], keys that nobody sees (bad pages)."""
    B, Sq = q.shape[:2]
    klt = torch.tensor(kl, dtype=torch.int32, device=DEV)
    qlt = None if ql is None else torch.tensor(ql, dtype=torch.int32, device=DEV)
    got = T.paged_attention(q, kp, vp, table, klt, q_lens=qlt, **kw)
    i, j = torch.arange(Sq, device=DEV), torch.arange(k.shape[1], device=DEV)
    nq = torch.tensor([Sq] * B if ql is None else ql, device=DEV).clamp(0, Sq)
    at = i[None] + (klt.long() - nq)[:, None]
    vis = (j[None, None] < klt.long()[:, None, None]) & (i[None, :, None] < nq[:, None, None])
    if kw.get("causal", True):
        vis &= j[None, None] <= at[:, :, None]
    if hidden is not None:
        vis &= ~hidden[:, None]
    dist = (at[:, :, None] - j).abs().double()[:, None]
    ref = attn_ref(q, k, v, vis, kw.get("scale"), kw.get("softcap", 0.0), kw.get("slopes"), dist=dist)
    within(got, *ref["o"], "o")
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("page,D", [(1, 64), (16, 64), (7, 40), (64, 128), (100, 64), (256, 96)])
def test_paged_single_tokens(dt, page, D):
    lens = [1, 2, 63, 64, 65, 301, 777, 0]
    kp, vp, table, k, v = _pages(len(lens), lens, page, 2, D, dt, seed=page)
    q = randn(len(lens), 1, 8, D, dtype=dt, seed=5)
    check_paged(q, kp, vp, table, lens, k, v)
    check_paged(q, kp, vp, table, lens, k, v, causal=False, softcap=2.0, slopes=torch.linspace(0, 0.3, 8, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("Sq,causal", [(5, True), (37, True), (200, True), (200, False), (130, True)])
def test_paged_chunks_of_ragged_lengths(dt, Sq, causal):
    lens, ql = [Sq, 400, 3 * Sq, 1, 0, 350], [Sq, Sq, max(1, Sq // 2), 1, 0, 0]
    kp, vp, table, k, v = _pages(6, lens, 48, 2, 64, dt, seed=Sq)
    q = randn(6, Sq, 4, 64, dtype=dt, seed=6)
    for b in range(6):
        q[b, ql[b]:] = float("nan")
    check_paged(q, kp, vp, table, lens, k, v, ql, causal=causal)


@pytest.mark.gpu
def test_paged_long_history_is_split_and_pool_passes_32_bits():
    """One token over 20000 keys on pages at the far end of a pool of 6 GB; 2 sequences whose first is tiny."""
    page, Hk, D = 256, 4, 128
    n = 6 * (1 << 30) // (page * Hk * D * 2)
    kp = torch.empty(n, page, Hk, D, dtype=torch.bfloat16, device=DEV)
    vp = torch.empty(n, page, Hk, D, dtype=torch.bfloat16, device=DEV)
    lens = [3, 20000]
    M = -(-lens[1] // page)
    k, v = randn(2, lens[1], Hk, D, dtype=torch.bfloat16, seed=1), randn(2, lens[1], Hk, D, dtype=torch.bfloat16, seed=2)
    table = torch.stack([torch.arange(M), n - 1 - torch.arange(M)]).to(DEV, torch.int32)
    for b in range(2):
        pad = torch.zeros(M * page - lens[1], Hk, D, dtype=torch.bfloat16, device=DEV)
        kp[table[b].long()] = torch.cat((k[b], pad)).view(M, page, Hk, D)
        vp[table[b].long()] = torch.cat((v[b], pad)).view(M, page, Hk, D)
    check_paged(randn(2, 1, 16, D, dtype=torch.bfloat16, seed=3), kp, vp, table, lens, k, v)


def test_paged_bad_pages_are_outside_the_pools_on_paper():
    """The kernel takes a page number as unsigned and compares it with the pool's size before any address is made:
    -1, the pool's size and the extremes all fail that comparison."""
    for bad in (-1, 10, 2 ** 31 - 1, -2 ** 31):
        assert (bad & 0xffffffff) >= 10


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 50])
def test_paged_bad_pages_and_lengths(Sq):
    """Page numbers outside the pools hide their keys; lengths past the table's room are cut to it."""
    page, lens = 16, [100, 64]
    kp, vp, table, k, v = _pages(2, lens, page, 1, 64, torch.bfloat16, seed=3)
    hidden = torch.zeros(2, 100, dtype=torch.bool, device=DEV)
    for b, j, bad in ((0, 0, -1), (0, 3, kp.shape[0]), (1, 2, 2 ** 31 - 1), (1, 1, -2 ** 31)):
        table[b, j] = bad
        hidden[b, j * page:(j + 1) * page] = True
    q = randn(2, Sq, 2, 64, dtype=torch.bfloat16, seed=4)
    check_paged(q, kp, vp, table, lens, k, v, hidden=hidden, causal=False)
    check_paged(q, kp, vp, table, lens, k, v, hidden=hidden)
    cut = table[:, :4].contiguous()               # room for 64 keys of 100
    hidden[:, 64:] = True
    check_paged(q, kp, vp, cut, lens, k, v, hidden=hidden, causal=False)
    none = T.paged_attention(q, kp, vp, table, torch.tensor([-5, 0], dtype=torch.int32, device=DEV))
    assert not none.any()


@pytest.mark.gpu
def test_paged_equals_attention_on_a_dense_history():
    """A chunk over pages gives what attention gives for the same rows (both causal with the last query at the last key)."""
    kp, vp, table, k, v = _pages(2, [300, 300], 64, 2, 64, torch.float32, seed=1)
    q = randn(2, 40, 4, 64, seed=2)
    a = T.attention(q, k, v, causal=True)
    b = T.paged_attention(q, kp, vp, table, torch.tensor([300, 300], dtype=torch.int32, device=DEV))
    within(b, a.double(), torch.full((1,), 1e-5, dtype=torch.float64, device=DEV), "o")


# -------------------------------------------------------------------------------------------------
# together, streams, graphs
# -------------------------------------------------------------------------------------------------

def _block(qkv, pos, wq, wk, heads, D, **kw):
    """The attention of a transformer block over a channels-last map [B, 3 heads D, H, W]."""
    B, _, H, W = qkv.shape
    q, k, v = qkv.permute(0, 2, 3, 1).reshape(B, H * W, 3, heads, D).unbind(2)
    q, k = T.qk_norm_rope(q, k, pos, wq, wk, (D // 4 // 2 * 2, D // 8 * 2, D // 8 * 2))
    return T.attention(q, k, v, **kw), k, v


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_block_trains_through_all_operators(dt):
    """Norm, rotation and attention in one graph: the gradients of the map and the gains against autograd on the fp64
    definitions. Tolerance: the chain rounds q', k' (u each, which moves scores by u sum|q k| scale) and every gradient
    once, so a relative error (Frobenius) under 16 u plus the fp32 arithmetic's 1e-5."""
    B, H, W, heads, D = 2, 5, 9, 2, 64
    ax = (D // 4 // 2 * 2, D // 8 * 2, D // 8 * 2)
    qkv = randn(B, 3 * heads * D, H, W, dtype=dt, seed=1).to(memory_format=torch.channels_last).requires_grad_(True)
    pos = _grid(H * W, 3)
    wq, wk = (1 + 0.1 * randn(D, seed=2)).requires_grad_(True), (1 + 0.1 * randn(D, seed=3)).requires_grad_(True)
    do = randn(B, H * W, heads, D, dtype=dt, seed=4)
    o, _, _ = _block(qkv, pos, wq, wk, heads, D, causal=True, prefix=9)
    got = torch.autograd.grad(o, (qkv, wq, wk), do)

    x, a, b = (t.detach().double().requires_grad_(True) for t in (qkv, wq, wk))
    q, k, v = x.permute(0, 2, 3, 1).reshape(B, H * W, 3, heads, D).unbind(2)
    def nr(t, w):
        z = t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w
        c, parts = 0, []
        for i, d in enumerate(ax):
            th = pos[:, i, None].double() * 10000.0 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
            z0, z1 = z[..., c:c + d:2], z[..., c + 1:c + d:2]
            co, si = th.cos()[:, None], th.sin()[:, None]
            parts.append(torch.stack((z0 * co - z1 * si, z0 * si + z1 * co), -1).flatten(-2))
            c += d
        return torch.cat(parts + [z[..., c:]], -1)
    q, k = nr(q, a).transpose(1, 2), nr(k, b).transpose(1, 2)
    s = (q @ k.transpose(2, 3) * D ** -0.5).masked_fill(~visible_ref(B, H * W, H * W, True, 9)[:, None], -math.inf)
    ref = (torch.softmax(s, -1) @ v.transpose(1, 2)).transpose(1, 2)
    want = torch.autograd.grad(ref, (x, a, b), do.double())
    tol = 16 * unit(dt) + 1e-5
    for n, g, r in zip(("o", "dqkv", "dwq", "dwk"), (o, *got), (ref, *want)):
        rel = float((g.detach().double() - r.detach()).norm() / r.detach().norm())
        assert rel <= tol, (n, rel)


@pytest.mark.gpu
def test_serving_frames_over_a_paged_history():
    """Frame by frame with a page for each frame equals the whole clip at once: tokens of a frame see all of their own
    and of earlier frames (a document per prefix is the frame-causal mask, here by keys up to the frame's end)."""
    heads, D, n, frames = 2, 64, 30, 4
    qkv = randn(1, frames * n, 3, heads, D, dtype=torch.bfloat16, seed=1)
    pos = torch.stack((torch.arange(frames).repeat_interleave(n), torch.arange(n).repeat(frames)), 1).to(DEV)
    w = 1 + 0.1 * randn(D, seed=2)
    q, k = T.qk_norm_rope(qkv[:, :, 0], qkv[:, :, 1], pos, w, w, (32, 32))
    v = qkv[:, :, 2]
    kp, vp = torch.full((6, n, heads, D), float("nan"), dtype=torch.bfloat16, device=DEV), torch.full((6, n, heads, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    table = torch.tensor([[4, 0, 5, 2]], dtype=torch.int32, device=DEV)
    for f in range(frames):
        sl = slice(f * n, (f + 1) * n)
        qf, kf = T.qk_norm_rope(qkv[:, sl, 0], qkv[:, sl, 1], pos[sl], w, w, (32, 32))
        assert torch.equal(qf, q[:, sl]) and torch.equal(kf, k[:, sl])
        kp[table[0, f].long()], vp[table[0, f].long()] = kf[0], v[0, sl]
        o = T.paged_attention(qf, kp, vp, table, torch.tensor([(f + 1) * n], dtype=torch.int32, device=DEV), causal=False)
        e = (f + 1) * n
        ref = attn_ref(q[:, sl], k[:, :e], v[:, :e], torch.ones(1, n, e, dtype=torch.bool, device=DEV))
        within(o, *ref["o"], f"frame {f}")


@pytest.mark.gpu
def test_operators_on_another_stream():
    q, k, v = (randn(1, 300, 2, 64, dtype=torch.bfloat16, seed=i) for i in range(3))
    pos = _grid(300, 3)
    want = T.attention(*T.qk_norm_rope(q, k, pos, None, None, (16, 24, 24)), v)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = T.attention(*T.qk_norm_rope(q, k, pos, None, None, (16, 24, 24)), v)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_inference_in_a_graph_follows_its_inputs():
    """A captured step - rotation, cache write, paged attention, dense attention with documents - replayed with other
    tokens, lengths, tables and documents, with eager work between the replays."""
    B, heads, D, page, M = 3, 2, 64, 16, 8
    kp, vp = torch.zeros(B * M, page, heads, D, dtype=torch.bfloat16, device=DEV), torch.zeros(B * M, page, heads, D, dtype=torch.bfloat16, device=DEV)
    x = randn(B, 1, 3, heads, D, dtype=torch.bfloat16, seed=1)
    pos = torch.zeros(B, 1, 1, dtype=torch.int32, device=DEV)
    table = torch.arange(B * M, device=DEV, dtype=torch.int32).view(B, M)
    lens = torch.ones(B, dtype=torch.int32, device=DEV)
    seq = randn(1, 600, 3, heads, D, dtype=torch.bfloat16, seed=2)
    doc = torch.zeros(1, 600, dtype=torch.int32, device=DEV)

    def step():
        q, k = T.qk_norm_rope(x[:, :, 0], x[:, :, 1], pos, None, None, (64,))
        slot = table.gather(1, (pos[:, :, 0] // page).long()).long() * page + pos[:, :, 0] % page
        kp.view(-1, heads, D).index_copy_(0, slot[:, 0], k[:, 0])
        vp.view(-1, heads, D).index_copy_(0, slot[:, 0], x[:, 0, 2])
        return T.paged_attention(q, kp, vp, table, lens), T.attention(seq[:, :, 0], seq[:, :, 1], seq[:, :, 2], q_doc=doc)

    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        for n in range(20):
            x.copy_(randn(B, 1, 3, heads, D, dtype=torch.bfloat16, seed=100 + n))
            pos.fill_(n)
            lens.fill_(n + 1)
            doc.copy_((torch.arange(600, device=DEV) // (50 + 10 * n))[None])
            g.replay()
            got = [t.clone() for t in out]
            torch.cuda.synchronize()
            want = step()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), n


@pytest.mark.gpu
def test_training_step_in_a_graph():
    """Forward and backward captured together, replayed on other data; two graphs of their own do not disturb each other."""
    def make(seed):
        leaves = [randn(1, 333, 2, 64, dtype=torch.bfloat16, seed=seed + i).requires_grad_(True) for i in range(3)]
        w = torch.ones(64, device=DEV, requires_grad=True)
        do, pos = randn(1, 333, 2, 64, dtype=torch.bfloat16, seed=seed + 5), _grid(333, 2)

        def step():
            q, k = T.qk_norm_rope(leaves[0], leaves[1], pos, w, None, (32, 32))
            o = T.attention(q, k, leaves[2], causal=True, softcap=5.0)
            return (o.detach(),) + torch.autograd.grad(o, (*leaves, w), do)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        return leaves, do, g, out, step
    a, b = make(1), make(50)
    for n in range(4):
        for leaves, do, g, out, step in (a, b):
            with torch.no_grad():
                for i, t in enumerate(leaves):
                    t.copy_(randn(*t.shape, dtype=t.dtype, seed=200 + n * 10 + i))
        a[2].replay()
        b[2].replay()
        torch.cuda.synchronize()
        for leaves, do, g, out, step in (a, b):
            got = [t.detach().clone() for t in out]
            assert all(torch.equal(x, y.detach()) for x, y in zip(got, step()))


@pytest.mark.gpu
def test_op_set_takes_the_autocast_type():
    """HipOps, the training graph's op set: fp32 tensors under bf16 autocast give the bf16 call's results."""
    from turtlevsr_amd.train_ops import HipOps
    q, k, v = (randn(1, 50, 2, 64, seed=i) for i in range(3))
    b = [t.bfloat16() for t in (q, k, v)]
    pos = _grid(50, 3)
    ax = (16, 24, 24)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        x = HipOps.axial_rope(q, pos, ax)
        y = HipOps.qk_norm_rope(q, k, pos, None, None, ax)
        z = HipOps.attention(q, k, v, causal=True)
        table, lens = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([50], dtype=torch.int32, device=DEV)
        p = HipOps.paged_attention(q, b[1], b[2], table, lens)
    assert torch.equal(x, T.axial_rope(b[0], pos, ax))
    assert all(torch.equal(a, c) for a, c in zip(y, T.qk_norm_rope(b[0], b[1], pos, None, None, ax)))
    assert torch.equal(z, T.attention(*b, causal=True)) and torch.equal(p, T.paged_attention(b[0], b[1], b[2], table, lens))
    assert HipOps.attention(q, k, v).dtype == torch.float32


def _masked(kind, B, Sq, Sk, Hq):
    if kind == "causal_prefix":
        return dict(causal=True, prefix=torch.tensor([(Sk * b) // (2 * B) for b in range(B)], device=DEV))
    if kind == "bias_cap":
        return dict(softcap=2.0, slopes=torch.linspace(0.0, 0.3, Hq, device=DEV))
    if kind == "docs":
        d = _docs(B, max(Sq, Sk), B, 0)
        d[:, Sk - 21:] = -1
        d[B // 2] = -1                         # a sequence of padding alone
        return dict(q_doc=d[:, :Sq], k_doc=d[:, :Sk], causal=Sq == Sk, softcap=3.0)
    return {}


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [40, 64, 104, 128])
@pytest.mark.parametrize("kind", ["full", "causal_prefix", "bias_cap", "docs"])
def test_attention_large_grids(dt, D, kind):
    """Enough sequences that blocks of 128 rows (keys) fill the card: forward, dk and dv, dq with a block's waves side by
    side, ragged last tiles, three query heads a key head; queries and keys of one length and of two."""
    for Sq, Sk in ((300, 300), (261, 300)):
        B, Hq, Hk = 45, 6, 2
        q, k, v = (randn(B, s, h, D, dtype=dt, seed=i) for i, (s, h) in enumerate(((Sq, Hq), (Sk, Hk), (Sk, Hk))))
        check_attention(q, k, v, randn(B, Sq, Hq, D, dtype=dt, seed=9), **_masked(kind, B, Sq, Sk, Hq))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Sk,B", [(130, 8200, 8), (70, 100, 3), (60, 200, 140), (9, 30, 300)])
def test_attention_middle_shapes(dt, D, Sq, Sk, B):
    """Many rows whose long keys are split, few keys in small and large grids."""
    for kind in ("full", "bias_cap"):
        q, k, v = (randn(B, s, h, D, dtype=dt, seed=i) for i, (s, h) in enumerate(((Sq, 2), (Sk, 2), (Sk, 2))))
        check_attention(q, k, v, randn(B, Sq, 2, D, dtype=dt, seed=9), **_masked(kind, B, Sq, Sk, 2))
    q, k, v = (randn(B, s, h, D, dtype=dt, seed=i) for i, (s, h) in enumerate(((Sq, 2), (Sk, 1), (Sk, 1))))
    check_attention(q, k, v, randn(B, Sq, 2, D, dtype=dt, seed=9), **_masked("docs", B, Sq, Sk, 2))
    check_attention(q, k, v, randn(B, Sq, 2, D, dtype=dt, seed=9), causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hk,Sq,Sk", [(4, 4, 260, 260), (8, 2, 700, 700), (48, 2, 300, 300), (8, 1, 100, 900), (2, 4, 3, 4000)])
def test_attention_causal_key_heads_in_eights(dt, D, B, Hk, Sq, Sk):
    """Key heads a multiple of eight, few blocks each: the order in which causal blocks go out."""
    q, k, v = randn(B, Sq, 2 * Hk, D, dtype=dt, seed=1), randn(B, Sk, Hk, D, dtype=dt, seed=2), randn(B, Sk, Hk, D, dtype=dt, seed=3)
    check_attention(q, k, v, randn(B, Sq, 2 * Hk, D, dtype=dt, seed=4), causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 104])
@pytest.mark.parametrize("Sq,Sk", [(3000, 40), (2500, 1), (6, 2000), (900, 900)])
def test_attention_gradients_of_long_walks(dt, D, Sq, Sk):
    """Few keys under many queries and the reverse, one pair of heads: the walks split over blocks and added up."""
    q, k, v = (randn(1, s, h, D, dtype=dt, seed=i) for i, (s, h) in enumerate(((Sq, 2), (Sk, 1), (Sk, 1))))
    do = randn(1, Sq, 2, D, dtype=dt, seed=9)
    check_attention(q, k, v, do, softcap=2.0, slopes=torch.tensor([0.3, 0.0], device=DEV))
    check_attention(q, k, v, do, causal=True, prefix=torch.tensor([Sk // 2], device=DEV))
    g = torch.Generator().manual_seed(Sq)
    docs = [(torch.arange(s) * 5 // s - (torch.rand(s, generator=g) < 0.1).int() * 9)[None].to(DEV) for s in (Sq, Sk)]
    check_attention(q, k, v, do, q_doc=docs[0], k_doc=docs[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_attention_many_heads_share_a_key(dt):
    """80 query heads on one key head: more rows of one query than a tile has, 27 of them: a share that divides nothing."""
    for Hq, Hk, S in ((80, 1, 7), (54, 2, 33)):
        q, k, v = randn(2, S, Hq, 64, dtype=dt, seed=1), randn(2, S + 3, Hk, 64, dtype=dt, seed=2), randn(2, S + 3, Hk, 64, dtype=dt, seed=3)
        check_attention(q, k, v, randn(2, S, Hq, 64, dtype=dt, seed=4), causal=True, slopes=torch.linspace(0, 0.5, Hq, device=DEV))


@pytest.mark.gpu
def test_more_sequences_than_a_grid_axis_has_blocks():
    B = 70000
    q, k = randn(B, 1, 3, 8, dtype=torch.bfloat16, seed=1).requires_grad_(True), randn(B, 1, 1, 8, dtype=torch.bfloat16, seed=2)
    pos, w = torch.arange(B, device=DEV).view(B, 1, 1), torch.linspace(0.5, 2, 8, device=DEV)
    flat = lambda t: t.reshape(1, B, *t.shape[2:])
    assert torch.equal(flat(T.axial_rope(q, pos, (8,))), T.axial_rope(flat(q), flat(pos), (8,)))
    dy = randn(B, 1, 3, 8, dtype=torch.bfloat16, seed=3)
    a, b = T.qk_norm_rope(q, k, pos, w, w, (8,)), T.qk_norm_rope(flat(q), flat(k), flat(pos), w, w, (8,))
    assert torch.equal(flat(a[0]), b[0]) and torch.equal(flat(a[1]), b[1])
    (da,), (db,) = torch.autograd.grad(a[0], q, dy), torch.autograd.grad(b[0], q, flat(dy))
    assert torch.equal(da, db)
    kv = randn(B, 2, 1, 8, dtype=torch.bfloat16, seed=4)
    check_attention(q.detach(), kv[..., :1, :], kv[..., :1, :], dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D,Sq,n,B", [(64, 200, 4300, 8), (128, 200, 4300, 8), (64, 65, 300, 130), (104, 130, 340, 70), (64, 70, 120, 4)])
def test_paged_large_grids(dt, D, Sq, n, B):
    """Blocks of 128 rows over a cache, with its keys split and whole; caches of few keys; ragged lengths."""
    lens = [max(0, n - 37 * (b % 9)) if b % 5 else min(n, 3 + b) for b in range(B)]
    ql = [min(Sq, lens[b]) - (b % 3 if lens[b] > 3 else 0) for b in range(B)]
    kp, vp, table, k, v = _pages(B, lens, 50, 2, D, dt, seed=Sq)
    q = randn(B, Sq, 4, D, dtype=dt, seed=6)
    check_paged(q, kp, vp, table, lens, k, v, ql)
    check_paged(q, kp, vp, table, lens, k, v, ql, causal=False, softcap=2.0, slopes=torch.linspace(0, 0.3, 4, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G,D", [(33, 64), (40, 128), (64, 64)])
def test_attention_bias_of_half_a_wave_and_more_sharing_heads(dt, G, D):
    """Gradients of every sharing head under its own slope, where more heads share a key than a tile has rows."""
    q, k, v = randn(2, 9, G, D, dtype=dt, seed=1), randn(2, 50, 1, D, dtype=dt, seed=2), randn(2, 50, 1, D, dtype=dt, seed=3)
    check_attention(q, k, v, randn(2, 9, G, D, dtype=dt, seed=4), slopes=torch.linspace(0.01, 0.7, G, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,Sk,B", [(3, 9000, 1), (70, 100, 2), (200, 300, 70), (130, 8200, 8)])
def test_attention_not_a_number_stays_in_its_row(Sq, Sk, B):
    """A query that is not a number gives such a row - its keys split over blocks or not - and no other."""
    q, k, v = (randn(B, s, 2, 64, dtype=torch.bfloat16, seed=i) for i, s in enumerate((Sq, Sk, Sk)))
    want = T.attention(q, k, v)
    q[0, 1, 1] = float("nan")
    got = T.attention(q, k, v)
    assert got[0, 1, 1].isnan().all()
    got[0, 1, 1] = want[0, 1, 1]
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("Sq,B", [(5, 2), (200, 2), (200, 70)])
def test_rows_that_see_nothing_are_zero_beside_infinite_values(dt, Sq, B):
    """The rows that do see the infinite value are not finite; infinity or not a number is left open: p may be multiplied as
    hi + lo, and hi inf + lo inf with lo < 0 or lo = 0 is not a number."""
    q, k, v = (randn(B, s, 2, 64, dtype=dt, seed=i) for i, s in enumerate((Sq, 300, 300)))
    v[:, 7] = float("inf")
    doc = torch.zeros(B, 300, dtype=torch.int64, device=DEV)
    qd = doc[:, :Sq].clone()
    qd[:, 2], qd[:, 3] = 5, -1
    o = T.attention(q, k, v, q_doc=qd, k_doc=doc)
    assert not o[:, 2:4].any() and not o[:, 4].isfinite().any()
    lens = torch.full((B,), 300, dtype=torch.int32, device=DEV)
    table = torch.arange(B * 3, dtype=torch.int32, device=DEV).view(B, 3)
    ql = torch.full((B,), Sq - 2, dtype=torch.int32, device=DEV)
    o = T.paged_attention(q, k.view(B * 3, 100, 2, 64), v.view(B * 3, 100, 2, 64), table, lens, q_lens=ql, causal=False)
    assert not o[:, Sq - 2:].any() and not o[:, :Sq - 2].isfinite().any()


@pytest.mark.gpu
def test_attention_rules_at_the_ends_of_their_range():
    """Prefixes below zero and past every key, 64-bit ones past 32 bits; document numbers at the top of 32 bits; padding
    numbers below them."""
    q, k, v = (randn(2, s, 2, 64, seed=i) for i, s in enumerate((40, 70, 70)))
    do = randn(2, 40, 2, 64, seed=5)
    ints = lambda *x: torch.tensor(x, device=DEV)
    for got, same in ((ints(-2 ** 31, 2 ** 31 - 1).int(), ints(0, 70)), (ints(-2 ** 40, 2 ** 40), ints(0, 70)), (-7, 0), (10 ** 12, 70)):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        a, b = T.attention(*leaves, causal=True, prefix=got), T.attention(*leaves, causal=True, prefix=same)
        assert torch.equal(a, b)
        assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(a, leaves, do), torch.autograd.grad(b, leaves, do)))
    qd, kd = torch.zeros(2, 40, dtype=torch.int64, device=DEV), torch.zeros(2, 70, dtype=torch.int64, device=DEV)
    qd[:, ::2], kd[:, ::3], kd[:, 1::3] = 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 2
    check_attention(q, k, v, do, q_doc=qd, k_doc=kd)
    low = kd.clone()
    low[:, 5:60], kd[:, 5:60] = -2 ** 40, -1
    assert torch.equal(T.attention(q, k, v, q_doc=qd, k_doc=low), T.attention(q, k, v, q_doc=qd, k_doc=kd))


@pytest.mark.gpu
def test_one_forward_walked_backward_by_two_graphs():
    """Two captured backward passes of one forward, replayed on two streams at once."""
    side = torch.cuda.Stream()
    leaves = [randn(2, 500, 4, 64, dtype=torch.bfloat16, seed=i).requires_grad_(True) for i in range(3)]
    dos = [randn(2, 500, 4, 64, dtype=torch.bfloat16, seed=5 + i) for i in range(2)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = T.attention(*leaves, causal=True)
        want = [torch.autograd.grad(o, leaves, do, retain_graph=True) for do in dos]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for do in dos:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(torch.autograd.grad(o, leaves, do, retain_graph=True))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in dos]
    for _ in range(4):
        for out in outs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_rope_rows_past_32_bit_offsets():
    """Tokens 5 GB apart, and a dense result of 5 GB."""
    S, D, stride = 40001, 64, 65536
    big = torch.empty(S * stride, dtype=torch.bfloat16, device=DEV)
    x = big.as_strided((1, S, 2, D), (0, stride, D, 1))
    x.copy_(randn(1, S, 2, D, dtype=torch.bfloat16, seed=1))
    pos, w = _grid(S, 3), torch.linspace(0.5, 2, D, device=DEV)
    assert torch.equal(T.axial_rope(x, pos, (16, 24, 24)), T.axial_rope(x.contiguous(), pos, (16, 24, 24)))
    ends = [T.qk_norm_rope(t, t[:, :, :1], pos, w, w, (16, 24, 24)) for t in (x, x.contiguous())]
    assert all(torch.equal(a, b) for a, b in zip(*ends))
    del big, x
    x = torch.empty(1, 300000, 64, 128, dtype=torch.bfloat16, device=DEV).normal_()
    pos = _grid(300000, 3)
    y = T.axial_rope(x, pos, (32, 48, 48))
    for at in (0, 131071, 262140, 299990):
        assert torch.equal(y[:, at:at + 10], T.axial_rope(x[:, at:at + 10], pos[at:at + 10], (32, 48, 48)))


def test_refusals_of_scales_and_caps():
    q = _cpu(1, 4, 2, 64)
    for c in (1e-9, 1e31, float("inf")):
        with pytest.raises(ValueError, match="softcap"):
            T.attention(q, q, q, softcap=c)
    for s in (1e31, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            T.attention(q, q, q, scale=s)


def test_backward_workspace_sizes_and_their_check():
    """The cached sizes are the C entry's, and a call without the scratch is refused before anything runs."""
    L, some = T.lib(), 0
    for B, Sq, Sk, Hq, Hk, D in ((1, 3, 9000, 8, 2, 64), (1, 8192, 64, 2, 1, 128), (8, 2048, 2048, 8, 8, 64), (1, 8192, 8192, 16, 4, 128)):
        for docs in (False, True):
            q, k = torch.zeros(B, Sq, Hq, D, dtype=torch.bfloat16), torch.zeros(B, Sk, Hk, D, dtype=torch.bfloat16)
            m = torch.zeros(B * max(Sq, Sk), dtype=torch.int32)
            room = torch.zeros(64, dtype=torch.float32)
            blk = T._attn_block(q, k, k, (1.0, 0.0, 0), (None, None, m, m) if docs else (None,) * 4, q, Sk, lse=room.data_ptr(), ranges=m.data_ptr())
            n = T._bwd_workspace_bytes(q.shape, Hk, Sk, docs, 1)
            assert n == L.turtle_token_attn_bwd_workspace(blk, 1)
            some += n > 0
            if n:
                blk += T._GRADS.pack(q.data_ptr(), *T._strides(q), q.data_ptr(), k.data_ptr(), k.data_ptr(), room.data_ptr())
                assert L.turtle_token_attn_bwd(blk, 1, None) == -1
    assert some > 3


def test_workspace_sizes_from_python_are_the_library_s():
    """The cached sizes: what the C entry says for the same call, dense and paged."""
    L = T.lib()
    for B, Sq, Sk, Hq, Hk, D in ((1, 1, 9000, 8, 2, 64), (2, 700, 2100, 4, 4, 128), (16, 64, 64, 2, 1, 40)):
        q = torch.zeros(B, Sq, Hq, D, dtype=torch.bfloat16)
        k = torch.zeros(B, Sk, Hk, D, dtype=torch.bfloat16)
        blk = T._attn_block(q, k, k, (1.0, 0.0, 0), (None,) * 4, q, Sk)
        assert T._workspace_bytes(q.shape, Hk, Sk, (0, 0, 0), 1) == L.turtle_token_attn_workspace(blk, 1)
        table = torch.zeros(B, 40, dtype=torch.int32)
        blk = T._attn_block(q, k, k, (1.0, 0.0, 1), (None,) * 4, q, 0, (256, 9, 40), (table, table, None))
        assert T._workspace_bytes(q.shape, Hk, 0, (256, 9, 40), 1) == L.turtle_token_attn_workspace(blk, 1)
    assert T._workspace_bytes(torch.Size((1, 1, 8, 64)), 2, 9000, (0, 0, 0), 1) > 0
    assert T._norm_workspace(5000, 64) == L.turtle_token_norm_rope_workspace(5000, 64)


# -------------------------------------------------------------------------------------------------
# forward mode
# -------------------------------------------------------------------------------------------------

def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A tensor that carries a tangent (with or without requires_grad) is refused by every operator, wherever it
    enters: a result without a tangent would be a wrong derivative. Tensors without one pass at the same level."""
    import torch.autograd.forward_ad as fw
    monkeypatch.setattr(T, "_device", lambda t: None)
    monkeypatch.setattr(T, "_run", lambda *a: None)             # no launch: what the calls would enqueue is not of interest
    x, w = torch.zeros(2, 5, 4, 64), torch.ones(64)
    pos, ax = torch.zeros(5, 3, dtype=torch.int32), (16, 24, 24)
    tab, kl = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    calls = {
        "rope x": (T.axial_rope, (x, pos, ax), {}, [0]),
        "norm q, k, gains": (T.qk_norm_rope, (x, x.clone(), pos, w, w.clone(), ax), {}, [0, 1, 3, 4]),
        "attention q, k, v": (T.attention, (x, x.clone(), x.clone()), {}, [0, 1, 2]),
        "attention slopes": (T.attention, (x, x, x), {"slopes": torch.ones(4)}, ["slopes"]),
        "attention without keys": (T.attention, (x, x[:, :0], x[:, :0]), {}, [0]),
        "paged q, pools": (T.paged_attention, (x, torch.zeros(6, 16, 2, 64), torch.zeros(6, 16, 2, 64), tab, kl), {}, [0, 1, 2]),
        "paged slopes": (T.paged_attention, (x, torch.zeros(6, 16, 2, 64), torch.zeros(6, 16, 2, 64), tab, kl), {"slopes": torch.ones(4)}, ["slopes"]),
    }
    for name, (f, args, kw, at) in calls.items():
        with torch.no_grad():
            f(*args, **kw)
        for i in at:
            for rg in (False, True):
                if rg and (i == "slopes" or f is T.paged_attention):
                    continue                                     # refused for its gradient already
                a, k = list(args), dict(kw)
                with fw.dual_level():
                    plain = (a if i != "slopes" else k)[i]
                    dual = fw.make_dual(plain.clone().requires_grad_(rg), torch.ones_like(plain))
                    if i == "slopes":
                        k[i] = dual
                    else:
                        a[i] = dual
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        f(*a, **k)
                    f(*args, **kw)


# -------------------------------------------------------------------------------------------------
# sizes of gradients
# -------------------------------------------------------------------------------------------------

def _fp16_grads(q, k, v, do, scale):
    """dq and dk of one head in fp64 and bounds on the sums of squared errors by element. dS = p (dP - delta) is rounded
    once, p carries the scores' error E, so a dS is off by at most s = sqrt(u^2 + E^2) of itself, independently of the
    others; delta by the same roundings of p: s^2 sum (p (|dP| + |delta|))^2, and dP by fp32 arithmetic. Errors of
    independent roundings add in squares, and a rounding's variance is a third of its bound's square; results are rounded
    once more, by u or half of fp16's smallest step."""
    u = unit(torch.float16)
    Q, K, V, g = (t.double() for t in (q, k, v, do))
    D = Q.shape[-1]
    raw = Q @ K.transpose(-1, -2) * scale
    p = torch.softmax(raw, -1)
    e32 = (D / 2 + 8) * 2.0 ** -23
    E = e32 * float((Q.abs() @ K.abs().transpose(-1, -2)).max()) * abs(scale) + 2.0 ** -20
    dp = g @ V.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    s2 = u * u + E * E
    edl2 = s2 * (p * (dp.abs() + delta.abs())).square().sum(-1, keepdim=True) + ((e32 + 2 * u * u) * (g.abs() * (p @ V.abs())).sum(-1, keepdim=True)).square()
    eds2 = s2 * ds.square() + (p * e32 * (g.abs() @ V.abs().transpose(-1, -2))).square()
    last = lambda r: (u * r).square() + 2.0 ** -50
    dq, dk = ds @ K * scale, ds.transpose(-1, -2) @ Q * scale
    dq2 = (eds2 @ K.square() + edl2 * (p @ K).square()) * scale ** 2 + last(dq)
    dk2 = (eds2 + edl2 * p.square()).transpose(-1, -2) @ Q.square() * scale ** 2 + last(dk)
    return (dq, dq2), (dk, dk2)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("n,Sq,Sk", [(1, 96, 4096), (1, 4096, 96), (2, 700, 3000), (24, 1200, 1100), (32, 900, 1000)])
@pytest.mark.parametrize("kind", ["1e-3", "1e-4", "rows", "keys"])
def test_attention_fp16_gradients_of_any_size(D, n, Sq, Sk, kind):
    """Gradients far from one: small ones over many keys, rows of 2^-12 to 2^9 in one call, growing along the walks, and
    values that grow along the keys. The norm of the error of all values, of the small rows and of the first keys is at
    most twice the bounds' (which are themselves 1.7 times what independent roundings give)."""
    q, k = randn(n, Sq, 1, D, seed=1).mul(2.0 ** -8).half(), randn(n, Sk, 1, D, seed=2).mul(2.0 ** -8).half()
    v, do = randn(n, Sk, 1, D, seed=3), randn(n, Sq, 1, D, seed=4)
    ramp = lambda s, lo, hi: torch.linspace(lo, hi, s, device=DEV).exp2().view(1, s, 1, 1)
    if kind == "rows":
        do = do * ramp(Sq, -12, 9) * 1e-2
    elif kind == "keys":
        v, do = v * ramp(Sk, -6, 6), do * 1e-3
    else:
        do = do * float(kind)
    v, do, scale = v.half(), do.half(), 2.0 ** 16 * D ** -0.5
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dq, dk, _ = torch.autograd.grad(T.attention(*leaves, scale=scale), leaves, do)
    ref = _fp16_grads(*(t.detach()[:, :, 0] for t in (q, k, v, do)), scale)
    for name, got, (want, e2), part in (("dq", dq, ref[0], Sq // 4), ("dk", dk, ref[1], Sk // 4)):
        err = got[:, :, 0].double() - want
        assert torch.isfinite(err).all(), name
        for what, x in (("all", slice(None)), ("first quarter", slice(0, part))):
            a, b = float(err[:, x].norm()), 2 * float(e2[:, x].sum().sqrt())
            assert a <= b, (name, what, a, b, float(want[:, x].norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 300])
def test_attention_fp16_gradients_past_the_type_s_range_inside(D, n):
    """dO of 2e4 on three keys: dS passes 65504, the gradients do not."""
    q, k, v = (randn(n, s, 1, D, dtype=torch.float16, seed=i) for i, s in enumerate((4, 3, 3)))
    do = (randn(n, 4, 1, D, seed=4) * 2e4).clamp(-5e4, 5e4).half()
    scale = 2.0 ** -8
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(T.attention(*leaves, scale=scale), leaves, do)
    ref = _fp16_grads(*(t.detach()[:, :, 0] for t in (q, k, v, do)), scale)
    p = torch.softmax(q.detach()[:, :, 0].double() @ k.detach()[:, :, 0].double().transpose(1, 2) * scale, -1)
    ds = p * (do[:, :, 0].double() @ v.detach()[:, :, 0].double().transpose(1, 2))
    assert float(ds.abs().max()) > 65504
    for name, got, (want, e2) in (("dq", grads[0], ref[0]), ("dk", grads[1], ref[1])):
        assert float(want.abs().max()) < 60000
        err = got[:, :, 0].double() - want
        assert torch.isfinite(err).all(), name
        assert float(err.norm()) <= 2 * float(e2.sum().sqrt()), name


# -------------------------------------------------------------------------------------------------
# the library and its header
# -------------------------------------------------------------------------------------------------

def test_a_changed_header_makes_the_built_library_stale(tmp_path, monkeypatch):
    """The argument blocks' layout stands in include/: a library built from another header is another library."""
    import shutil
    from turtlevsr_amd import build as B
    (tmp_path / "turtlevsr_amd").mkdir()
    for d, src in (("turtlevsr_amd/csrc", B.CSRC), ("include", os.path.join(REPO, "include"))):
        shutil.copytree(src, tmp_path / d)
    shutil.copy(os.path.join(REPO, "turtlevsr_amd", "build.py"), tmp_path / "turtlevsr_amd")
    monkeypatch.setattr(B, "REPO", str(tmp_path))
    monkeypatch.setattr(B, "CSRC", str(tmp_path / "turtlevsr_amd" / "csrc"))
    seen = {B.source_hash()}
    for h in sorted(os.listdir(tmp_path / "include")):
        with open(tmp_path / "include" / h, "a") as f:
            f.write("/* */\n")
        seen.add(B.source_hash())
    assert len(seen) == 1 + len(os.listdir(tmp_path / "include"))


def test_packed_blocks_have_the_header_s_layout(tmp_path):
    """Every field of include/turtle_token.h's structs against the formats the calls are packed with, by the C compiler."""
    import shutil
    import struct
    import subprocess
    cc = shutil.which("gcc") or shutil.which("cc") or shutil.which("clang")
    assert cc, "no C compiler"
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", "turtle_token.h")).read(), flags=re.S)
    body = {}
    for m in re.finditer(r"typedef struct \{([^{}]*)\} (turtle_token_\w+);", hdr):
        names = []
        for decl in filter(None, (d.strip() for d in m.group(1).split(";"))):
            names += [re.search(r"(\w+)(?:\[\d+\])?\s*$", part).group(1) for part in decl.split(",")]
        body[m.group(2)] = names
    assert set(body) == {"turtle_token_axes", "turtle_token_side", "turtle_token_attn_args", "turtle_token_attn_grads"}
    src = '#include <stdio.h>\n#include "turtle_token.h"\nint main(void) {\n'
    for s, names in body.items():
        src += f'printf("{s} %zu", sizeof({s}));\n' + "".join(f'printf(" %zu", offsetof({s}, {n}));\n' for n in names) + 'puts("");\n'
    (tmp_path / "a.c").write_text(src + "return 0; }\n")
    subprocess.run([cc, "-I", os.path.join(REPO, "include"), str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    c = {x.split()[0]: [int(n) for n in x.split()[1:]] for x in subprocess.run([str(tmp_path / "a")], check=True, capture_output=True, text=True).stdout.splitlines()}

    def offsets(fmt):
        at, out = 0, []
        for n, t in re.findall(r"(\d*)([A-Za-z])", fmt):
            size = struct.calcsize("@" + t)
            at = -(-at // size) * size
            out += [at + size * i for i in range(int(n or 1))]
            at += size * int(n or 1)
        return out
    side, attn = offsets(T._SIDE.format), offsets(T._ATTN.format)
    assert c["turtle_token_side"] == [T._SIDE.size] + side
    assert c["turtle_token_axes"][0] == T._AXES.size
    q, b, i = re.findall(r"\d*[A-Za-z]", T._AXES.format)
    assert (q, b, i) == ("64Q", "64B", "2i") and c["turtle_token_axes"][1:] == [0, 512, 576, 580]
    assert c["turtle_token_attn_args"] == [T._ATTN.size] + attn
    assert c["turtle_token_attn_grads"] == [T._ATTN.size + T._GRADS.size, 0] + [T._ATTN.size + o for o in offsets(T._GRADS.format)]


# -------------------------------------------------------------------------------------------------
# far positions
# -------------------------------------------------------------------------------------------------

def _turns(pos, j, d, base):
    """pos base^(-j / d) / 2 pi mod 1 (nearest to zero), in 60 digits; pi from Machin's formula."""
    from decimal import Decimal, getcontext, localcontext
    with localcontext() as c:
        c.prec = 60

        def arctan_inverse(n):
            x, s, k = Decimal(1) / n, Decimal(0), 0
            while abs(x) > Decimal(10) ** -58:
                s += x / (2 * k + 1) * (-1) ** k
                x, k = x / (n * n), k + 1
            return s
        pi = 16 * arctan_inverse(5) - 4 * arctan_inverse(239)
        r = Decimal(pos) * (-Decimal(j) / d * Decimal(base).ln()).exp() / (2 * pi)
        return float(r - r.to_integral_value())


FAR = [0, 1, -1, 10 ** 6, 2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7, 10 ** 12, -10 ** 12 - 1, 2 ** 45 + 3, 2 ** 50, -2 ** 50 + 1]


@pytest.mark.parametrize("base,d", [(10000.0, 24), (10000.0, 64), (100.5, 16), (1.0, 8), (1e30, 128)])
def test_frequencies_hold_for_far_positions(base, d):
    """Revolutions of every pair from the table, pos * freq mod 2^64: off by at most |pos| / 2 of the 2^-64 that freq is
    rounded to, besides the comparison's own 2^-50."""
    tab = T._AXES.unpack(T._axes((d,), base, 128)[0])
    for i in range(d // 2):
        for pos in FAR:
            got = (pos * tab[i] % 2 ** 64) / 2 ** 64
            off = abs(got - _turns(pos, 2 * i, d, base)) % 1.0
            assert min(off, 1 - off) <= abs(pos) * 2.0 ** -65 + 2.0 ** -50, (i, pos)


@pytest.mark.gpu
def test_axial_rope_turns_far_64_bit_positions_rightly():
    """fp32: the functions' error of the other fp32 test (2^-22 of the pair), the angle's 2^-32 revolutions and the table's
    |pos| 2^-65."""
    d = 24
    pos = torch.tensor(FAR, dtype=torch.int64, device=DEV)[:, None]
    x = randn(1, len(FAR), 2, d, seed=1)
    turns = torch.tensor([[_turns(p, 2 * i, d, 10000.0) for i in range(d // 2)] for p in FAR], dtype=torch.float64, device=DEV)
    th = (turns * 2 * math.pi)[:, None]
    x0, x1 = x.double()[..., ::2], x.double()[..., 1::2]
    ref = torch.stack((x0 * th.cos() - x1 * th.sin(), x0 * th.sin() + x1 * th.cos()), -1).flatten(-2)
    pair = (x0.abs() + x1.abs()).repeat_interleave(2, -1)
    far = pos.double().abs()[:, None] * 2.0 ** -65 * 2 * math.pi
    within(T.axial_rope(x, pos, (d,)), ref, (2.0 ** -22 + 2.0 ** -29 + far) * pair, "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_qk_norm_of_rows_past_the_range_of_squares(dt):
    """A head whose squares pass fp32's range has a norm of infinity: zeros, zero gradients and nothing in the gain's, as from
    x * rsqrt(mean(x^2) + eps) in fp32; the other heads are as without it. Values whose squares just fit are normed."""
    q, k = randn(2, 9, 3, 64, dtype=dt, seed=1), randn(2, 9, 1, 64, dtype=dt, seed=2)
    pos, w = _grid(9, 3), torch.linspace(0.5, 2, 64, device=DEV)
    g = randn(2, 9, 3, 64, dtype=dt, seed=3), randn(2, 9, 1, 64, dtype=dt, seed=4)

    def call(q, k):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, w, w)]
        y = T.qk_norm_rope(leaves[0], leaves[1], pos, leaves[2], leaves[3], (16, 24, 24))
        return [t.detach() for t in y] + list(torch.autograd.grad(y, leaves, g))
    small = q.clone()
    small[0, 4, 1] = 0
    want = call(small, k)
    for big in (1e20, 3e38):
        huge = q.clone()
        huge[0, 4, 1] = big
        got = call(huge, k)
        assert not got[0][0, 4, 1].any() and not got[2][0, 4, 1].any()
        for a, b in zip(got, want):
            assert torch.isfinite(a).all()
        got[2][0, 4, 1] = want[2][0, 4, 1] = 0
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    edge = q.clone()
    edge[0, 4, 1] = 2e18                                       # 64 squares of 4e36 add up to 2.6e38
    y = call(edge, k)[0][0, 4, 1].double()
    ref = rope_ref(w.double().expand(1, 1, 1, 64).clone(), pos[4:5], (16, 24, 24))[0, 0, 0]
    within(y, ref, (unit(dt) + 2.0 ** -18) * 4 + 0 * ref, "edge")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Sq,Sk,n", [(20, 300, 1), (100, 200, 3), (200, 300, 70)])
def test_attention_cap_keeps_small_scores_beside_large_ones(dt, Sq, Sk, n):
    """A cap of 10^6 that one query reaches: the scores of the other rows, which it leaves as they are (tanh x = x to
    (s / 10^6)^2 / 3), keep fp32's relative accuracy. tanh's part of their error is 2^-20 of the largest, a fifth of the
    bound on the fp32 sums. The one query has no gradient, so those of the keys are of the other rows too. fp16 results under
    2^-14 are rounded to multiples of 2^-24, by 2^-25 at most however small they are: added to the relative bounds."""
    q, k, v = (randn(n, s, 2, 64, dtype=dt, seed=i) for i, s in enumerate((Sq, Sk, Sk)))
    do = randn(n, Sq, 2, 64, dtype=dt, seed=5)
    q[:, 3], do[:, 3] = 6e4 * q[:, 3].sign(), 0
    assert float((q[:, 3].double()[:, None] * k.double()).sum(-1).abs().max()) > 5e5
    rest = [i for i in range(Sq) if i != 3]
    ref = attn_ref(q[:, rest], k, v, torch.ones(n, Sq - 1, Sk, dtype=torch.bool, device=DEV), scale=1.0, do=do[:, rest])
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = T.attention(*leaves, scale=1.0, softcap=1e6)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    for name, got in (("o", o[:, rest]), ("dq", dq[:, rest]), ("dk", dk), ("dv", dv)):
        within(got, ref[name][0], 1.2 * ref[name][1] + (2.0 ** -25 if dt == torch.float16 else 0.0), name)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("cap", [0.5, 64.0, 64.5])
def test_attention_caps_that_scores_reach(dt, cap):
    """Scores of up to a few caps, under the cap where a 16-bit tanh changes its form and over it."""
    q, k, v = (randn(2, s, 2, 64, dtype=dt, seed=i) for i, s in enumerate((70, 150, 150)))
    check_attention(q, k, v, randn(2, 70, 2, 64, dtype=dt, seed=5), scale=cap / 8, softcap=cap)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,Sq,Sk,D", [(1, 3, 9000, 64), (2, 70, 100, 64), (2, 70, 100, 128), (70, 200, 300, 64), (40, 300, 300, 104)])
@pytest.mark.parametrize("what", ["key", "query"])
def test_gradients_that_depend_on_a_number_that_is_none_are_none(dt, B, Sq, Sk, D, what):
    """A key that is not a number makes the softmax of every query of its sequence so: no gradient of them comes out finite.
    A query: no gradient of its sequence's keys; its neighbours' stay as they are."""
    q, k, v = (randn(B, s, 2, D, dtype=dt, seed=i) for i, s in enumerate((Sq, Sk, Sk)))
    do = randn(B, Sq, 2, D, dtype=dt, seed=5)
    def grads():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(T.attention(*leaves), leaves, do)
    want = grads()
    (k if what == "key" else q)[0, 1, 1, 3] = float("nan")
    got = grads()
    for n, a, b in zip(("dq", "dk", "dv"), got, want):
        if n == "dq" and what == "query":
            assert not a[0, 1, 1].isfinite().any()
            a, b = a.clone(), b.clone()
            a[0, 1, 1] = b[0, 1, 1] = 0
            assert torch.equal(a, b)
        else:
            assert not a[0, :, 1].isfinite().any(), n
            assert torch.equal(a[:, :, 0], b[:, :, 0]) and torch.equal(a[1:], b[1:]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,Sq,Sk,Hq,Hk,D", [(2, 150, 333, 4, 2, 64), (1, 60, 90, 2, 1, 128), (40, 300, 300, 6, 2, 64), (24, 261, 300, 6, 2, 104), (1, 3000, 40, 2, 1, 40)])
@pytest.mark.parametrize("causal", [False, True])
def test_queries_that_see_nothing_pass_no_gradient_whatever_they_hold(dt, B, Sq, Sk, Hq, Hk, D, causal):
    """Queries of documents that no key has, or (causal, documents out of order) has later only: their rows and the gradients
    that arrive there hold not-a-numbers and infinities, and nothing of them comes out."""
    q, k, v = (randn(B, s, h, D, dtype=dt, seed=i) for i, (s, h) in enumerate(((Sq, Hq), (Sk, Hk), (Sk, Hk))))
    do = randn(B, Sq, Hq, D, dtype=dt, seed=9)
    g = torch.Generator().manual_seed(Sq)
    qd = (torch.arange(Sq)[None] * -(-Sk // 40) // Sq).repeat(B, 1)
    qd[torch.rand(B, Sq, generator=g) < 0.1] = 1000            # single ones, a whole tile, a last piece
    qd[:, 64:130], qd[:, -5:] = 1001, 1002
    kd = (torch.arange(Sk)[None] // 40).repeat(B, 1)
    if causal:
        kd = kd.flip(1)
    qd, kd = qd.to(DEV), kd.to(DEV)
    blind = ~visible_ref(B, Sq, Sk, causal, None, qd, kd).any(2)
    assert blind.any() and not blind.all()
    q[blind], do[blind] = float("nan"), float("inf")
    check_attention(q, k, v, do, q_doc=qd, k_doc=kd, causal=causal)


def test_the_caller_s_decimal_context_does_not_matter():
    import decimal
    T._axes_table.cache_clear()
    want = T._axes_table((16, 24), 10000.0)
    T._axes_table.cache_clear()
    with decimal.localcontext() as c:
        c.prec, c.rounding = 3, decimal.ROUND_UP
        c.traps[decimal.Inexact] = c.traps[decimal.FloatOperation] = True
        assert T._axes_table((16, 24), 10000.0) == want


# -------------------------------------------------------------------------------------------------
# combinations
# -------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,Sq,Sk,Hq,Hk,D", [(2, 90, 130, 4, 2, 64), (1, 300, 200, 3, 1, 128), (45, 300, 290, 6, 2, 40), (1, 5, 2500, 8, 2, 96), (1, 2500, 70, 2, 2, 64)])
def test_attention_all_rules_at_once(dt, B, Sq, Sk, Hq, Hk, D):
    """Documents in any order, causal, a prefix for each sequence, a bias and a cap, a scale below zero."""
    q, k, v = (randn(B, s, h, D, dtype=dt, seed=i) for i, (s, h) in enumerate(((Sq, Hq), (Sk, Hk), (Sk, Hk))))
    g = torch.Generator().manual_seed(Sq)
    n = max(Sq, Sk)
    doc = torch.randint(0, 4, (B, n // 20 + 1), generator=g).repeat_interleave(20, 1)[:, :n]
    doc[torch.rand(B, n, generator=g) < 0.05] = -3
    check_attention(q, k, v, randn(B, Sq, Hq, D, dtype=dt, seed=9), causal=True, prefix=torch.tensor([(7 * b) % Sk for b in range(B)], device=DEV),
                    q_doc=doc[:, :Sq].to(DEV), k_doc=doc[:, -Sk:].to(DEV), slopes=torch.linspace(-0.02, 0.2, Hq, device=DEV), softcap=4.0, scale=-0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G,Sq,D", [(40, 1, 64), (96, 1, 128), (33, 7, 40), (64, 3, 64)])
def test_paged_many_heads_share_a_key(dt, G, Sq, D):
    lens = [700, 33, Sq]
    kp, vp, table, k, v = _pages(3, lens, 24, 1, D, dt, seed=G)
    check_paged(randn(3, Sq, G, D, dtype=dt, seed=6), kp, vp, table, lens, k, v, slopes=torch.linspace(0, 0.3, G, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 70])
@pytest.mark.parametrize("causal", [True, False])
def test_paged_lengths_at_the_ends_of_their_range(Sq, causal):
    """More keys than 32 bits count past the table's room, fewer than none, more queries than the chunk has or than keys,
    fewer than none: keys are cut to [0, room], queries to [0, Sq], a query's place is kv_lens - queries + i."""
    most, least = 2 ** 31 - 1, -2 ** 31
    lens, ql = [most, least, 64, 5, 64, -1, most], [Sq, Sq, most, Sq, least, most, least]
    page = 16
    kp, vp, table, k, v = _pages(7, [64] * 7, page, 2, 64, torch.bfloat16, seed=1)
    q = randn(7, Sq, 4, 64, dtype=torch.bfloat16, seed=2)
    check_paged(q, kp, vp, table, lens, k, v, ql, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_qk_norm_rope_with_more_key_heads(dt):
    """Heads of k past q's: as k's own call gives them; gradients too."""
    q, k = randn(2, 31, 1, 40, dtype=dt, seed=1), randn(2, 31, 5, 40, dtype=dt, seed=2)
    pos, w = _grid(31, 2), torch.linspace(0.5, 2, 40, device=DEV)
    g = randn(2, 31, 5, 40, dtype=dt, seed=3)
    a, b = k.detach().requires_grad_(True), k.detach().requires_grad_(True)
    wa, wb = w.clone().requires_grad_(True), w.clone().requires_grad_(True)
    x, y = T.qk_norm_rope(q, a, pos, None, wa, (16, 8))[1], T.qk_norm_rope(b, k, pos, wb, None, (16, 8))[0]
    assert torch.equal(x, y)
    da, dwa = torch.autograd.grad(x, (a, wa), g)
    db, dwb = torch.autograd.grad(y, (b, wb), g)
    assert torch.equal(da, db) and torch.equal(dwa, dwb)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_training_step_with_documents_in_a_graph(D):
    """Forward and backward captured, replayed with other documents: queries that see nothing in one replay (and hold
    not-a-numbers there) are ordinary ones in the next."""
    leaves = [randn(2, 333, h, D, dtype=torch.float16, seed=i).requires_grad_(True) for i, h in enumerate((4, 2, 2))]
    do = randn(2, 333, 4, D, dtype=torch.float16, seed=5)
    qd, kd = torch.zeros(2, 333, dtype=torch.int32, device=DEV), torch.zeros(2, 333, dtype=torch.int32, device=DEV)

    def step():
        o = T.attention(*leaves, q_doc=qd, k_doc=kd, causal=True)
        return (o.detach(),) + torch.autograd.grad(o, leaves, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for n in range(5):
        with torch.no_grad():
            for i, t in enumerate(leaves):
                t.copy_(randn(*t.shape, dtype=t.dtype, seed=100 + 10 * n + i))
            do.copy_(randn(*do.shape, dtype=do.dtype, seed=100 + 10 * n + 7))
            kd.copy_((torch.arange(333, device=DEV) // (20 + 30 * n))[None].expand(2, -1))
            qd.copy_(kd)
            qd[:, 40 * n:40 * n + 70] = 500
            if n % 2:
                leaves[0][:, 40 * n:40 * n + 70], do[:, 40 * n:40 * n + 70] = float("nan"), float("inf")
        g.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.isfinite(t).all() for t in got)
        assert not got[0][:, 40 * n:40 * n + 70].any() and not got[1][:, 40 * n:40 * n + 70].any()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    check_attention(*(t.detach() for t in leaves), do, q_doc=qd, k_doc=kd, causal=True)
