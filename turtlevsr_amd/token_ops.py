"""Token attention on the HIP kernels (include/turtle_token.h): rotary positions over several axes, the per-head
norm of queries and keys with that rotation in the same pass, masked attention with its gradients, and attention
of a chunk of new tokens over a paged history cache.

Tokens are ``[B, S, heads, D]`` tensors with the channels contiguous (D a multiple of 8, at most 128); any other
strides do, so q, k and v can be slices of one channels-last 1x1 projection: ``qkv`` of shape [B, 3 C, H, W] in
``torch.channels_last`` is ``qkv.permute(0, 2, 3, 1).reshape(B, H * W, 3, heads, D).unbind(2)`` without a copy.
A tensor whose rows do not start at multiples of 16 bytes is copied first. Activations are fp32, bf16 or fp16;
results have the inputs' type and are dense. Everything runs on the caller's current stream of the tensors'
device and can be captured into a graph. There is no CPU path: a CPU tensor or a missing library raises.

* ``axial_rope(x, pos, axes)``: channel pairs turned by the token's place on several axes (time, height, width);
* ``qk_norm_rope(q, k, pos, q_weight, k_weight, axes)``: RMS norm of every head, gain, rotation, in one pass;
* ``attention(q, k, v, ...)``: softmax(q k^T) v with shared key heads, a tanh cap, a distance bias, causal, prefix
  and document masks;
* ``paged_attention(q, k_pages, v_pages, block_table, kv_lens, ...)``: the serving form, no gradient.

The first three are differentiable (first order); sums run in a fixed order, so results repeat bit for bit.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .train_ops import _check, _dt, _p, _stream

MAX_D = 128


class _Axes(C.Structure):
    _fields_ = [("freq", C.c_uint64 * 64), ("axis", C.c_uint8 * 64), ("npair", C.c_int32), ("naxis", C.c_int32)]


class _Side(C.Structure):
    _fields_ = [("x", C.c_void_p), ("dy", C.c_void_p), ("y", C.c_void_p), ("w", C.c_void_p)] + \
               [(n, C.c_int64) for n in ("sb", "ss", "sh", "gb", "gs", "gh")] + [("H", C.c_int32), ("pad", C.c_int32)]


class _Attn(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v")] + \
               [(n, C.c_int64) for n in ("qb", "qs", "qh", "kb", "ks", "kh", "vb", "vs", "vh")] + \
               [(n, C.c_int32) for n in ("B", "Sq", "Sk", "Hq", "Hk", "D")] + [("scale", C.c_float), ("softcap", C.c_float)] + \
               [(n, C.c_void_p) for n in ("slopes", "prefix", "qdoc", "kdoc")] + \
               [(n, C.c_int32) for n in ("causal", "page", "npages", "maxpages")] + \
               [(n, C.c_void_p) for n in ("table", "kv_lens", "q_lens", "o", "o_lo", "lse", "ranges", "ws")] + [("ws_bytes", C.c_size_t)]


class _Grads(C.Structure):
    _fields_ = [("f", _Attn), ("dout", C.c_void_p)] + [(n, C.c_int64) for n in ("gb", "gs", "gh")] + \
               [(n, C.c_void_p) for n in ("dq", "dk", "dv", "delta")]


_bound = None


def lib():
    global _bound
    if _bound is not None:
        return _bound
    L = _lib.lib()
    vp, i64, ci, sz, P = C.c_void_p, C.c_int64, C.c_int, C.c_size_t, C.POINTER
    rope = [P(_Side), P(_Side), P(_Axes), vp, i64, ci, i64, i64, ci]
    L.turtle_token_rope.argtypes = rope + [ci, ci, vp]
    L.turtle_token_norm_rope_fwd.argtypes = rope + [C.c_float, ci, vp]
    L.turtle_token_norm_rope_workspace.argtypes = [i64, ci]
    L.turtle_token_norm_rope_workspace.restype = sz
    L.turtle_token_norm_rope_bwd.argtypes = rope + [C.c_float, vp, vp, sz, ci, vp]
    L.turtle_token_attn_ranges.argtypes = [P(_Attn)]
    L.turtle_token_attn_ranges.restype = sz
    L.turtle_token_attn_workspace.argtypes = [P(_Attn), ci]
    L.turtle_token_attn_workspace.restype = sz
    L.turtle_token_attn_fwd.argtypes = [P(_Attn), ci, vp]
    L.turtle_token_attn_bwd.argtypes = [P(_Grads), ci, vp]
    _bound = L
    return L


# -------------------------------------------------------------------------------------------------
# arguments
# -------------------------------------------------------------------------------------------------

def _tokens(t, name: str) -> torch.Tensor:
    """``t`` itself when the kernels can read it: channels contiguous, rows at multiples of 16 bytes; else a copy."""
    es = t.element_size()
    ok = t.data_ptr() % 16 == 0 and (t.shape[3] == 1 or t.stride(3) == 1)
    for i in range(3):
        ok = ok and (t.shape[i] == 1 or (t.stride(i) * es) % 16 == 0)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    """(batch, token, head) strides in elements; 0 along a dimension of one (it may have any stride)."""
    return tuple(t.stride(i) if t.shape[i] > 1 else 0 for i in range(3))


def _check_tokens(t, name: str, D=None):
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise ValueError(f"{name}: expected a [B, S, heads, D] tensor")
    _dt(t)
    d = t.shape[3]
    if d % 8 or not 8 <= d <= MAX_D:
        raise ValueError(f"{name}: D = {d}, must be a multiple of 8, at most {MAX_D}")
    if t.shape[2] < 1:
        raise ValueError(f"{name}: no heads")


def _device(t):
    if t.device.type != "cuda":
        raise RuntimeError("turtle token kernels run on a ROCm device only")


def _same(a, b, name: str):
    if b.device != a.device:
        raise ValueError(f"{name}: on {b.device}, expected {a.device}")


def _ints(t, shape, name: str, like):
    """An int32 tensor of ``shape`` on ``like``'s device from an integer tensor."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: expected an int32 or int64 tensor")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    _same(like, t, name)
    return t.to(torch.int32).contiguous()


def _slopes(t, H: int, like):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or not t.is_floating_point():
        raise TypeError("slopes: expected a floating-point tensor")
    if tuple(t.shape) != (H,):
        raise ValueError(f"slopes: shape {tuple(t.shape)}, expected {(H,)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("slopes: the distance bias has no gradient (pass slopes.detach())")
    _same(like, t, "slopes")
    return t.float().contiguous()


def _cap(softcap) -> float:
    c = float(softcap)
    if not 0.0 <= c < float("inf"):
        raise ValueError(f"softcap = {softcap}, must be finite and not negative (0: none)")
    return c


def _scale(scale, D: int) -> float:
    s = D ** -0.5 if scale is None else float(scale)
    if not abs(s) < float("inf"):
        raise ValueError(f"scale = {scale}, must be finite")
    return s


class _on:
    """The tensors' device as the current one (a no-op where it already is)."""

    def __init__(self, t):
        self.to = None if torch.cuda.current_device() == t.device.index else torch.cuda.device(t.device)

    def __enter__(self):
        if self.to is not None:
            self.to.__enter__()

    def __exit__(self, *e):
        if self.to is not None:
            self.to.__exit__(*e)
        return False


# -------------------------------------------------------------------------------------------------
# rotation
# -------------------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=64)
def _axes_table(axes, base: float):
    """Every rotated pair's axis and its revolutions per unit of position in 64-bit fixed point: with it
    pos * freq mod 2^64 is the exact angle, however far the position."""
    t = _Axes()
    i = 0
    for a, d in enumerate(axes):
        for j in range(0, d, 2):
            f = base ** (-j / d) / 6.283185307179586476925
            t.freq[i], t.axis[i] = int(f * 2.0 ** 64), a
            i += 1
    t.npair, t.naxis = i, len(axes)
    return t


def _axes(axes, base, D: int):
    ax = tuple(int(d) for d in axes)
    if not 1 <= len(ax) <= 4 or any(d < 0 or d % 2 for d in ax) or sum(ax) > D:
        raise ValueError(f"axes = {tuple(axes)}: one to four even channel counts, together at most D = {D}")
    base = float(base)
    if not 1.0 <= base < float("inf"):
        raise ValueError(f"base = {base}, must be at least 1")
    return _axes_table(ax, base)


def _pos(pos, B: int, S: int, naxis: int, like):
    """(pos, elements between batches, is int64)"""
    if not isinstance(pos, torch.Tensor) or pos.dtype not in (torch.int32, torch.int64):
        raise TypeError("pos: expected an int32 or int64 tensor")
    if tuple(pos.shape) not in ((S, naxis), (B, S, naxis)):
        raise ValueError(f"pos: shape {tuple(pos.shape)}, expected {(S, naxis)} or {(B, S, naxis)}")
    _same(like, pos, "pos")
    pos = pos.contiguous()
    return pos, (S * naxis if pos.dim() == 3 else 0), int(pos.dtype == torch.int64)


def _side(x, y, w=None, dy=None):
    s = _Side()
    if x is None:
        return s
    s.x, s.y, s.H = x.data_ptr(), y.data_ptr(), x.shape[2]
    s.sb, s.ss, s.sh = _strides(x)
    if w is not None:
        s.w = w.data_ptr()
    if dy is not None:
        s.dy = dy.data_ptr()
        s.gb, s.gs, s.gh = _strides(dy)
    return s


def _dense(x):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, pos_b, pos64, tab):
        ctx.save_for_backward(pos)
        ctx.rest = (pos_b, pos64, tab)
        return _Rope.turn(x, pos, pos_b, pos64, tab, 0)

    @staticmethod
    def turn(x, pos, pos_b, pos64, tab, inverse):
        x = _tokens(x, "x")
        y = _dense(x)
        B, S, _, D = x.shape
        if x.numel():
            with _on(x):
                _check(lib().turtle_token_rope(_side(x, y), None, tab, _p(pos), pos_b, pos64, B, S, D, inverse, _dt(x), _stream(x)),
                       "token_rope")
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (pos,) = ctx.saved_tensors
        return _Rope.turn(dy, pos, *ctx.rest, 1), None, None, None, None


def axial_rope(x, pos, axes, base: float = 10000.0):
    """Rotary positions over several axes: the first ``axes[0]`` channels of every head turn with the token's
    place on axis 0, the next ``axes[1]`` with its place on axis 1, and so on; channels past ``sum(axes)`` pass
    unchanged. Within an axis of d channels, pair i - channels (2 i, 2 i + 1) - turns by the angle
    ``pos[axis] * base ** (-2 i / d)``.

    x [B, S, heads, D]; pos int32 or int64 [S, len(axes)] or [B, S, len(axes)] (any sign, exact at any
    distance); axes one to four even numbers. Returns a dense tensor of x's type."""
    _check_tokens(x, "x")
    B, S, _, D = x.shape
    tab = _axes(axes, base, D)
    p, pos_b, pos64 = _pos(pos, B, S, tab.naxis, x)
    _device(x)
    return _Rope.apply(x, p, pos_b, pos64, tab)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, pos, pos_b, pos64, tab, eps):
        q, k = _tokens(q, "q"), _tokens(k, "k")
        yq, yk = _dense(q), _dense(k)
        B, S, _, D = q.shape
        w = [None if t is None else t.detach().float().contiguous() for t in (wq, wk)]
        if q.numel():
            with _on(q):
                _check(lib().turtle_token_norm_rope_fwd(_side(q, yq, w[0]), _side(k, yk, w[1]), tab, _p(pos), pos_b, pos64, B, S, D, eps,
                                                        _dt(q), _stream(q)), "token_norm_rope_fwd")
        ctx.save_for_backward(q, k, pos, *[t for t in w if t is not None])
        ctx.has_w = [t is not None for t in w]
        ctx.w_dt = [None if t is None else t.dtype for t in (wq, wk)]
        ctx.rest = (pos_b, pos64, tab, eps)
        return yq, yk

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, pos, *ws = ctx.saved_tensors
        w = [ws.pop(0) if has else None for has in ctx.has_w]
        pos_b, pos64, tab, eps = ctx.rest
        B, S, _, D = q.shape
        gq, gk = _tokens(gq, "dq"), _tokens(gk, "dk")
        dq, dk = _dense(q), _dense(k)
        want = any(ctx.has_w[i] and ctx.needs_input_grad[2 + i] for i in range(2))
        dw = torch.zeros(2, D, dtype=torch.float32, device=q.device) if want and not q.numel() else \
            (torch.empty(2, D, dtype=torch.float32, device=q.device) if want else None)
        if q.numel():
            L = lib()
            n = int(L.turtle_token_norm_rope_workspace(B * S, D)) if want else 0
            ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
            with _on(q):
                _check(L.turtle_token_norm_rope_bwd(_side(q, dq, w[0], gq), _side(k, dk, w[1], gk), tab, _p(pos), pos_b, pos64, B, S, D,
                                                    eps, _p(dw), _p(ws), n, _dt(q), _stream(q)), "token_norm_rope_bwd")
        g = [dw[i].to(ctx.w_dt[i]) if want and ctx.has_w[i] else None for i in range(2)]
        return dq, dk, g[0], g[1], None, None, None, None, None


def qk_norm_rope(q, k, pos, q_weight, k_weight, axes, base: float = 10000.0, eps: float = 1e-6):
    """(q', k'): every head's RMS norm over its D channels, x / sqrt(mean(x^2) + eps) times the gain (``q_weight``
    / ``k_weight`` [D], or None), then ``axial_rope``, in one pass over q and k.

    q [B, S, Hq, D], k [B, S, Hk, D] of one type at the same tokens; pos, axes and base as in ``axial_rope``.
    Gradients go to q, k and the gains."""
    _check_tokens(q, "q")
    _check_tokens(k, "k")
    B, S, _, D = q.shape
    if (k.shape[0], k.shape[1], k.shape[3]) != (B, S, D):
        raise ValueError(f"k: shape {tuple(k.shape)} does not match q {tuple(q.shape)}")
    if k.dtype != q.dtype:
        raise TypeError(f"q is {q.dtype}, k is {k.dtype}")
    _same(q, k, "k")
    for w, n in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is None:
            continue
        if not isinstance(w, torch.Tensor) or not w.is_floating_point():
            raise TypeError(f"{n}: expected a floating-point tensor")
        if tuple(w.shape) != (D,):
            raise ValueError(f"{n}: shape {tuple(w.shape)}, expected {(D,)}")
        _same(q, w, n)
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps = {eps}, must be finite and not negative")
    tab = _axes(axes, base, D)
    p, pos_b, pos64 = _pos(pos, B, S, tab.naxis, q)
    _device(q)
    return _QkNormRope.apply(q, k, q_weight, k_weight, p, pos_b, pos64, tab, eps)


# -------------------------------------------------------------------------------------------------
# attention
# -------------------------------------------------------------------------------------------------

def _set(a, **kw):
    for n, v in kw.items():
        setattr(a, n, v.data_ptr() if isinstance(v, torch.Tensor) else v)


def _attn_args(q, k, v, scale, softcap, causal, slopes, prefix, q_doc, k_doc):
    a = _Attn()
    (a.qb, a.qs, a.qh), (a.kb, a.ks, a.kh), (a.vb, a.vs, a.vh) = _strides(q), _strides(k), _strides(v)
    a.B, a.Sq, a.Hq, a.D = q.shape
    a.Sk, a.Hk = k.shape[1], k.shape[2]
    _set(a, q=q, k=k, v=v, scale=scale, softcap=softcap, causal=int(causal), slopes=slopes, prefix=prefix, qdoc=q_doc, kdoc=k_doc)
    return a


def _workspace(a, dt: int, dev):
    n = int(lib().turtle_token_attn_workspace(a, dt))
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _set(a, ws=ws, ws_bytes=n)
    return ws


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, softcap, causal, slopes, prefix, q_doc, k_doc):
        q, k, v = _tokens(q, "q"), _tokens(k, "k"), _tokens(v, "v")
        ctx.rest = (scale, softcap, causal)
        opt = (slopes, prefix, q_doc, k_doc)
        if q.numel() == 0 or k.numel() == 0:
            ctx.save_for_backward(q, k, v)
            return torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        a = _attn_args(q, k, v, *ctx.rest, *opt)
        grad = any(ctx.needs_input_grad[:3])
        o = _dense(q)
        lo = _dense(q) if grad and q.dtype != torch.float32 else None
        lse = torch.empty(q.shape[0] * q.shape[1] * q.shape[2], dtype=torch.float32, device=q.device) if grad else None
        n = int(lib().turtle_token_attn_ranges(a))
        ranges = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        _set(a, o=o, o_lo=lo, lse=lse, ranges=ranges)
        dt = _dt(q)
        ws = _workspace(a, dt, q.device)      # noqa: F841  (alive until the launch)
        with _on(q):
            _check(lib().turtle_token_attn_fwd(a, dt, _stream(q)), "token_attn_fwd")
        if grad:
            ctx.save_for_backward(q, k, v, o, lse, lo, ranges, *opt)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, *saved = ctx.saved_tensors
        need = ctx.needs_input_grad
        if not saved:
            return tuple(torch.zeros_like(t) if n else None for t, n in zip((q, k, v), need)) + (None,) * 7
        o, lse, lo, ranges, *opt = saved
        do = _tokens(do.to(q.dtype), "do")
        g = _Grads()
        g.f = _attn_args(q, k, v, *ctx.rest, *opt)
        _set(g.f, o=o, o_lo=lo, lse=lse, ranges=ranges)
        dq = _dense(q) if need[0] else None
        dk, dv = (_dense(k), _dense(v)) if need[1] or need[2] else (None, None)
        delta = torch.empty_like(lse)
        g.gb, g.gs, g.gh = _strides(do)
        _set(g, dout=do, dq=dq, dk=dk, dv=dv, delta=delta)
        with _on(q):
            _check(lib().turtle_token_attn_bwd(g, _dt(q), _stream(q)), "token_attn_bwd")
        return (dq, dk if need[1] else None, dv if need[2] else None) + (None,) * 7


def _check_qkv(q, k, v):
    _check_tokens(q, "q")
    _check_tokens(k, "k")
    _check_tokens(v, "v")
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"q is {q.dtype}, k is {k.dtype}, v is {v.dtype}")
    _same(q, k, "k")
    _same(q, v, "v")
    if tuple(k.shape) != tuple(v.shape) or k.shape[3] != q.shape[3]:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have one shape, and q's D ({q.shape[3]})")
    if q.shape[2] % k.shape[2]:
        raise ValueError(f"{q.shape[2]} query heads over {k.shape[2]} key heads: not a multiple")


def attention(q, k, v, *, scale=None, softcap: float = 0.0, slopes=None, causal: bool = False, prefix=None, q_doc=None, k_doc=None):
    """o = softmax(s) v over the visible keys, differentiable in q, k and v.

    q [B, Sq, Hq, D], k, v [B, Sk, Hk, D], Hq a multiple of Hk: query head h reads key head h // (Hq // Hk).
    Query i stands at place i + Sk - Sq among the keys (the last query at the last key). Scores:

    * z = scale q.k (scale: D ** -0.5 unless given); softcap > 0: z = softcap tanh(z / softcap);
    * slopes (fp32 [Hq]): z -= slopes[head] * |distance of the places|;
    * causal: a query sees the keys up to its own place, and the first ``prefix`` keys (int, or [B] integers) of its
      sequence in any case;
    * q_doc [B, Sq], k_doc [B, Sk] (k_doc None: q_doc, with Sq == Sk): integers; a query sees only keys of its own
      document. Negative: padding, which sees nothing and is seen by nobody - its rows may hold anything.

    A query that sees nothing gives zeros and passes no gradient. A value that is not finite in a key or value
    that ANY query may see can reach every query of its tile. Returns a dense [B, Sq, Hq, D] of q's type."""
    _check_qkv(q, k, v)
    B, Sq, Hq, D = q.shape
    Sk = k.shape[1]
    if k.shape[0] != B:
        raise ValueError(f"q has {B} sequences, k {k.shape[0]}")
    if prefix is not None:
        if not causal:
            raise ValueError("prefix: only with causal (without, every key is visible)")
        prefix = torch.full((B,), prefix, dtype=torch.int32, device=q.device) if isinstance(prefix, int) else _ints(prefix, (B,), "prefix", q)
    if q_doc is None and k_doc is not None:
        raise ValueError("k_doc without q_doc")
    if q_doc is not None:
        if k_doc is None and Sq != Sk:
            raise ValueError(f"q_doc alone needs Sq == Sk ({Sq}, {Sk}): pass k_doc")
        q_doc = _ints(q_doc, (B, Sq), "q_doc", q)
        k_doc = q_doc if k_doc is None else _ints(k_doc, (B, Sk), "k_doc", q)
    scale, softcap, slopes = _scale(scale, D), _cap(softcap), _slopes(slopes, Hq, q)
    _device(q)
    return _Attention.apply(q, k, v, scale, softcap, bool(causal), slopes, prefix, q_doc, k_doc)


def paged_attention(q, k_pages, v_pages, block_table, kv_lens, *, q_lens=None, scale=None, softcap: float = 0.0, slopes=None,
                    causal: bool = True):
    """Attention of a chunk of new tokens over a paged history: the serving form, from one token a sequence on.

    q [B, Sq, Hq, D]; k_pages, v_pages [pages, page, Hk, D] (pages of any size: one can hold a frame); block_table
    int32 [B, max pages]: key j of sequence b is row j % page of page block_table[b, j // page]; kv_lens int32 [B]:
    keys of every sequence, the chunk's own - written to the cache before the call - included; q_lens int32 [B] or
    None (all Sq): queries of every sequence. Query i stands at place kv_lens - q_lens + i; rows past q_lens give
    zeros. scale, softcap, slopes and causal as in ``attention``. Lengths past the table's room are cut to it; keys
    of a page number outside the pools are seen by nobody; what the pools hold past a sequence's length is never
    read. Lengths and tables stay on the device, so a captured call follows their contents. No gradient."""
    _check_qkv(q, k_pages, v_pages)
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad):
        raise RuntimeError("paged_attention has no gradient: call it under torch.no_grad()")
    B, Sq, Hq, D = q.shape
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError(f"block_table: expected an int32 [{B}, pages] tensor")
    for t, n in ((block_table, "block_table"), (kv_lens, "kv_lens"), (q_lens, "q_lens")):
        if t is None and n == "q_lens":
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
            raise TypeError(f"{n}: expected an int32 tensor")
        if n != "block_table" and tuple(t.shape) != (B,):
            raise ValueError(f"{n}: shape {tuple(t.shape)}, expected {(B,)}")
        _same(q, t, n)
    scale, softcap, slopes = _scale(scale, D), _cap(softcap), _slopes(slopes, Hq, q)
    _device(q)
    if q.numel() == 0 or k_pages.numel() == 0 or block_table.numel() == 0:
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    q, kp, vp = _tokens(q, "q"), _tokens(k_pages, "k_pages"), _tokens(v_pages, "v_pages")
    table, kv_lens = block_table.contiguous(), kv_lens.contiguous()
    q_lens = None if q_lens is None else q_lens.contiguous()
    a = _attn_args(q, kp, vp, scale, softcap, causal, slopes, None, None, None)
    o = _dense(q)
    a.Sk = 0
    _set(a, o=o, page=kp.shape[1], npages=kp.shape[0], maxpages=table.shape[1], table=table, kv_lens=kv_lens, q_lens=q_lens)
    dt = _dt(q)
    ws = _workspace(a, dt, q.device)          # noqa: F841  (alive until the launch)
    with _on(q):
        _check(lib().turtle_token_attn_fwd(a, dt, _stream(q)), "token_attn_fwd")
    return o
