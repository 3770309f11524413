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

The first three are differentiable (first order, reverse mode; a tensor with a forward-mode tangent is refused); sums run
in a fixed order, so results repeat bit for bit.
"""
from __future__ import annotations

import ctypes as C
import decimal
import functools
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .train_ops import _check, _dt

MAX_D = 128

# the argument blocks of include/turtle_token.h, packed in one go (a small call is bound by its host work)
_SIDE = struct.Struct("@4P6q2i")
_AXES = struct.Struct("@64Q64B2i")
_ATTN = struct.Struct("@3P9q6i2f4P4i8PN")
_GRADS = struct.Struct("@P3q4P")
_NO_SIDE = bytes(_SIDE.size)

_bound = None


def lib():
    global _bound
    if _bound is not None:
        return _bound
    L = _lib.lib()
    vp, i64, ci, sz, blk = C.c_void_p, C.c_int64, C.c_int, C.c_size_t, C.c_char_p
    rope = [blk, blk, blk, vp, i64, ci, i64, i64, ci]
    L.turtle_token_rope.argtypes = rope + [ci, ci, vp]
    L.turtle_token_norm_rope_fwd.argtypes = rope + [C.c_float, ci, vp]
    L.turtle_token_norm_rope_workspace.argtypes = [i64, ci]
    L.turtle_token_norm_rope_workspace.restype = sz
    L.turtle_token_norm_rope_bwd.argtypes = rope + [C.c_float, vp, vp, sz, ci, vp]
    L.turtle_token_attn_ranges.argtypes = [blk]
    L.turtle_token_attn_ranges.restype = sz
    L.turtle_token_attn_workspace.argtypes = [blk, ci]
    L.turtle_token_attn_workspace.restype = sz
    L.turtle_token_attn_bwd_workspace.argtypes = [blk, ci]
    L.turtle_token_attn_bwd_workspace.restype = sz
    L.turtle_token_attn_fwd.argtypes = [blk, ci, vp]
    L.turtle_token_attn_bwd.argtypes = [blk, ci, vp]
    _bound = L
    return L


# -------------------------------------------------------------------------------------------------
# arguments
# -------------------------------------------------------------------------------------------------

def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _tokens(t) -> torch.Tensor:
    """``t`` itself when the kernels can read it: channels contiguous, rows at multiples of 16 bytes; else a copy."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        n, st, per = t.shape, t.stride(), 16 // t.element_size()
        if st[3] == 1 and (st[0] % per == 0 or n[0] == 1) and (st[1] % per == 0 or n[1] == 1) and (st[2] % per == 0 or n[2] == 1):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    """(batch, token, head) strides in elements; 0 along a dimension of one (it may have any stride)."""
    n, st = t.shape, t.stride()
    return (st[0] if n[0] > 1 else 0, st[1] if n[1] > 1 else 0, st[2] if n[2] > 1 else 0)


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
    """An int32 tensor of ``shape`` on ``like``'s device from an integer tensor (64-bit values are cut to the range)."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: expected an int32 or int64 tensor")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    _same(like, t, name)
    return (t if t.dtype == torch.int32 else t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)).contiguous()


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
    if not (c == 0.0 or 1e-6 <= c <= 1e30):
        raise ValueError(f"softcap = {softcap}, must be 0 (none) or of 1e-6 to 1e30")
    return c


def _scale(scale, D: int) -> float:
    s = D ** -0.5 if scale is None else float(scale)
    if not abs(s) <= 1e30:
        raise ValueError(f"scale = {scale}, must be finite and at most 1e30")
    return s


_device_now, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _run(t, what: str, entry, *args):
    """One library call on ``t``'s device (made the current one where it is not) and its current stream."""
    i = t.device.index
    if _device_now() == i:
        rc = entry(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            rc = entry(*args, _raw_stream(i))
    if rc:
        _check(rc, what)


def _no_tangents(*ts):
    """Refuses tensors with a tangent: whether they require a gradient or not, the result would have none."""
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("turtle token operators have no forward-mode derivative")


def _wants_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# -------------------------------------------------------------------------------------------------
# rotation
# -------------------------------------------------------------------------------------------------

_TWO_PI = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


@functools.lru_cache(maxsize=64)
def _axes_table(axes, base: float):
    """Every rotated pair's axis and its revolutions per unit of position in 64-bit fixed point, rounded once: pos * freq
    mod 2^64 is the angle but for |pos| 2^-65 revolutions (a double has 53 bits: at 2^50 it would be arbitrary to 0.03)."""
    freq, axis = [0] * 64, [0] * 64
    i = 0
    with decimal.localcontext(decimal.Context(prec=50)):
        ln = decimal.Decimal(base).ln()
        for a, d in enumerate(axes):
            for j in range(0, d, 2):
                freq[i], axis[i] = int((2 ** 64 * (-ln * j / d).exp() / _TWO_PI).to_integral_value()), a
                i += 1
    return _AXES.pack(*freq, *axis, i, len(axes))


def _axes(axes, base, D: int):
    ax = tuple(int(d) for d in axes)
    if not 1 <= len(ax) <= 4 or any(d < 0 or d % 2 for d in ax) or sum(ax) > D:
        raise ValueError(f"axes = {tuple(axes)}: one to four even channel counts, together at most D = {D}")
    base = float(base)
    if not 1.0 <= base < float("inf"):
        raise ValueError(f"base = {base}, must be at least 1")
    return _axes_table(ax, base), len(ax)


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
    return _SIDE.pack(x.data_ptr(), _ptr(dy), y.data_ptr(), _ptr(w), *_strides(x), *((0, 0, 0) if dy is None else _strides(dy)), x.shape[2], 0)


def _dense(x):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _turn(x, pos, pos_b, pos64, tab, inverse):
    x = _tokens(x)
    y = _dense(x)
    B, S, H, D = x.shape
    if B and S:
        _run(x, "token_rope", lib().turtle_token_rope, _side(x, y), _NO_SIDE, tab, pos.data_ptr(), pos_b, pos64, B, S, D, inverse, _dt(x))
    return y


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, pos_b, pos64, tab):
        ctx.save_for_backward(pos)
        ctx.rest = (pos_b, pos64, tab)
        return _turn(x, pos, pos_b, pos64, tab, 0)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return _turn(dy, ctx.saved_tensors[0], *ctx.rest, 1), None, None, None, None


def axial_rope(x, pos, axes, base: float = 10000.0):
    """Rotary positions over several axes: the first ``axes[0]`` channels of every head turn with the token's
    place on axis 0, the next ``axes[1]`` with its place on axis 1, and so on; channels past ``sum(axes)`` pass
    unchanged. Within an axis of d channels, pair i - channels (2 i, 2 i + 1) - turns by the angle
    ``pos[axis] * base ** (-2 i / d)``.

    x [B, S, heads, D]; pos int32 or int64 [S, len(axes)] or [B, S, len(axes)] (any sign; an angle is off by at most
    2^-23 and ``|pos| 2^-62`` rad, the latter 6e-5 at 2^48); axes one to four even numbers. Returns a dense tensor of x's type."""
    _check_tokens(x, "x")
    B, S, _, D = x.shape
    tab, naxis = _axes(axes, base, D)
    p, pos_b, pos64 = _pos(pos, B, S, naxis, x)
    _device(x)
    _no_tangents(x)
    return _Rope.apply(x, p, pos_b, pos64, tab) if _wants_grad(x) else _turn(x, p, pos_b, pos64, tab, 0)


def _gain(w):
    return None if w is None else w.detach().float().contiguous()


def _norm_turn(q, k, wq, wk, pos, pos_b, pos64, tab, eps):
    """(q', k') from readable q, k and fp32 gains."""
    yq, yk = _dense(q), _dense(k)
    B, S, _, D = q.shape
    if B and S:
        _run(q, "token_norm_rope_fwd", lib().turtle_token_norm_rope_fwd, _side(q, yq, wq), _side(k, yk, wk), tab, pos.data_ptr(), pos_b,
             pos64, B, S, D, eps, _dt(q))
    return yq, yk


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, *rest):
        q, k = _tokens(q), _tokens(k)
        gq, gk = _gain(wq), _gain(wk)
        ctx.save_for_backward(q, k, rest[0], gq, gk)
        ctx.rest = rest[1:]
        ctx.w_dt = (None if wq is None else wq.dtype, None if wk is None else wk.dtype)
        return _norm_turn(q, k, gq, gk, *rest)

    @staticmethod
    @once_differentiable
    def backward(ctx, dyq, dyk):
        q, k, pos, wq, wk = ctx.saved_tensors
        pos_b, pos64, tab, eps = ctx.rest
        B, S, _, D = q.shape
        dyq, dyk = _tokens(dyq), _tokens(dyk)
        dq, dk = _dense(q), _dense(k)
        need = ctx.needs_input_grad
        nq, nk = need[2] and wq is not None, need[3] and wk is not None
        dw, ws, n = None, None, 0
        if nq or nk:
            n = _norm_workspace(B * S, D)
            dw = torch.empty(2 * D, dtype=torch.float32, device=q.device)
            ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        if B and S:
            _run(q, "token_norm_rope_bwd", lib().turtle_token_norm_rope_bwd, _side(q, dq, wq, dyq), _side(k, dk, wk, dyk), tab,
                 pos.data_ptr(), pos_b, pos64, B, S, D, eps, _ptr(dw), _ptr(ws), n, _dt(q))
        elif dw is not None:
            dw.zero_()
        return (dq, dk, dw[:D].to(ctx.w_dt[0]) if nq else None, dw[D:].to(ctx.w_dt[1]) if nk else None, None, None, None, None, None)


@functools.lru_cache(maxsize=256)
def _norm_workspace(tokens: int, D: int) -> int:
    return lib().turtle_token_norm_rope_workspace(tokens, D)


def qk_norm_rope(q, k, pos, q_weight, k_weight, axes, base: float = 10000.0, eps: float = 1e-6):
    """(q', k'): every head's RMS norm over its D channels, x / sqrt(mean(x^2) + eps) times the gain (``q_weight``
    / ``k_weight`` [D], or None), then ``axial_rope``, in one pass over q and k.

    q [B, S, Hq, D], k [B, S, Hk, D] of one type at the same tokens; pos, axes and base as in ``axial_rope``.
    Gradients go to q, k and the gains. Squares are fp32: a head whose mean square passes that range gives zeros and
    passes no gradient."""
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
    if not 1e-30 <= eps < float("inf"):
        raise ValueError(f"eps = {eps}, must be finite and at least 1e-30")
    tab, naxis = _axes(axes, base, D)
    rest = (*_pos(pos, B, S, naxis, q), tab, eps)
    _device(q)
    _no_tangents(q, k, q_weight, k_weight)
    if _wants_grad(q, k, q_weight, k_weight):
        return _QkNormRope.apply(q, k, q_weight, k_weight, *rest)
    return _norm_turn(_tokens(q), _tokens(k), _gain(q_weight), _gain(k_weight), *rest)


# -------------------------------------------------------------------------------------------------
# attention
# -------------------------------------------------------------------------------------------------

def _attn_block(q, k, v, rules, masks, o, Sk, pages=(0, 0, 0), cache=(None, None, None), lo=0, lse=0, ranges=0, ws=0, ws_bytes=0):
    """turtle_token_attn_args. rules: (scale, softcap, causal); masks: (slopes, prefix, q_doc, k_doc)."""
    scale, softcap, causal = rules
    B, Sq, Hq, D = q.shape
    return _ATTN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), *_strides(q), *_strides(k), *_strides(v), B, Sq, Sk, Hq, k.shape[2], D,
                      scale, softcap, *map(_ptr, masks), causal, *pages, *map(_ptr, cache), o.data_ptr(), lo, lse, ranges, ws, ws_bytes)


def _attn_forward(q, k, v, rules, masks, grad):
    """(o, aux) of readable, non-empty q, k, v; aux (or None): what the backward needs besides - o's rounding remainder
    (16-bit types), the rows' softmax sums, the document ranges - in one buffer."""
    o = _dense(q)
    n, Sk, dt = q.shape[0] * q.shape[1] * q.shape[2], k.shape[1], _dt(q)
    lo = lse = ranges = 0
    aux = None
    docs = masks[2] is not None
    if grad or docs:
        nr = lib().turtle_token_attn_ranges(_attn_block(q, k, v, rules, masks, o, Sk)) if docs else 0
        parts = _aux_parts(n, q.shape[3], dt, nr) if grad else (0, 0, nr)
        aux = torch.empty(parts[2], dtype=torch.uint8, device=q.device)
        p = aux.data_ptr()
        ranges = p + parts[1] if docs else 0
        if grad:
            lo, lse = (p if dt else 0), p + parts[0]
    ws, nws = _attn_workspace(q.shape, k.shape[2], Sk, (0, 0, 0), dt, q.device)
    blk = _attn_block(q, k, v, rules, masks, o, Sk, lo=lo, lse=lse, ranges=ranges, ws=_ptr(ws), ws_bytes=nws)
    _run(q, "token_attn_fwd", lib().turtle_token_attn_fwd, blk, dt)
    return o, aux


def _aux_parts(n: int, D: int, dt: int, nr: int):
    """Byte offsets of (sums, ranges, end) for n rows, behind the remainder."""
    a = 2 * n * D if dt else 0
    b = (a + 4 * n + 15) // 16 * 16
    return a, b, b + nr


@functools.lru_cache(maxsize=256)
def _workspace_bytes(q_shape, Hk: int, Sk: int, pages, dt: int) -> int:
    """The library's answer for these sizes (it goes by nothing else)."""
    B, Sq, Hq, D = q_shape
    a = [0] * 37
    a[12:18], a[25:28], a[28] = (B, Sq, Sk, Hq, Hk, D), pages, 1 if pages[0] else 0
    return lib().turtle_token_attn_workspace(_ATTN.pack(*a), dt)


def _attn_workspace(q_shape, Hk: int, Sk: int, pages, dt: int, device):
    n = _workspace_bytes(q_shape, Hk, Sk, pages, dt)
    return (torch.empty(n, dtype=torch.uint8, device=device), n) if n else (None, 0)


@functools.lru_cache(maxsize=256)
def _bwd_workspace_bytes(q_shape, Hk: int, Sk: int, docs: bool, dt: int) -> int:
    B, Sq, Hq, D = q_shape
    a = [0] * 37
    a[12:18], a[22] = (B, Sq, Sk, Hq, Hk, D), 1 if docs else 0
    return lib().turtle_token_attn_bwd_workspace(_ATTN.pack(*a), dt)


class _NoKeys(torch.autograd.Function):
    """Attention where there are no keys, or no queries: zeros, and zero gradients."""

    @staticmethod
    def forward(ctx, q, k, v):
        ctx.save_for_backward(q, k, v)
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device)

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        return tuple(torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t in ctx.saved_tensors)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, rules, *masks):
        q, k, v = _tokens(q), _tokens(k), _tokens(v)
        o, aux = _attn_forward(q, k, v, rules, masks, True)
        ctx.save_for_backward(q, k, v, o, aux, *masks)
        ctx.rules = rules
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, aux, *masks = ctx.saved_tensors
        need = ctx.needs_input_grad
        do = _tokens(do)
        n, dt, p = q.shape[0] * q.shape[1] * q.shape[2], _dt(q), aux.data_ptr()
        lse, ranges, _ = _aux_parts(n, q.shape[3], dt, 0)
        dq = _dense(q) if need[0] else None
        dk, dv = (_dense(k), _dense(v)) if need[1] or need[2] else (None, None)
        docs = masks[2] is not None
        nws = _bwd_workspace_bytes(q.shape, k.shape[2], k.shape[1], docs, dt)
        # the split sums, then the rows' deltas: this run's own, a graph may be walked twice at once
        ws = torch.empty(nws + 4 * n, dtype=torch.uint8, device=q.device)
        pws = ws.data_ptr()
        blk = _attn_block(q, k, v, ctx.rules, masks, o, k.shape[1], lo=p if dt else 0, lse=p + lse, ranges=p + ranges if docs else 0, ws=pws,
                          ws_bytes=nws)
        blk += _GRADS.pack(do.data_ptr(), *_strides(do), _ptr(dq), _ptr(dk), _ptr(dv), pws + nws)
        _run(q, "token_attn_bwd", lib().turtle_token_attn_bwd, blk, dt)
        return (dq, dk if need[1] else None, dv if need[2] else None) + (None,) * 5


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
    * q_doc [B, Sq], k_doc [B, Sk] (k_doc None: q_doc, with Sq == Sk): integers below 2^31; a query sees only keys
      of its own document. Negative: padding, which sees nothing and is seen by nobody - its rows may hold anything.

    A query that sees nothing gives zeros and passes no gradient, whatever it and its gradient hold (so does one whose
    every visible score is minus infinity). Elsewhere what is not finite makes the results that depend on it infinite or
    not a number, and can reach further within its tile (32 to 64 tokens, those it is hidden from included): a key or
    value - of any document but padding - the results of queries and their dq, a query or its gradient the dk and dv of
    keys; a query's own result stays in its row. Returns a dense
    [B, Sq, Hq, D] of q's type."""
    _check_qkv(q, k, v)
    B, Sq, Hq, D = q.shape
    Sk = k.shape[1]
    if k.shape[0] != B:
        raise ValueError(f"q has {B} sequences, k {k.shape[0]}")
    if prefix is not None:
        if not causal:
            raise ValueError("prefix: only with causal (without, every key is visible)")
        prefix = torch.full((B,), max(0, min(prefix, 2 ** 31 - 1)), dtype=torch.int32, device=q.device) if isinstance(prefix, int) else _ints(prefix, (B,), "prefix", q)
    if q_doc is None and k_doc is not None:
        raise ValueError("k_doc without q_doc")
    if q_doc is not None:
        if k_doc is None and Sq != Sk:
            raise ValueError(f"q_doc alone needs Sq == Sk ({Sq}, {Sk}): pass k_doc")
        q_doc = _ints(q_doc, (B, Sq), "q_doc", q)
        k_doc = q_doc if k_doc is None else _ints(k_doc, (B, Sk), "k_doc", q)
    _no_tangents(q, k, v, slopes)
    scale, softcap, slopes = _scale(scale, D), _cap(softcap), _slopes(slopes, Hq, q)
    _device(q)
    rules, masks = (scale, softcap, 1 if causal else 0), (slopes, prefix, q_doc, k_doc)
    if B == 0 or Sq == 0 or Sk == 0:
        return _NoKeys.apply(q, k, v)
    if _wants_grad(q, k, v):
        return _Attention.apply(q, k, v, rules, *masks)
    return _attn_forward(_tokens(q), _tokens(k), _tokens(v), rules, masks, False)[0]


def paged_attention(q, k_pages, v_pages, block_table, kv_lens, *, q_lens=None, scale=None, softcap: float = 0.0, slopes=None,
                    causal: bool = True):
    """Attention of a chunk of new tokens over a paged history: the serving form, from one token a sequence on.

    q [B, Sq, Hq, D]; k_pages, v_pages [pages, page, Hk, D] (pages of any size: one can hold a frame); block_table
    int32 [B, max pages]: key j of sequence b is row j % page of page block_table[b, j // page]; kv_lens int32 [B]:
    keys of every sequence, the chunk's own - written to the cache before the call - included; q_lens int32 [B] or
    None (all Sq): queries of every sequence. Query i stands at place kv_lens - q_lens + i; rows past q_lens give
    zeros. scale, softcap, slopes and causal as in ``attention``. Lengths past the table's room are cut to it (a
    query's place goes by kv_lens as it is), those below zero count as zero; keys of a page number outside the pools are
    seen by nobody; what the pools hold past a sequence's length is never read. Lengths and
    tables stay on the device, so a captured call follows their contents. No gradient."""
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
    _no_tangents(q, k_pages, v_pages, slopes)
    scale, softcap, slopes = _scale(scale, D), _cap(softcap), _slopes(slopes, Hq, q)
    _device(q)
    if q.numel() == 0 or k_pages.numel() == 0 or block_table.numel() == 0:
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    q, kp, vp = _tokens(q), _tokens(k_pages), _tokens(v_pages)
    cache = (block_table.contiguous(), kv_lens.contiguous(), None if q_lens is None else q_lens.contiguous())
    rules, masks, pages = (scale, softcap, 1 if causal else 0), (slopes, None, None, None), (kp.shape[1], kp.shape[0], block_table.shape[1])
    o, dt = _dense(q), _dt(q)
    ws, nws = _attn_workspace(q.shape, kp.shape[2], 0, pages, dt, q.device)
    _run(q, "token_attn_fwd", lib().turtle_token_attn_fwd, _attn_block(q, kp, vp, rules, masks, o, 0, pages, cache, ws=_ptr(ws), ws_bytes=nws), dt)
    return o
