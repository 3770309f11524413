"""Autograd Functions over the hand-written HIP training kernels (include/turtle_train.h).

The training graph (turtlevsr_amd/train.py) keeps its activations channels-last (torch
``channels_last``: NHWC storage, the inference path's layout) and runs these op families through
libturtle_hip.so, forward and backward:

* ``conv1x1``      pointwise convolutions (217 per frame, 87 % of the MACs): the inference GEMM
                   family forward and for the input gradient (W transposed); the weight gradient
                   dW = dY^T X as a reduction GEMM over pixels on the matrix cores; bias gradients as
                   column sums. Per-image weight sets (channel attention W_eff = project_out .
                   blockdiag(A), turtle_t1_arch.py:694-702) use the same kernels;
* ``gram``         the channel-attention Gram q^T k over HW per head (turtle_t1_arch.py:694-697) as a
                   reduction GEMM; its backward as GEMMs with block-diagonal per-image weights;
* ``layer_norm``   per-pixel LayerNorm over channels (turtle_t1_arch.py:67-112), 98 per frame;
* ``dwconv3x3``    depthwise 3x3 / pad 1 convolutions (99 per frame);
* ``gelu_gate``    gelu(x1) * x2 of the GatedFeedForward (turtle_t1_arch.py:176);
* ``gelu``         the plain GELU of FeedForward / ReducedAttn (turtle_t1_arch.py:181-210, 704-742);
* ``norm_cols`` / ``cross_gram``  the FHR / CHM attention with its caches (turtle_t1_arch.py:218-286,
                   612-662): per-channel L2 normalisation over HW and the q [k_cache ; k]^T scores;
* ``conv3x3``      the dense 3x3 convolutions of Down / Upsample (turtle_t1_arch.py:136-154), forward,
                   input and weight gradients;
* ``window_conv``  the SAB window convolutions k2_dwconv / q2_dwconv (ws x ws, stride ws, pad 1, one group
                   per channel: turtle_t1_arch.py:306-308), forward, input and weight gradients.

They run on the caller's current HIP stream; weights and their gradients are fp32, activations
fp32 or bf16 (autocast), fp16 for the elementwise kernels; the GEMMs take fp16 autocast operands
as bf16 (cast in, cast back). There is no CPU path: a CPU tensor or a missing library raises.
"""
from __future__ import annotations

import ctypes as C
import torch
from torch.utils.weak import WeakIdKeyDictionary

from . import _lib

_train = None
CL = torch.channels_last


def lib():
    global _train
    if _train is not None:
        return _train
    L = _lib.lib()
    vp, i64, ci, sz = C.c_void_p, C.c_int64, C.c_int, C.c_size_t
    L.turtle_train_ln_fwd.argtypes = [vp, i64, vp, vp, vp, i64, vp, vp, i64, ci, ci, ci, vp]
    L.turtle_train_ln_bwd.argtypes = [vp, i64, vp, vp, vp, vp, i64, vp, i64, vp, i64, vp, vp, i64, ci, ci, ci, vp]
    L.turtle_train_dw3x3_fwd.argtypes = [vp, i64, vp, vp, vp, i64, i64, ci, ci, ci, ci, ci, vp]
    L.turtle_train_dw3x3_wgrad.argtypes = [vp, i64, vp, i64, vp, vp, i64, ci, ci, ci, ci, vp]
    L.turtle_train_gate_fwd.argtypes = [vp, i64, vp, i64, i64, ci, ci, vp]
    L.turtle_train_gate_bwd.argtypes = [vp, i64, vp, i64, vp, i64, i64, ci, ci, vp]
    L.turtle_train_colsum.argtypes = [vp, i64, vp, i64, ci, ci, vp]
    L.turtle_train_gemm.argtypes = [vp, i64, vp, i64, i64, vp, vp, i64, vp, i64, i64, ci, ci, ci, vp]
    L.turtle_train_rgemm_workspace.argtypes = [i64, ci, ci, i64]
    L.turtle_train_rgemm_workspace.restype = sz
    L.turtle_train_rgemm.argtypes = [vp, i64, vp, i64, vp, i64, ci, ci, i64, ci, ci, vp, sz, vp]
    L.turtle_train_colsumsq.argtypes = [vp, i64, vp, i64, ci, i64, ci, vp]
    L.turtle_train_gram_wd.argtypes = [vp, vp, vp, vp, i64, ci, ci, ci, vp]
    L.turtle_train_gelu_fwd.argtypes = [vp, i64, vp, i64, i64, ci, ci, vp]
    L.turtle_train_gelu_bwd.argtypes = [vp, i64, vp, i64, vp, i64, i64, ci, ci, vp]
    L.turtle_train_window_fwd.argtypes = [vp, i64, vp, vp, vp, i64, i64, ci, ci, ci, ci, ci, ci, ci, vp]
    L.turtle_train_window_dgrad.argtypes = [vp, i64, vp, vp, i64, i64, ci, ci, ci, ci, ci, ci, ci, vp]
    L.turtle_train_window_wgrad.argtypes = [vp, i64, vp, i64, vp, i64, ci, ci, ci, ci, ci, ci, ci, vp]
    L.turtle_train_conv3x3.argtypes = [vp, i64, vp, vp, vp, i64, i64, ci, ci, ci, ci, ci, vp]
    L.turtle_train_coldot.argtypes = [vp, i64, vp, i64, vp, i64, ci, i64, ci, vp]
    L.turtle_train_sab_softmax_fwd.argtypes = [vp, i64, ci, ci, ci, vp, vp, vp, ci, vp]
    L.turtle_train_sab_softmax_bwd.argtypes = [vp, vp, vp, i64, ci, vp, ci, vp]
    L.turtle_train_colscale.argtypes = [vp, i64, vp, vp, i64, i64, ci, i64, ci, vp]
    L.turtle_train_l2n_bwd.argtypes = [vp, i64, vp, i64, vp, vp, vp, i64, i64, ci, i64, ci, vp]
    L.turtle_train_conv3x3_wgrad_workspace.argtypes = [i64, ci, ci]
    L.turtle_train_conv3x3_wgrad_workspace.restype = sz
    L.turtle_train_conv3x3_wgrad.argtypes = [vp, i64, vp, i64, vp, i64, ci, ci, ci, ci, ci, vp, sz, vp]
    _train = L
    return L


def _p(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return 0
    if t.dtype == torch.bfloat16:
        return 1
    if t.dtype == torch.float16:
        return 2
    raise TypeError(f"training kernels take fp32 / bf16 / fp16 activations, got {t.dtype}")


def _stream(t):
    if t.device.type != "cuda":
        raise RuntimeError("turtle training kernels run on a ROCm device only")
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _check(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} failed ({rc})")


def rows(t: torch.Tensor):
    """(tensor, ld): a [B, C, H, W] tensor as NHWC pixel rows - channel stride 1, images and rows
    contiguous with pixel stride ld, 16-byte aligned - copied to channels_last when it is not."""
    if t.dim() != 4:
        raise ValueError("expected a [B, C, H, W] tensor")
    B, Cc, H, W = t.shape
    s = t.stride()
    es = t.element_size()
    ld = s[3] if W > 1 else (s[2] if H > 1 else (s[0] if B > 1 else Cc))
    ok = (Cc == 1 or s[1] == 1) and ld >= Cc and (W == 1 or s[3] == ld) and (H == 1 or s[2] == W * ld) and \
         (B == 1 or s[0] == H * W * ld) and t.data_ptr() % 16 == 0 and (ld * es) % 16 == 0
    if ok:
        return t, ld
    return t.contiguous(memory_format=CL), Cc


def _empty(B, Cc, H, W, like):
    return torch.empty((B, Cc, H, W), dtype=like.dtype, device=like.device, memory_format=CL)


def _gemm_dt(x: torch.Tensor) -> torch.dtype:
    return torch.float32 if x.dtype == torch.float32 else torch.bfloat16


class ParamGradAccumulator:
    """In-place parameter-gradient accumulation over one training step.

    A clip of T frames uses every weight T times (plus the reference's 0 * sum(p) term,
    video_restoration_model.py:99), so autograd builds T per-use fp32 gradients of each parameter
    and adds them pairwise in the AccumulateGrad input buffer - about 4 000 fp32 adds, 1 300 fills
    and the term's 633 sums / expands / adds per GoPro step (profiles/r06f_train_sites.txt). Inside
    ``step()`` the HIP ops instead accumulate each use's weight / bias gradient in place into one
    zero-filled fp32 arena (the reduction GEMM's accumulate mode, the atomics of the LayerNorm /
    depthwise / window / column-sum reductions), return None for every use but the last backward one
    of a parameter, and hand autograd the finished sum there: one AccumulateGrad per parameter, as
    before, with no adds. Uses are counted in the forward; a use whose backward never runs leaves a
    count behind and ``step()`` raises rather than dropping that parameter's gradient.

    ``zero_term(params)`` is the reference's 0 * sum(p) term with the same (zero) gradient for the
    parameters no HIP op reported, and none for the others - they receive a real gradient anyway."""

    def __init__(self, params):
        self.slot, off = {}, 0
        for p in params:
            if p.requires_grad and p.dtype == torch.float32 and id(p) not in self.slot:
                self.slot[id(p)] = (p, off)
                off += (p.numel() + 15) // 16 * 16             # 64-byte aligned slices
        self.total = off
        self.arena, self.count = None, {}

    def use(self, w):
        """The parameter behind ``w`` (itself or the base of a view of it) when its gradient is
        accumulated here - one more pending use - else None."""
        if w is None or not w.requires_grad:
            return None
        base = w if w.is_leaf else w._base
        s = self.slot.get(id(base))
        if s is None or s[0] is not base:
            return None
        self.count[id(base)] = self.count.get(id(base), 0) + 1
        return base

    def buf(self, p, n: int):
        """The parameter's first ``n`` fp32 accumulators (flat)."""
        off = self.slot[id(p)][1]
        return self.arena[off:off + n]

    def done(self, p, make):
        """One use's backward finished: None, or ``make(flat slot)`` after the last one."""
        k = id(p)
        self.count[k] -= 1
        if self.count[k]:
            return None
        del self.count[k]
        return make(self.buf(p, p.numel()))

    def zero_term(self, params):
        return _ZeroTerm.apply(self, *params)

    def step(self):
        return _AccStep(self)


class _AccStep:
    def __init__(self, acc):
        self.acc = acc

    def __enter__(self):
        global _ACC
        if _ACC is not None:
            raise RuntimeError("nested ParamGradAccumulator steps")
        a = self.acc
        dev = next(iter(a.slot.values()))[0].device if a.slot else None
        a.arena = torch.zeros(max(a.total, 16), dtype=torch.float32, device=dev)
        a.count = {}
        _ACC = a
        return a

    def __exit__(self, et, ev, tb):
        global _ACC
        _ACC = None
        a = self.acc
        left, a.count, a.arena = a.count, {}, None
        if et is None and left:
            names = sorted(tuple(a.slot[k][0].shape) for k in left)[:4]
            raise RuntimeError(f"{len(left)} parameters kept gradient uses whose backward never ran (shapes {names})")
        return False


_ACC = None


def _acc_use(ctx, i: int, w):
    """(accumulator, parameter) for input ``i`` (= ``w``) of an autograd Function's forward inside an
    accumulating step when that input takes a gradient (forward runs in no-grad mode: the
    Function's needs_input_grad says whether this use will see a backward), else None."""
    a = _ACC
    if a is None or not ctx.needs_input_grad[i]:
        return None
    p = a.use(w)
    return None if p is None else (a, p)


def _acc_dst(acc, n: int):
    """A use's gradient destination: the parameter's fp32 arena slice (accumulated into), or None."""
    return None if acc is None else acc[0].buf(acc[1], n)


def _acc_done(acc, make):
    return acc[0].done(acc[1], make)


class _ZeroTerm(torch.autograd.Function):
    """0 * sum(p.sum()) over ``params`` (video_restoration_model.py:99) as far as the step sees it:
    a zero added to the loss and a zero gradient for the parameters not accumulated by ``acc``.
    (The reference's term would also turn the - never used - total loss value into NaN for a
    non-finite parameter; the loss reported is l_pix in both.)"""

    @staticmethod
    def forward(ctx, acc, *params):
        ctx.covered = [id(p) in acc.count for p in params]
        ctx.shapes = [(p.shape, p.dtype, p.device) for p in params]
        dev = params[0].device if params else None
        return torch.zeros((), dtype=torch.float32, device=dev)

    @staticmethod
    def backward(ctx, g):
        return (None,) + tuple(None if c else torch.zeros(s, dtype=d, device=dv)
                               for c, (s, d, dv) in zip(ctx.covered, ctx.shapes))


class _LayerNorm(torch.autograd.Function):
    """y = LayerNorm(x) in ``out_dtype``: an fp32 x (the residual stream under autocast, promoted by
    the fp32 gamma / beta scales as in the reference) is read as fp32 and y written in the autocast
    dtype by the kernel itself, and the backward writes dx in fp32 - no cast passes either way.

    ``residual``: also return x itself (an alias) for the block's residual use, x + branch(LN(x))
    (turtle_t1_arch.py:808-809). Its gradient then comes back into this backward, which the kernel
    adds into dx - autograd would otherwise sum x's two gradients with a separate full-size add."""

    @staticmethod
    def forward(ctx, x, w, b, biasfree: bool, out_dtype, residual: bool = False):
        x_in = x
        x, ldx = rows(x)
        B, Cc, H, W = x.shape
        P = B * H * W
        y = torch.empty((B, Cc, H, W), dtype=out_dtype, device=x.device, memory_format=CL)
        mu = torch.empty(P, dtype=torch.float32, device=x.device)
        rs = torch.empty_like(mu)
        w32 = w.float().contiguous()
        b32 = None if b is None else b.float().contiguous()
        dt = _dt(x) | ((_dt(y) + 1) << 4 if y.dtype != x.dtype else 0)
        _check(lib().turtle_train_ln_fwd(_p(x), ldx, _p(w32), _p(b32), _p(y), Cc, _p(mu), _p(rs), P, Cc, int(biasfree), dt,
                                         _stream(x)), "ln_fwd")
        ctx.save_for_backward(x, w32, mu, rs)
        ctx.biasfree, ctx.has_b, ctx.ldx, ctx.ydt = biasfree, b is not None, ldx, y.dtype
        ctx.acc_w, ctx.acc_b, ctx.w_shape = _acc_use(ctx, 1, w), _acc_use(ctx, 2, b), w.shape
        return (y, x_in.view_as(x_in)) if residual else y

    @staticmethod
    def backward(ctx, dy, dres=None):
        x, w32, mu, rs = ctx.saved_tensors
        dy, lddy = rows(dy.to(ctx.ydt))
        if dres is not None:
            dres, lddres = rows(dres.to(x.dtype))
        B, Cc, H, W = x.shape
        P = B * H * W
        dx = _empty(B, Cc, H, W, x)
        aw, ab = ctx.acc_w, ctx.acc_b
        dw, db = _acc_dst(aw, Cc), (_acc_dst(ab, Cc) if ctx.has_b else None)
        nz = (Cc if dw is None else 0) + (Cc if ctx.has_b and db is None else 0)
        if nz:
            z = torch.zeros(nz, dtype=torch.float32, device=x.device)                    # one fill for both
            dw = z[:Cc] if dw is None else dw
            db = z[nz - Cc:] if ctx.has_b and db is None else db
        dt = _dt(x) | ((_dt(dy) + 1) << 4 if dy.dtype != x.dtype else 0)
        _check(lib().turtle_train_ln_bwd(_p(x), ctx.ldx, _p(w32), _p(mu), _p(rs), _p(dy), lddy, _p(dx), Cc, _p(dres),
                                         lddres if dres is not None else 0, _p(dw), _p(db), P, Cc, int(ctx.biasfree), dt,
                                         _stream(x)), "ln_bwd")
        shape = ctx.w_shape
        dw = _acc_done(aw, lambda f: f.view(shape)) if aw else dw
        db = _acc_done(ab, lambda f: f.view(shape)) if ab else db
        return dx, dw, db, None, None, None


_DWCACHE = WeakIdKeyDictionary()


def _dw_taps(w):
    """(w9, w9 flipped): the depthwise weight [C, 1, 3, 3] as fp32 tap-major [9, C] tables for the
    forward and the data gradient, built once per parameter version (5 frames x forward + backward
    reuse them) - the same validity rule as the GEMM weight casts (_WCast)."""
    if not isinstance(w, torch.nn.Parameter):
        w9 = w.detach().float().reshape(w.shape[0], 9).t().contiguous()
        return w9, w9.flip(0).contiguous()
    e = _DWCACHE.get(w)
    if e is None or e[0] != w._version or e[1] != w.data_ptr() or e[2].device != w.device:
        w9 = w.detach().float().reshape(w.shape[0], 9).t().contiguous()
        e = _DWCACHE[w] = (w._version, w.data_ptr(), w9, w9.flip(0).contiguous())
    return e[2], e[3]


class _DWConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b):
        x, ldx = rows(x)
        B, Cc, H, W = x.shape
        w9, ctx.w9f = _dw_taps(w)
        b32 = None if b is None else b.float().contiguous()
        y = _empty(B, Cc, H, W, x)
        _check(lib().turtle_train_dw3x3_fwd(_p(x), ldx, _p(w9), _p(b32), _p(y), Cc, B, Cc, H, W, 0, _dt(x), _stream(x)), "dw_fwd")
        ctx.save_for_backward(x, w9)
        ctx.has_b, ctx.ldx = b is not None, ldx
        ctx.acc_w, ctx.acc_b = _acc_use(ctx, 1, w), _acc_use(ctx, 2, b)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w9 = ctx.saved_tensors
        dy, lddy = rows(dy.to(x.dtype))
        B, Cc, H, W = x.shape
        dx = _empty(B, Cc, H, W, x)
        st = _stream(x)
        # dx = depthwise of dy with the taps flipped (correlation transposed); the flipped table is
        # passed as a plain forward so the row-sweeping kernel takes it
        w9f = ctx.w9f
        _check(lib().turtle_train_dw3x3_fwd(_p(dy), lddy, _p(w9f), None, _p(dx), Cc, B, Cc, H, W, 0, _dt(x), st), "dw_dgrad")
        aw, ab = ctx.acc_w, ctx.acc_b
        dw9, db = _acc_dst(aw, 9 * Cc), (_acc_dst(ab, Cc) if ctx.has_b else None)
        nz = (9 * Cc if dw9 is None else 0) + (Cc if ctx.has_b and db is None else 0)
        if nz:
            z = torch.zeros(nz, dtype=torch.float32, device=x.device)                    # one fill for both
            dw9 = z[:9 * Cc] if dw9 is None else dw9
            db = z[nz - Cc:] if ctx.has_b and db is None else db
        _check(lib().turtle_train_dw3x3_wgrad(_p(x), ctx.ldx, _p(dy), lddy, _p(dw9), _p(db), B, Cc, H, W, _dt(x), st), "dw_wgrad")
        tap_major = lambda f: f.view(9, Cc).t().reshape(Cc, 1, 3, 3)     # the kernel's [9][C] -> [C, 1, 3, 3]
        dw = _acc_done(aw, tap_major) if aw else tap_major(dw9)
        db = _acc_done(ab, lambda f: f) if ab else db
        return dx, dw, db


class _Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        x, ldx = rows(x)
        B, C2, H, W = x.shape
        h = C2 // 2
        y = _empty(B, h, H, W, x)
        _check(lib().turtle_train_gate_fwd(_p(x), ldx, _p(y), h, B * H * W, h, _dt(x), _stream(x)), "gate_fwd")
        ctx.save_for_backward(x)
        ctx.ldx = ldx
        return y

    @staticmethod
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        dy, lddy = rows(dy.to(x.dtype))
        B, C2, H, W = x.shape
        dx = _empty(B, C2, H, W, x)
        _check(lib().turtle_train_gate_bwd(_p(x), ctx.ldx, _p(dy), lddy, _p(dx), C2, B * H * W, C2 // 2, _dt(x), _stream(x)),
               "gate_bwd")
        return dx


class _Gelu(torch.autograd.Function):
    """y = gelu(x) (exact erf form) on NHWC rows; backward dx = dy gelu'(x) (turtle_train_gelu_*)."""

    @staticmethod
    def forward(ctx, x):
        x, ldx = rows(x)
        B, Cc, H, W = x.shape
        y = _empty(B, Cc, H, W, x)
        _check(lib().turtle_train_gelu_fwd(_p(x), ldx, _p(y), Cc, B * H * W, Cc, _dt(x), _stream(x)), "gelu_fwd")
        ctx.save_for_backward(x)
        ctx.ldx = ldx
        return y

    @staticmethod
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        dy, lddy = rows(dy.to(x.dtype))
        B, Cc, H, W = x.shape
        dx = _empty(B, Cc, H, W, x)
        _check(lib().turtle_train_gelu_bwd(_p(x), ctx.ldx, _p(dy), lddy, _p(dx), Cc, B * H * W, Cc, _dt(x), _stream(x)), "gelu_bwd")
        return dx


def window_grid(H: int, W: int, ws: int):
    """Token grid of nn.Conv2d(kernel ws, stride ws, padding 1): ((H + 2 - ws) // ws + 1, ...)."""
    return (H + 2 - ws) // ws + 1, (W + 2 - ws) // ws + 1


class _WinConv(torch.autograd.Function):
    """SAB window convolution nn.Conv2d(C, C, ws, stride=ws, padding=1, groups=C) (k2_dwconv /
    q2_dwconv, turtle_t1_arch.py:306-308) on NHWC rows, forward and both gradients on the HIP
    kernels (turtle_train_window_*); the bias gradient is a column sum of dy."""

    @staticmethod
    def forward(ctx, x, w, b, ws: int):
        x, ldx = rows(x)
        B, Cc, H, W = x.shape
        th, tw = window_grid(H, W, ws)
        wt = w.detach().float().reshape(Cc, ws * ws).t().contiguous()          # [ws*ws][C]
        b32 = None if b is None else b.detach().float().contiguous()
        y = _empty(B, Cc, th, tw, x)
        _check(lib().turtle_train_window_fwd(_p(x), ldx, _p(wt), _p(b32), _p(y), Cc, B, Cc, H, W, ws, th, tw, _dt(x), _stream(x)),
               "window_fwd")
        ctx.save_for_backward(x, wt)
        ctx.ldx, ctx.ws, ctx.has_b, ctx.w_dt = ldx, ws, b is not None, w.dtype
        ctx.acc_w, ctx.acc_b = _acc_use(ctx, 1, w), _acc_use(ctx, 2, b)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, wt = ctx.saved_tensors
        B, Cc, H, W = x.shape
        ws = ctx.ws
        th, tw = window_grid(H, W, ws)
        dy, lddy = rows(dy.to(x.dtype))
        st = _stream(x)
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = _empty(B, Cc, H, W, x)
            _check(lib().turtle_train_window_dgrad(_p(dy), lddy, _p(wt), _p(dx), Cc, B, Cc, H, W, ws, th, tw, _dt(x), st),
                   "window_dgrad")
        if ctx.needs_input_grad[1]:
            aw = ctx.acc_w
            dwt = _acc_dst(aw, ws * ws * Cc)
            dwt = torch.zeros(ws * ws * Cc, dtype=torch.float32, device=x.device) if dwt is None else dwt
            _check(lib().turtle_train_window_wgrad(_p(x), ctx.ldx, _p(dy), lddy, _p(dwt), B, Cc, H, W, ws, th, tw, _dt(x), st),
                   "window_wgrad")
            tap_major = lambda f: f.view(ws * ws, Cc).t().reshape(Cc, 1, ws, ws).to(ctx.w_dt)
            dw = _acc_done(aw, tap_major) if aw else tap_major(dwt)
        if ctx.has_b and ctx.needs_input_grad[2]:
            db = _acc_dst(ctx.acc_b, Cc)
            db = torch.zeros(Cc, dtype=torch.float32, device=x.device) if db is None else db
            _check(lib().turtle_train_colsum(_p(dy), lddy, _p(db), B * th * tw, Cc, _dt(dy), st), "colsum")
            db = _acc_done(ctx.acc_b, lambda f: f) if ctx.acc_b else db
        return dx, dw, db, None


class _Conv3x3(torch.autograd.Function):
    """Dense 3x3 convolution, stride 1, padding 1 (Down / Upsample body[0], turtle_t1_arch.py:136-154) on
    NHWC rows: forward and input gradient on the inference implicit-GEMM family (turtle_train_conv3x3;
    the input gradient with the rotated, transposed weights), weight gradient by the tap-shifted
    reduction GEMM (turtle_train_conv3x3_wgrad). No NCHW copies, no MIOpen."""

    @staticmethod
    def forward(ctx, x, w, b):
        gdt = _gemm_dt(x)
        out_dt = x.dtype
        xg, ldx = rows(x.to(gdt))
        B, Cin, H, W = xg.shape
        N = w.shape[0]
        wf = w.detach().permute(0, 2, 3, 1).reshape(N, 9 * Cin).to(gdt).contiguous()     # [N][tap][Cin]
        b32 = None if b is None else b.detach().float().contiguous()
        y = _empty(B, N, H, W, xg)
        _check(lib().turtle_train_conv3x3(_p(xg), ldx, _p(wf), _p(b32), _p(y), N, B, H, W, Cin, N, _dt(xg), _stream(xg)), "conv3x3")
        ctx.save_for_backward(xg, w)
        ctx.ldx, ctx.has_b, ctx.in_dt = ldx, b is not None, x.dtype
        return y.to(out_dt)

    @staticmethod
    def backward(ctx, dy):
        xg, w = ctx.saved_tensors
        B, Cin, H, W = xg.shape
        N = w.shape[0]
        P = B * H * W
        dy, lddy = rows(dy.to(xg.dtype))
        st = _stream(xg)
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            wr = w.detach().flip(2, 3).permute(1, 2, 3, 0).reshape(Cin, 9 * N).to(xg.dtype).contiguous()   # [Cin][tap][N]
            dx = _empty(B, Cin, H, W, xg)
            _check(lib().turtle_train_conv3x3(_p(dy), lddy, _p(wr), None, _p(dx), Cin, B, H, W, N, Cin, _dt(xg), st), "conv3x3_dgrad")
            dx = dx.to(ctx.in_dt)
        if ctx.needs_input_grad[1]:
            L = lib()
            nws = L.turtle_train_conv3x3_wgrad_workspace(P, N, Cin)
            ws = torch.empty(max(int(nws), 16), dtype=torch.uint8, device=xg.device)
            dw9 = torch.empty(9, N, Cin, dtype=torch.float32, device=xg.device)
            _check(L.turtle_train_conv3x3_wgrad(_p(dy), lddy, _p(xg), ctx.ldx, _p(dw9), B, H, W, N, Cin, _dt(xg), _p(ws), ws.numel(), st),
                   "conv3x3_wgrad")
            dw = dw9.permute(1, 2, 0).reshape(N, Cin, 3, 3).to(w.dtype)
        if ctx.has_b and ctx.needs_input_grad[2]:
            db = torch.zeros(N, dtype=torch.float32, device=xg.device)
            _check(lib().turtle_train_colsum(_p(dy), lddy, _p(db), P, N, _dt(dy), st), "colsum")
        return dx, dw, db


class _NormCols(torch.autograd.Function):
    """Per-image, per-channel L2 normalisation over the pixels on NHWC rows: F.normalize(t, dim=-1) of the
    [b, heads, ch, HW] view of q / k (turtle_t1_arch.py:236-237, 649-651), y = x / max(|x|, 1e-12), in
    x's dtype. Forward: column sums of squares + one scaling pass; backward dx = (dy - y sum(dy y)) / |x|
    (turtle_train_colsumsq / colscale / coldot / l2n_bwd) - no fp32 copies, no NCHW re-layout."""

    @staticmethod
    def forward(ctx, x):
        x, ldx = rows(x)
        B, Cc, H, W = x.shape
        HW, P = H * W, B * H * W
        st = _stream(x)
        ss = torch.zeros(B, Cc, dtype=torch.float32, device=x.device)
        _check(lib().turtle_train_colsumsq(_p(x), ldx, _p(ss), P, Cc, HW, _dt(x), st), "colsumsq")
        n = ss.sqrt()
        inv = 1.0 / n.clamp_min(L2N_EPS)
        y = _empty(B, Cc, H, W, x)
        _check(lib().turtle_train_colscale(_p(x), ldx, _p(inv), _p(y), Cc, P, Cc, HW, _dt(x), st), "colscale")
        ctx.save_for_backward(y, inv, (n > L2N_EPS).float())
        return y

    @staticmethod
    def backward(ctx, dy):
        y, inv, live = ctx.saved_tensors
        B, Cc, H, W = y.shape
        HW, P = H * W, B * H * W
        st = _stream(y)
        dy, lddy = rows(dy.to(y.dtype))
        d = torch.zeros(B, Cc, dtype=torch.float32, device=y.device)
        _check(lib().turtle_train_coldot(_p(dy), lddy, _p(y), Cc, _p(d), P, Cc, HW, _dt(y), st), "coldot")
        d = (d * live).contiguous()
        dx = _empty(B, Cc, H, W, y)
        _check(lib().turtle_train_l2n_bwd(_p(dy), lddy, _p(y), Cc, _p(d), _p(inv), _p(dx), Cc, P, Cc, HW, _dt(y), st), "l2n_bwd")
        return dx


L2N_EPS = 1e-12


def _gemm_rows(x2d, w3d, bias=None):
    """y [P, N] = x2d [P, K] w3d[img]^T with one weight set per run of P / nimg rows (turtle_train_gemm)."""
    P, K = x2d.shape
    nimg, N, _ = w3d.shape
    y = torch.empty(P, N, dtype=x2d.dtype, device=x2d.device)
    _check(lib().turtle_train_gemm(_p(x2d), K, _p(w3d), N * K, P // nimg, _p(bias), None, 0, _p(y), N, P, K, N, _dt(x2d), _stream(x2d)),
           "gemm")
    return y


def _rgemm_rows(a2d, b2d, nimg):
    """c [nimg, N, K] fp32 = sum over each image's rows of a2d[p]^T b2d[p] (turtle_train_rgemm)."""
    P, N = a2d.shape
    K = b2d.shape[1]
    return _rgemm(a2d, N, b2d, K, P, N, K, P // nimg)


class _SabAttn(torch.autograd.Function):
    """The StateAlignBlock attention core (turtle_t1_arch.py:585-599) on the HIP kernels: s = q k^T per
    frame (one GEMM with a weight set per (image, frame)), the top-5 + ball clipped softmax
    (turtle_train_sab_softmax_*), o = a v (one GEMM with the per-frame values, held transposed [D, n]:
    the dilated value tokens are written that way, so no operand is transposed in the forward);
    backward: da = dO v^T and ds -> dq = ds k as GEMMs, dk = ds^T q and dv^T = dO^T a as reduction GEMMs
    over the query rows. q [b, n, g], K [b, t, n, g], VT [b, t, D, n] (activation dtype), temperature
    [1, 1, 1] -> o [b, t, n, D]."""

    @staticmethod
    def forward(ctx, q, K, VT, temp, tw: int, radius: int):
        b, t, n, g = K.shape
        D = VT.shape[2]
        dt = K.dtype
        q_rep = q.to(dt)[:, None].expand(b, t, n, g).reshape(b * t * n, g).contiguous()
        Kc = K.contiguous()
        VTc = VT.contiguous()
        S = _gemm_rows(q_rep, Kc.view(b * t, n, g))                          # [btn, n] raw scores
        sc = S.float() * temp.reshape(()).float()
        a = torch.empty(b * t * n, n, dtype=dt, device=K.device)
        a32 = torch.empty(b * t * n, n, dtype=torch.float32, device=K.device)
        m = torch.empty(b * t * n, n, dtype=torch.uint8, device=K.device)
        _check(lib().turtle_train_sab_softmax_fwd(_p(sc), b * t * n, n, tw, radius, _p(a), _p(a32), _p(m), _dt(a), _stream(K)),
               "sab_softmax_fwd")
        o = _gemm_rows(a, VTc.view(b * t, D, n))                             # [btn, D]
        ctx.save_for_backward(q_rep, Kc, VTc, S, a, a32, m, temp)
        ctx.dims, ctx.q_dt = (b, t, n, g, D), q.dtype
        return o.view(b, t, n, D)

    @staticmethod
    def backward(ctx, dO):
        q_rep, Kc, VTc, S, a, a32, m, temp = ctx.saved_tensors
        b, t, n, g, D = ctx.dims
        dt = Kc.dtype
        R = b * t * n
        dO = dO.to(dt).reshape(R, D).contiguous()
        V = VTc.view(b * t, D, n).transpose(1, 2).contiguous()              # [bt, n, D]
        da = _gemm_rows(dO, V)                                               # [R, n]
        ds = torch.empty(R, n, dtype=torch.float32, device=dO.device)
        _check(lib().turtle_train_sab_softmax_bwd(_p(da), _p(a32), _p(m), R, n, _p(ds), _dt(da), _stream(dO)), "sab_softmax_bwd")
        tau = temp.reshape(()).float()
        dtemp = (ds * S.float()).sum().reshape(temp.shape).to(temp.dtype)
        dS = (ds * tau).to(dt)
        KT = Kc.view(b * t, n, g).transpose(1, 2).contiguous()              # [bt, g, n]
        dq = _gemm_rows(dS, KT).view(b, t, n, g).float().sum(1).to(ctx.q_dt)
        dK = _rgemm_rows(dS, q_rep, b * t).view(b, t, n, g).to(dt)           # sum_i ds[i][j] q[i]
        dVT = _rgemm_rows(dO, a, b * t).view(b, t, D, n).to(dt)               # sum_i dO[i][d] a[i][j]
        return dq, dK, dVT, dtemp, None, None


class _SabSoftmax(torch.autograd.Function):
    """StateAlignBlock scores -> attention (turtle_t1_arch.py:585-599): top-5 mask + L1 ball (radius on
    the th x tw token grid), s * (top + ball), clipped softmax (115-132), renormalised - one HIP kernel
    each way (turtle_train_sab_softmax_*) in place of topk / scatter / masks / softmax / sum / div and their
    backward. s fp32 [..., n] (last dim keys); a in ``out_dtype``."""

    @staticmethod
    def forward(ctx, s, tw: int, radius: int, out_dtype):
        s = s.float().contiguous()
        n = s.shape[-1]
        R = s.numel() // n
        a = torch.empty(s.shape, dtype=out_dtype, device=s.device)
        a32 = torch.empty(s.shape, dtype=torch.float32, device=s.device)
        m = torch.empty(s.shape, dtype=torch.uint8, device=s.device)
        _check(lib().turtle_train_sab_softmax_fwd(_p(s), R, n, tw, radius, _p(a), _p(a32), _p(m), _dt(a), _stream(s)), "sab_softmax_fwd")
        ctx.save_for_backward(a32, m)
        return a

    @staticmethod
    def backward(ctx, da):
        a32, m = ctx.saved_tensors
        n = a32.shape[-1]
        R = a32.numel() // n
        da = da.contiguous()
        if da.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            da = da.float()
        ds = torch.empty(a32.shape, dtype=torch.float32, device=a32.device)
        _check(lib().turtle_train_sab_softmax_bwd(_p(da), _p(a32), _p(m), R, n, _p(ds), _dt(da), _stream(da)), "sab_softmax_bwd")
        return ds, None, None, None


class _CrossGram(torch.autograd.Function):
    """G[b] [cq, cK] fp32 = sum over image b's pixels of q[p]^T K[p] (NHWC rows): the FHR / CHM attention
    scores q_hat [k_cache ; k_hat]^T of every head pair (turtle_t1_arch.py:238-241, 649-660; the caller
    takes the per-head blocks). Reduction GEMM forward; backward dq = K dG^T, dK = q dG as GEMMs with one
    weight set per image."""

    @staticmethod
    def forward(ctx, q, K):
        gdt = _gemm_dt(q)
        in_q, in_k = q.dtype, K.dtype
        q, ldq = rows(q.to(gdt))
        K, ldk = rows(K.to(gdt))
        B, cq, H, W = q.shape
        cK = K.shape[1]
        P, HW = B * H * W, H * W
        G = _rgemm(q, ldq, K, ldk, P, cq, cK, HW)                       # [B, cq, cK]
        ctx.save_for_backward(q, K)
        ctx.ldq, ctx.ldk, ctx.in_q, ctx.in_k = ldq, ldk, in_q, in_k
        return G

    @staticmethod
    def backward(ctx, dG):
        q, K = ctx.saved_tensors
        B, cq, H, W = q.shape
        cK = K.shape[1]
        P, HW = B * H * W, H * W
        dG = dG.float()
        dq = dk = None
        if ctx.needs_input_grad[0]:
            dq = _gemm_into(K, ctx.ldk, dG.to(K.dtype).contiguous(), HW, None, P, cK, cq).to(ctx.in_q)
        if ctx.needs_input_grad[1]:
            dk = _gemm_into(q, ctx.ldq, dG.transpose(1, 2).to(q.dtype).contiguous(), HW, None, P, cq, cK).to(ctx.in_k)
        return dq, dk


def _rgemm(a, lda, b, ldb, P, N, K, img_px, acc_into=None):
    """c [nimg, N, K] fp32 = sum over each image's pixels (all pixels when img_px = 0) of
    a[p][n] b[p][k]; a, b are pixel-row tensors (or head slices of one). ``acc_into``: a contiguous
    fp32 tensor of N K elements (img_px = 0) the sum is added to instead (returned)."""
    L = lib()
    nimg = P // img_px if img_px else 1
    if acc_into is not None:
        if img_px or acc_into.numel() != N * K or acc_into.dtype != torch.float32 or not acc_into.is_contiguous():
            raise ValueError("rgemm accumulation target must be a contiguous fp32 [N, K] tensor")
        c = acc_into
    else:
        c = torch.empty(nimg, N, K, dtype=torch.float32, device=a.device)
    nws = L.turtle_train_rgemm_workspace(P, N, K, img_px)
    ws = torch.empty(max(int(nws), 16), dtype=torch.uint8, device=a.device)
    _check(L.turtle_train_rgemm(_p(a), lda, _p(b), ldb, _p(c), P, N, K, img_px, int(acc_into is not None), _dt(a), _p(ws),
                                ws.numel(), _stream(a)), "rgemm")
    return c


def _gemm_into(x, ldx, w, img_px, bias, P, K, N, out=None, res=None):
    """y = x w^T (+ bias) (+ res): x rows [P][ldx] of a [B, K, H, W] tensor; w [N, K] or [nimg, N, K] in
    x's dtype; res (x's dtype, [B, N, H, W]) added in the epilogue; returns a channels_last
    [B, N, H, W] tensor, or writes ``out`` (NHWC rows with their own pixel stride: a channel slice of
    a wider tensor) and returns it."""
    B, _, H, W = x.shape
    if out is None:
        y, ldy = _empty(B, N, H, W, x), N
    else:
        y, ldy = rows(out)
        if y is not out:
            raise ValueError("gemm output slice is not NHWC rows")
    wstride = (N * K) if w.dim() == 3 else 0
    ldr = 0
    if res is not None:
        res, ldr = rows(res)
        if res.dtype != x.dtype or tuple(res.shape) != (B, N, H, W):
            raise ValueError("gemm residual must match the output's shape and dtype")
    _check(lib().turtle_train_gemm(_p(x), ldx, _p(w), wstride, img_px if wstride else 0, _p(bias), _p(res), ldr, _p(y), ldy, P,
                                   K, N, _dt(x), _stream(x)), "gemm")
    return y


class GradSink:
    """One input-gradient buffer for the channel slices of a channels-last tensor (the qkv map of a
    channel attention, split into [q | k] and v: turtle_t1_arch.py:688-689). The HIP ops consuming
    the slices write their input gradients straight into their channel range of the buffer (the
    GEMM's output pixel stride is the full width), and the split's backward returns the buffer when
    every slice gradient is that range, untouched - no concatenation pass. A slice claimed twice in
    one backward (two consumers), or a gradient autograd had to accumulate, falls back to the
    split's concatenation."""

    def __init__(self, x):
        self.shape, self.dtype, self.device = tuple(x.shape), x.dtype, x.device
        self.buf, self.claimed = None, set()

    def claim(self, off: int, n: int, dtype):
        if dtype != self.dtype or off in self.claimed:
            return None
        if self.buf is None:
            self.buf = torch.empty(self.shape, dtype=self.dtype, device=self.device, memory_format=CL)
        self.claimed.add(off)
        return self.buf.narrow(1, off, n)

    def take(self, grads, sizes):
        """The buffer if ``grads`` are exactly its claimed slices (then the sink resets), else None."""
        buf, off = self.buf, 0
        self.buf, self.claimed = None, set()
        if buf is None:
            return None
        for g, n in zip(grads, sizes):
            ref = buf.narrow(1, off, n)
            if g is None or g.data_ptr() != ref.data_ptr() or g.shape != ref.shape or g.stride() != ref.stride():
                return None
            off += n
        return buf


def _sink_out(sink, n, dtype):
    return None if sink is None else sink[0].claim(sink[1], n, dtype)


class _WCast:
    """A shared weight in the GEMM dtype (`wg`) and its transpose for the input gradient (`wt`,
    built on first use). One entry per leaf parameter (or a view of one: the [N, K] reshape of a
    conv weight), reused while the parameter's version and storage are unchanged: the 5 frames of
    a clip (and the forward / backward of each) stop re-casting and re-transposing the same weight;
    the optimizer's in-place update bumps the version (a view shares its base's counter), a
    ``p.data = t`` rebinding changes the data pointer. Writes through ``p.data.copy_()`` bump
    neither: call ``clear_weight_cache()`` after such a write (training ABI)."""
    __slots__ = ("version", "ptr", "dtype", "wg", "wt")

    def __init__(self, w, gdt):
        self.version, self.ptr, self.dtype = w._version, w.data_ptr(), gdt
        self.wg = w.detach().to(gdt).contiguous()
        self.wt = None

    def transposed(self):
        if self.wt is None:
            self.wt = self.wg.transpose(-1, -2).contiguous()
        return self.wt


# keyed weakly on the base Parameter (identity, not tensor equality): an entry - and the device
# memory of its casts - goes with its parameter, so `del net` frees everything
_WCACHE = WeakIdKeyDictionary()


def clear_weight_cache():
    """Drop every cached weight cast (after parameter writes that bypass the version counter)."""
    _WCACHE.clear()
    _DWCACHE.clear()


def _weight_cast(w, gdt):
    """(wg, entry): the cached cast of a 2-D weight that is a leaf parameter or a view of one, or a
    fresh cast (entry None) for computed weights (scaled, per-image)."""
    base = w if w.is_leaf else w._base
    if w.dim() != 2 or not isinstance(base, torch.nn.Parameter):
        return w.to(gdt).contiguous(), None
    per = _WCACHE.get(base)
    if per is None:
        per = _WCACHE[base] = {}
    key = (tuple(w.shape), w.stride(), w.storage_offset())
    e = per.get(key)
    if e is None or e.version != w._version or e.ptr != w.data_ptr() or e.dtype != gdt or e.wg.device != w.device:
        e = per[key] = _WCast(w, gdt)
    return e.wg, e


class _Conv1x1(torch.autograd.Function):
    """y = x W^T + b (+ res) on NHWC rows; W [N, K] (shared) or [B, N, K] (one set per image). ``res``
    (the block's residual stream in the output dtype, turtle_t1_arch.py:808-809) is added in the
    GEMM epilogue; its gradient is dy itself."""

    @staticmethod
    def forward(ctx, x, w, b, sink=None, res=None):
        gdt = _gemm_dt(x)
        out_dt = x.dtype
        ctx.sink = sink
        xg, ldx = rows(x.to(gdt))
        B, K, H, W = xg.shape
        N = w.shape[-2]
        wg, ctx.wcache = _weight_cast(w, gdt)
        b32 = None if b is None else b.float().contiguous()
        if res is not None and (res.dtype != gdt or out_dt != gdt):
            raise ValueError("conv1x1 residual fusion needs the residual in the GEMM dtype")
        y = _gemm_into(xg, ldx, wg, H * W, b32, B * H * W, K, N, res=res)
        ctx.save_for_backward(xg, wg)
        ctx.ldx, ctx.has_b, ctx.in_dt, ctx.w_dt = ldx, b is not None, x.dtype, w.dtype
        ctx.acc_w, ctx.acc_b, ctx.w_shape = (_acc_use(ctx, 1, w) if w.dim() == 2 else None), _acc_use(ctx, 2, b), w.shape
        return y.to(out_dt)

    @staticmethod
    def backward(ctx, dy):
        xg, wg = ctx.saved_tensors
        B, K, H, W = xg.shape
        N = wg.shape[-2]
        P, HW = B * H * W, H * W
        dres = dy if len(ctx.needs_input_grad) > 4 and ctx.needs_input_grad[4] else None
        dy, lddy = rows(dy.to(xg.dtype))
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            wt = ctx.wcache.transposed() if ctx.wcache is not None else wg.transpose(-1, -2).contiguous()   # [.., K, N]
            dst = _sink_out(ctx.sink, K, ctx.in_dt) if xg.dtype == ctx.in_dt else None
            dx = _gemm_into(dy, lddy, wt, HW, None, P, N, K, out=dst).to(ctx.in_dt)
        if ctx.needs_input_grad[1]:
            if ctx.acc_w is not None:                      # in-place accumulation over the step's uses
                _rgemm(dy, lddy, xg, ctx.ldx, P, N, K, 0, acc_into=_acc_dst(ctx.acc_w, N * K))
                shape = ctx.w_shape
                dw = _acc_done(ctx.acc_w, lambda f: f.view(shape))
            elif wg.dim() == 3:
                dw = _rgemm(dy, lddy, xg, ctx.ldx, P, N, K, HW).to(ctx.w_dt)  # [B, N, K]
            else:
                dw = _rgemm(dy, lddy, xg, ctx.ldx, P, N, K, 0)[0].to(ctx.w_dt)
        if ctx.has_b and ctx.needs_input_grad[2]:
            db = _acc_dst(ctx.acc_b, N)
            db = torch.zeros(N, dtype=torch.float32, device=dy.device) if db is None else db
            _check(lib().turtle_train_colsum(_p(dy), lddy, _p(db), P, N, _dt(dy), _stream(dy)), "colsum")
            db = _acc_done(ctx.acc_b, lambda f: f) if ctx.acc_b else db
        return dx, dw, db, None, dres


class _Gram(torch.autograd.Function):
    """G[b, h] = sum over HW of q[b, head h channels] k[b, head h channels]^T (fp32)."""

    @staticmethod
    def forward(ctx, q, k, heads: int):
        gdt = _gemm_dt(q)
        q, ldq = rows(q.to(gdt))
        k, ldk = rows(k.to(gdt))
        B, Cc, H, W = q.shape
        ch = Cc // heads
        P, HW = B * H * W, H * W
        G = torch.empty(B, heads, ch, ch, dtype=torch.float32, device=q.device)
        for h in range(heads):
            G[:, h] = _rgemm(q[:, h * ch:(h + 1) * ch], ldq, k[:, h * ch:(h + 1) * ch], ldk, P, ch, ch, HW)
        ctx.save_for_backward(q, k)
        ctx.heads, ctx.ldq, ctx.ldk = heads, ldq, ldk
        return G

    @staticmethod
    def backward(ctx, dG):
        q, k = ctx.saved_tensors
        B, Cc, H, W = q.shape
        heads, ch = ctx.heads, Cc // ctx.heads
        HW, P = H * W, B * H * W
        # block-diagonal per-image weights D[b][i][j] = dG[b, h, i', j'] inside head h:
        # dq = k D^T, dk = q D (GEMMs over the pixels with one weight set per image)
        D = torch.zeros(B, Cc, Cc, dtype=torch.float32, device=q.device)
        for h in range(heads):
            D[:, h * ch:(h + 1) * ch, h * ch:(h + 1) * ch] = dG[:, h]
        dq = _gemm_into(k, ctx.ldk, D.to(k.dtype).contiguous(), HW, None, P, Cc, Cc)
        dk = _gemm_into(q, ctx.ldq, D.transpose(1, 2).to(q.dtype).contiguous(), HW, None, P, Cc, Cc)
        return dq, dk, None


class _NormGram(torch.autograd.Function):
    """Gn[b, h] = normalize(q_h) normalize(k_h)^T over HW (F.normalize, eps 1e-12:
    turtle_t1_arch.py:690-697) from the channel-adjacent [q | k] rows of qkv. Forward: the Gram by
    the reduction GEMM, the L2 norms by one column sum-of-squares pass over [q | k]. Backward: one
    GEMM over the same [q | k] rows with per-image weights [[diag(a_q), D], [D^T, diag(a_k)]] (D =
    dGn / (|q| |k|^T) block-diagonal per head, a = the norms' gradient / |x|), so neither the fp32
    copies of q and k nor the norm ops' elementwise passes of the ATen formulation exist."""

    @staticmethod
    def forward(ctx, qk, heads: int, sink=None):
        gdt = _gemm_dt(qk)
        in_dt = qk.dtype
        ctx.sink = sink
        qk, ld = rows(qk.to(gdt))
        B, C2, H, W = qk.shape
        c = C2 // 2
        ch = c // heads
        P, HW = B * H * W, H * W
        if heads == 1:
            G = _rgemm(qk[:, :c], ld, qk[:, c:], ld, P, c, c, HW).view(B, 1, c, c)
        else:
            # one reduction GEMM over all c x c channel pairs, then the heads' diagonal blocks: the
            # GEMM is bound by reading q and k (read once either way), and one launch pair replaces
            # `heads` GEMM + reduce + block-copy triples
            Gf = _rgemm(qk[:, :c], ld, qk[:, c:], ld, P, c, c, HW)                  # [B, c, c]
            G = Gf.view(B, heads, ch, heads, ch).diagonal(dim1=1, dim2=3).permute(0, 3, 1, 2).contiguous()
        ss = torch.zeros(B, C2, dtype=torch.float32, device=qk.device)
        _check(lib().turtle_train_colsumsq(_p(qk), ld, _p(ss), P, C2, HW, _dt(qk), _stream(qk)), "colsumsq")
        n = ss.sqrt()
        nc = n.clamp_min(1e-12)
        nq, nk = nc[:, :c].view(B, heads, ch), nc[:, c:].view(B, heads, ch)
        Gn = G / (nq[..., :, None] * nk[..., None, :])
        ctx.save_for_backward(qk, Gn, nq, nk, n)
        ctx.heads, ctx.ld, ctx.in_dt = heads, ld, in_dt
        return Gn

    @staticmethod
    def backward(ctx, dGn):
        qk, Gn, nq, nk, n = ctx.saved_tensors
        B, C2, H, W = qk.shape
        c, heads = C2 // 2, ctx.heads
        ch = c // heads
        P, HW = B * H * W, H * W
        dGn = dGn.float()
        D = dGn / (nq[..., :, None] * nk[..., None, :])                  # dL/dG
        t = dGn * Gn
        live = (n > 1e-12).float()
        aq = (-t.sum(-1) / (nq * nq)).reshape(B, c) * live[:, :c]          # dL/d|q_i| / |q_i|
        ak = (-t.sum(-2) / (nk * nk)).reshape(B, c) * live[:, c:]
        # Wd [B, 2c, 2c] = [[diag(aq), D], [D^T, diag(ak)]] built densely in the GEMM dtype by one
        # kernel (no fp32 zero-fill, block scatter and cast passes)
        Wd = torch.empty(B, C2, C2, dtype=qk.dtype, device=qk.device)
        D, aq, ak = D.contiguous(), aq.contiguous(), ak.contiguous()
        _check(lib().turtle_train_gram_wd(_p(D), _p(aq), _p(ak), _p(Wd), B, c, heads, _dt(qk), _stream(qk)), "gram_wd")
        dst = _sink_out(ctx.sink, C2, ctx.in_dt) if qk.dtype == ctx.in_dt else None
        dqk = _gemm_into(qk, ctx.ld, Wd, HW, None, P, C2, C2, out=dst)
        return dqk.to(ctx.in_dt), None, None


class _AttnWeff(torch.autograd.Function):
    """The channel-attention / FHR finalize (turtle_t1_arch.py:697-702, 240-244): A = softmax(G * t) per
    head (G [b, heads, ch, L] fp32, t = the temperature [heads, 1, 1]) and the per-image weight set
    W_eff[b, o, (h, k)] = sum_i wp[o, h, i] A[b, h, i, k] (wp = project_out's weight as [c, heads, ch]) that
    the conv1x1 applies to v (A v followed by project_out as one GEMM), in fp32 with a hand-written
    backward: one op chain instead of autograd's softmax / einsum / cast / view nodes (~20 small
    launches per site and step)."""

    @staticmethod
    def forward(ctx, G, temp, wp, out_dtype):
        Gf = G.float()
        t = temp.float()
        a = torch.softmax(Gf * t, dim=-1)
        weff = torch.einsum("ohi,bhik->bohk", wp.float(), a)
        ctx.save_for_backward(Gf, t, wp, a)
        ctx.g_dt, ctx.t_dt, ctx.w_dt = G.dtype, temp.dtype, wp.dtype
        b, h, ch, L = G.shape
        return weff.reshape(b, wp.shape[0], h * L).to(out_dtype)

    @staticmethod
    def backward(ctx, dweff):
        Gf, t, wp, a = ctx.saved_tensors
        b, h, ch, L = Gf.shape
        dW = dweff.float().view(b, wp.shape[0], h, L)
        dG = dt = dwp = None
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            da = torch.einsum("ohi,bohk->bhik", wp.float(), dW)
            ds = a * (da - (da * a).sum(-1, keepdim=True))                     # softmax backward
            if ctx.needs_input_grad[0]:
                dG = (ds * t).to(ctx.g_dt)
            if ctx.needs_input_grad[1]:
                dt = (ds * Gf).sum(dim=(0, 2, 3)).view(t.shape).to(ctx.t_dt)
        if ctx.needs_input_grad[2]:
            dwp = torch.einsum("bohk,bhik->ohi", dW, a).to(ctx.w_dt)
        return dG, dt, dwp, None


def _act_dtype(x: torch.Tensor) -> torch.dtype:
    if torch.is_autocast_enabled("cuda") and x.dtype == torch.float32:
        return torch.get_autocast_dtype("cuda")
    return x.dtype


def _act(x: torch.Tensor) -> torch.Tensor:
    """Activations enter the kernels in the autocast dtype (bf16 / fp16 under autocast)."""
    if torch.is_autocast_enabled("cuda") and x.dtype == torch.float32:
        return x.to(torch.get_autocast_dtype("cuda"))
    return x


class HipOps:
    """The op set of the training graph, on the HIP kernels (channels-last activations)."""

    channels_last = True
    param_grad_accumulator = ParamGradAccumulator      # Trainer: in-place weight-gradient accumulation
    fused_residual = True                              # layer_norm(residual=True) + conv1x1(res=): train.py _block

    @staticmethod
    def layer_norm(x, w, b, biasfree: bool, residual: bool = False):
        """LayerNorm(x); ``residual``: (LayerNorm(x), x) with x's second gradient (its residual use)
        summed inside the LayerNorm backward."""
        out = _act_dtype(x)                          # an fp32 x under autocast: cast inside the kernel
        return _LayerNorm.apply(x, w, b, biasfree, out, residual)

    @staticmethod
    def dwconv3x3(x, w, b):
        return _DWConv.apply(_act(x), w, b)

    @staticmethod
    def gelu_gate(x):
        return _Gate.apply(_act(x))

    @staticmethod
    def gelu(x):
        return _Gelu.apply(_act(x))

    @staticmethod
    def window_conv(x, w, b, ws: int):
        """nn.Conv2d(C, C, ws, stride=ws, padding=1, groups=C)(x), channels-last in and out."""
        return _WinConv.apply(_act(x), w, b, ws)

    @staticmethod
    def norm_cols(x):
        """x / max(|x|, 1e-12) per image and channel over H x W (F.normalize of the [b, heads, ch, HW] view)."""
        return _NormCols.apply(_act(x))

    @staticmethod
    def cross_gram(q, K):
        """[b, cq, cK] fp32: sum over each image's pixels of q[p]^T K[p] (channels-last q, K)."""
        return _CrossGram.apply(_act(q), _act(K))

    @staticmethod
    def sab_attention(q, K, VT, temp, tw: int, radius: int):
        """StateAlignBlock core: q [b, n, g], K [b, t, n, g], VT [b, t, D, n] -> a v [b, t, n, D] with a the
        top-5 + ball clipped softmax of q k^T * temp (n, g, D multiples of 8)."""
        dt = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else K.dtype
        gdt = _gemm_dt(torch.empty(0, dtype=dt))        # fp16 autocast: the GEMMs take bf16 (as _Conv1x1)
        return _SabAttn.apply(q, K.to(gdt), VT.to(gdt), temp, tw, radius).to(dt)

    @staticmethod
    def sab_softmax(s, tw: int, radius: int):
        """The StateAlignBlock's s * (top5 + ball) clipped softmax (fp32 s [..., n keys])."""
        out = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else torch.float32
        return _SabSoftmax.apply(s, tw, radius, out)

    @staticmethod
    def conv3x3(x, w, b=None):
        """nn.Conv2d(Cin, N, 3, 1, 1)(x) with Cin % 8 == N % 8 == 0, channels-last in and out."""
        return _Conv3x3.apply(_act(x), w, b)

    grad_sink = GradSink

    @staticmethod
    def conv1x1(x, w, b, sink=None, res=None):
        """nn.Conv2d(K, N, 1)(x) (+ res): w [N, K, 1, 1] (or [B, N, K]: one weight set per image).
        ``sink`` (GradSink, channel offset): write the input gradient into that slice of the sink's
        buffer. ``res``: the block's residual stream, res + conv(x) (turtle_t1_arch.py:808-809) - in
        the GEMM's epilogue when it already has the output dtype, else the add as written."""
        xa = _act(x)
        w2 = w.reshape(w.shape[0], w.shape[1]) if w.dim() == 4 else w
        if res is not None and res.dtype == _gemm_dt(xa) == xa.dtype and res.dim() == 4 and \
                tuple(res.shape) == (xa.shape[0], w2.shape[-2], xa.shape[2], xa.shape[3]):
            return _Conv1x1.apply(xa, w2, b, sink, res)
        y = _Conv1x1.apply(xa, w2, b, sink)
        return y if res is None else res + y

    @staticmethod
    def gram(q, k, heads: int):
        return _Gram.apply(_act(q), _act(k), heads)

    @staticmethod
    def attn_weff(G, temp, wp, out_dtype):
        """softmax(G * temp) per head and W_eff = project_out . blockdiag(A) as one op (_AttnWeff)."""
        return _AttnWeff.apply(G, temp, wp, out_dtype)

    @staticmethod
    def norm_gram(qk, heads: int, sink=None):
        """[b, heads, ch, ch] Gram of the L2-normalised (over HW) q and k, the first / second half of
        qk's channels (``sink`` as in conv1x1)."""
        return _NormGram.apply(_act(qk), heads, sink)

    # token attention (turtlevsr_amd/token_ops.py): the same calls with activations in the autocast dtype

    @staticmethod
    def axial_rope(x, pos, axes, base: float = 10000.0):
        from . import token_ops
        return token_ops.axial_rope(_act(x), pos, axes, base)

    @staticmethod
    def qk_norm_rope(q, k, pos, q_weight, k_weight, axes, base: float = 10000.0, eps: float = 1e-6):
        from . import token_ops
        return token_ops.qk_norm_rope(_act(q), _act(k), pos, q_weight, k_weight, axes, base, eps)

    @staticmethod
    def attention(q, k, v, **kw):
        from . import token_ops
        return token_ops.attention(_act(q), _act(k), _act(v), **kw)

    @staticmethod
    def paged_attention(q, k_pages, v_pages, block_table, kv_lens, **kw):
        from . import token_ops
        return token_ops.paged_attention(_act(q).to(k_pages.dtype), k_pages, v_pages, block_table, kv_lens, **kw)
