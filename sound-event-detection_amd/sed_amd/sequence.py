"""Sequence operators between the front-ends and the decoders: what the networks that read this package's features need besides
matrix products, with gradients, and in the form a stream calls frame by frame.

`gated_scan` is the gated linear recurrence along the frames that the Audio-Mamba classifier mixes its patches with
(external/audio_mamba imports it from a native extension that is not in its tree), `causal_conv` the short depthwise
convolution in front of it, `group_norm_act` a group norm with an activation on channels-last feature maps (B, T, F, C) or
sequences (B, T, C).  All take `frames`, the clips' own row counts, as reshape_wav2img does: rows behind a clip's own are never
read, and are zero in every output and gradient.  Arithmetic, states and sums are fp32 whatever the element type (fp32, bf16,
fp16); every output is rounded once.  Derivatives are first ones in reverse mode: a tensor with a forward-mode tangent is refused.  There
is no CPU path.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib as L

_DTYPES = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}
_ACTIVATIONS = {None: L.ACT_NONE, "silu": L.ACT_SILU, "relu": L.ACT_RELU, "gelu": L.ACT_GELU}


# The one-frame forms are called once per frame and layer, so what every call does on the host is kept short: argument structs
# are filled by position, and a check looks at everything at once and finds out what is wrong only if something is.


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """t with a contiguous last axis and rows at most 2^26 elements apart (views of a joint projection are read in place)."""
    if t is None:
        return t
    st = t.stride()
    if (st[-1] == 1 or t.shape[-1] == 1) and (len(st) < 3 or st[1] <= 1 << 26):
        return t
    return t.contiguous()


def _new(t):
    """An output of t's shape and type, contiguous whatever t's strides."""
    return None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)


def _param(t):
    """A parameter as the kernels read it; its gradient comes back in the parameter's own type."""
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.float().contiguous()


def _check_x(what, x, dim):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError(f"{what}: x is on {getattr(x, 'device', type(x))}; the sequence operators run only on a ROCm device (no CPU path)")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what}: x is {x.dtype}; fp32, bf16 and fp16 are supported")
    if x.dim() != dim or x.shape[-1] < 1:
        raise ValueError(f"{what}: x has shape {tuple(x.shape)}; {dim} axes with at least one channel are needed")


def _check(what, name, t, x, shape, dtype=None):
    """t: a tensor of this shape on x's device, of x's type (dtype None), of one type, or of any floating type ('float')."""
    if isinstance(t, torch.Tensor) and t.shape == shape and t.device == x.device and (
            t.is_floating_point() if dtype == "float" else t.dtype is (dtype or x.dtype)):
        return
    if not isinstance(t, torch.Tensor) or t.device != x.device:
        raise RuntimeError(f"{what}: {name} has to be a tensor on {x.device}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}; {tuple(shape)} is needed")
    raise TypeError(f"{what}: {name} is {t.dtype}; {'a floating type' if dtype == 'float' else dtype or x.dtype} is needed")


def _check_frames(what, frames, x):
    if frames is not None and not (isinstance(frames, torch.Tensor) and frames.device == x.device and frames.dtype == torch.int32 and
                                   frames.shape == (x.shape[0],) and frames.is_contiguous()):
        raise TypeError(f"{what}: frames: a contiguous int32 tensor with one entry per clip on x's device")


def _workspace(nbytes, x):
    L.check(nbytes, "workspace")
    return x.new_empty(max(int(nbytes), 16), dtype=torch.uint8)


def _call(fn, args, dev, what):
    stream = torch._C._cuda_getCurrentRawStream(dev.index)
    if torch.cuda.current_device() == dev.index:
        L.check(fn(args, stream), what)
    else:
        with torch.cuda.device(dev):
            L.check(fn(args, stream), what)


def _no_tangent(what, *tensors):
    """A dual tensor of forward-mode differentiation need not require grad; its tangent would get lost without a word."""
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled() and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative")


def _no_grad_only(what, *tensors):
    _no_tangent(what, *tensors)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} updates the state in place and keeps nothing for a gradient: call it under torch.no_grad()")


def _moved_on(state):
    """state was written in place: a gradient that kept it as an input notices (tensors of inference mode have no such count)."""
    torch._C._increment_version((state,))


def _wants_grad(what, *tensors):
    _no_tangent(what, *tensors)
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- gated linear recurrence --------------------------------------------------------------------------------------------


def _scan_args(x, dt, A, B, Cm, D, z, dt_bias, softplus, frames, reverse, state):
    b, n_frames, d = x.shape
    xs, ds, zs, bs, cs = x.stride(), dt.stride(), (0, 0) if z is None else z.stride(), B.stride(), Cm.stride()
    return L.ScanArgs(b, n_frames, d, A.shape[1], B.shape[2], _DTYPES[x.dtype], int(softplus), int(reverse), _ptr(frames),
                      x.data_ptr(), dt.data_ptr(), _ptr(z), B.data_ptr(), Cm.data_ptr(), xs[0], xs[1], ds[0], ds[1], zs[0], zs[1],
                      bs[0], bs[1], bs[2], cs[0], cs[1], cs[2], A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(state))


def _scan_forward(x, dt, A, B, Cm, D, z, dt_bias, softplus, frames, reverse, state, want_last, want_saved):
    b, n_frames, d = x.shape
    n = B.shape[3]
    dev = x.device
    y = _new(x)
    last = x.new_empty((b, d, n), dtype=torch.float32) if want_last else None
    saved = None
    if b == 0 or n_frames == 0:
        if want_last:
            last.zero_() if state is None else last.copy_(state)
        return y, last, saved
    a = _scan_args(x, dt, A, B, Cm, D, z, dt_bias, softplus, frames, reverse, state)
    if want_saved:
        saved = x.new_empty(L.lib.sed_gated_scan_saved_floats(b, n_frames, d, n), dtype=torch.float32)
        a.saved = saved.data_ptr()
    nbytes = L.lib.sed_gated_scan_workspace(a, 0)
    if nbytes:
        ws = _workspace(nbytes, x)
        a.ws, a.ws_bytes = ws.data_ptr(), nbytes
    a.y, a.h_last = y.data_ptr(), _ptr(last)
    _call(L.lib.sed_gated_scan_forward, a, dev, "sed_gated_scan_forward")
    return y, last, saved


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, Cm, D, z, dt_bias, state, softplus, frames, reverse, want_last):
        y, last, saved = _scan_forward(x, dt, A, B, Cm, D, z, dt_bias, softplus, frames, reverse, state, want_last, True)
        ctx.save_for_backward(x, dt, A, B, Cm, D, z, dt_bias, frames, saved)
        # the state in front is part of `saved`: it may move on before the gradient is taken
        ctx.rest = (softplus, reverse, None if state is None else state.shape)
        ctx.set_materialize_grads(False)
        return (y, last) if want_last else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast=None):
        _no_tangent("the gradient of gated_scan", dy, dlast)
        x, dt, A, B, Cm, D, z, dt_bias, frames, saved = ctx.saved_tensors
        softplus, reverse, state_shape = ctx.rest
        b, n_frames, d = x.shape
        dev = x.device
        dx, ddt, dA, dB, dC, dD, dz, dbias = (_new(t) for t in (x, dt, A, B, Cm, D, z, dt_bias))
        dstate = None if state_shape is None else x.new_empty(state_shape, dtype=torch.float32)
        if b == 0 or n_frames == 0:
            for t in (dA, dD, dbias, dstate):
                if t is not None:
                    t.zero_()
            if dstate is not None and dlast is not None:
                dstate.copy_(dlast)
            return dx, ddt, dA, dB, dC, dD, dz, dbias, dstate, None, None, None, None
        dy = torch.zeros((b, n_frames, d), dtype=x.dtype, device=dev) if dy is None else _rows(dy)
        dlast = None if dlast is None else dlast.contiguous()
        a = _scan_args(x, dt, A, B, Cm, D, z, dt_bias, softplus, frames, reverse, None)
        a.saved = saved.data_ptr()
        a.dy, a.dy_b, a.dy_t, a.dh_last = dy.data_ptr(), dy.stride(0), dy.stride(1), _ptr(dlast)
        a.dx, a.ddt, a.dz, a.dB, a.dC = dx.data_ptr(), ddt.data_ptr(), _ptr(dz), dB.data_ptr(), dC.data_ptr()
        a.dA, a.dskip, a.ddt_bias, a.dh0 = dA.data_ptr(), _ptr(dD), _ptr(dbias), _ptr(dstate)
        nbytes = L.lib.sed_gated_scan_workspace(a, 1)
        ws = _workspace(nbytes, x)
        a.ws, a.ws_bytes = ws.data_ptr(), nbytes
        _call(L.lib.sed_gated_scan_backward, a, dev, "sed_gated_scan_backward")
        return dx, ddt, dA, dB, dC, dD, dz, dbias, dstate, None, None, None, None


def _scan_checks(what, x, dt, A, B, Cm, D, z, dt_bias, lead):
    d = x.shape[-1]
    _check(what, "dt", dt, x, x.shape)
    if not torch.is_tensor(A) or A.dim() != 2:
        raise ValueError(f"{what}: A: a (channels, states) tensor")
    n = A.shape[1]
    if not 1 <= n <= 32:
        raise ValueError(f"{what}: {n} states a channel; 1 to 32 are supported")
    _check(what, "A", A, x, (d, n), "float")
    if not torch.is_tensor(B) or B.dim() not in (lead + 1, lead + 2):
        raise ValueError(f"{what}: B: {'(clips, frames, [groups,] states)' if lead == 2 else '(streams, [groups,] states)'}")
    g = B.shape[lead] if B.dim() == lead + 2 else 1
    if g < 1 or d % g:
        raise ValueError(f"{what}: {d} channels do not divide into {g} groups")
    shape = (*x.shape[:lead], g, n) if B.dim() == lead + 2 else (*x.shape[:lead], n)
    _check(what, "B", B, x, shape)
    _check(what, "C", Cm, x, shape)
    if D is not None:
        _check(what, "D", D, x, (d,), "float")
    if z is not None:
        _check(what, "z", z, x, x.shape)
    if dt_bias is not None:
        _check(what, "dt_bias", dt_bias, x, (d,), "float")
    return g, n


def gated_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False, frames=None, reverse=False, state=None, return_state=False):
    """The gated linear recurrence along the frames, with a gradient for every tensor but `frames`:

        delta_t[d] = softplus(dt_t[d] + dt_bias[d])          (softplus=False: dt + dt_bias)
        h_t[d,n]   = exp(delta_t[d] A[d,n]) h_{t-1}[d,n] + delta_t[d] B_t[g,n] x_t[d]
        y_t[d]     = (sum_n C_t[g,n] h_t[d,n] + D[d] x_t[d]) * silu(z_t[d])

    x, dt, z (clips, frames, channels); B, C (clips, frames, states) or (clips, frames, groups, states), channel d reading group
    d // (channels // groups); all of one type (fp32, bf16, fp16) and of any strides.  A (channels, states), 1 to 32 states;
    D, dt_bias (channels,): any floating type, read as fp32.
    frames (clips,) int32 on the device: the clips' own row counts; rows behind them give zero and are not read.
    reverse: from a clip's last own row to its first.  state (clips, channels, states) fp32: h in front of the first row walked.
    Returns y (clips, frames, channels), and with return_state also h behind the last row walked (fp32): passing it on as the
    next call's state continues the sequence."""
    what = "gated_scan"
    _check_x(what, x, 3)
    g, n = _scan_checks(what, x, dt, A, B, C, D, z, dt_bias, 2)
    _check_frames(what, frames, x)
    if state is not None:
        _check(what, "state", state, x, (x.shape[0], x.shape[2], n), torch.float32)
        state = state.contiguous()
    if B.dim() == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    x, dt, z, B, C = (_rows(t) for t in (x, dt, z, B, C))
    A, D, dt_bias = _param(A), _param(D), _param(dt_bias)
    if _wants_grad(what, x, dt, A, B, C, D, z, dt_bias, state):
        return _GatedScan.apply(x, dt, A, B, C, D, z, dt_bias, state, bool(softplus), frames, bool(reverse), bool(return_state))
    y, last, _ = _scan_forward(x, dt, A, B, C, D, z, dt_bias, softplus, frames, reverse, state, return_state, False)
    return (y, last) if return_state else y


def gated_scan_step(state, x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False):
    """One frame of gated_scan for a batch of streams: state (streams, channels, states) fp32, contiguous, is updated in place;
    x, dt, z (streams, channels), B, C (streams, states) or (streams, groups, states).  Returns y (streams, channels).  For
    inference: it has no gradient, and a gradient that kept this state as an input raises afterwards."""
    what = "gated_scan_step"
    _check_x(what, x, 2)
    g, n = _scan_checks(what, x, dt, A, B, C, D, z, dt_bias, 1)
    _check(what, "state", state, x, (x.shape[0], x.shape[1], n), torch.float32)
    if not state.is_contiguous():
        raise ValueError(f"{what}: state is updated in place and has to be contiguous")
    _no_grad_only(what, state, x, dt, A, B, C, D, z, dt_bias)
    y = _new(x)
    if x.shape[0] == 0:
        return y
    x, dt, z, B, C = (_rows(t) for t in (x, dt, z, B, C))
    A, D, dt_bias = _param(A), _param(D), _param(dt_bias)
    bs, cs = B.stride(), C.stride()
    wide = len(bs) == 3
    a = L.ScanArgs(x.shape[0], 1, x.shape[1], n, g, _DTYPES[x.dtype], int(softplus), 0, None, x.data_ptr(), dt.data_ptr(), _ptr(z), B.data_ptr(),
                   C.data_ptr(), x.stride(0), 0, dt.stride(0), 0, 0 if z is None else z.stride(0), 0, bs[0], 0, bs[1] if wide else 0, cs[0], 0,
                   cs[1] if wide else 0, A.data_ptr(), _ptr(D), _ptr(dt_bias), None, state.data_ptr(), y.data_ptr())
    _call(L.lib.sed_gated_scan_step, a, x.device, "sed_gated_scan_step")
    _moved_on(state)
    return y


# ---- causal convolution -------------------------------------------------------------------------------------------------


def _conv_args(x, weight, bias, act, frames, reverse, state):
    b, n_frames, d = x.shape
    xs = x.stride()
    return L.ConvArgs(b, n_frames, d, weight.shape[1], _DTYPES[x.dtype], act, int(reverse), _ptr(frames), x.data_ptr(), xs[0], xs[1],
                      weight.data_ptr(), _ptr(bias), _ptr(state))


def _conv_forward(x, weight, bias, act, frames, reverse, state, want_last):
    b, n_frames, d = x.shape
    y = _new(x)
    last = x.new_empty((b, weight.shape[1] - 1, d)) if want_last else None
    if b == 0 or n_frames == 0:
        if want_last:
            last.zero_() if state is None else last.copy_(state)
        return y, last
    a = _conv_args(x, weight, bias, act, frames, reverse, state)
    a.y, a.state_out = y.data_ptr(), _ptr(last)
    _call(L.lib.sed_causal_conv_forward, a, x.device, "sed_causal_conv_forward")
    return y, last


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, act, frames, reverse, want_last):
        y, last = _conv_forward(x, weight, bias, act, frames, reverse, state, want_last)
        ctx.save_for_backward(x, weight, bias, state, frames)
        ctx.flags = (act, reverse)
        ctx.set_materialize_grads(False)
        return (y, last) if want_last else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast=None):
        _no_tangent("the gradient of causal_conv", dy, dlast)
        x, weight, bias, state, frames = ctx.saved_tensors
        act, reverse = ctx.flags
        b, n_frames, d = x.shape
        dev = x.device
        dx, dw, db, dstate = (_new(t) for t in (x, weight, bias, state))
        if b == 0 or n_frames == 0:
            for t in (dw, db, dstate):
                if t is not None:
                    t.zero_()
            if dstate is not None and dlast is not None:
                dstate.copy_(dlast)
            return dx, dw, db, dstate, None, None, None, None
        dy = torch.zeros((b, n_frames, d), dtype=x.dtype, device=dev) if dy is None else _rows(dy)
        dlast = None if dlast is None else dlast.contiguous()
        a = _conv_args(x, weight, bias, act, frames, reverse, state)
        a.dy, a.dy_b, a.dy_t, a.dstate_out = dy.data_ptr(), dy.stride(0), dy.stride(1), _ptr(dlast)
        a.dx, a.dw, a.db, a.dstate = dx.data_ptr(), dw.data_ptr(), _ptr(db), _ptr(dstate)
        nbytes = L.lib.sed_causal_conv_workspace(b, n_frames, d, weight.shape[1])
        ws = _workspace(nbytes, x)
        a.ws, a.ws_bytes = ws.data_ptr(), nbytes
        _call(L.lib.sed_causal_conv_backward, a, dev, "sed_causal_conv_backward")
        return dx, dw, db, dstate, None, None, None, None


def _conv_checks(what, x, weight, bias, activation):
    if activation not in (None, "silu"):
        raise ValueError(f"{what}: activation {activation!r}; None and 'silu' are supported")
    if torch.is_tensor(weight) and weight.dim() == 3 and weight.shape[1] == 1:  # as a depthwise convolution layer holds it
        weight = weight.squeeze(1)
    if not torch.is_tensor(weight) or weight.dim() != 2 or not 1 <= weight.shape[1] <= 8:
        raise ValueError(f"{what}: weight: a (channels, taps) tensor of 1 to 8 taps")
    _check(what, "weight", weight, x, (x.shape[-1], weight.shape[1]), "float")
    if bias is not None:
        _check(what, "bias", bias, x, (x.shape[-1],), "float")
    return weight


def causal_conv(x, weight, bias=None, activation=None, frames=None, reverse=False, state=None, return_state=False):
    """Depthwise convolution of every channel with its own taps over the frames in front, with a gradient for every tensor but
    `frames`: y_t = act(bias + sum_k weight[:, k] x_{t - W + 1 + k}).

    x (clips, frames, channels) fp32, bf16 or fp16, any strides; weight (channels, W) or (channels, 1, W), 1 to 8 taps; bias
    (channels,); activation None or "silu".  frames: the clips' own row counts.  reverse: the window looks to later frames.
    state (clips, W - 1, channels): the rows in front of the first row walked, oldest first (zero if None).  With return_state
    also returns the last W - 1 rows seen, the next call's state."""
    what = "causal_conv"
    _check_x(what, x, 3)
    weight = _conv_checks(what, x, weight, bias, activation)
    _check_frames(what, frames, x)
    if state is not None:
        _check(what, "state", state, x, (x.shape[0], weight.shape[1] - 1, x.shape[2]))
        state = state.contiguous()
    x, weight, bias, act = _rows(x), _param(weight), _param(bias), _ACTIVATIONS[activation]
    if _wants_grad(what, x, weight, bias, state):
        return _CausalConv.apply(x, weight, bias, state, act, frames, bool(reverse), bool(return_state))
    y, last = _conv_forward(x, weight, bias, act, frames, reverse, state, return_state)
    return (y, last) if return_state else y


def causal_conv_step(state, x, weight, bias=None, activation=None):
    """One frame of causal_conv for a batch of streams: state (streams, W - 1, channels) of x's type, contiguous, moves up by the
    new row in place; x (streams, channels).  Returns y (streams, channels).  For inference: it has no gradient, and a gradient that
    kept this state as an input (causal_conv's does) raises afterwards."""
    what = "causal_conv_step"
    _check_x(what, x, 2)
    weight = _conv_checks(what, x, weight, bias, activation)
    _check(what, "state", state, x, (x.shape[0], weight.shape[1] - 1, x.shape[1]))
    if not state.is_contiguous():
        raise ValueError(f"{what}: state is updated in place and has to be contiguous")
    _no_grad_only(what, state, x, weight, bias)
    y = _new(x)
    if x.shape[0] == 0:
        return y
    x, weight, bias = _rows(x), _param(weight), _param(bias)
    a = L.ConvArgs(x.shape[0], 1, x.shape[1], weight.shape[1], _DTYPES[x.dtype], _ACTIVATIONS[activation], 0, None, x.data_ptr(), x.stride(0), 0,
                   weight.data_ptr(), _ptr(bias), None, y.data_ptr(), _ptr(state))
    _call(L.lib.sed_causal_conv_step, a, x.device, "sed_causal_conv_step")
    _moved_on(state)
    return y


# ---- group norm ---------------------------------------------------------------------------------------------------------


def _norm_args(x, shape, groups, weight, bias, act, eps, frames, stats, y, ws):
    """stats: mean and rstd, one behind the other; ws: (bytes, tensor) of the workspace."""
    at = stats.data_ptr()
    return L.NormArgs(*shape, groups, _DTYPES[x.dtype], act, eps, _ptr(frames), x.data_ptr(), _ptr(weight), _ptr(bias), _ptr(y), at,
                      at + 4 * shape[0] * groups, None, None, None, None, ws[1].data_ptr(), ws[0])


def _norm_workspace(shape, groups, x):
    nbytes = L.lib.sed_group_norm_workspace(*shape, groups)
    return nbytes, _workspace(nbytes, x)


def _norm_forward(x, groups, weight, bias, eps, act, frames):
    n = x.numel()
    shape = (x.shape[0], x.shape[1], n // (x.shape[0] * x.shape[1] * x.shape[-1]) if n else 1, x.shape[-1])
    y = torch.empty_like(x)
    stats = x.new_empty(2 * shape[0] * groups, dtype=torch.float32)
    if n:
        ws = _norm_workspace(shape, groups, x)  # held until the kernels are launched
        a = _norm_args(x, shape, groups, weight, bias, act, eps, frames, stats, y, ws)
        _call(L.lib.sed_group_norm_forward, a, x.device, "sed_group_norm_forward")
    return y, stats, shape


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, frames):
        y, stats, shape = _norm_forward(x, groups, weight, bias, eps, act, frames)
        ctx.save_for_backward(x, weight, bias, frames, stats)
        ctx.rest = (shape, groups, eps, act)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _no_tangent("the gradient of group_norm_act", dy)
        x, weight, bias, frames, stats = ctx.saved_tensors
        shape, groups, eps, act = ctx.rest
        dx, dw, db = (_new(t) for t in (x, weight, bias))
        if x.numel() == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
            return dx, dw, db, None, None, None, None
        dy = dy.contiguous()
        ws = _norm_workspace(shape, groups, x)
        a = _norm_args(x, shape, groups, weight, bias, act, eps, frames, stats, None, ws)
        a.dy, a.dx, a.dw, a.db = dy.data_ptr(), dx.data_ptr(), _ptr(dw), _ptr(db)
        _call(L.lib.sed_group_norm_backward, a, x.device, "sed_group_norm_backward")
        return dx, dw, db, None, None, None, None


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, activation=None, frames=None):
    """act(group norm of x) on channels-last data, with a gradient for x, weight and bias.

    x (clips, frames, ..., channels) fp32, bf16 or fp16: mean and (biased) variance are taken per clip and group of
    channels // groups neighbouring channels over the clip's own frames and all axes in between.  weight, bias (channels,), any
    floating type, or None; activation None, "silu", "relu" or "gelu" (the exact one).  frames (clips,) int32 on the device:
    rows behind a clip's own give zero and are not read.  At most 65535 clips and 2^19 channels."""
    what = "group_norm_act"
    if not torch.is_tensor(x) or x.dim() < 3:
        raise ValueError(f"{what}: x: (clips, frames, ..., channels)")
    _check_x(what, x, x.dim())
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: activation {activation!r}; None, 'silu', 'relu' and 'gelu' are supported")
    groups, c = int(groups), x.shape[-1]
    if groups < 1 or c % groups:
        raise ValueError(f"{what}: {c} channels do not divide into {groups} groups")
    if not float(eps) >= 0:
        raise ValueError(f"{what}: eps {eps} is negative")
    if x.shape[0] > 65535:
        raise ValueError(f"{what}: {x.shape[0]} clips; 65535 at most")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check(what, name, t, x, (c,), "float")
    _check_frames(what, frames, x)
    x, weight, bias, act = x.contiguous(), _param(weight), _param(bias), _ACTIVATIONS[activation]
    if _wants_grad(what, x, weight, bias):
        return _GroupNormAct.apply(x, weight, bias, groups, float(eps), act, frames)
    return _norm_forward(x, groups, weight, bias, float(eps), act, frames)[0]
