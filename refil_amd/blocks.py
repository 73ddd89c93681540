"""The residual temporal block as torch functions over librefil_hip.so: a gated linear recurrence over an episode (an alternative to the
GRU cell whose steps do not wait for each other), the norms before and after a block fused with the block's gate and residual scale, and a
gated feed-forward block (include/refil_hip.h section 4 has the formulas).

    y, h_last = linear_recurrence(x, decay_gate, input_gate, decay)          # autograd; linrec_forward / linrec_backward underneath
    y         = linrec_step(x, decay_gate, input_gate, decay, state)         # one acting step, state in place
    y, n      = norm_gate_residual(x, o, gate, post_weight=..., ...)         # autograd; norm_gate_forward / norm_gate_backward
    h         = gated_ff(x, w_gate, w_up)                                    # autograd; gated_ff_forward / gated_ff_backward

Activations are fp32, bf16 or fp16 (all of one call alike); decay, norm weights, hidden states and their gradients are fp32. Work is enqueued on
the current stream of the tensors' device, outputs and workspaces come from torch's allocator for that stream (one call's workspace is never
another's). A tensor whose inner dimensions are not dense is copied; CPU tensors are refused: there is no host path.

The explicit forward / backward functions can be captured into a HIP graph. Running the AUTOGRAD backward under capture is refused: with an
eager graph of the same leaves alive, torch would join the capture from the stream that graph recorded and end the process."""
from __future__ import annotations

import ctypes as C
from collections import namedtuple

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib
from ._lib import GatedFfDesc, LinrecDesc, LinrecStepDesc, NormGateDesc, check

__all__ = ["linear_recurrence", "linrec_forward", "linrec_backward", "linrec_step", "norm_gate_residual", "norm_gate_forward",
           "norm_gate_backward", "NormGateGrads", "gated_ff", "gated_ff_forward", "gated_ff_backward"]

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_ACTS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}


def _require_gpu(t, who):
    if not t.is_cuda:
        raise ValueError(f"{who}: tensors live on {t.device}: refil_amd.blocks has no host path")


def _launch(fn, desc, dev, what):
    if dev.type == "cuda":
        i = dev.index
        if i != torch._C._cuda_getDevice():
            with torch.cuda.device(dev):
                rc = fn(C.byref(desc), torch._C._cuda_getCurrentRawStream(i))
        else:
            rc = fn(C.byref(desc), torch._C._cuda_getCurrentRawStream(i))
    else:
        rc = fn(C.byref(desc), _lib.current_stream_ptr())
    if rc:
        check(rc, what)


def _first(x, who):
    """dtype code of the call's activations"""
    _require_gpu(x, who)
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"{who}: dtype {x.dtype}; float32, bfloat16 and float16 are supported")
    return code


def _like(t, x, name, who, shape=None):
    """an activation tensor beside x: same device and dtype, the given shape (x's)"""
    want = x.shape if shape is None else shape
    if t.shape == want and t.dtype is x.dtype and t.get_device() == x.get_device():
        return t
    if t.device != x.device:
        raise ValueError(f"{who}: {name} is on {t.device}, the other tensors on {x.device}")
    if t.dtype != x.dtype:
        raise TypeError(f"{who}: {name} is {t.dtype}, the other activations {x.dtype}")
    raise ValueError(f"{who}: {name} has shape {tuple(t.shape)}, expected {tuple(want)}")


def _f32(t, x, name, who, shape):
    """an fp32 parameter / state tensor, dense"""
    if t is None:
        return None
    if t.shape == shape and t.dtype is torch.float32 and t.get_device() == x.get_device():
        return t if t.is_contiguous() else t.contiguous()
    if t.device != x.device:
        raise ValueError(f"{who}: {name} is on {t.device}, the other tensors on {x.device}")
    if t.dtype != torch.float32:
        raise TypeError(f"{who}: {name} is {t.dtype}, expected float32")
    raise ValueError(f"{who}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _bytes(t, x, name, who, shape):
    """a uint8 / bool mask"""
    if t is None:
        return None
    if t.dtype is torch.bool:
        t = t.view(torch.uint8)
    if t.shape == shape and t.dtype is torch.uint8 and t.get_device() == x.get_device():
        return t
    if t.device != x.device:
        raise ValueError(f"{who}: {name} is on {t.device}, the other tensors on {x.device}")
    if t.dtype != torch.uint8:
        raise TypeError(f"{who}: {name} is {t.dtype}, expected uint8 or bool")
    raise ValueError(f"{who}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _new(x):
    """an uninitialised dense tensor of x's shape, type and device"""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _p(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes, x):
    return x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _grad(who, *tensors):
    """whether autograd has to record this call. A forward-mode tangent, which a call without a recorded gradient would drop, is refused"""
    if _forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{who}: an input carries a forward-mode tangent; forward-mode derivatives are not supported")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_capture(who):
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{who}: the autograd backward cannot run under graph capture (an eager graph of the same leaves would make torch end the "
                           f"process); capture the explicit {who}_forward / {who}_backward calls instead")


# ------------------------------------------------------------------------------------------------ gated linear recurrence
def _seq(t):
    """[B, T, ..., D] with its inner dimensions dense; (tensor, stride of B, stride of T)"""
    st = t.stride()
    if st[-1] != 1 or (len(st) == 4 and st[2] != t.shape[3]):
        t = t.contiguous()
        st = t.stride()
    return t, st[0], st[1]


def _linrec_desc(who, x, decay_gate, input_gate, decay, scale, h0, reset, lengths):
    code = _first(x, who)
    if x.dim() not in (3, 4):
        raise ValueError(f"{who}: x has shape {tuple(x.shape)}, expected [B, T, D] or [B, T, n_agents, D]")
    _like(decay_gate, x, "decay_gate", who)
    _like(input_gate, x, "input_gate", who)
    B, T, D = x.shape[0], x.shape[1], x.shape[-1]
    inner = tuple(x.shape[2:])
    decay = _f32(decay, x, "decay", who, (D,))
    h0 = _f32(h0, x, "h0", who, (B, *inner))
    reset = _bytes(reset, x, "reset", who, (B, T))
    if lengths is not None:
        if lengths.device != x.device or lengths.shape != (B,) or lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{who}: lengths must be an integer tensor of shape ({B},) on {x.device}")
        lengths = (lengths if lengths.dtype is torch.int32 else lengths.clamp(0, T).to(torch.int32)).contiguous()
    x, xb, xt = _seq(x)
    decay_gate, ab, at = _seq(decay_gate)
    input_gate, ib, it = _seq(input_gate)
    d = LinrecDesc(x.data_ptr(), xb, xt, decay_gate.data_ptr(), ab, at, input_gate.data_ptr(), ib, it, decay.data_ptr(), _p(h0))
    d.lengths = _p(lengths)
    if reset is not None:
        d.reset, d.rs_sB, d.rs_sT = reset.data_ptr(), reset.stride(0), reset.stride(1)
    width = 1
    for n in inner:
        width *= n
    d.B, d.T, d.C, d.D, d.dtype, d.scale = B, T, width, D, code, scale
    if D == 0:
        raise ValueError(f"{who}: D must be positive")
    d._keep = [x, decay_gate, input_gate, decay, h0, reset, lengths]
    return d


def linrec_forward(x, decay_gate, input_gate, decay, *, scale=8.0, h0=None, reset=None, lengths=None, save=False):
    """y [like x], h_last [B, ..., D] fp32, saved (None unless `save`: the states the backward restarts from). x, decay_gate, input_gate
    [B, T, D] or [B, T, n_agents, D], decay [D], h0 [B, ..., D] fp32, reset [B, T] uint8 / bool (1: the state is dropped in front of that
    step), lengths [B] (steps behind an episode's length are not read; their y is 0)."""
    who = "linrec_forward"
    d = _linrec_desc(who, x, decay_gate, input_gate, decay, scale, h0, reset, lengths)
    L = _lib.lib()
    y = _new(x)
    h_last = torch.empty((x.shape[0], *x.shape[2:]), dtype=torch.float32, device=x.device)
    saved = torch.empty(L.refil_linrec_saved_floats(C.byref(d)), dtype=torch.float32, device=x.device) if save else None
    ws = _workspace(L.refil_linrec_workspace_bytes(C.byref(d), 0), x)
    d.y, d.y_sB, d.y_sT, d.h_last, d.saved = y.data_ptr(), y.stride(0), y.stride(1), h_last.data_ptr(), _p(saved)
    d.workspace, d.workspace_bytes = _p(ws), 0 if ws is None else ws.numel()
    _launch(L.refil_linrec_forward, d, x.device, who)
    return y, h_last, saved


def linrec_backward(dy, x, decay_gate, input_gate, decay, saved, *, scale=8.0, h0=None, reset=None, lengths=None, dh_last=None):
    """(dx, d decay_gate, d input_gate, d decay [D] fp32, d h0 fp32) of linrec_forward(..., save=True) with the same arguments."""
    who = "linrec_backward"
    d = _linrec_desc(who, x, decay_gate, input_gate, decay, scale, h0, reset, lengths)
    L = _lib.lib()
    _like(dy, x, "dy", who)
    state = (x.shape[0], *x.shape[2:])
    dh_last = _f32(dh_last, x, "dh_last", who, state)
    saved = _f32(saved, x, "saved", who, (L.refil_linrec_saved_floats(C.byref(d)),))
    dy, d.dy_sB, d.dy_sT = _seq(dy)
    dx, dga, dgi = (_new(x) for _ in range(3))
    ddecay = _new(decay)
    dh0 = torch.empty(state, dtype=torch.float32, device=x.device)
    ws = _workspace(L.refil_linrec_workspace_bytes(C.byref(d), 1), x)
    d.dy, d.dh_last, d.saved = dy.data_ptr(), _p(dh_last), saved.data_ptr()
    d.dx, d.dga, d.dgi, d.d_sB, d.d_sT, d.ddecay, d.dh0 = dx.data_ptr(), dga.data_ptr(), dgi.data_ptr(), dx.stride(0), dx.stride(1), ddecay.data_ptr(), dh0.data_ptr()
    d.workspace, d.workspace_bytes = _p(ws), 0 if ws is None else ws.numel()
    _launch(L.refil_linrec_backward, d, x.device, who)
    return dx, dga, dgi, ddecay, dh0


def linrec_step(x, decay_gate, input_gate, decay, state, *, scale=8.0, slots=None, state_out=None):
    """One step for the rows of x [B, D] / [B, n_agents, D]; returns y. state [n, ..., D] fp32, dense, is advanced in place, or into state_out of
    the same shape. slots [B] int32: the state row of each x row (None: row b is state b); a slot outside [0, n) marks a padded row (y = 0),
    rows that name one slot are consecutive steps of it in row order. No gradient: inputs that require one are refused outside torch.no_grad()."""
    who = "linrec_step"
    if _grad(who, x, decay_gate, input_gate, decay, state, state_out):
        raise RuntimeError(f"{who}: an input requires a gradient, which an acting step does not have: call it under torch.no_grad(), or train through "
                           "linear_recurrence")
    code = _first(x, who)
    if x.dim() not in (2, 3):
        raise ValueError(f"{who}: x has shape {tuple(x.shape)}, expected [B, D] or [B, n_agents, D]")
    _like(decay_gate, x, "decay_gate", who)
    _like(input_gate, x, "input_gate", who)
    B, D = x.shape[0], x.shape[-1]
    decay = _f32(decay, x, "decay", who, (D,))
    out = state if state_out is None else state_out
    inner = x.shape[1:]
    for name, t in ((("state", state),) if out is state else (("state", state), ("state_out", out))):
        if t.get_device() != x.get_device() or t.dtype is not torch.float32 or t.shape[1:] != inner or not t.is_contiguous():
            raise ValueError(f"{who}: {name} must be a dense float32 tensor [n, {', '.join(map(str, inner))}] on {x.device}")
    if out is not state and out.shape != state.shape:
        raise ValueError(f"{who}: state_out has shape {tuple(out.shape)}, state {tuple(state.shape)}")
    a, b, n = state.data_ptr(), out.data_ptr(), 4 * state.numel()
    if a != b and a < b + n and b < a + n:
        raise ValueError(f"{who}: state_out overlaps state without being it")
    if slots is not None:
        if slots.shape != (B,) or slots.dtype is not torch.int32 or slots.get_device() != x.get_device():
            raise ValueError(f"{who}: slots must be an int32 tensor of shape ({B},) on {x.device}")
        slots = slots.contiguous()
    elif state.shape[0] < B:
        raise ValueError(f"{who}: {B} rows, {state.shape[0]} states")
    if D == 0:
        raise ValueError(f"{who}: D must be positive")

    def rows(t):
        return t if t.is_contiguous() or (t.stride(-1) == 1 and (t.dim() == 2 or t.stride(1) == D)) else t.contiguous()
    x, decay_gate, input_gate = rows(x), rows(decay_gate), rows(input_gate)
    y = _new(x)
    width = D if x.dim() == 2 else D * x.shape[1]
    d = LinrecStepDesc(x.data_ptr(), x.stride(0), decay_gate.data_ptr(), decay_gate.stride(0), input_gate.data_ptr(), input_gate.stride(0), decay.data_ptr(),
                       a, b, _p(slots), y.data_ptr(), width, B, width, D, state.shape[0], code, scale)
    _launch(_lib.lib().refil_linrec_step, d, x.device, who)
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)         # (written behind torch's back: a graph that kept it has to notice)
    return y


class _LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, decay_gate, input_gate, decay, h0, reset, lengths, scale):
        y, h_last, saved = linrec_forward(x, decay_gate, input_gate, decay, scale=scale, h0=h0, reset=reset, lengths=lengths, save=True)
        ctx.save_for_backward(x, decay_gate, input_gate, decay, h0, reset, lengths, saved)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return y, h_last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh_last):
        _no_capture("linrec")
        x, ga, gi, decay, h0, reset, lengths, saved = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(x)
        dx, dga, dgi, dd, dh0 = linrec_backward(dy, x, ga, gi, decay, saved, scale=ctx.scale, h0=h0, reset=reset, lengths=lengths, dh_last=dh_last)
        return dx, dga, dgi, dd, (dh0 if h0 is not None else None), None, None, None


def linear_recurrence(x, decay_gate, input_gate, decay, *, scale=8.0, h0=None, reset=None, lengths=None):
    """(y, h_last) of linrec_forward, differentiable in x, decay_gate, input_gate, decay and h0."""
    if not _grad("linear_recurrence", x, decay_gate, input_gate, decay, h0):
        return linrec_forward(x, decay_gate, input_gate, decay, scale=scale, h0=h0, reset=reset, lengths=lengths)[:2]
    return _LinearRecurrence.apply(x, decay_gate, input_gate, decay, h0, reset, lengths, scale)


# ------------------------------------------------------------------------------------- norms, gate and residual scale
NormGateGrads = namedtuple("NormGateGrads", "dx do dgate dpost_weight dres_scale dpre_weight")


def _rows(t, D):
    """[..., D] as rows with a dense last dimension; (tensor kept alive, row stride)"""
    if t is None:
        return None, 0
    if t.dim() != 2:
        t = t.reshape(-1, D)
    st = t.stride()
    if st[1] != 1 and D > 1:
        t = t.contiguous()
        return t, D
    return t, st[0]


def _norm_desc(who, x, o, gate, post_weight, res_scale, pre_weight, alpha, eps, row_mask):
    code = _first(x, who)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{who}: x has shape {tuple(x.shape)}, expected [..., D] with D > 0")
    D = x.shape[-1]
    if o is not None:
        _like(o, x, "o", who)
    if gate is not None:
        if o is None:
            raise ValueError(f"{who}: a gate needs the block's output o")
        _like(gate, x, "gate", who)
    one = (D,)
    post_weight, res_scale, pre_weight = _f32(post_weight, x, "post_weight", who, one), _f32(res_scale, x, "res_scale", who, one), _f32(pre_weight, x, "pre_weight", who, one)
    if not 1.17549435e-38 <= eps < 1e30:
        raise ValueError(f"{who}: eps must be positive (a normal fp32 number) and finite")
    row_mask = _bytes(row_mask, x, "row_mask", who, x.shape[:-1])
    x2, xs = _rows(x, D)
    o2, os_ = _rows(o, D)
    g2, gs = _rows(gate, D)
    if row_mask is not None and (row_mask.dim() != 1 or not row_mask.is_contiguous()):
        row_mask = row_mask.reshape(-1).contiguous()
    d = NormGateDesc(x2.data_ptr(), xs, _p(o2), os_, _p(g2), gs, _p(post_weight), _p(res_scale), _p(pre_weight), _p(row_mask))
    d.N, d.D, d.dtype, d.alpha, d.eps = x2.shape[0], D, code, alpha, eps
    d._keep = [x2, o2, g2, post_weight, res_scale, pre_weight, row_mask]
    return d


def norm_gate_forward(x, o=None, gate=None, *, post_weight=None, res_scale=None, pre_weight=None, alpha=1.0, eps=1e-6, row_mask=None,
                      want_y=True, want_n=True):
    """(y, n): y = alpha x + res_scale sigmoid(gate) N(o; post_weight), n = N(y; pre_weight), N(v; w) = v w / sqrt(mean(v^2) + eps) over the last
    dimension D <= 16384. x, o, gate [..., D]; weights [D] fp32 (None: ones); row_mask [...] uint8 / bool: rows with 1 are not read, their
    outputs are 0. Without o it is the plain norm in front of a block. want_y / want_n: None is returned for the one not asked for."""
    who = "norm_gate_forward"
    d = _norm_desc(who, x, o, gate, post_weight, res_scale, pre_weight, alpha, eps, row_mask)
    if not (want_y or want_n):
        raise ValueError(f"{who}: neither y nor n is asked for")
    y = _new(x) if want_y else None
    n = _new(x) if want_n else None
    d.y, d.n, d.y_stride, d.n_stride = _p(y), _p(n), d.D, d.D
    _launch(_lib.lib().refil_norm_gate_forward, d, x.device, who)
    return y, n


def norm_gate_backward(dy, dn, x, o=None, gate=None, *, post_weight=None, res_scale=None, pre_weight=None, alpha=1.0, eps=1e-6, row_mask=None):
    """NormGateGrads of norm_gate_forward with the same arguments; dy or dn may be None. Gradients of absent inputs are None."""
    who = "norm_gate_backward"
    d = _norm_desc(who, x, o, gate, post_weight, res_scale, pre_weight, alpha, eps, row_mask)
    if dy is None and dn is None:
        raise ValueError(f"{who}: neither dy nor dn is given")
    L, D = _lib.lib(), d.D
    dy2, d.dy_stride = _rows(None if dy is None else _like(dy, x, "dy", who), D)
    dn2, d.dn_stride = _rows(None if dn is None else _like(dn, x, "dn", who), D)
    dx = _new(x)
    do = None if o is None else _new(x)
    dg = None if gate is None else _new(x)
    dwp, dsc, dwq = (None if t is None else _new(t) for t in (post_weight, res_scale, pre_weight))
    ws = _workspace(L.refil_norm_gate_workspace_bytes(C.byref(d)), x)
    d.dy, d.dn, d.dx, d.d_o, d.dgate, d.dx_stride, d.do_stride, d.dgate_stride = _p(dy2), _p(dn2), dx.data_ptr(), _p(do), _p(dg), D, D, D
    d.dpost_weight, d.dres_scale, d.dpre_weight = _p(dwp), _p(dsc), _p(dwq)
    d.workspace, d.workspace_bytes = _p(ws), 0 if ws is None else ws.numel()
    _launch(L.refil_norm_gate_backward, d, x.device, who)
    return NormGateGrads(dx, do, dg, dwp, dsc, dwq)


class _NormGate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, o, gate, post_weight, res_scale, pre_weight, alpha, eps, row_mask):
        y, n = norm_gate_forward(x, o, gate, post_weight=post_weight, res_scale=res_scale, pre_weight=pre_weight, alpha=alpha, eps=eps, row_mask=row_mask,
                                 want_y=o is not None)
        ctx.save_for_backward(x, o, gate, post_weight, res_scale, pre_weight, row_mask)
        ctx.alpha, ctx.eps = alpha, eps
        ctx.set_materialize_grads(False)
        return y, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dn):
        if dy is None and dn is None:
            return (None,) * 9
        _no_capture("norm_gate")
        x, o, gate, wp, sc, wq, mask = ctx.saved_tensors
        r = norm_gate_backward(dy, dn, x, o, gate, post_weight=wp, res_scale=sc, pre_weight=wq, alpha=ctx.alpha, eps=ctx.eps, row_mask=mask)
        return (*r, None, None, None)


def norm_gate_residual(x, o=None, gate=None, *, post_weight=None, res_scale=None, pre_weight=None, alpha=1.0, eps=1e-6, row_mask=None):
    """(y, n) of norm_gate_forward, differentiable in the tensors and the weights. Without o: (None, N(alpha x; pre_weight))."""
    if not _grad("norm_gate_residual", x, o, gate, post_weight, res_scale, pre_weight):
        return norm_gate_forward(x, o, gate, post_weight=post_weight, res_scale=res_scale, pre_weight=pre_weight, alpha=alpha, eps=eps, row_mask=row_mask,
                                 want_y=o is not None)
    return _NormGate.apply(x, o, gate, post_weight, res_scale, pre_weight, alpha, eps, row_mask)


# ------------------------------------------------------------------------------------------------ gated feed-forward block
def _ff_desc(who, x, w_gate, w_up, act):
    code = _first(x, who)
    if act not in _ACTS:
        raise ValueError(f"{who}: act {act!r} is none of {sorted(_ACTS)}")
    if w_gate.dim() != 2 or x.dim() < 1 or x.shape[-1] != w_gate.shape[1] or 0 in w_gate.shape:
        raise ValueError(f"{who}: x {tuple(x.shape)} and w_gate {tuple(w_gate.shape)}, expected [..., D] and [F, D]")
    F, D = w_gate.shape
    _like(w_gate, x, "w_gate", who, (F, D))
    _like(w_up, x, "w_up", who, (F, D))
    ws = w_gate.stride()
    if ws != w_up.stride() or ws[1] != 1 or ws[0] < D:
        w_gate, w_up, ws = w_gate.contiguous(), w_up.contiguous(), (D, 1)
    x2, xs = _rows(x, D)
    if xs < D:                            # (one row, or rows expanded over one another)
        x2, xs = x2.contiguous(), D
    d = GatedFfDesc(x2.data_ptr(), xs, w_gate.data_ptr(), w_up.data_ptr(), ws[0])
    d.N, d.D, d.F, d.act, d.dtype = x2.shape[0], D, F, _ACTS[act], code
    d._keep = [x2, w_gate, w_up]
    return d


def gated_ff_forward(x, w_gate, w_up, b_gate=None, b_up=None, *, act="silu", save=False):
    """(h, saved): h = act(x w_gate^T + b_gate) * (x w_up^T + b_up). x [..., D], w_* [F, D], b_* [F], one dtype; act "silu" or "gelu" (tanh form);
    saved (None unless `save`): the two pre-activations, fp32, for the backward."""
    who = "gated_ff_forward"
    d = _ff_desc(who, x, w_gate, w_up, act)
    L = _lib.lib()
    keep = []
    for name, t in (("b_gate", b_gate), ("b_up", b_up)):
        if t is not None:
            t = _like(t, x, name, who, (d.F,)).contiguous()
            keep.append(t)
            setattr(d, name, t.data_ptr())
    h = torch.empty((*x.shape[:-1], d.F), dtype=x.dtype, device=x.device)
    saved = torch.empty((2, d.N, d.F), dtype=torch.float32, device=x.device) if save else None
    ws = _workspace(L.refil_gated_ff_workspace_bytes(C.byref(d), 0), x)
    d.h, d.h_stride, d.saved = h.data_ptr(), d.F, _p(saved)
    d.workspace, d.workspace_bytes = _p(ws), 0 if ws is None else ws.numel()
    _launch(L.refil_gated_ff_forward, d, x.device, who)
    return h, saved


def gated_ff_backward(dh, x, w_gate, w_up, saved, *, act="silu", bias=False):
    """(dx, dw_gate, dw_up, db_gate, db_up) of gated_ff_forward(..., save=True); the bias gradients are None unless `bias`. In 16 bits the gradients
    of the two pre-activations are rounded to the type once on the way to dx and the weight gradients, inside fp16's range whatever dh's."""
    who = "gated_ff_backward"
    d = _ff_desc(who, x, w_gate, w_up, act)
    L, F, D = _lib.lib(), d.F, d.D
    _like(dh, x, "dh", who, (*x.shape[:-1], F))
    saved = _f32(saved, x, "saved", who, (2, d.N, F))
    new = torch.empty if d.N else torch.zeros
    dx = _new(x)
    dwg, dwu = (new((F, D), dtype=x.dtype, device=x.device) for _ in range(2))
    dbg, dbu = (new(F, dtype=x.dtype, device=x.device) if bias else None for _ in range(2))
    if d.N:
        dh2, d.dh_stride = _rows(dh, F)
        ws = _workspace(L.refil_gated_ff_workspace_bytes(C.byref(d), 1), x)
        d.dh, d.saved, d.dx, d.dx_stride = dh2.data_ptr(), saved.data_ptr(), dx.data_ptr(), D
        d.dw_gate, d.dw_up, d.db_gate, d.db_up = dwg.data_ptr(), dwu.data_ptr(), _p(dbg), _p(dbu)
        d.workspace, d.workspace_bytes = _p(ws), 0 if ws is None else ws.numel()
        _launch(L.refil_gated_ff_backward, d, x.device, who)
    return dx, dwg, dwu, dbg, dbu


class _GatedFf(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        h, saved = gated_ff_forward(x, w_gate, w_up, b_gate, b_up, act=act, save=True)
        ctx.save_for_backward(x, w_gate, w_up, saved)
        ctx.act, ctx.biases = act, (b_gate is not None, b_up is not None)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        _no_capture("gated_ff")
        x, w_gate, w_up, saved = ctx.saved_tensors
        dx, dwg, dwu, dbg, dbu = gated_ff_backward(dh, x, w_gate, w_up, saved, act=ctx.act, bias=any(ctx.biases))
        return dx, dwg, dwu, (dbg if ctx.biases[0] else None), (dbu if ctx.biases[1] else None), None


def gated_ff(x, w_gate, w_up, b_gate=None, b_up=None, *, act="silu"):
    """h of gated_ff_forward, differentiable in x, the weights and the biases."""
    if not _grad("gated_ff", x, w_gate, w_up, b_gate, b_up):
        return gated_ff_forward(x, w_gate, w_up, b_gate, b_up, act=act)[0]
    return _GatedFf.apply(x, w_gate, w_up, b_gate, b_up, act)
