"""Sequence operators over packed clips: a short causal convolution, a selective state-space scan and a root-mean-square
norm (csrc/seqconv.hip, seqscan.hip, rmsnorm.hip) -- what a state-space block over a clip's events or nodes needs beside its
matrix products.  The reference's temporal part is the GRU of its head (models/EventAD.py:62-97); these have no counterpart
there.

Rows are packed: activations are [rows, channels], clip s owns rows clip_start[s] .. clip_start[s+1]-1 (int32 on the device,
not decreasing, within 0..rows; None = all rows are one clip); rows of no clip give zeros and take no part in a gradient.
Activations are float32, bfloat16 or float16, all of one call alike; parameters and scan states are float32.  A row may be a
slice of a wider array (any row stride); an array whose channels are not adjacent is copied first.

Every function launches on the current stream of its tensors' device, waits for nothing, and can be captured into a graph;
workspaces come from torch's allocator per call, so captured graphs do not share one.  The functions are differentiable
(except the single-token and 8-bit forms, which refuse inputs that need a gradient); gradients are not differentiable
again.  There is no CPU path: tensors must be on a GPU."""
import contextlib
import ctypes

import torch
from torch.autograd.function import once_differentiable

from ._lib import call, stream_handle

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACT = {None: 0, "silu": 1}
MAX_TAPS, MAX_STATE = 8, 64


def _fail(msg, *args):
    raise RuntimeError("eventad_amd.sequence: " + msg % args)


_MAX_LD = 1 << 24               # row strides above this are taken by copying the array


def _activation(name, t, rows, width, like=None):
    """Checks t [rows, width] (None: any); returns it with adjacent channels."""
    if not isinstance(t, torch.Tensor):
        _fail("%s must be a tensor", name)
    if like is not None:
        if t.dtype != like.dtype or t.device != like.device:
            _fail("%s is %s on %s, expected %s on %s", name, t.dtype, t.device, like.dtype, like.device)
    elif t.dtype not in _DTYPE:
        _fail("%s must be float32, bfloat16 or float16, not %s", name, t.dtype)
    shape = t.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (width is not None and shape[1] != width):
        _fail("%s has shape %s, expected %s", name, tuple(shape), ("*" if rows is None else rows, "*" if width is None else width))
    ld, step = t.stride()
    if step == 1 and (shape[1] <= ld <= _MAX_LD or shape[0] <= 1):
        return t
    return t.contiguous()


def _tensor(name, t, shape, dtype, device):
    """Checks a parameter or a state; returns it contiguous."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device:
        _fail("%s must be a %s tensor on %s", name, dtype, device)
    if t.shape != shape:
        _fail("%s has shape %s, expected %s", name, tuple(t.shape), shape)
    return t if t.is_contiguous() else t.contiguous()


def _ld(t):
    """Row stride in elements (an array of at most one row may have any)."""
    if t is None:
        return 0
    ld, width = t.stride(0), t.shape[1]
    return ld if width <= ld <= _MAX_LD else width


def _p(t):
    return None if t is None else t.data_ptr()


def _clips(clip_start, rows, device):
    if clip_start is None:
        return None, 1
    if not isinstance(clip_start, torch.Tensor) or clip_start.dtype != torch.int32 or clip_start.device != device or \
            clip_start.dim() != 1 or clip_start.numel() < 2:
        _fail("clip_start must be int32[clips + 1] on %s", device)
    return clip_start.contiguous(), clip_start.numel() - 1


def _gpu(t):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _fail("tensors must be on a GPU (there is no CPU path)")
    return t.device


def _needs_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _bytes(name, *shape):
    n = ctypes.c_int64(0)
    call(name, *shape, ctypes.byref(n))
    return n.value


def _workspace(nbytes, device):
    return torch.empty(max(16, nbytes), dtype=torch.uint8, device=device)


_HERE = contextlib.nullcontext()


def _on(device):
    """Makes the tensors' device current for the launches."""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


# ---------------------------------------------------------------------------------------------------- causal convolution
def _conv_fwd(x, w, bias, starts, clips, state, act, want_state):
    rows, D = x.shape
    y = torch.empty((rows, D), dtype=x.dtype, device=x.device)
    final = torch.empty((clips, w.shape[1] - 1, D), dtype=x.dtype, device=x.device) if want_state else None
    call("eventad_causal_conv_fwd", _p(x), _ld(x), _p(w), _p(bias), _p(starts), clips, _p(state), _p(final), _p(y), D, rows, D,
         w.shape[1], act, _DTYPE[x.dtype], stream_handle())
    return y, final


class _ConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, starts, clips, state, act, want_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, w, bias, starts, state)
        ctx.clips, ctx.act = clips, act
        return _conv_fwd(x, w, bias, starts, clips, state, act, want_state)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        x, w, bias, starts, state = ctx.saved_tensors
        rows, D = x.shape
        K = w.shape[1]
        with _on(x.device):
            dy = torch.zeros_like(x) if dy is None else _activation("the gradient", dy, rows, D, x)
            dfinal = None if dfinal is None else dfinal.contiguous()
            dx = torch.empty((rows, D), dtype=x.dtype, device=x.device)
            dstate = torch.empty_like(state) if state is not None and ctx.needs_input_grad[5] else None
            dp = torch.empty(D * (K + 1), device=x.device)
            n = _bytes("eventad_causal_conv_workspace", rows, D, K)
            ws = _workspace(n, x.device)
            call("eventad_causal_conv_bwd", _p(x), _ld(x), _p(w), _p(bias), _p(starts), ctx.clips, _p(state), _p(dy), _ld(dy), _p(dfinal),
                 _p(dx), D, _p(dstate), _p(dp), _p(ws), ws.numel(), rows, D, K, ctx.act, _DTYPE[x.dtype], stream_handle())
        return dx, dp[:D * K].view(D, K), dp[D * K:] if bias is not None else None, None, None, dstate, None, None


def _conv_args(x, weight, bias, state, activation, clips):
    dev = _gpu(x)
    if activation not in _ACT:
        _fail("activation must be None or 'silu', not %r", activation)
    x = _activation("x", x, None, None)
    D = x.shape[1]
    taps = weight.shape[1] if isinstance(weight, torch.Tensor) and weight.dim() == 2 else 0
    if D < 1 or not 1 <= taps <= MAX_TAPS:
        _fail("weight must be [channels, taps] with 1..%d taps, x [rows, channels] with at least one channel", MAX_TAPS)
    weight = _tensor("weight", weight, (D, taps), torch.float32, dev)
    bias = _tensor("bias", bias, (D,), torch.float32, dev)
    state = _tensor("state", state, (clips, taps - 1, D), x.dtype, dev)
    return x, weight, bias, state, _ACT[activation]


def causal_conv(x, weight, bias=None, clip_start=None, state=None, activation="silu", return_state=False):
    """y_t = act(bias + sum_k weight[:, k] x_{t-(taps-1)+k}) per channel, inside every clip.

    x [rows, channels]; weight float32 [channels, taps], taps 1..8, weight[:, -1] multiplies the row itself; bias float32
    [channels]; activation None or "silu" (x sigmoid(x)).  state [clips, taps - 1, channels], of x's type, holds the inputs in
    front of each clip's first row, oldest first (None: zeros).
    -> y, or (y, final_state) with return_state: the inputs in front of the row that would follow each clip."""
    starts, clips = _clips(clip_start, x.shape[0] if isinstance(x, torch.Tensor) else 0, _gpu(x))
    x, weight, bias, state, act = _conv_args(x, weight, bias, state, activation, clips)
    with _on(x.device):
        if _needs_grad(x, weight, bias, state):
            y, final = _ConvFn.apply(x, weight, bias, starts, clips, state, act, return_state)
        else:
            y, final = _conv_fwd(x, weight, bias, starts, clips, state, act, return_state)
    return (y, final) if return_state else y


def causal_conv_step(x, weight, state, bias=None, activation="silu", state_out=None):
    """One row per clip: x [clips, channels], state [clips, taps - 1, channels] contiguous.  The state is moved on in place, or
    -- state_out given, a contiguous tensor like it that does not overlap it -- written there and left as it was.  -> y [clips,
    channels]."""
    if _needs_grad(x, weight, state, bias):
        _fail("the single-token form has no gradient: use causal_conv, or torch.no_grad()")
    x, weight, bias, checked, act = _conv_args(x, weight, bias, state, activation, x.shape[0])
    if checked is not state or checked is None:
        _fail("state must be contiguous, of x's type, [clips, taps - 1, channels]")
    out = _state_out(state, state_out)
    with _on(x.device):
        y = torch.empty((x.shape[0], x.shape[1]), dtype=x.dtype, device=x.device)
        call("eventad_causal_conv_step", _p(x), _ld(x), _p(weight), _p(bias), _p(state), _p(out), _p(y), x.shape[1], x.shape[0],
             x.shape[1], weight.shape[1], act, _DTYPE[x.dtype], stream_handle())
        torch.autograd.graph.increment_version(out)              # written behind autograd's back
    return y


def _state_out(state, out):
    if out is None or out is state:
        return state
    if not isinstance(out, torch.Tensor) or out.dtype != state.dtype or out.device != state.device or out.shape != state.shape or \
            not out.is_contiguous():
        _fail("state_out must be a contiguous tensor like state")
    size = state.numel() * state.element_size()
    if abs(out.data_ptr() - state.data_ptr()) < size and out.data_ptr() != state.data_ptr():
        _fail("state_out overlaps state")
    return out


# -------------------------------------------------------------------------------------------------------- selective scan
def _scan_fwd(u, delta, A, B, C, D, z, bias, starts, clips, state, softplus, want_state, want_checkpoint):
    rows, ch = u.shape
    N = A.shape[1]
    y = torch.empty((rows, ch), dtype=u.dtype, device=u.device)
    final = torch.empty((clips, ch, N), device=u.device) if want_state else None
    ckpt = _workspace(_bytes("eventad_selective_scan_checkpoint", rows, ch, N), u.device) if want_checkpoint else None
    ws = _workspace(_bytes("eventad_selective_scan_workspace", rows, ch, N, 0), u.device)
    call("eventad_selective_scan_fwd", _p(u), _ld(u), _p(delta), _ld(delta), _p(A), _p(B), _ld(B), _p(C), _ld(C), _p(D), _p(z), _ld(z),
         _p(bias), _p(starts), clips, _p(state), _p(final), _p(y), ch, _p(ckpt), _p(ws), ws.numel(), rows, ch, N, softplus,
         _DTYPE[u.dtype], stream_handle())
    return y, final, ckpt


class _ScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, bias, starts, clips, state, softplus, want_state):
        ctx.set_materialize_grads(False)
        y, final, ckpt = _scan_fwd(u, delta, A, B, C, D, z, bias, starts, clips, state, softplus, want_state, True)
        ctx.save_for_backward(u, delta, A, B, C, D, z, bias, starts, state, ckpt)
        ctx.clips, ctx.softplus = clips, softplus
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        u, delta, A, B, C, D, z, bias, starts, state, ckpt = ctx.saved_tensors
        rows, ch = u.shape
        N = A.shape[1]
        with _on(u.device):
            dy = torch.zeros_like(u) if dy is None else _activation("the gradient", dy, rows, ch, u)
            dfinal = None if dfinal is None else dfinal.contiguous()
            new = lambda n: torch.empty((rows, n), dtype=u.dtype, device=u.device)
            du, dd, dB, dC, dz = new(ch), new(ch), new(N), new(N), new(ch) if z is not None else None
            dstate = torch.empty_like(state) if state is not None and ctx.needs_input_grad[10] else None
            dp = torch.empty(ch * (N + 2), device=u.device)
            ws = _workspace(_bytes("eventad_selective_scan_workspace", rows, ch, N, 1), u.device)
            call("eventad_selective_scan_bwd", _p(u), _ld(u), _p(delta), _ld(delta), _p(A), _p(B), _ld(B), _p(C), _ld(C), _p(D), _p(z),
                 _ld(z), _p(bias), _p(starts), ctx.clips, _p(state), _p(ckpt), _p(dy), _ld(dy), _p(dfinal), _p(du), ch, _p(dd), ch,
                 _p(dB), N, _p(dC), N, _p(dz), ch, _p(dstate), _p(dp), _p(ws), ws.numel(), rows, ch, N, ctx.softplus,
                 _DTYPE[u.dtype], stream_handle())
        dA = dp[:ch * N].view(ch, N)
        return (du, dd, dA, dB, dC, dp[ch * N:ch * (N + 1)] if D is not None else None, dz,
                dp[ch * (N + 1):] if bias is not None else None, None, None, dstate, None, None)


def _scan_args(u, delta, A, B, C, D, z, bias, state, clips):
    dev, f32 = _gpu(u), torch.float32
    u = _activation("u", u, None, None)
    rows, ch = u.shape
    if ch < 1 or not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATE:
        _fail("A must be [channels, states] with 1..%d states, u [rows, channels] with at least one channel", MAX_STATE)
    N = A.shape[1]
    delta = _activation("delta", delta, rows, ch, u)
    A = _tensor("A", A, (ch, N), f32, dev)
    B, C = _activation("B", B, rows, N, u), _activation("C", C, rows, N, u)
    D, bias = _tensor("D", D, (ch,), f32, dev), _tensor("delta_bias", bias, (ch,), f32, dev)
    z = None if z is None else _activation("z", z, rows, ch, u)
    state = _tensor("state", state, (clips, ch, N), f32, dev)
    return u, delta, A, B, C, D, z, bias, state


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=True, clip_start=None, state=None,
                   return_state=False):
    """s_t = softplus(delta_t + delta_bias);  h_t = exp(s_t A) h_{t-1} + s_t u_t B_t;  y_t = (C_t . h_t + D u_t) silu(z_t).

    u, delta, z [rows, channels]; B, C [rows, states], shared by the channels; A float32 [channels, states], states 1..64;
    D, delta_bias float32 [channels].  D, z and delta_bias may be None; delta_softplus=False takes delta + delta_bias as the step
    itself.  state float32 [clips, channels, states] = h in front of each clip's first row (None: zeros).
    -> y, or (y, final_state) with return_state: h behind each clip's last row (an empty clip keeps its state)."""
    starts, clips = _clips(clip_start, u.shape[0] if isinstance(u, torch.Tensor) else 0, _gpu(u))
    u, delta, A, B, C, D, z, delta_bias, state = _scan_args(u, delta, A, B, C, D, z, delta_bias, state, clips)
    with _on(u.device):
        if _needs_grad(u, delta, A, B, C, D, z, delta_bias, state):
            y, final = _ScanFn.apply(u, delta, A, B, C, D, z, delta_bias, starts, clips, state, int(bool(delta_softplus)), return_state)
        else:
            y, final, _ = _scan_fwd(u, delta, A, B, C, D, z, delta_bias, starts, clips, state, int(bool(delta_softplus)), return_state, False)
    return (y, final) if return_state else y


def selective_scan_step(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, delta_softplus=True, state_out=None):
    """One row per clip: u, delta, z [clips, channels], B, C [clips, states], state float32 [clips, channels, states] contiguous.
    The state is moved on in place, or -- state_out given, a contiguous tensor like it that does not overlap it -- written there
    and left as it was.  -> y [clips, channels]."""
    if _needs_grad(u, delta, A, B, C, state, D, z, delta_bias):
        _fail("the single-token form has no gradient: use selective_scan, or torch.no_grad()")
    u, delta, A, B, C, D, z, delta_bias, checked = _scan_args(u, delta, A, B, C, D, z, delta_bias, state, u.shape[0])
    if checked is not state or checked is None:
        _fail("state must be contiguous float32 [clips, channels, states]")
    out = _state_out(state, state_out)
    clips, ch = u.shape
    with _on(u.device):
        y = torch.empty((clips, ch), dtype=u.dtype, device=u.device)
        call("eventad_selective_scan_step", _p(u), _ld(u), _p(delta), _ld(delta), _p(A), _p(B), _ld(B), _p(C), _ld(C), _p(D), _p(z), _ld(z),
             _p(delta_bias), _p(state), _p(out), _p(y), ch, clips, ch, A.shape[1], int(bool(delta_softplus)), _DTYPE[u.dtype],
             stream_handle())
        torch.autograd.graph.increment_version(out)
    return y


# ------------------------------------------------------------------------------------------------------------- RMS norm
def _norm_args(x, weight, residual, eps):
    dev = _gpu(x)
    x = _activation("x", x, None, None)
    if x.shape[1] < 1:
        _fail("x must have at least one channel")
    if not float(eps) >= 0.0:
        _fail("eps must not be negative")
    if weight is None:
        _fail("weight must be a float32 tensor")
    weight = _tensor("weight", weight, (x.shape[1],), torch.float32, dev)
    residual = None if residual is None else _activation("residual", residual, x.shape[0], x.shape[1], x)
    return x, weight, residual, float(eps)


def _norm_fwd(x, weight, residual, eps):
    rows, D = x.shape
    y = torch.empty((rows, D), dtype=x.dtype, device=x.device)
    total = torch.empty_like(y) if residual is not None else None
    call("eventad_rms_norm_fwd", _p(x), _ld(x), _p(residual), _ld(residual), _p(weight), _p(total), D, _p(y), D, rows, D, eps,
         _DTYPE[x.dtype], stream_handle())
    return y, total


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        y, total = _norm_fwd(x, weight, residual, eps)
        ctx.save_for_backward(x if total is None else total, weight)
        ctx.eps = eps
        return y, total

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dtotal):
        h, weight = ctx.saved_tensors
        rows, D = h.shape
        with _on(h.device):
            dy = torch.zeros_like(h) if dy is None else _activation("the gradient", dy, rows, D, h)
            dtotal = None if dtotal is None else _activation("the gradient", dtotal, rows, D, h)
            dh = torch.empty((rows, D), dtype=h.dtype, device=h.device)
            dw = torch.empty(D, device=h.device)
            ws = _workspace(_bytes("eventad_rms_norm_workspace", rows, D), h.device)
            call("eventad_rms_norm_bwd", _p(h), _ld(h), _p(weight), _p(dy), _ld(dy), _p(dtotal), _ld(dtotal), _p(dh), D, _p(dw), _p(ws),
                 ws.numel(), rows, D, ctx.eps, _DTYPE[h.dtype], stream_handle())
        return dh, dw, dh if ctx.needs_input_grad[2] else None, None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the channels of a row, weight float32 [channels].  With a residual (like x)
    h = x + residual rounded to their type -- the norm and its gradient are those of the stored sum -- and the result is (y, h);
    without one h = x and the result is y."""
    x, weight, residual, eps = _norm_args(x, weight, residual, eps)
    with _on(x.device):
        y, total = _NormFn.apply(x, weight, residual, eps) if _needs_grad(x, weight, residual) else _norm_fwd(x, weight, residual, eps)
    return y if residual is None else (y, total)


def rms_norm_fp8(x, weight, residual=None, eps=1e-6):
    """rms_norm's y in 8 bits for a scaled matrix product: scale float32 [rows] = max|y| / 448 of the row (1 for a row of zeros),
    q torch.float8_e4m3fn [rows, channels] = y / scale rounded to nearest even.  -> (q, scale), or (q, scale, h) with a residual."""
    if _needs_grad(x, weight, residual):
        _fail("the 8-bit form has no gradient: use rms_norm, or torch.no_grad()")
    x, weight, residual, eps = _norm_args(x, weight, residual, eps)
    rows, D = x.shape
    with _on(x.device):
        q = torch.empty((rows, D), dtype=torch.float8_e4m3fn, device=x.device)
        scale = torch.empty(rows, device=x.device)
        total = torch.empty((rows, D), dtype=x.dtype, device=x.device) if residual is not None else None
        call("eventad_rms_norm_fp8", _p(x), _ld(x), _p(residual), _ld(residual), _p(weight), _p(total), D, _p(q), D, _p(scale), rows, D, eps,
             _DTYPE[x.dtype], stream_handle())
    return (q, scale) if residual is None else (q, scale, total)
