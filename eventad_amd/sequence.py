"""Sequence operators over packed clips: a short causal convolution, a selective state-space scan and a root-mean-square
norm (csrc/seqconv.hip, seqscan.hip, rmsnorm.hip) -- what a state-space block over a clip's events or nodes needs beside its
matrix products.  The reference's temporal part is the GRU of its head (models/EventAD.py:62-97); these have no counterpart
there.

Rows are packed: activations are [rows, channels], clip s owns rows clip_start[s] .. clip_start[s+1]-1 (int32 on the device,
not decreasing; below 0 counts as 0, above rows as rows; None = all rows are one clip); rows of no clip give zeros and take
no part in a gradient.
Activations are float32, bfloat16 or float16, all of one call alike; parameters and scan states are float32.  A row may be a
slice of a wider array (any row stride); an array whose channels are not adjacent is copied first.  Up to 2^20 channels (the
norm: 2^24), 2^31 rows and 2^30 clips.

Every function launches on the current stream of its tensors' device, waits for nothing, and can be captured into a graph;
workspaces come from torch's allocator per call, so captured graphs do not share one.  torch.jit.trace and make_fx cannot record
the functions and are refused.  The functions are differentiable
(except the single-token and 8-bit forms, which refuse inputs that need a gradient); gradients are not differentiable
again, and there are no forward-mode derivatives.  There is no CPU path: tensors must be on a GPU."""
import contextlib
import ctypes
import functools

import torch
from torch.autograd import forward_ad

from ._lib import NativeError, load

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACT = {None: 0, "silu": 1}
_F32, _I32 = torch.float32, torch.int32
_Tensor = torch.Tensor
_tracing, _modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack
MAX_TAPS, MAX_STATE = 8, 64
_MAX_LD = 1 << 24               # row strides above this are taken by copying the array; no more channels than that
_MAX_CLIPS = (1 << 30) - 1      # (the library numbers clips, and bisects their offsets, in 32 bits)

# A single-token call is bound by this file: the checks below compare identities and device numbers, read each attribute once
# and pass plain integers to the library.
#
# A backward pass checks its saved tensors like a call's arguments and takes their strides anew: what a saved-tensor hook gives back
# (torch.autograd.graph.save_on_cpu, say) need not be laid out as what it was given.


def _fail(msg, *args):
    raise RuntimeError("eventad_amd.sequence: " + msg % args)


_functions = {}


def _call(name, *args):
    f = _functions.get(name)
    if f is None:
        f = _functions[name] = getattr(load(), name)
    rc = f(*args)
    if rc:
        raise NativeError("%s failed with code %d%s" % (name, rc, {-1: " (bad argument)", -3: " (too large for one launch)"}.get(rc, " (hipError_t)")))


def _device(t):
    """The GPU's number."""
    if not isinstance(t, _Tensor):
        _fail("expected a tensor, got %s", type(t).__name__)
    index = t.get_device() if t.is_cuda else -1
    if index < 0:
        _fail("tensors must be on a GPU (there is no CPU path)")
    return index


def _elsewhere(index):
    return index != torch._C._cuda_getDevice()


_here = contextlib.nullcontext()


def _on(index):
    return torch.cuda.device(index) if _elsewhere(index) else _here


def _stream(index):
    return torch._C._cuda_getCurrentRawStream(index)


def _rows(name, t, shape, dtype, index):
    """Checks an array [rows, channels] (shape None: any) -> it with adjacent channels, and its row stride in elements."""
    if not (t.__class__ is _Tensor or isinstance(t, _Tensor)) or t.dtype is not dtype or t.get_device() != index:
        _fail("%s must be a %s tensor on GPU %d", name, dtype, index)
    if shape is None:
        shape = t.shape
        if len(shape) != 2:
            _fail("%s has %d dimensions, expected [rows, channels]", name, len(shape))
    elif t.shape != shape:
        _fail("%s has shape %s, expected %s", name, tuple(t.shape), shape)
    n, m = shape
    ld, step = t.stride()
    if step == 1 and m <= ld <= _MAX_LD:
        return t, ld
    if m > _MAX_LD:
        _fail("%s has %d channels, more than 2^24", name, m)
    if n <= 1 and (step == 1 or m <= 1):                         # (one row: any stride)
        return t, m
    return t.contiguous(), m


def _tensor(name, t, shape, dtype, index):
    """Checks a parameter or a state -> it, contiguous (None stays None)."""
    if t is None:
        return None
    if not (t.__class__ is _Tensor or isinstance(t, _Tensor)) or t.dtype is not dtype or t.get_device() != index:
        _fail("%s must be a %s tensor on GPU %d", name, dtype, index)
    if t.shape != shape:
        _fail("%s has shape %s, expected %s", name, tuple(t.shape), shape)
    return t if t.is_contiguous() else t.contiguous()


def _gradient(g, like, shape, index):
    """An incoming gradient as an array [rows, channels] of like's type, zeros for None; with its row stride."""
    if g is None:
        g = torch.zeros_like(like, memory_format=torch.contiguous_format)
    return _rows("the gradient", g, shape, like.dtype, index)


def _p(t):
    return None if t is None else t.data_ptr()


def _clips(clip_start, index):
    if clip_start is None:
        return None, 1
    if not isinstance(clip_start, torch.Tensor) or clip_start.dtype is not _I32 or clip_start.get_device() != index or \
            clip_start.dim() != 1 or not 2 <= clip_start.numel() <= _MAX_CLIPS + 1:
        _fail("clip_start must be int32[clips + 1] on GPU %d, with 1..%d clips", index, _MAX_CLIPS)
    return clip_start.contiguous(), clip_start.numel() - 1


def _proxies():
    from torch.fx.experimental.proxy_tensor import get_proxy_mode
    return get_proxy_mode() is not None


def _needs_grad(*tensors):
    # A tracer records torch's own operations: of these calls the allocation of the result, and nothing that fills it.
    if _tracing() or (_modes() and _proxies()):
        _fail("the call cannot be recorded by torch.jit.trace or make_fx")
    if forward_ad._current_level >= 0:                           # (inside forward_ad.dual_level or torch.func.jvp)
        for t in tensors:
            if isinstance(t, _Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                _fail("there is no forward-mode derivative")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and isinstance(t, _Tensor) and t.requires_grad:
                return True
    return False


@functools.lru_cache(maxsize=4096)
def _bytes(name, *shape):
    """What the library's size function says for a shape."""
    n = ctypes.c_int64(0)
    _call(name, *shape, ctypes.byref(n))
    return n.value


def _workspace(nbytes, like):
    return like.new_empty(max(16, nbytes), dtype=torch.uint8)


def _state_out(state, out):
    if out is None or out is state:
        return state
    if not isinstance(out, torch.Tensor) or out.dtype is not state.dtype or out.get_device() != state.get_device() or \
            out.shape != state.shape or not out.is_contiguous():
        _fail("state_out must be a contiguous tensor like state")
    if abs(out.data_ptr() - state.data_ptr()) < state.numel() * state.element_size() and out.data_ptr() != state.data_ptr():
        _fail("state_out overlaps state")
    return out


class _Final(torch.autograd.Function):
    """Gradients as they are; an error where something is differentiated through them."""
    @staticmethod
    def forward(ctx, *grads):
        return grads

    @staticmethod
    def backward(ctx, *grads):
        _fail("gradients are not differentiable again")


def _once(backward):
    """For a backward pass with a graph of its own pending (create_graph): torch's once_differentiable, but its error comes whether or not
    the incoming gradient needs one, as these gradients depend on the saved inputs too."""
    def run(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        return _Final.apply(*(g if g is None else g.detach().requires_grad_() for g in out))
    return run


# ---------------------------------------------------------------------------------------------------- causal convolution
def _conv_args(x, weight, bias, state, activation, clips, index):
    if activation not in _ACT:
        _fail("activation must be None or 'silu', not %r", activation)
    if x.dtype not in _DTYPE:
        _fail("x must be float32, bfloat16 or float16, not %s", x.dtype)
    x, ldx = _rows("x", x, None, x.dtype, index)
    D = x.shape[1]
    taps = weight.shape[1] if isinstance(weight, torch.Tensor) and weight.dim() == 2 else 0
    if D < 1 or not 1 <= taps <= MAX_TAPS:
        _fail("weight must be [channels, taps] with 1..%d taps, x [rows, channels] with at least one channel", MAX_TAPS)
    weight = _tensor("weight", weight, (D, taps), _F32, index)
    bias = _tensor("bias", bias, (D,), _F32, index)
    state = _tensor("state", state, (clips, taps - 1, D), x.dtype, index)
    return x, ldx, weight, bias, state, taps


def _conv_fwd(x, ldx, w, bias, starts, clips, state, act, want_state):
    rows, D = x.shape
    taps = w.shape[1]
    y = x.new_empty((rows, D))
    final = x.new_empty((clips, taps - 1, D)) if want_state else None
    _call("eventad_causal_conv_fwd", _p(x), ldx, _p(w), _p(bias), _p(starts), clips, _p(state), _p(final), _p(y), D, rows, D, taps, act,
          _DTYPE[x.dtype], _stream(x.get_device()))
    return y, final


class _ConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, state, ldx, starts, clips, act, want_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, w, bias, state, starts)
        ctx.act = act
        return _conv_fwd(x, ldx, w, bias, starts, clips, state, act, want_state)

    @staticmethod
    @_once
    def backward(ctx, dy, dfinal):
        x, w, bias, state, starts = ctx.saved_tensors
        index = _device(x)
        with _on(index):
            starts, clips = _clips(starts, index)
            x, ldx, w, bias, state, K = _conv_args(x, w, bias, state, None, clips, index)
            rows, D = x.shape
            dy, ldy = _gradient(dy, x, (rows, D), index)
            dfinal = _tensor("the final state's gradient", dfinal, (clips, K - 1, D), x.dtype, index)
            dx = x.new_empty((rows, D))
            dstate = torch.empty_like(state) if state is not None and ctx.needs_input_grad[3] else None
            dp = w.new_empty(D * (K + 1))
            ws = _workspace(_bytes("eventad_causal_conv_workspace", rows, D, K), x)
            _call("eventad_causal_conv_bwd", _p(x), ldx, _p(w), _p(bias), _p(starts), clips, _p(state), _p(dy), ldy, _p(dfinal),
                  _p(dx), D, _p(dstate), _p(dp), _p(ws), ws.numel(), rows, D, K, ctx.act, _DTYPE[x.dtype], _stream(index))
        return dx, dp.as_strided((D, K), (K, 1)), dp.as_strided((D,), (1,), D * K) if bias is not None else None, dstate, None, None, None, None, None


def causal_conv(x, weight, bias=None, clip_start=None, state=None, activation="silu", return_state=False):
    """y_t = act(bias + sum_k weight[:, k] x_{t-(taps-1)+k}) per channel, inside every clip.

    x [rows, channels]; weight float32 [channels, taps], taps 1..8, weight[:, -1] multiplies the row itself; bias float32
    [channels]; activation None or "silu" (x sigmoid(x)).  state [clips, taps - 1, channels], of x's type, holds the inputs in
    front of each clip's first row, oldest first (None: zeros).
    -> y, or (y, final_state) with return_state: the inputs in front of the row that would follow each clip."""
    index = _device(x)
    if _elsewhere(index):
        with torch.cuda.device(index):
            return causal_conv(x, weight, bias, clip_start, state, activation, return_state)
    starts, clips = _clips(clip_start, index)
    x, ldx, weight, bias, state, _ = _conv_args(x, weight, bias, state, activation, clips, index)
    if _needs_grad(x, weight, bias, state):
        y, final = _ConvFn.apply(x, weight, bias, state, ldx, starts, clips, _ACT[activation], return_state)
    else:
        y, final = _conv_fwd(x, ldx, weight, bias, starts, clips, state, _ACT[activation], return_state)
    return (y, final) if return_state else y


def causal_conv_step(x, weight, state, bias=None, activation="silu", state_out=None):
    """One row per clip: x [clips, channels], state [clips, taps - 1, channels] contiguous.  The state is moved on in place, or
    -- state_out given, a contiguous tensor like it that does not overlap it -- written there and left as it was.  -> y [clips,
    channels]."""
    if _needs_grad(x, weight, state, bias, state_out):
        _fail("the single-token form has no gradient: use causal_conv, or torch.no_grad()")
    index = _device(x)
    if _elsewhere(index):
        with torch.cuda.device(index):
            return causal_conv_step(x, weight, state, bias, activation, state_out)
    x, ldx, weight, bias, checked, taps = _conv_args(x, weight, bias, state, activation, x.shape[0] if x.dim() else 0, index)
    if checked is not state or checked is None:
        _fail("state must be contiguous, of x's type, [clips, taps - 1, channels]")
    out = _state_out(state, state_out)
    clips, D = x.shape
    if clips > _MAX_CLIPS:
        _fail("%d clips, more than %d", clips, _MAX_CLIPS)
    y = x.new_empty((clips, D))
    _call("eventad_causal_conv_step", x.data_ptr(), ldx, weight.data_ptr(), _p(bias), state.data_ptr(), out.data_ptr(), y.data_ptr(), D, clips,
          D, taps, _ACT[activation], _DTYPE[x.dtype], _stream(index))
    torch.autograd.graph.increment_version(out)                  # (written behind autograd's back)
    return y


# -------------------------------------------------------------------------------------------------------- selective scan
def _scan_args(u, delta, A, B, C, D, z, bias, state, clips, index):
    """-> the checked tensors, and the row strides of u, delta, B, C, z"""
    dt = u.dtype
    if dt not in _DTYPE:
        _fail("u must be float32, bfloat16 or float16, not %s", dt)
    u, ldu = _rows("u", u, None, dt, index)
    wide = rows, ch = u.shape
    N = A.shape[1] if isinstance(A, torch.Tensor) and A.dim() == 2 else 0
    if ch < 1 or not 1 <= N <= MAX_STATE:
        _fail("A must be [channels, states] with 1..%d states, u [rows, channels] with at least one channel", MAX_STATE)
    delta, ldd = _rows("delta", delta, wide, dt, index)
    A = _tensor("A", A, (ch, N), _F32, index)
    B, ldb = _rows("B", B, (rows, N), dt, index)
    C, ldc = _rows("C", C, (rows, N), dt, index)
    D = _tensor("D", D, (ch,), _F32, index)
    z, ldz = (None, 0) if z is None else _rows("z", z, wide, dt, index)
    bias = _tensor("delta_bias", bias, (ch,), _F32, index)
    state = _tensor("state", state, (clips, ch, N), _F32, index)
    return (u, delta, A, B, C, D, z, bias, state), (ldu, ldd, ldb, ldc, ldz)


def _scan_fwd(u, delta, A, B, C, D, z, bias, state, lds, starts, clips, softplus, want_state, want_checkpoint):
    rows, ch = u.shape
    N = A.shape[1]
    ldu, ldd, ldb, ldc, ldz = lds
    y = u.new_empty((rows, ch))
    final = A.new_empty((clips, ch, N)) if want_state else None
    ckpt = _workspace(_bytes("eventad_selective_scan_checkpoint", rows, ch, N), u) if want_checkpoint else None
    ws = _workspace(_bytes("eventad_selective_scan_workspace", rows, ch, N, 0), u)
    _call("eventad_selective_scan_fwd", _p(u), ldu, _p(delta), ldd, _p(A), _p(B), ldb, _p(C), ldc, _p(D), _p(z), ldz, _p(bias), _p(starts), clips,
          _p(state), _p(final), _p(y), ch, _p(ckpt), _p(ws), ws.numel(), rows, ch, N, softplus, _DTYPE[u.dtype], _stream(u.get_device()))
    return y, final, ckpt


class _ScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, bias, state, lds, starts, clips, softplus, want_state):
        ctx.set_materialize_grads(False)
        y, final, ckpt = _scan_fwd(u, delta, A, B, C, D, z, bias, state, lds, starts, clips, softplus, want_state, True)
        ctx.save_for_backward(u, delta, A, B, C, D, z, bias, state, starts, ckpt)
        ctx.softplus = softplus
        return y, final

    @staticmethod
    @_once
    def backward(ctx, dy, dfinal):
        *t, starts, ckpt = ctx.saved_tensors
        index = _device(t[0])
        with _on(index):
            starts, clips = _clips(starts, index)
            (u, delta, A, B, C, D, z, bias, state), (ldu, ldd, ldb, ldc, ldz) = _scan_args(*t, clips, index)
            rows, ch = u.shape
            N = A.shape[1]
            ckpt = _tensor("the checkpoint", ckpt, (max(16, _bytes("eventad_selective_scan_checkpoint", rows, ch, N)),), torch.uint8, index)
            dy, ldy = _gradient(dy, u, (rows, ch), index)
            dfinal = _tensor("the final state's gradient", dfinal, (clips, ch, N), _F32, index)
            new = lambda n: u.new_empty((rows, n))
            du, dd, dB, dC, dz = new(ch), new(ch), new(N), new(N), new(ch) if z is not None else None
            dstate = torch.empty_like(state) if state is not None and ctx.needs_input_grad[8] else None
            dp = A.new_empty(ch * (N + 2))
            ws = _workspace(_bytes("eventad_selective_scan_workspace", rows, ch, N, 1), u)
            _call("eventad_selective_scan_bwd", _p(u), ldu, _p(delta), ldd, _p(A), _p(B), ldb, _p(C), ldc, _p(D), _p(z), ldz, _p(bias), _p(starts),
                  clips, _p(state), _p(ckpt), _p(dy), ldy, _p(dfinal), _p(du), ch, _p(dd), ch, _p(dB), N, _p(dC), N, _p(dz), ch,
                  _p(dstate), _p(dp), _p(ws), ws.numel(), rows, ch, N, ctx.softplus, _DTYPE[u.dtype], _stream(index))
        return (du, dd, dp.as_strided((ch, N), (N, 1)), dB, dC, dp.as_strided((ch,), (1,), ch * N) if D is not None else None, dz,
                dp.as_strided((ch,), (1,), ch * (N + 1)) if bias is not None else None, dstate, None, None, None, None, None)


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=True, clip_start=None, state=None,
                   return_state=False):
    """s_t = softplus(delta_t + delta_bias);  h_t = exp(s_t A) h_{t-1} + s_t u_t B_t;  y_t = (C_t . h_t + D u_t) silu(z_t).

    u, delta, z [rows, channels]; B, C [rows, states], shared by the channels; A float32 [channels, states], states 1..64;
    D, delta_bias float32 [channels].  D, z and delta_bias may be None; delta_softplus=False takes delta + delta_bias as the step
    itself.  An A of -inf is a state that forgets at once: it counts as -2.36e38, which every step of 1e-36 or more takes to
    exp(s A) = 0; a step of 0 leaves the state as it is.  state float32 [clips, channels, states] = h in front of each clip's
    first row (None: zeros).
    -> y, or (y, final_state) with return_state: h behind each clip's last row (an empty clip keeps its state).

    Every clip's end inside a group of 16 rows costs that group another turn: a batch whose clips are all a row or two long is
    better served by selective_scan_step.  With a gradient pending, the call keeps 2 x channels x (states, rounded up to a power of
    two from 4 to 64) bytes per 4 rows, and the backward pass takes 2 bytes per row and channel up to 16 states (8 up to 32, 32 up to
    64) for as long as it runs."""
    index = _device(u)
    if _elsewhere(index):
        with torch.cuda.device(index):
            return selective_scan(u, delta, A, B, C, D, z, delta_bias, delta_softplus, clip_start, state, return_state)
    starts, clips = _clips(clip_start, index)
    t, lds = _scan_args(u, delta, A, B, C, D, z, delta_bias, state, clips, index)
    softplus = int(bool(delta_softplus))
    if _needs_grad(*t):
        y, final = _ScanFn.apply(*t, lds, starts, clips, softplus, return_state)
    else:
        y, final, _ = _scan_fwd(*t, lds, starts, clips, softplus, return_state, False)
    return (y, final) if return_state else y


def selective_scan_step(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, delta_softplus=True, state_out=None):
    """One row per clip: u, delta, z [clips, channels], B, C [clips, states], state float32 [clips, channels, states] contiguous.
    The state is moved on in place, or -- state_out given, a contiguous tensor like it that does not overlap it -- written there
    and left as it was.  -> y [clips, channels]."""
    if _needs_grad(u, delta, A, B, C, state, D, z, delta_bias, state_out):
        _fail("the single-token form has no gradient: use selective_scan, or torch.no_grad()")
    index = _device(u)
    if _elsewhere(index):
        with torch.cuda.device(index):
            return selective_scan_step(u, delta, A, B, C, state, D, z, delta_bias, delta_softplus, state_out)
    (u, delta, A, B, C, D, z, delta_bias, checked), (ldu, ldd, ldb, ldc, ldz) = \
        _scan_args(u, delta, A, B, C, D, z, delta_bias, state, u.shape[0] if u.dim() else 0, index)
    if checked is not state or checked is None:
        _fail("state must be contiguous float32 [clips, channels, states]")
    out = _state_out(state, state_out)
    clips, ch = u.shape
    if clips > _MAX_CLIPS:
        _fail("%d clips, more than %d", clips, _MAX_CLIPS)
    y = u.new_empty((clips, ch))
    _call("eventad_selective_scan_step", u.data_ptr(), ldu, delta.data_ptr(), ldd, A.data_ptr(), B.data_ptr(), ldb, C.data_ptr(), ldc, _p(D),
          _p(z), ldz, _p(delta_bias), state.data_ptr(), out.data_ptr(), y.data_ptr(), ch, clips, ch, A.shape[1], 1 if delta_softplus else 0,
          _DTYPE[u.dtype], _stream(index))
    torch.autograd.graph.increment_version(out)
    return y


# ------------------------------------------------------------------------------------------------------------- RMS norm
def _norm_args(x, weight, residual, eps, index):
    if x.dtype not in _DTYPE:
        _fail("x must be float32, bfloat16 or float16, not %s", x.dtype)
    x, ldx = _rows("x", x, None, x.dtype, index)
    rows, D = x.shape
    if D < 1 or weight is None:
        _fail("x must have at least one channel, and weight must be a float32 tensor")
    eps = float(eps)
    if not eps >= 0.0:
        _fail("eps must not be negative")
    weight = _tensor("weight", weight, (D,), _F32, index)
    residual, ldr = (None, 0) if residual is None else _rows("residual", residual, (rows, D), x.dtype, index)
    return x, ldx, weight, residual, ldr, eps


def _norm_fwd(x, ldx, weight, residual, ldr, eps):
    rows, D = x.shape
    y = x.new_empty((rows, D))
    total = x.new_empty((rows, D)) if residual is not None else None
    _call("eventad_rms_norm_fwd", x.data_ptr(), ldx, _p(residual), ldr, weight.data_ptr(), _p(total), D, y.data_ptr(), D, rows, D, eps,
          _DTYPE[x.dtype], _stream(x.get_device()))
    return y, total


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, ldx, ldr, eps):
        ctx.set_materialize_grads(False)
        y, total = _norm_fwd(x, ldx, weight, residual, ldr, eps)
        ctx.save_for_backward(x if total is None else total, weight)
        ctx.eps = eps
        return y, total

    @staticmethod
    @_once
    def backward(ctx, dy, dtotal):
        h, weight = ctx.saved_tensors
        index = _device(h)
        with _on(index):
            h, ldh, weight, _, _, eps = _norm_args(h, weight, None, ctx.eps, index)
            rows, D = h.shape
            dy, ldy = _gradient(dy, h, (rows, D), index)
            dtotal, ldt = (None, 0) if dtotal is None else _gradient(dtotal, h, (rows, D), index)
            dh = h.new_empty((rows, D))
            dw = weight.new_empty(D)
            ws = _workspace(_bytes("eventad_rms_norm_workspace", rows, D), h)
            _call("eventad_rms_norm_bwd", _p(h), ldh, _p(weight), _p(dy), ldy, _p(dtotal), ldt, _p(dh), D, _p(dw), _p(ws), ws.numel(), rows,
                  D, eps, _DTYPE[h.dtype], _stream(index))
        return dh, dw, dh if ctx.needs_input_grad[2] else None, None, None, None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the channels of a row, weight float32 [channels].  With a residual (like x)
    h = x + residual rounded to their type -- the norm and its gradient are those of the stored sum -- and the result is (y, h);
    without one h = x and the result is y."""
    index = _device(x)
    if _elsewhere(index):
        with torch.cuda.device(index):
            return rms_norm(x, weight, residual, eps)
    x, ldx, weight, residual, ldr, eps = _norm_args(x, weight, residual, eps, index)
    if _needs_grad(x, weight, residual):
        y, total = _NormFn.apply(x, weight, residual, ldx, ldr, eps)
    else:
        y, total = _norm_fwd(x, ldx, weight, residual, ldr, eps)
    return y if residual is None else (y, total)


def rms_norm_fp8(x, weight, residual=None, eps=1e-6):
    """rms_norm's y in 8 bits for a scaled matrix product: scale float32 [rows] = max|y| / 448 of the row (1 where that is below the
    smallest normal number, 1.2e-38: a row of zeros comes back as zeros), q torch.float8_e4m3fn [rows, channels] = y / scale
    rounded to nearest even.  -> (q, scale), or (q, scale, h) with a residual."""
    if _needs_grad(x, weight, residual):
        _fail("the 8-bit form has no gradient: use rms_norm, or torch.no_grad()")
    index = _device(x)
    if _elsewhere(index):
        with torch.cuda.device(index):
            return rms_norm_fp8(x, weight, residual, eps)
    x, ldx, weight, residual, ldr, eps = _norm_args(x, weight, residual, eps, index)
    rows, D = x.shape
    q = x.new_empty((rows, D), dtype=torch.float8_e4m3fn)
    scale = x.new_empty(rows, dtype=_F32)
    total = x.new_empty((rows, D)) if residual is not None else None
    _call("eventad_rms_norm_fp8", x.data_ptr(), ldx, _p(residual), ldr, weight.data_ptr(), _p(total), D, q.data_ptr(), D, scale.data_ptr(), rows,
          D, eps, _DTYPE[x.dtype], _stream(index))
    return (q, scale) if residual is None else (q, scale, total)
