"""What eventad_amd/sequence.py hands to the library, on the CPU: the library's calls are replaced by a record of their arguments."""
import pytest
import torch

from eventad_amd import sequence as S


@pytest.fixture
def calls(monkeypatch):
    """The calls made, as (name, arguments); tensors of the CPU pass the checks in the place of a GPU's."""
    made = []
    monkeypatch.setattr(S, "_device", lambda t: t.get_device())
    monkeypatch.setattr(S, "_elsewhere", lambda index: False)
    monkeypatch.setattr(S, "_stream", lambda index: 0)
    monkeypatch.setattr(S, "_bytes", lambda name, *shape: 64)
    monkeypatch.setattr(S, "_call", lambda name, *args: made.append((name, args)))
    return made


ROWS, CH, N, TAPS, CLIPS = 6, 4, 3, 4, 2


def run(op, state=True):
    """One differentiable call on column slices of wider arrays -> (outputs, inputs that need a gradient)"""
    wide = torch.randn(ROWS, 5 * CH + 2 * N, requires_grad=True)
    at = lambda c, n: wide[:, c:c + n]
    starts = torch.tensor([0, 2, ROWS], dtype=torch.int32)
    x = at(1, CH)
    if op == "conv":
        s = torch.randn(CLIPS, TAPS - 1, CH, requires_grad=True) if state else None
        return S.causal_conv(x, torch.randn(CH, TAPS), torch.randn(CH), starts, s, return_state=True), [t for t in (wide, s) if t is not None]
    if op == "scan":
        s = torch.randn(CLIPS, CH, N, requires_grad=True) if state else None
        return S.selective_scan(x, at(CH, CH), -torch.ones(CH, N), at(3 * CH, N), at(4 * CH, N), torch.ones(CH), at(2 * CH, CH), torch.ones(CH), True,
                                starts, s, True), [t for t in (wide, s) if t is not None]
    return (S.rms_norm(x, torch.ones(CH)),), [wide]


# (array, row stride) as positions in the arguments of each backward call
STRIDED = {"conv": [(0, 1), (7, 8)], "scan": [(0, 1), (2, 3), (5, 6), (7, 8), (10, 11), (17, 18)], "norm": [(0, 1), (3, 4)]}


@pytest.mark.parametrize("op", ["conv", "scan", "norm"])
@pytest.mark.parametrize("spread", [False, True])
def test_backward_takes_the_strides_of_what_saved_tensor_hooks_return(calls, op, spread):
    """A hook (offloading, say) may give back a packed copy of a slice, or a slice of an array wider still."""
    back = []

    def unpack(t):
        if t.dim() == 2 and t.dtype == torch.float32:
            t = torch.cat([t, torch.zeros(t.shape[0], 7)], 1)[:, :t.shape[1]] if spread else t.clone().contiguous()
        back.append(t)
        return t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out, leaves = run(op)
    back.clear()
    kept = [torch.randn_like(o) for o in out]
    torch.autograd.grad(out, leaves, kept)
    name, args = next(c for c in calls if c[0].endswith("_bwd"))
    strides = {t.data_ptr(): t.stride(0) for t in back + kept if t.dim() == 2}
    for p, ld in STRIDED[op]:
        assert args[p] in strides, (name, p)
        assert args[ld] == strides[args[p]], (name, p, args[ld], strides[args[p]])
    for t in back:                                               # parameters and states: no strides are passed for them
        if t.dim() == 3 or (t.dim() == 2 and t.shape[0] == CH):
            assert t.data_ptr() not in args or t.is_contiguous()


@pytest.mark.parametrize("op", ["conv", "scan", "norm"])
def test_backward_refuses_what_is_no_copy_of_the_saved_tensor(calls, op):
    for change in (lambda t: t.half() if t.dtype == torch.float32 else t, lambda t: t[:-1], lambda t: t.new_zeros(t.numel())):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            out, leaves = run(op)
        with pytest.raises(RuntimeError, match="eventad_amd.sequence"):
            torch.autograd.grad(out, leaves, [torch.randn_like(o) for o in out])


def every_form():
    """(name, tensors, call of those tensors): each entry point with every tensor that it takes a derivative of"""
    r, starts = torch.randn, torch.tensor([0, 2, ROWS], dtype=torch.int32)
    rows = dict(u=r(ROWS, CH), delta=r(ROWS, CH), A=r(CH, N), B=r(ROWS, N), C=r(ROWS, N), D=r(CH), z=r(ROWS, CH), delta_bias=r(CH))
    norm = dict(x=r(ROWS, CH), weight=r(CH), residual=r(ROWS, CH))
    return [("causal_conv", dict(x=r(ROWS, CH), weight=r(CH, TAPS), bias=r(CH), state=r(CLIPS, TAPS - 1, CH)), lambda **t: S.causal_conv(clip_start=starts, **t)),
            ("causal_conv_step", dict(x=r(ROWS, CH), weight=r(CH, TAPS), state=r(ROWS, TAPS - 1, CH), bias=r(CH)), S.causal_conv_step),
            ("selective_scan", dict(rows, state=r(CLIPS, CH, N)), lambda **t: S.selective_scan(clip_start=starts, **t)),
            ("selective_scan_step", dict(rows, state=r(ROWS, CH, N)), S.selective_scan_step), ("rms_norm", norm, S.rms_norm), ("rms_norm_fp8", norm, S.rms_norm_fp8)]


def test_forward_mode_derivatives_are_refused(calls):
    for name, tensors, f in every_form():
        for dual in tensors:
            with torch.autograd.forward_ad.dual_level():
                t = dict(tensors)
                t[dual] = torch.autograd.forward_ad.make_dual(t[dual], torch.ones_like(t[dual]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(**t)
        with torch.autograd.forward_ad.dual_level():
            f(**tensors)                                         # nothing dual among them
    assert len(calls) == 6


@pytest.mark.parametrize("pending", [False, True])
def test_tracers_are_refused(calls, pending):
    """They would record the result's allocation and nothing that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    for name, tensors, f in every_form():
        if pending and (name.endswith("_step") or name.endswith("_fp8")):
            continue
        keys = list(tensors)
        call = lambda *t: f(**dict(zip(keys, t)))
        args = tuple(t.clone().requires_grad_(pending) for t in tensors.values())
        for record in (lambda: torch.jit.trace(call, args, check_trace=False), lambda: make_fx(call)(*args), lambda: make_fx(call, tracing_mode="fake")(*args)):
            with pytest.raises(RuntimeError, match="recorded by torch.jit.trace or make_fx"):
                record()
    assert not calls


def test_state_out_that_needs_a_gradient_is_refused(calls):
    """Nothing may be written into a leaf, or into a tensor of a graph, behind autograd's back."""
    for name, tensors, f in every_form():
        if name.endswith("_step"):
            out = torch.zeros_like(tensors["state"], requires_grad=True)
            for t in (out, out * 1.0):
                with pytest.raises(RuntimeError, match="has no gradient"):
                    f(state_out=t, **tensors)
            with torch.no_grad():
                f(state_out=out, **tensors)
    assert len(calls) == 2


@pytest.mark.parametrize("op", ["conv", "scan", "norm"])
def test_differentiating_twice_is_an_error_and_never_a_silent_zero(calls, op):
    out, leaves = run(op)
    loss = sum(o.sum() for o in out)
    plain = torch.autograd.grad(loss, leaves, retain_graph=True)
    grads = torch.autograd.grad(loss, leaves, create_graph=True)                # by itself it may be asked for
    assert all(g.requires_grad for g in grads) and not any(g.requires_grad for g in plain)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        (loss + sum(g.sum() for g in grads)).backward()
    for t in leaves:
        t.grad = None
    out, leaves = run(op)
    sum(o.sum() for o in out).backward(create_graph=True)
    with torch.no_grad():
        torch.nn.utils.clip_grad_norm_(leaves, 1.0)


def batch_of(sizes):
    from eventad_amd.batch import EventBatch
    clip = lambda n: dict(x=torch.zeros(n, 1), pos=torch.rand(n, 2), t=torch.zeros(n), bbox=torch.zeros(1, 5), bbox0=torch.zeros(1, 5), width=64, height=64, time_window=1)
    return EventBatch.from_clips([clip(n) for n in sizes])


def test_offsets_from_a_batch_of_events():
    """Made from the index per event, empty clips at the ends and in between included."""
    for sizes in ([3, 5, 1], [0, 4, 0, 0, 2, 0], [7], [0, 0]):
        b = batch_of(sizes)
        clip_start = torch.searchsorted(b.batch, torch.arange(b.num_graphs + 1, device=b.batch.device)).int()
        assert clip_start.tolist() == [sum(sizes[:i]) for i in range(len(sizes) + 1)]


def test_launches_past_the_stated_sizes_are_refused():
    import ctypes
    from eventad_amd import _lib
    lib, buf = _lib.load(), ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)     # only ever compared with NULL
    norm = lambda rows, ch: lib.eventad_rms_norm_fwd(buf, ch, None, 0, buf, None, 0, buf, ch, rows, ch, 1e-6, 0, None)
    for rows, ch in ((268435441, 1), (268435441, 64), (16777216, 4096)):
        assert norm(rows, ch) == -3
    step = lambda clips, ch: lib.eventad_causal_conv_step(buf, ch, buf, None, buf, buf, buf, ch, clips, ch, 4, 1, 0, None)
    assert step(4294967296 // 31 + 1, 31) == -3 and step(4294967296 // 8 + 1, 32) == -3


def test_sizes_past_32_bits_are_refused_and_not_cut_short(calls):
    """ctypes passes the low 32 bits of an int.  The arrays are one element each, repeated."""
    r, big = lambda *s: torch.zeros(1).expand(*s), (1 << 32) + 2
    clips = torch.zeros(1, dtype=torch.int32).expand(big + 1)
    x, w, A, B = r(6, CH), r(CH, TAPS), r(CH, N), r(6, N)
    for f in (lambda: S.rms_norm(r(1, big), r(big)), lambda: S.rms_norm_fp8(r(1, big), r(big)), lambda: S.causal_conv(r(1, big), r(big, TAPS)),
              lambda: S.causal_conv(x, w, clip_start=clips), lambda: S.selective_scan(x, x, A, B, B, clip_start=clips)):
        with pytest.raises(RuntimeError, match="more than 2\\^24|1\\.\\.1073741823 clips"):
            f()

    many = 1 << 30                                               # rows of a single-token call; memory that nobody touches
    u, h = torch.empty(many, 1, dtype=torch.bfloat16), torch.empty(many, 1, 1)
    for f in (lambda: S.causal_conv_step(u, r(1, 1), torch.empty(many, 0, 1, dtype=torch.bfloat16)), lambda: S.selective_scan_step(u, u, r(1, 1), u, u, h)):
        with pytest.raises(RuntimeError, match="1073741824 clips"):
            f()
    assert not calls


def test_more_clips_than_can_be_bisected_are_refused_by_the_library():
    import ctypes
    from eventad_amd import _lib
    lib, buf = _lib.load(), ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)     # only ever compared with NULL
    for clips in (1 << 30, (1 << 31) - 1):
        assert lib.eventad_causal_conv_fwd(buf, 8, buf, None, buf, clips, None, None, buf, 8, 4, 8, 4, 1, 0, None) == -1
        assert lib.eventad_causal_conv_bwd(buf, 8, buf, None, buf, clips, None, buf, 8, None, buf, 8, None, buf, buf, 1 << 20, 4, 8, 4, 1, 0, None) == -1
        assert lib.eventad_selective_scan_fwd(buf, 8, buf, 8, buf, buf, 16, buf, 16, None, None, 0, None, buf, clips, None, None, buf, 8, None, buf, 1 << 16, 4, 8, 16, 1,
                                              0, None) == -1
        assert lib.eventad_selective_scan_bwd(buf, 8, buf, 8, buf, buf, 16, buf, 16, None, None, 0, None, buf, clips, None, buf, buf, 8, None, buf, 8, buf, 8, buf, 16,
                                              buf, 16, None, 0, None, buf, buf, 1 << 20, 4, 8, 16, 1, 0, None) == -1
