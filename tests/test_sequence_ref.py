"""The float64 restatement of the sequence operators against autograd and finite differences, and the library's refusals that
need no GPU."""
import ctypes

import pytest
import torch

from oracle import sequence_ref as R


def _autograd_conv(L, starts, silu):
    rows, K = L["x"].shape[0], L["weight"].shape[1]
    outs, finals = [torch.zeros_like(L["x"][0])] * rows, []
    for s, (lo, hi) in enumerate(R.clips_of(starts, rows)):
        ext = torch.cat([L["state"][s], L["x"][lo:hi]])
        finals.append(ext[hi - lo:])
        for t in range(hi - lo):
            p = (ext[t:t + K] * L["weight"].t()).sum(0) + L["bias"]
            outs[lo + t] = torch.nn.functional.silu(p) if silu else p
    return torch.stack(outs), torch.stack(finals)


def _autograd_scan(L, starts, softplus):
    rows = L["u"].shape[0]
    outs, finals = [torch.zeros_like(L["u"][0])] * rows, []
    for s, (lo, hi) in enumerate(R.clips_of(starts, rows)):
        h = L["state"][s]
        for t in range(lo, hi):
            d = L["delta"][t] + L["delta_bias"]
            d = torch.nn.functional.softplus(d) if softplus else d
            h = torch.exp(d[:, None] * L["A"]) * h + (d * L["u"][t])[:, None] * L["B"][t]
            outs[t] = ((h * L["C"][t]).sum(1) + L["D"] * L["u"][t]) * torch.nn.functional.silu(L["z"][t])
        finals.append(h)
    return torch.stack(outs), torch.stack(finals)


def _leaves(gen, **shapes):
    return {k: torch.randn(s, generator=gen, dtype=torch.float64).requires_grad_() for k, s in shapes.items()}


STARTS = [1, 4, 4, 9, 10, 12]                                     # a row in front, an empty clip, a single row, two rows behind


@pytest.mark.parametrize("flag", [True, False])
@pytest.mark.parametrize("op", ["conv", "scan"])
def test_restated_gradients_equal_autograd_and_differences(op, flag):
    gen = torch.Generator().manual_seed(5)
    if op == "conv":
        L = _leaves(gen, x=(14, 3), weight=(3, 4), bias=(3,), state=(5, 3, 3))
        f = lambda: _autograd_conv(L, STARTS, flag)
        ref = lambda **k: R.conv(L["x"], L["weight"], L["bias"], STARTS, L["state"], flag, **k)
    else:
        L = _leaves(gen, u=(14, 3), delta=(14, 3), A=(3, 4), B=(14, 4), C=(14, 4), D=(3,), z=(14, 3), delta_bias=(3,), state=(5, 3, 4))
        f = lambda: _autograd_scan(L, STARTS, flag)
        ref = lambda **k: R.scan(L["u"], L["delta"], L["A"], L["B"], L["C"], L["D"], L["z"], L["delta_bias"], flag, STARTS, L["state"], **k)
    y, final = f()
    dy, df = torch.randn(y.shape, generator=gen, dtype=torch.float64), torch.randn(final.shape, generator=gen, dtype=torch.float64)
    grads = dict(zip(L, torch.autograd.grad([y, final], list(L.values()), [dy, df])))
    got = ref(dy=dy, dfinal=df)
    for k, v in dict(grads, y=y, final=final).items():
        assert torch.allclose(got[k][0], v, rtol=1e-10, atol=1e-10), k
    with torch.no_grad():                                        # central differences, error O(step^2)
        for k, t in L.items():
            v = torch.randn(t.shape, generator=gen, dtype=torch.float64)
            t += 1e-5 * v
            a = ref()
            t -= 2e-5 * v
            b = ref()
            t += 1e-5 * v
            slope = (((a["y"][0] - b["y"][0]) * dy).sum() + ((a["final"][0] - b["final"][0]) * df).sum()) / 2e-5
            assert abs(float(slope - (got[k][0] * v).sum())) < 1e-6 * (1 + float((got[k][0] * v).abs().sum())), k


def test_restated_norm_gradient_equals_autograd():
    gen = torch.Generator().manual_seed(6)
    L = _leaves(gen, x=(5, 7), w=(7,), res=(5, 7))
    h = L["x"] + L["res"]
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-3) * L["w"]
    dy, ds = torch.randn(y.shape, generator=gen, dtype=torch.float64), torch.randn(y.shape, generator=gen, dtype=torch.float64)
    gx, gw = torch.autograd.grad([y, h], [L["x"], L["w"]], [dy, ds])
    got = R.norm(L["x"], L["w"], L["res"], 1e-3, dy, ds)
    assert torch.allclose(got["h"][0], gx, atol=1e-12) and torch.allclose(got["weight"][0], gw, atol=1e-12)


def test_sequence_entry_points_refuse_bad_arguments_without_touching_the_gpu():
    from eventad_amd import _lib
    lib = _lib.load()
    n = ctypes.c_int64(0)
    ref = ctypes.byref(n)
    assert lib.eventad_causal_conv_workspace(10, 4, 9, ref) == -1 and lib.eventad_causal_conv_workspace(10, 0, 4, ref) == -1
    assert lib.eventad_causal_conv_workspace(-1, 4, 4, ref) == -1 and lib.eventad_causal_conv_workspace(10, 4, 4, None) == -1
    assert lib.eventad_selective_scan_workspace(10, 4, 65, 0, ref) == -1 and lib.eventad_selective_scan_workspace(10, 4, 0, 1, ref) == -1
    assert lib.eventad_selective_scan_checkpoint(1 << 31, 4, 16, ref) == -1
    assert lib.eventad_rms_norm_workspace(10, 0, ref) == -1
    assert lib.eventad_causal_conv_workspace(100, 8, 4, ref) == 0 and n.value > 0
    buf = ctypes.cast(ctypes.create_string_buffer(1 << 16), ctypes.c_void_p)      # only ever compared with NULL
    conv = lambda **k: lib.eventad_causal_conv_fwd(*[k.get(a, d) for a, d in (
        ("x", buf), ("ldx", 8), ("w", buf), ("bias", None), ("starts", None), ("clips", 1), ("state", None), ("final", None), ("y", buf),
        ("ldy", 8), ("rows", 4), ("channels", 8), ("taps", 4), ("act", 1), ("dtype", 0), ("stream", None))])
    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(ldx=7), dict(ldy=7), dict(rows=-1), dict(rows=1 << 31), dict(channels=0),
                dict(taps=0), dict(taps=9), dict(act=2), dict(dtype=3), dict(clips=0), dict(clips=2)):
        assert conv(**bad) == -1, bad
    assert conv(rows=(1 << 31) - 16, channels=1 << 16, ldx=1 << 16, ldy=1 << 16) == -3       # too many threads for one launch
    assert lib.eventad_causal_conv_step(buf, 64, buf, None, buf, buf, buf, 64, 1 << 30, 64, 4, 1, 0, None) == -3
    assert lib.eventad_rms_norm_fwd(buf, 5000, None, 0, buf, None, 0, buf, 5000, 1 << 30, 5000, 1e-6, 0, None) == -3
    assert conv(rows=0) == 0                                     # nothing to do, nothing launched
    assert lib.eventad_causal_conv_bwd(buf, 8, buf, None, None, 1, None, buf, 8, None, buf, 8, None, buf, buf, 16, 4, 8, 4, 1, 0, None) == -1
    assert lib.eventad_causal_conv_step(buf, 8, buf, None, None, None, buf, 8, 2, 8, 4, 1, 0, None) == -1
    scan = lambda **k: lib.eventad_selective_scan_fwd(*[k.get(a, d) for a, d in (
        ("u", buf), ("ldu", 8), ("delta", buf), ("ldd", 8), ("A", buf), ("B", buf), ("ldb", 16), ("C", buf), ("ldc", 16), ("D", None),
        ("z", None), ("ldz", 0), ("bias", None), ("starts", None), ("clips", 1), ("state", None), ("final", None), ("y", buf), ("ldy", 8),
        ("ckpt", None), ("ws", buf), ("wsb", 1 << 16), ("rows", 4), ("channels", 8), ("n", 16), ("softplus", 1), ("dtype", 0), ("stream", None))])
    for bad in (dict(u=None), dict(delta=None), dict(A=None), dict(B=None), dict(C=None), dict(y=None), dict(ws=None), dict(wsb=8),
                dict(ldu=7), dict(ldu=(1 << 24) + 1), dict(ldb=15), dict(ldc=15), dict(z=buf, ldz=7), dict(clips=2), dict(clips=0), dict(n=0), dict(n=65),
                dict(softplus=2), dict(dtype=-1), dict(rows=-1), dict(ckpt=ctypes.c_void_p(8 + 1))):
        assert scan(**bad) == -1, bad
    assert lib.eventad_selective_scan_bwd(*([None] * 1 + [8] + [None] * 1 + [8] + [None] * 2 + [16, None, 16, None, None, 0, None, None, 1, None,
                                           None, None, 8, None, None, 8, None, 8, None, 16, None, 16, None, 0, None, None, None, 0, 4, 8, 16, 1, 0, None])) == -1
    assert lib.eventad_selective_scan_step(buf, 8, buf, 8, buf, buf, 16, buf, 16, None, None, 0, None, None, None, buf, 8, 2, 8, 16, 1, 0, None) == -1
    assert lib.eventad_rms_norm_fwd(buf, 8, buf, 8, buf, None, 8, buf, 8, 4, 8, 1e-6, 0, None) == -1
    assert lib.eventad_rms_norm_fwd(buf, 8, None, 0, buf, None, 0, buf, 8, 4, 8, -1.0, 0, None) == -1
    assert lib.eventad_rms_norm_fp8(buf, 8, None, 0, buf, None, 0, buf, 7, buf, 4, 8, 1e-6, 0, None) == -1
    assert lib.eventad_rms_norm_bwd(buf, 8, buf, buf, 8, None, 0, buf, 8, buf, buf, 4, 4, 8, 1e-6, 0, None) == -1


def test_sequence_operators_have_no_cpu_path():
    from eventad_amd import sequence as S
    x = torch.zeros(4, 8)
    for f in (lambda: S.causal_conv(x, torch.zeros(8, 4)), lambda: S.causal_conv_step(x, torch.zeros(8, 4), torch.zeros(4, 3, 8)),
              lambda: S.selective_scan(x, x, torch.zeros(8, 4), torch.zeros(4, 4), torch.zeros(4, 4)),
              lambda: S.selective_scan_step(x, x, torch.zeros(8, 4), torch.zeros(4, 4), torch.zeros(4, 4), torch.zeros(4, 8, 4)),
              lambda: S.rms_norm(x, torch.ones(8)), lambda: S.rms_norm_fp8(x, torch.ones(8))):
        with pytest.raises(RuntimeError, match="GPU"):
            f()


def test_sequence_operators_take_only_tensors():
    from eventad_amd import sequence as S
    x = [[0.0] * 8] * 4
    for f in (lambda: S.causal_conv(x, x), lambda: S.causal_conv_step(x, x, x), lambda: S.selective_scan(x, x, x, x, x),
              lambda: S.selective_scan_step(x, x, x, x, x, x), lambda: S.rms_norm(x, x), lambda: S.rms_norm_fp8(x, x), lambda: S.rms_norm(None, None)):
        with pytest.raises(RuntimeError, match="expected a tensor"):
            f()
