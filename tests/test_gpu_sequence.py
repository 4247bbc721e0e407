"""The sequence operators (eventad_amd/sequence.py) against their float64 restatement (oracle/sequence_ref.py).

Tolerances: an output is rounded to its type once, half a step (finfo.eps / 2 relative to the value, 2^-25 absolute for
float16's subnormals), and float32 arithmetic in front of that may be off by the restatement's bound in units of 2^-24."""
import pytest
import torch

from oracle import sequence_ref as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = 2.0 ** -24


@pytest.fixture(scope="module")
def S():
    from eventad_amd import sequence
    return sequence


def close(name, got, want, units):
    """got within half a step of its type plus units x 2^-24 of want (both tensors, float64 on the CPU)."""
    g = got.detach().double().cpu()
    assert g.shape == want.shape, (name, g.shape, want.shape)
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -7) + 1.01 * UNIT * units
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    if got.dtype == torch.float32:
        tol = tol + 1e-37                                        # (subnormal results are flushed)
    over = (g - want).abs() - tol
    assert bool((over <= 0).all()), "%s: %d of %d entries off, worst by %.3g at %s: got %r want %r" % (
        name, int((~(over <= 0)).sum()), over.numel(), float(over.max()), int(over.argmax()), float(g.reshape(-1)[int(over.argmax())]),
        float(want.reshape(-1)[int(over.argmax())]))


def rnd(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen) * scale).to(dtype).cuda()


def starts_of(bounds):
    return None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")


def leaf(t):
    return None if t is None else t.clone().requires_grad_()


# clip bounds by name; the last entry may be short of the rows (rows behind the last clip), the first above 0
def bounds_of(kind, rows):
    return {"one": None, "all": [0, rows], "three": [0, rows // 3, rows // 2, rows], "empties": [0, 0, 0, rows // 2, rows // 2, rows, rows],
            "gaps": [min(2, rows), rows // 2, rows // 2, max(min(2, rows), rows - 3)], "singles": list(range(rows + 1)),
            "tiles": sorted({0, min(16, rows), min(63, rows), min(64, rows), min(65, rows), min(128, rows), rows})}[kind]


# ---------------------------------------------------------------------------------------------------- causal convolution
def conv_units(K, rows):
    return K + 16, K + 16 + rows                                 # per row: K products and the activation; sums over the rows


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,channels,taps,kind,silu,state,bias", [
    (1, 1, 1, "one", True, False, True), (1, 8, 4, "all", True, True, True), (2, 16, 4, "singles", True, True, True),
    (33, 8, 4, "three", True, True, True), (70, 24, 3, "empties", False, True, False), (131, 40, 4, "tiles", True, False, True),
    (64, 7, 2, "gaps", True, True, True), (97, 16, 8, "three", True, True, False), (40, 5, 6, "singles", False, True, True),
    (200, 64, 5, "tiles", True, True, True), (65, 16, 7, "gaps", True, False, True), (32, 8, 1, "empties", True, True, True)])
def test_causal_conv_and_gradient(S, dtype, rows, channels, taps, kind, silu, state, bias):
    gen, dt = torch.Generator().manual_seed(rows * 31 + channels), DTYPES[dtype]
    b = bounds_of(kind, rows)
    clips = 1 if b is None else len(b) - 1
    x, w = rnd(gen, rows, channels, dtype=dt), rnd(gen, channels, taps)
    bs = rnd(gen, channels) if bias else None
    st = rnd(gen, clips, taps - 1, channels, dtype=dt) if state else None
    dy, df = rnd(gen, rows, channels, dtype=dt), rnd(gen, clips, taps - 1, channels, dtype=dt)
    act = "silu" if silu else None
    want = R.conv(x, w, bs, b, st, silu, dy, df)
    row_units, sum_units = conv_units(taps, rows)
    with torch.no_grad():
        y, final = S.causal_conv(x, w, bs, starts_of(b), st, act, True)
        assert torch.equal(y, S.causal_conv(x, w, bs, starts_of(b), st, act))
    close("y", y, want["y"][0], row_units * want["y"][1])
    assert torch.equal(final.double().cpu(), want["final"][0])    # copies
    L = [leaf(t) for t in (x, w, bs, st)]
    y2, f2 = S.causal_conv(L[0], L[1], L[2], starts_of(b), L[3], act, True)
    assert torch.equal(y2, y) and torch.equal(f2, final)
    grads = torch.autograd.grad([y2, f2], [t for t in L if t is not None], [dy, df])
    names = [k for k, t in zip(("x", "weight", "bias", "state"), L) if t is not None]
    for k, g in zip(names, grads):
        close("d" + k, g, want[k][0], (sum_units if k in ("weight", "bias") else row_units + taps) * want[k][1])


def conv_by_shifts(x, w, bs, b, st, dy, df):
    """R.conv for arrays of any length: float64 on the GPU, clip by clip, tap by tap."""
    x, w, bs, st, dy, df = (t.detach().double() for t in (x, w, bs, st, dy, df))
    K = w.shape[1]
    out = {k: [torch.zeros_like(t), torch.zeros_like(t)] for k, t in (("y", x), ("x", x), ("weight", w), ("bias", bs), ("state", st))}
    final = st.clone()
    for s, (lo, hi) in enumerate(zip(b, b[1:])):
        n = hi - lo
        ext = torch.cat([st[s], x[lo:hi]])
        pre, mag = bs + sum(ext[k:k + n] * w[:, k] for k in range(K)), bs.abs() + sum(ext[k:k + n].abs() * w[:, k].abs() for k in range(K))
        sg = torch.sigmoid(pre)
        out["y"][0][lo:hi], out["y"][1][lo:hi] = pre * sg, mag
        final[s] = ext[n:]
        d, dm = dy[lo:hi] * sg * (1 + pre * (1 - sg)), dy[lo:hi].abs() * (1 + mag)
        dext, dextm = torch.zeros_like(ext), torch.zeros_like(ext)
        dext[n:] += df[s]
        dextm[n:] += df[s].abs()
        for k in range(K):
            dext[k:k + n] += d * w[:, k]
            dextm[k:k + n] += dm * w[:, k].abs()
            out["weight"][0][:, k] += (ext[k:k + n] * d).sum(0)
            out["weight"][1][:, k] += (ext[k:k + n].abs() * dm).sum(0)
        out["bias"][0] += d.sum(0)
        out["bias"][1] += dm.sum(0)
        out["state"][0][s], out["state"][1][s] = dext[:K - 1], dextm[:K - 1]
        out["x"][0][lo:hi], out["x"][1][lo:hi] = dext[K - 1:], dextm[K - 1:]
    return {k: tuple(t.cpu() for t in v) for k, v in out.items()}, final.cpu()


@pytest.mark.parametrize("dtype,rows,channels,taps", [("f32", 60001, 512, 4), ("bf16", 50003, 300, 4), ("f16", 40001, 513, 3), ("f32", 30011, 131, 2),
                                                      ("bf16", 40007, 256, 6), ("f32", 300001, 64, 4), ("bf16", 200003, 31, 8)])
def test_causal_conv_over_long_chunks(S, dtype, rows, channels, taps):
    """Arrays long enough for chunks of many groups of rows: the unbroken groups, their borders with clips and chunks, waves
    that are not full, and several chunks per wave."""
    gen, dt = torch.Generator().manual_seed(rows), DTYPES[dtype]
    b = [0, 1, 7, 1000, 1000, rows // 2 + 1, rows - 66, rows - 5, rows]
    clips = len(b) - 1
    x, w, bs = rnd(gen, rows, channels, dtype=dt), rnd(gen, channels, taps), rnd(gen, channels)
    st, dy, df = rnd(gen, clips, taps - 1, channels, dtype=dt), rnd(gen, rows, channels, dtype=dt), rnd(gen, clips, taps - 1, channels, dtype=dt)
    want, final = conv_by_shifts(x, w, bs, b, st, dy, df)
    L = [leaf(t) for t in (x, w, bs, st)]
    y, f = S.causal_conv(L[0], L[1], L[2], starts_of(b), L[3], "silu", True)
    close("y", y, want["y"][0], (taps + 16) * want["y"][1])
    assert torch.equal(f.double().cpu(), final)
    # sums over the rows: 4..128 in sequence per chunk, the chunks shared out among 64 workgroups of 4 x 4 sums
    depth = 2 * taps + 16 + 128 + 2 * rows / 4 / 64 / 16
    for k, g in zip(("x", "weight", "bias", "state"), torch.autograd.grad([y, f], L, [dy, df])):
        close("d" + k, g, want[k][0], (depth if k in ("weight", "bias") else 2 * taps + 16) * want[k][1])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("channels", [1, 6, 67, 259, 1023])
@pytest.mark.parametrize("taps", [4, 7])
def test_causal_conv_rows_of_any_start_and_length(S, dtype, channels, taps):
    """Rows inside wider arrays that start at any element: results as those of packed rows, and nothing written beside them."""
    gen, dt, rows, wide = torch.Generator().manual_seed(channels + taps), DTYPES[dtype], 77, channels + 3
    code, bounds = {"f32": 0, "bf16": 1, "f16": 2}[dtype], [2, 31, 31, 32, 75]
    starts, clips = starts_of(bounds), len(bounds) - 1
    inner = lambda: torch.full((rows, wide), 7.0, device="cuda", dtype=dt)
    x, dy, y, dx = (inner() for _ in range(4))
    mine, at = (lambda t: t[:, 1:1 + channels]), (lambda t: t.data_ptr() + t.element_size())
    for t in (x, dy):
        mine(t).copy_(rnd(gen, rows, channels, dtype=dt))
    w, b = rnd(gen, channels, taps), rnd(gen, channels)
    st, df = rnd(gen, clips, taps - 1, channels, dtype=dt), rnd(gen, clips, taps - 1, channels, dtype=dt)
    guard = lambda: torch.full((clips * (taps - 1) * channels + 8,), 7.0, device="cuda", dtype=dt)
    final, dst = guard(), guard()
    dp = torch.empty(channels * (taps + 1), device="cuda")
    ws = torch.empty(S._bytes("eventad_causal_conv_workspace", rows, channels, taps), device="cuda", dtype=torch.uint8)
    stream = torch.cuda.current_stream().cuda_stream
    S._call("eventad_causal_conv_fwd", at(x), wide, w.data_ptr(), b.data_ptr(), starts.data_ptr(), clips, st.data_ptr(), final.data_ptr(), at(y), wide,
            rows, channels, taps, 1, code, stream)
    S._call("eventad_causal_conv_bwd", at(x), wide, w.data_ptr(), b.data_ptr(), starts.data_ptr(), clips, st.data_ptr(), at(dy), wide, df.data_ptr(),
            at(dx), wide, dst.data_ptr(), dp.data_ptr(), ws.data_ptr(), ws.numel(), rows, channels, taps, 1, code, stream)
    for t in (y, dx):
        assert bool((t[:, 0] == 7).all()) and bool((t[:, 1 + channels:] == 7).all())
    for t in (final, dst):
        assert bool((t[-8:] == 7).all())
    want = R.conv(mine(x).cpu(), w, b, bounds, st, True, mine(dy).cpu(), df)
    row_units, sum_units = conv_units(taps, rows)
    close("y", mine(y), want["y"][0], row_units * want["y"][1])
    close("final", final[:-8].view(clips, taps - 1, channels), want["final"][0], 0)
    close("dx", mine(dx), want["x"][0], row_units * want["x"][1])
    close("dstate", dst[:-8].view(clips, taps - 1, channels), want["state"][0], row_units * want["state"][1])
    close("dweight", dp[:channels * taps].view(channels, taps), want["weight"][0], sum_units * want["weight"][1])
    close("dbias", dp[channels * taps:], want["bias"][0], sum_units * want["bias"][1])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("clips,channels,taps", [(1, 1, 1), (1, 8, 4), (6, 256, 4), (5, 13, 3), (33, 40, 8), (3, 16, 2)])
def test_causal_conv_step(S, dtype, clips, channels, taps):
    gen, dt = torch.Generator().manual_seed(clips), DTYPES[dtype]
    x, w, bs, st = rnd(gen, clips, channels, dtype=dt), rnd(gen, channels, taps), rnd(gen, channels), rnd(gen, clips, taps - 1, channels, dtype=dt)
    want = R.conv(x, w, bs, list(range(clips + 1)), st, True)
    kept, out = st.clone(), torch.empty_like(st)
    y = S.causal_conv_step(x, w, st, bs, state_out=out)
    assert torch.equal(st, kept)
    close("y", y, want["y"][0], (taps + 16) * want["y"][1])
    assert torch.equal(out.double().cpu(), want["final"][0])
    assert torch.equal(S.causal_conv_step(x, w, st, bs), y) and torch.equal(st, out)          # in place


# -------------------------------------------------------------------------------------------------------- selective scan
def scan_inputs(gen, rows, channels, N, dt, clips, D=True, z=True, bias=True, state=True, decay=1.0):
    return dict(u=rnd(gen, rows, channels, dtype=dt), delta=rnd(gen, rows, channels, dtype=dt),
                A=-torch.exp(rnd(gen, channels, N)) * decay, B=rnd(gen, rows, N, dtype=dt), C=rnd(gen, rows, N, dtype=dt),
                D=rnd(gen, channels) if D else None, z=rnd(gen, rows, channels, dtype=dt) if z else None,
                delta_bias=rnd(gen, channels) - 2.0 if bias else None, state=rnd(gen, clips, channels, N) if state else None)


SCAN_CASES = [  # rows, channels, states, clips, softplus, which of D z bias state
    (1, 1, 1, "one", True, "Dzbs"), (1, 3, 16, "all", True, "Dzbs"), (5, 16, 4, "singles", True, "zbs"), (15, 17, 16, "three", True, "Dbs"),
    (16, 64, 16, "gaps", True, "Dzb"), (17, 70, 5, "empties", True, "Dzbs"), (64, 20, 16, "one", True, "Dzbs"), (65, 66, 16, "tiles", True, "Dzbs"),
    (200, 33, 16, "tiles", True, "Dzbs"), (200, 65, 16, "all", True, "zb"), (197, 16, 13, "empties", True, "Dzbs"), (150, 9, 24, "three", True, "Dzbs"),
    (130, 40, 32, "tiles", True, "Dzb"), (131, 18, 64, "three", True, "Dzbs"), (66, 5, 33, "gaps", True, "s"), (140, 12, 16, "gaps", True, ""),
    (400, 6, 16, "tiles", True, "Dzbs"), (390, 5, 20, "one", True, "zbs"), (300, 3, 7, "empties", True, "Dzbs"), (260, 2, 50, "all", True, "Dzs"),
    (90, 8, 8, "all", False, "Dzs"), (260, 4, 1, "one", True, "Dzbs")]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,channels,N,kind,softplus,given", SCAN_CASES)
def test_selective_scan_and_gradient(S, dtype, rows, channels, N, kind, softplus, given):
    gen, dt = torch.Generator().manual_seed(rows * 17 + channels * 3 + N), DTYPES[dtype]
    b = bounds_of(kind, rows)
    clips = 1 if b is None else len(b) - 1
    a = scan_inputs(gen, rows, channels, N, dt, clips, "D" in given, "z" in given, "b" in given, "s" in given)
    if not softplus:
        a["delta"] = (a["delta"].abs() * 0.3).to(dt)
    dy, df = rnd(gen, rows, channels, dtype=dt), rnd(gen, clips, channels, N)
    want = R.scan(softplus=softplus, clip_start=b, dy=dy, dfinal=df, **a)
    with torch.no_grad():
        y, final = S.selective_scan(delta_softplus=softplus, clip_start=starts_of(b), return_state=True, **a)
        assert torch.equal(y, S.selective_scan(delta_softplus=softplus, clip_start=starts_of(b), **a))
    close("y", y, *want["y"])
    close("final", final, *want["final"])
    L = {k: leaf(t) for k, t in a.items()}
    y2, f2 = S.selective_scan(delta_softplus=softplus, clip_start=starts_of(b), return_state=True, **L)
    assert torch.equal(y2, y) and torch.equal(f2, final)
    have = [k for k, t in L.items() if t is not None]
    first = torch.autograd.grad([y2, f2], [L[k] for k in have], [dy, df], retain_graph=True)
    for k, g in zip(have, first):
        close("d" + k, g, *want[k])
    for g, again in zip(first, torch.autograd.grad([y2, f2], [L[k] for k in have], [dy, df])):
        assert torch.equal(g, again)                             # reproducible bit for bit


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,channels,N,kind", [(100, 5, 2, "tiles"), (333, 67, 4, "three"), (260, 1, 3, "gaps"), (70, 130, 4, "empties"),
                                                  (333, 65, 8, "three"), (260, 3, 6, "gaps"), (90, 130, 5, "tiles"), (40, 3, 8, "singles"), (40, 9, 4, "singles")])
def test_selective_scan_with_few_states(S, dtype, rows, channels, N, kind):
    test_selective_scan_and_gradient(S, dtype, rows, channels, N, kind, True, "Dzbs")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("clips,channels,N", [(1, 1, 1), (6, 256, 16), (5, 13, 5), (3, 33, 24), (2, 7, 64), (17, 20, 8)])
def test_selective_scan_step(S, dtype, clips, channels, N):
    gen, dt = torch.Generator().manual_seed(clips + N), DTYPES[dtype]
    a = scan_inputs(gen, clips, channels, N, dt, clips)
    want = R.scan(clip_start=list(range(clips + 1)), **a)
    st = a.pop("state")
    kept, out = st.clone(), torch.empty_like(st)
    y = S.selective_scan_step(state=st, state_out=out, **a)
    assert torch.equal(st, kept)
    close("y", y, *want["y"])
    close("state", out, *want["final"])
    assert torch.equal(S.selective_scan_step(state=st, **a), y) and torch.equal(st, out)       # in place


def test_scan_extreme_steps_and_decays(S):
    """Steps from underflow to saturation of softplus, decays that vanish in one row, states that never decay (A = 0)."""
    gen = torch.Generator().manual_seed(3)
    rows, ch, N = 80, 6, 16
    a = scan_inputs(gen, rows, ch, N, torch.float32, 1)
    a["delta"] = torch.linspace(-90.0, 40.0, rows * ch).view(rows, ch)[torch.randperm(rows, generator=gen)].contiguous().cuda()
    a["A"][:, 0] = 0.0
    a["A"][:, 1] = -1e4
    dy = rnd(gen, rows, ch)
    want = R.scan(dy=dy, **a)
    L = {k: leaf(t) for k, t in a.items()}
    y = S.selective_scan(**L)
    close("y", y, *want["y"])
    for k, g in zip(L, torch.autograd.grad(y, list(L.values()), dy)):
        close("d" + k, g, *want[k])


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 1e30])
def test_rows_of_no_clip_are_not_looked_at(S, value):
    """Whatever stands in rows in front of the first and behind the last clip: zeros come out, and no gradient sees them."""
    gen = torch.Generator().manual_seed(4)
    rows, ch, N, b = 90, 20, 16, [5, 40, 70]
    a = scan_inputs(gen, rows, ch, N, torch.float32, 2)
    x, w, bs = rnd(gen, rows, ch), rnd(gen, ch, 4), rnd(gen, ch)
    dy = rnd(gen, rows, ch)
    dead = torch.ones(rows, dtype=torch.bool)
    dead[5:70] = False
    dead = dead.cuda()
    results = []
    for fill in (0.0, value):
        t = {k: (v.clone() if v is not None else None) for k, v in a.items()}
        for k in ("u", "delta", "B", "C", "z"):
            t[k][dead] = fill
        xx, g = x.clone(), dy.clone()
        xx[dead], g[dead] = fill, fill
        L = {k: leaf(v) for k, v in t.items()}
        y, f = S.selective_scan(clip_start=starts_of(b), return_state=True, **L)
        C = [leaf(v) for v in (xx, w, bs)]
        yc = S.causal_conv(C[0], C[1], C[2], starts_of(b))
        r = [y, f, yc] + list(torch.autograd.grad(y, list(L.values()), g)) + list(torch.autograd.grad(yc, C, g))
        results.append(r)
        assert bool((y[dead] == 0).all()) and bool((yc[dead] == 0).all())
    for p, q in zip(*results):
        assert torch.equal(p, q)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("channels,rows,bounds", [
    (8, 40, [0, 5, 11, 13, 16, 27, 40]),                         # several clips inside a tile
    (24, 700, [3, 130, 333, 340, 680, 690]),                     # a clip's end inside a tile of another chunk; rows of no clip
    (64, 6400, [0, 1000, 3011, 3500, 6400])])                    # clips over several groups of chunks
@pytest.mark.parametrize("bad", [0, 1, 2])
def test_a_clip_does_not_spoil_its_neighbours(S, value, channels, rows, bounds, bad):
    """With one clip's arrays full of NaN or infinities the other clips' results keep every bit."""
    gen, N, K, clips = torch.Generator().manual_seed(rows + bad), 16, 4, len(bounds) - 1
    starts, row = starts_of(bounds), torch.arange(rows, device="cuda")
    hit = (row >= bounds[bad]) & (row < bounds[bad + 1])
    good_clips = [i for i in range(clips) if i != bad]
    x, delta, z, dy = (rnd(gen, rows, channels) for _ in range(4))
    B, C = rnd(gen, rows, N), rnd(gen, rows, N)
    A, D, w = -rnd(gen, channels, N).abs(), rnd(gen, channels), rnd(gen, channels, K)
    h0, c0, dh, dc = rnd(gen, clips, channels, N), rnd(gen, clips, K - 1, channels), rnd(gen, clips, channels, N), rnd(gen, clips, K - 1, channels)
    runs = []
    for spoil in (False, True):
        t = [v.clone() for v in (x, delta, B, C, z, dy)]
        s = [v.clone() for v in (h0, c0, dh, dc)]
        if spoil:
            for v in t:
                v[hit] = value
            for v in s:
                v[bad] = value
        L = [v.requires_grad_() for v in t[:5]] + [s[0].requires_grad_(), s[1].requires_grad_()]
        y, h = S.selective_scan(L[0], L[1], A, L[2], L[3], D, L[4], clip_start=starts, state=L[5], return_state=True)
        v, c = S.causal_conv(L[0], w, None, starts, L[6], return_state=True)
        per_row = list(torch.autograd.grad([y, h], L[:6], [t[5], s[2]], retain_graph=True)) + list(torch.autograd.grad([v, c], [L[0], L[6]], [t[5], s[3]]))
        runs.append(([y, v, *per_row[:5], per_row[6]], [h, c, per_row[5], per_row[7]]))
    for a, b in zip(runs[0][0], runs[1][0]):
        assert torch.equal(a[~hit], b[~hit])
    for a, b in zip(runs[0][1], runs[1][1]):
        assert torch.equal(a[good_clips], b[good_clips])


def test_offsets_outside_the_array_reach_no_row_outside_it(S):
    """Offsets below 0, above the rows or decreasing give wrong numbers, made of the array's own rows and the given states."""
    gen, rows, ch, N, K = torch.Generator().manual_seed(4), 70, 8, 16, 4
    wide = lambda n: torch.full((rows + 64, n), float("nan"), device="cuda")
    held = [wide(n) for n in (ch, ch, N, N, ch)]
    t = [v[32:32 + rows] for v in held]
    for v in t:
        v.copy_(torch.randn(v.shape, generator=gen))
    A, w, norm_w = -rnd(gen, ch, N).abs(), rnd(gen, ch, K), rnd(gen, ch)
    for bounds in ([-5, 30, 75], [-3, -1, rows], [20, 10, 40, 5, 90], [60, 0, 70], [80, 90], [-9, -4]):
        clips, starts = len(bounds) - 1, starts_of(bounds)
        h0, c0 = rnd(gen, clips, ch, N), rnd(gen, clips, K - 1, ch)
        L = [v.detach().requires_grad_() for v in t] + [h0.requires_grad_(), c0.requires_grad_()]
        y = S.selective_scan(L[0], L[1], A, L[2], L[3], None, L[4], clip_start=starts, state=L[5])
        v = S.causal_conv(L[0], w, None, starts, L[6])
        rows_of = [y, v, *torch.autograd.grad(y.sum(), L[:5], retain_graph=True), *torch.autograd.grad(v.sum(), L[:1])]
        assert all(bool(torch.isfinite(r).all()) for r in rows_of), bounds


def test_no_rows_and_only_empty_clips(S):
    st, cs = torch.randn(3, 4, 16, device="cuda"), torch.randn(3, 2, 4, device="cuda")
    e = lambda n: torch.empty(0, n, device="cuda")
    b = starts_of([0, 0, 0, 0])
    L = [leaf(t) for t in (e(4), e(4), -torch.ones(4, 16, device="cuda"), e(16), e(16), st)]
    y, f = S.selective_scan(*L[:5], clip_start=b, state=L[5], return_state=True)
    assert y.shape == (0, 4) and torch.equal(f, st)
    g = torch.autograd.grad(f, L, st, allow_unused=True)
    assert torch.equal(g[5], st) and bool((g[2] == 0).all())
    C = [leaf(t) for t in (e(4), torch.ones(4, 3, device="cuda"), cs)]
    y, f = S.causal_conv(C[0], C[1], clip_start=b, state=C[2], return_state=True)
    assert y.shape == (0, 4) and torch.equal(f, cs)
    g = torch.autograd.grad(f, C, cs)
    assert torch.equal(g[2], cs) and bool((g[1] == 0).all())
    n = [leaf(e(4)), leaf(torch.ones(4, device="cuda"))]
    y = S.rms_norm(*n)
    assert y.shape == (0, 4) and bool((torch.autograd.grad(y, n, y)[1] == 0).all())
    q, s = S.rms_norm_fp8(e(4), torch.ones(4, device="cuda"))
    assert q.shape == (0, 4) and s.shape == (0,)
    assert S.causal_conv_step(e(4), torch.ones(4, 3, device="cuda"), torch.empty(0, 2, 4, device="cuda")).shape == (0, 4)
    assert S.selective_scan_step(e(4), e(4), -torch.ones(4, 16, device="cuda"), e(16), e(16), torch.empty(0, 4, 16, device="cuda")).shape == (0, 4)


# ------------------------------------------------------------------------------------------------------------- RMS norm
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,channels,residual", [(1, 1, True), (3, 7, True), (6, 256, True), (5, 128, False), (37, 64, True), (2, 1000, True),
                                                    (9, 2048, True), (3, 4104, True), (3, 5000, True), (2, 8192, False), (2, 9000, True), (2, 1027, True),
                                                    (1100, 24, True), (1, 20001, True)])
def test_rms_norm_and_gradient(S, dtype, rows, channels, residual):
    gen, dt = torch.Generator().manual_seed(rows + channels), DTYPES[dtype]
    x, w = rnd(gen, rows, channels, dtype=dt), rnd(gen, channels) + 1.0
    res = rnd(gen, rows, channels, dtype=dt, scale=2.0) if residual else None
    dy, ds = rnd(gen, rows, channels, dtype=dt), rnd(gen, rows, channels, dtype=dt)
    want = R.norm(x.cpu(), w, None if res is None else res.cpu(), 1e-5, dy, ds if residual else None)
    units = 2 * (channels / 16 + 24)                             # additions in sequence of a sum over the row
    with torch.no_grad():
        r = S.rms_norm(x, w, res, 1e-5)
    y, total = r if residual else (r, None)
    close("y", y, want["y"][0], units * want["y"][1])
    if residual:
        assert torch.equal(total.double().cpu(), want["sum"][0])
    L = [leaf(x), leaf(w), leaf(res)]
    r = S.rms_norm(L[0], L[1], L[2], 1e-5)
    outs = list(r) if residual else [r]
    grads = torch.autograd.grad(outs, [t for t in L if t is not None], [dy, ds][:len(outs)])
    close("dx", grads[0], want["h"][0], units * want["h"][1])
    close("dweight", grads[1], want["weight"][0], (units + rows) * want["weight"][1])
    if residual:
        assert torch.equal(grads[2], grads[0])
        only = torch.autograd.grad(S.rms_norm(L[0], L[1], L[2], 1e-5)[1], L[2], ds)[0]         # only the sum is used
        assert torch.equal(only, ds)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,channels,residual", [(1, 1, True), (3, 7, True), (6, 256, True), (37, 64, False), (9, 2048, True), (3, 4104, True), (2, 9000, True),
                                                    (3, 1030, True)])
def test_rms_norm_fp8_is_the_nearest_value(S, dtype, rows, channels, residual):
    gen, dt = torch.Generator().manual_seed(rows + channels), DTYPES[dtype]
    x, w = rnd(gen, rows, channels, dtype=dt), rnd(gen, channels)
    res = rnd(gen, rows, channels, dtype=dt) if residual else None
    x[0] = 0.0                                                   # a row of zeros (with a residual: of the residual alone)
    if res is not None and rows > 1:
        res[0] = 0.0
    want = R.norm(x.cpu(), w, None if res is None else res.cpu(), 1e-6)
    r = S.rms_norm_fp8(x, w, res)
    assert r[0].dtype == torch.float8_e4m3fn and r[1].dtype == torch.float32
    assert torch.equal(r[0].double().cpu(), want["q"])           # every value on the side the definition says
    close("scale", r[1], want["scale"][0], (channels / 16 + 28) * want["scale"][0])
    if residual:
        assert torch.equal(r[2].double().cpu(), want["sum"][0])


@pytest.mark.parametrize("channels", [40, 1030, 2048, 4104, 9000])
def test_rms_norm_fp8_next_to_every_border(S, channels):
    """Quotients within a few float32 units of the borders between neighbouring 8-bit values, subnormal ones among them."""
    gen, rows = torch.Generator().manual_seed(channels), 24
    grid = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    borders = (grid[1:] + grid[:-1]) / 2
    w = torch.randn(channels, generator=gen)
    pick = borders[torch.randint(0, len(borders), (rows, channels), generator=gen)] * (1 + torch.randint(-12, 13, (rows, channels), generator=gen) * 2.0 ** -24)
    sign = torch.randint(0, 2, (rows, channels), generator=gen) * 2.0 - 1
    x = torch.rand(rows, channels, generator=gen) + 0.5
    top = (x[:, :1].double() * w[0].double().abs())              # the row's largest |h w|
    x[:, 1:] = (pick * sign * top / 448 / w.double()).float()[:, 1:]
    want = R.norm(x, w.cuda(), None, 1e-6)
    q, _ = S.rms_norm_fp8(x.cuda(), w.cuda())
    assert torch.equal(q.double().cpu(), want["q"])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("channels", [5, 67, 257, 1027, 4611, 9001, 16390])
def test_rms_norm_rows_of_any_start_and_length(S, dtype, channels):
    """Rows inside wider arrays that start at any element: results as those of packed rows, and nothing written beside them."""
    gen, dt, rows, pad = torch.Generator().manual_seed(channels), DTYPES[dtype], 5, 3
    code, wide = {"f32": 0, "bf16": 1, "f16": 2}[dtype], channels + pad
    inner = lambda: torch.full((rows, wide), 7.0, device="cuda", dtype=dt)
    x, res, dy, ds = (inner() for _ in range(4))
    for t in (x, res, dy, ds):
        t[:, 1:1 + channels] = rnd(gen, rows, channels, dtype=dt)
    w = rnd(gen, channels)
    total, y, dh = inner(), inner(), inner()
    q = torch.full((rows, wide), 9, device="cuda", dtype=torch.uint8)
    scale, dw = torch.empty(rows, device="cuda"), torch.empty(channels, device="cuda")
    at = lambda t: t.data_ptr() + t.element_size()
    stream = torch.cuda.current_stream().cuda_stream
    ws = torch.empty(S._bytes("eventad_rms_norm_workspace", rows, channels), device="cuda", dtype=torch.uint8)
    S._call("eventad_rms_norm_fwd", at(x), wide, at(res), wide, w.data_ptr(), at(total), wide, at(y), wide, rows, channels, 1e-6, code, stream)
    S._call("eventad_rms_norm_bwd", at(total), wide, w.data_ptr(), at(dy), wide, at(ds), wide, at(dh), wide, dw.data_ptr(), ws.data_ptr(), ws.numel(),
            rows, channels, 1e-6, code, stream)
    kept = total.clone()
    S._call("eventad_rms_norm_fp8", at(x), wide, at(res), wide, w.data_ptr(), at(total), wide, at(q), wide, scale.data_ptr(), rows, channels, 1e-6, code, stream)
    assert torch.equal(total, kept)
    mine = lambda t: t[:, 1:1 + channels]
    for t, fill in ((total, 7), (y, 7), (dh, 7), (q, 9)):
        assert bool((t[:, 0] == fill).all()) and bool((t[:, 1 + channels:] == fill).all())
    want = R.norm(mine(x).cpu(), w, mine(res).cpu(), 1e-6, mine(dy).cpu(), mine(ds).cpu())
    assert torch.equal(mine(total).double().cpu(), want["sum"][0])
    assert torch.equal(mine(q).contiguous().view(torch.float8_e4m3fn).double().cpu(), want["q"])
    units = 2 * (channels / 16 + 24)
    close("y", mine(y), want["y"][0], units * want["y"][1])
    close("scale", scale, want["scale"][0], units * want["scale"][0])
    close("dh", mine(dh), want["h"][0], units * want["h"][1])
    close("dw", dw, want["weight"][0], (units + rows) * want["weight"][1])


def test_rms_norm_takes_any_number_as_eps(S):
    import numpy as np
    x, w = rnd(torch.Generator().manual_seed(8), 5, 24), torch.ones(24, device="cuda")
    want = S.rms_norm(x, w, eps=0.5)
    for eps in (np.float32(0.5), np.float64(0.5), torch.tensor(0.5)):
        assert torch.equal(S.rms_norm(x, w, eps=eps), want)
        assert torch.equal(S.rms_norm_fp8(x, w, eps=eps)[1], S.rms_norm_fp8(x, w, eps=0.5)[1])
    assert torch.equal(S.rms_norm(x, w, eps=1), S.rms_norm(x, w, eps=1.0))


def test_rms_norm_fp8_keeps_nan(S):
    x = torch.randn(4, 64, device="cuda")
    x[1, 3] = float("nan")
    q, s = S.rms_norm_fp8(x, torch.ones(64, device="cuda"))
    assert bool(torch.isnan(s[1])) and bool(torch.isnan(q[1].float()).all())
    assert not bool(torch.isnan(s[[0, 2, 3]]).any()) and not bool(torch.isnan(q[[0, 2, 3]].float()).any())


# -------------------------------------------------------------------------------------------------- how they are called
def block_weights(gen, D, E, N, K, rank):
    return dict(norm=rnd(gen, D, scale=0.1) + 1.0, w_in=rnd(gen, D, 2 * E, scale=D ** -0.5), conv=rnd(gen, E, K, scale=K ** -0.5), conv_b=rnd(gen, E, scale=0.1),
                w_x=rnd(gen, E, rank + 2 * N, scale=E ** -0.5), w_dt=rnd(gen, rank, E, scale=rank ** -0.5), dt_b=rnd(gen, E) - 2.0,
                A=-torch.exp(rnd(gen, E, N)), D=rnd(gen, E), w_out=rnd(gen, E, D, scale=E ** -0.5))


def block(S, p, x, res, starts=None, states=None, step=False):
    """norm(+residual) -> projection -> convolution -> step sizes, B, C -> scan with its gate -> projection; the operators read
    slices of the projections' outputs."""
    N, E = p["A"].shape[1], p["A"].shape[0]
    h, res = S.rms_norm(x, p["norm"], residual=res)
    xz = h @ p["w_in"]
    u, z = xz[:, :E], xz[:, E:]
    if step:
        u = S.causal_conv_step(u, p["conv"], states[0], p["conv_b"])
    else:
        u, cs = S.causal_conv(u, p["conv"], p["conv_b"], starts, None if states is None else states[0], return_state=True)
    dbc = u @ p["w_x"]
    rank = dbc.shape[1] - 2 * N
    dt, Bm, Cm = dbc[:, :rank] @ p["w_dt"], dbc[:, rank:rank + N], dbc[:, rank + N:]
    if step:
        y, new = S.selective_scan_step(u, dt, p["A"], Bm, Cm, states[1], p["D"], z, p["dt_b"]), states
    else:
        y, ss = S.selective_scan(u, dt, p["A"], Bm, Cm, p["D"], z, p["dt_b"], True, starts, None if states is None else states[1], True)
        new = [cs, ss]
    return y @ p["w_out"], res, new


def test_block_of_prompts_single_tokens_and_appended_rows_agree(S):
    gen = torch.Generator().manual_seed(8)
    D, E, N, K, rank, lens = 24, 40, 16, 4, 5, [37, 1, 80, 0, 20]
    p = block_weights(gen, D, E, N, K, rank)
    b = [0]
    for n in lens:
        b.append(b[-1] + n)
    x, res = rnd(gen, b[-1], D), rnd(gen, b[-1], D)
    with torch.no_grad():
        whole, wres, wst = block(S, p, x, res, starts_of(b))
        # each clip's first part as a prompt, the rest appended: by several rows at once, then row by row
        cut = [n // 2 for n in lens]
        idx = torch.cat([torch.arange(b[i], b[i] + cut[i]) for i in range(5)]).cuda()
        cb = [0]
        for n in cut:
            cb.append(cb[-1] + n)
        part, _, st = block(S, p, x[idx], res[idx], starts_of(cb))
        rest = [n - c for n, c in zip(lens, cut)]
        more = [max(0, r - 3) for r in rest]
        idx2 = torch.cat([torch.arange(b[i] + cut[i], b[i] + cut[i] + more[i]) for i in range(5)]).cuda()
        mb = [0]
        for n in more:
            mb.append(mb[-1] + n)
        part2, _, st = block(S, p, x[idx2], res[idx2], starts_of(mb), st)
        got = torch.empty_like(whole)
        got[idx], got[idx2] = part, part2
        for k in range(3):
            live = [i for i in range(5) if cut[i] + more[i] + k < lens[i]]
            rows = torch.tensor([b[i] + cut[i] + more[i] + k for i in live]).cuda()
            sub = [s[live].contiguous() for s in st]
            y, _, _ = block(S, p, x[rows], res[rows], states=sub, step=True)
            got[rows] = y
            for s, t in zip(st, sub):
                s[live] = t
    scale = float(whole.abs().max())
    assert float((got - whole).abs().max()) < 1e-4 * scale       # different orders of float32 sums over <= 80 rows
    for s, t in zip(st, wst):
        assert float((s - t).abs().max()) < 1e-4 * float(t.abs().max())


def test_block_gradients_against_differences(S):
    gen = torch.Generator().manual_seed(9)
    p = {k: leaf(v) for k, v in block_weights(gen, 12, 20, 16, 4, 3).items()}
    x, res, b = rnd(gen, 50, 12), rnd(gen, 50, 12), [0, 20, 20, 47]
    c1, c2 = rnd(gen, 50, 12), rnd(gen, 50, 12)
    loss = lambda q: sum((o.double() * c.double()).sum() for o, c in zip(block(S, q, x, res, starts_of(b))[:2], (c1, c2)))
    grads = torch.autograd.grad(loss(p), list(p.values()))
    for (k, t), g in zip(p.items(), grads):
        v = rnd(gen, *t.shape) * (t.detach().abs().mean() + 0.1)
        with torch.no_grad():
            q = {n: w.detach().clone() for n, w in p.items()}
            q[k] = t.detach() + 1e-2 * v
            up = loss(q)
            q[k] = t.detach() - 1e-2 * v
            slope = float(up - loss(q)) / 2e-2
        want = float((g.double() * v.double()).sum())
        # second-order differences of a smooth function at 1e-2 of the weights' size, and float32 losses divided by the step
        assert abs(slope - want) < 2e-2 * (abs(want) + float((g.double() * v.double()).norm())) + 1e-3, (k, slope, want)


def test_strides_orders_and_alignment(S):
    """Slices of wider rows, rows that start off a 16-byte border, transposed and broadcast arrays give what copies give."""
    gen = torch.Generator().manual_seed(10)
    rows, ch, N, b = 70, 24, 16, [0, 30, 70]
    for dt in DTYPES.values():
        wide = rnd(gen, rows, 3 * ch + 2 * N + 5, dtype=dt)
        for off in (0, 1, 8):
            u, z, d = wide[:, off:off + ch], wide[:, off + ch:off + 2 * ch], wide[:, off + ch + 3:off + 2 * ch + 3]
            Bm, Cm = wide[:, 2 * ch + off - 1 if off else 0:][:, :N], wide[:, 5:5 + N]
            A, D = -torch.exp(rnd(gen, ch, N)), rnd(gen, ch)
            view, flat = (u, d, A, Bm, Cm, D, z), tuple(t.contiguous().clone() for t in (u, d, A, Bm, Cm, D, z))
            dy = rnd(gen, rows, 2 * ch, dtype=dt)[:, ch:]
            outs = []
            for t in (view, flat, tuple(v.t().contiguous().t() if v.dim() == 2 else v for v in flat)):
                L = [v.detach().requires_grad_() for v in t]
                y = S.selective_scan(*L, clip_start=starts_of(b))
                outs.append([y] + list(torch.autograd.grad(y, L, dy)))
            for o in outs[1:]:
                for p, q in zip(outs[0], o):
                    assert torch.equal(p, q)
            w, res = rnd(gen, ch, 4), wide[:, 7:7 + ch]
            outs = []
            for xs, rs in ((u, res), (u.contiguous().clone(), res.contiguous().clone())):
                L = [xs.detach().requires_grad_(), w.detach().requires_grad_(), rs.detach().requires_grad_(), D.detach().requires_grad_()]
                y = S.causal_conv(L[0], L[1], clip_start=starts_of(b))
                n, t = S.rms_norm(L[0], L[3], L[2])
                q = S.rms_norm_fp8(xs, D, rs)
                outs.append([y, n, t, q[0].float(), q[1]] + list(torch.autograd.grad(y, L[:2], dy)) + list(torch.autograd.grad([n, t], [L[0], L[3], L[2]], [dy, dy])))
            # the 16-byte and the one-element form of the norm add a row in different orders
            for i, (p, q) in enumerate(zip(*outs)):
                p, q = p.detach(), q.detach()
                if i in (0, 5) and dt == torch.float16:
                    # the last fused multiply-add may be rounded to float16 at once or through float32: both are the rounding of
                    # numbers 2^-24 apart, hence equal or neighbours, at most eps |q| apart (2^-24 among the subnormals)
                    assert bool(((p.float() - q.float()).abs() <= torch.finfo(dt).eps * q.float().abs() + 2.0 ** -24).all()), i
                elif i in (0, 2, 5, 6):
                    assert torch.equal(p, q), i
                else:
                    assert float((p.float() - q.float()).abs().max()) <= 4 * torch.finfo(dt).eps * float(q.float().abs().max()), i
        row = rnd(gen, 1, ch, dtype=dt).expand(rows, ch)         # one row for all
        assert torch.equal(S.causal_conv(row, w, clip_start=starts_of(b)), S.causal_conv(row.contiguous(), w, clip_start=starts_of(b)))


def test_captured_calls_replay_and_two_graphs_do_not_share(S):
    gen = torch.Generator().manual_seed(11)
    rows, ch, N = 200, 32, 16
    bounds = [[0, 60, 60, 200], [3, 100, 130, 190]]
    a = scan_inputs(gen, rows, ch, N, torch.float32, 3, state=False)
    names = [k for k, t in a.items() if t is not None]
    static = {k: a[k].clone() for k in names}
    w, starts = rnd(gen, ch, 4), starts_of(bounds[0])
    dy = rnd(gen, rows, ch)

    def once():
        L = {k: t.detach().requires_grad_() for k, t in static.items()}
        u = S.causal_conv(L["u"], w, clip_start=starts)
        n, t = S.rms_norm(u, L["D"], residual=L["u"])
        y = S.selective_scan(n, L["delta"], L["A"], L["B"], L["C"], L["D"], L["z"], L["delta_bias"], clip_start=starts)
        return [y, t] + list(torch.autograd.grad([y, t], [L[k] for k in names], [dy, dy]))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        once()
    side.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = once()
        graphs.append((g, out))
    for it in range(4):
        for k in names:
            static[k].copy_(a[k] * (1.0 + 0.1 * it))
        starts.copy_(starts_of(bounds[it % 2]))
        want = [t.clone() for t in once()]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for p, q in zip(out, want):
                assert torch.equal(p, q), it


def test_two_streams_at_once(S):
    gen = torch.Generator().manual_seed(12)
    sets = [scan_inputs(gen, 3000, 48, 16, torch.float32, 1) for _ in range(2)]
    with torch.no_grad():
        want = [S.selective_scan(return_state=True, **a) for a in sets]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in sets]
        got = []
        for _ in range(5):
            for st, a in zip(streams, sets):
                with torch.cuda.stream(st):
                    got.append(S.selective_scan(return_state=True, **a))
        torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g[0], want[i % 2][0]) and torch.equal(g[1], want[i % 2][1])


def test_long_clip_against_float64_doubling(S):
    """60001 rows in many chunks, three clips, few channels."""
    gen = torch.Generator().manual_seed(13)
    rows, ch, N, b = 60001, 8, 16, [0, 20000, 20017, 60001]
    a = scan_inputs(gen, rows, ch, N, torch.float32, 3, decay=0.2)
    a["delta_bias"] -= 3.0
    dy = rnd(gen, rows, ch)
    L = {k: leaf(t) for k, t in a.items()}
    y, f = S.selective_scan(clip_start=starts_of(b), return_state=True, **L)
    got = dict(zip(L, torch.autograd.grad(y, list(L.values()), dy)))
    u, A, B, C, z = (a[k].double() for k in ("u", "A", "B", "C", "z"))
    raw = a["delta"].double() + a["delta_bias"].double()
    s = torch.nn.functional.softplus(raw)

    def doubled(p, q):
        d = 1
        while d < rows:
            q = torch.cat([q[:d], q[d:] + p[d:] * q[:-d]])
            p = torch.cat([p[:d], p[d:] * p[:-d]])
            d *= 2
        return q
    p, q = torch.exp(s[:, :, None] * A), (s * u)[:, :, None] * B[:, None]
    for i in range(3):
        q[b[i]] += p[b[i]] * a["state"][i].double()
    chain = p.clone()
    chain[torch.tensor(b[:3]).cuda()] = 0.0
    h = doubled(chain, q)
    gate = torch.nn.functional.silu(z)
    pre = (h * C[:, None]).sum(2) + a["D"].double() * u
    d = dy.double() * gate
    back = torch.cat([chain[1:], torch.zeros_like(chain[:1])])
    g = doubled(back.flip(0), (d[:, :, None] * C[:, None]).flip(0)).flip(0)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    for i in range(3):
        before[b[i]] = a["state"][i].double()
    flow = g * p * before
    dd = (u * (g * B[:, None]).sum(2) + (flow * A).sum(2)) * torch.sigmoid(raw)
    want = dict(u=a["D"].double() * d + s * (g * B[:, None]).sum(2), delta=dd, A=(flow * s[:, :, None]).sum(0), B=(g * (s * u)[:, :, None]).sum(1),
                C=(h * d[:, :, None]).sum(1), D=(d * u).sum(0), delta_bias=dd.sum(0),
                state=torch.stack([(g[b[i]] * p[b[i]]) for i in range(3)]))
    # memories of up to a few hundred rows, 2^-24 x (a few tens of units per row) each
    ok = lambda name, v, w: float((v.double() - w).norm()) <= 3e-5 * float(w.norm()) or pytest.fail("%s: %.3g" % (name, float((v.double() - w).norm() / w.norm())))
    ok("y", y, pre * gate)
    ok("final", f, torch.stack([h[b[i + 1] - 1] for i in range(3)]))
    for k, v in want.items():
        ok(k, got[k], v)


def test_offsets_past_32_bits(S):
    """Arrays of more than 2^31 elements: the last rows equal those of a call on their own."""
    rows, ch, tail = 70000, 32768, 20
    b = [0, rows - tail, rows]
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(rows, ch, dtype=torch.bfloat16, device="cuda")
    x.zero_()
    x[-tail:].normal_(generator=gen)
    last = x[-tail:].clone()
    w, nw = torch.randn(ch, 4, device="cuda", generator=gen), torch.rand(ch, device="cuda", generator=gen)
    A = -torch.rand(ch, 4, device="cuda", generator=gen)
    B = torch.randn(rows, 4, device="cuda", generator=gen).bfloat16()
    with torch.no_grad():
        assert torch.equal(S.causal_conv(x, w, clip_start=starts_of(b))[-tail:], S.causal_conv(last, w))
        y = S.rms_norm(x, nw)
        assert torch.equal(y[-tail:], S.rms_norm(last, nw))
        del y
        y = S.selective_scan(x, x, A, B, B, clip_start=starts_of(b))
        assert torch.equal(y[-tail:], S.selective_scan(last, last, A, B[-tail:].contiguous(), B[-tail:].contiguous()))


def test_refusals(S):
    x, w, st = torch.zeros(4, 8, device="cuda"), torch.zeros(8, 4, device="cuda"), torch.zeros(4, 3, 8, device="cuda")
    A, Bm, hs = torch.zeros(8, 16, device="cuda"), torch.zeros(4, 16, device="cuda"), torch.zeros(4, 8, 16, device="cuda")
    b = starts_of([0, 2, 4])
    bad = [lambda: S.causal_conv(x.double(), w), lambda: S.causal_conv(x, w.half()), lambda: S.causal_conv(x, w[:4]), lambda: S.causal_conv(x, torch.zeros(8, 9, device="cuda")),
           lambda: S.causal_conv(x[0], w), lambda: S.causal_conv(x, w, activation="relu"), lambda: S.causal_conv(x, w, clip_start=b.long()),
           lambda: S.causal_conv(x, w, clip_start=b.cpu()), lambda: S.causal_conv(x, w, clip_start=b[:1]), lambda: S.causal_conv(x, w, clip_start=b, state=st),
           lambda: S.causal_conv(x, w, clip_start=b, state=st[:2].half()), lambda: S.causal_conv(x, w, bias=torch.zeros(7, device="cuda")), lambda: S.causal_conv(x, w.cpu()),
           lambda: S.causal_conv_step(x, w, st.transpose(0, 1).contiguous().transpose(0, 1)), lambda: S.causal_conv_step(x, w, st[:3]), lambda: S.causal_conv_step(x, w, None),
           lambda: S.causal_conv_step(x.clone().requires_grad_(), w, st), lambda: S.causal_conv_step(x, w, torch.zeros(5, 3, 8, device="cuda")[:4], state_out=st.half()),
           lambda: S.selective_scan(x, x.half(), A, Bm, Bm), lambda: S.selective_scan(x, x, A.half(), Bm, Bm), lambda: S.selective_scan(x, x, A, Bm[:3], Bm),
           lambda: S.selective_scan(x, x, A, Bm, Bm[:, :8]), lambda: S.selective_scan(x, x, torch.zeros(8, 65, device="cuda"), Bm, Bm), lambda: S.selective_scan(x, x, A, Bm, Bm, z=x[:, :7]),
           lambda: S.selective_scan(x, x, A, Bm, Bm, D=torch.zeros(8, 1, device="cuda")), lambda: S.selective_scan(x, x, A, Bm, Bm, state=hs), lambda: S.selective_scan(x, x, A, Bm, Bm.cpu()),
           lambda: S.selective_scan_step(x, x, A, Bm, Bm, hs.half()), lambda: S.selective_scan_step(x, x, A, Bm, Bm, hs.transpose(1, 2).contiguous().transpose(1, 2)),
           lambda: S.selective_scan_step(x, x, A.clone().requires_grad_(), Bm, Bm, hs), lambda: S.rms_norm(x, w), lambda: S.rms_norm(x, None), lambda: S.rms_norm(x, torch.ones(8, device="cuda"), eps=-1.0),
           lambda: S.rms_norm(x, torch.ones(8, device="cuda"), residual=x.half()), lambda: S.rms_norm(x, torch.ones(8, device="cuda"), residual=x[:2]),
           lambda: S.rms_norm_fp8(x.clone().requires_grad_(), torch.ones(8, device="cuda")), lambda: S.rms_norm(x[:, :0], torch.ones(0, device="cuda"))]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail("refusal %d did not happen" % i)
    big = torch.zeros(8 * 3 * 8 + 4, device="cuda")              # state_out that overlaps the state
    with pytest.raises(RuntimeError, match="overlaps"):
        S.causal_conv_step(x, w, big[:96].view(4, 3, 8), state_out=big[4:100].view(4, 3, 8))
    # a state that a pending gradient needs may not be moved on behind autograd's back
    s0 = hs.clone().requires_grad_()
    s1 = (s0 * 1.0)
    y = S.selective_scan(x, x, A, Bm, Bm, clip_start=starts_of([0, 1, 2, 3, 4]), state=s1)
    with torch.no_grad():
        S.selective_scan_step(x, x, A, Bm, Bm, s1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_under_saved_tensor_hooks(S):
    """Offloading packs the slices that were saved, another hook spreads them out: the gradients are bit for bit those of calls
    on arrays that are laid out so from the start."""
    gen = torch.Generator().manual_seed(21)
    rows, ch, N, b = 75, 24, 16, [0, 30, 30, 71]
    packed = lambda t: t.contiguous().clone()
    spread = lambda t: torch.cat([t, torch.full_like(t[:, :1], float("nan")).expand(-1, 9)], 1)[:, :t.shape[1]]
    slices = lambda t: t if t.is_contiguous() else spread(t)     # (the norm's own sum, which it saves, stays packed)
    plain, on_cpu = torch.autograd.graph.saved_tensors_hooks, torch.autograd.graph.save_on_cpu
    for dt in DTYPES.values():
        wide = rnd(gen, rows, 4 * ch + 2 * N + 3, dtype=dt)
        at = lambda c, n: wide[:, c:c + n]
        acts = [at(0, ch), at(ch + 1, ch), at(4 * ch, N), at(4 * ch + N, N), at(2 * ch, ch), at(3, ch), at(5, ch), at(7, ch), at(ch, ch)]
        others = [-torch.exp(rnd(gen, ch, N)), rnd(gen, ch), rnd(gen, ch, 4), rnd(gen, ch), rnd(gen, 3, ch, N), rnd(gen, 3, 3, ch, dtype=dt)]
        dy, dh, dc = rnd(gen, rows, ch, dtype=dt), rnd(gen, 3, ch, N), rnd(gen, 3, 3, ch, dtype=dt)

        def gradients(hooks, lay=lambda t: t):
            L = [lay(t).detach().requires_grad_() for t in acts] + [t.detach().requires_grad_() for t in others]
            u, delta, B, C, z, x, n1, n2, res, A, D, w, bias, h0, c0 = L
            with hooks:
                y, h = S.selective_scan(u, delta, A, B, C, D, z, bias, clip_start=starts_of(b), state=h0, return_state=True)
                v, c = S.causal_conv(x, w, bias, starts_of(b), c0, return_state=True)
                n = S.rms_norm(n1, D)
                m, t = S.rms_norm(n2, D, res)
            return torch.autograd.grad([y, h, v, c, n, m, t], L, [dy, dh, dy, dc, dy, dy, dy])

        for lay, hooks in ((packed, on_cpu()), (packed, on_cpu(pin_memory=True)), (spread, plain(slices, lambda t: t))):
            want = gradients(plain(lambda t: t, lambda t: t), lay)
            for i, (p, q) in enumerate(zip(want, gradients(hooks))):
                assert torch.equal(p, q), (dt, lay is packed, i)


@pytest.mark.parametrize("N", [1, 3, 4, 8, 16, 24, 64])
def test_scan_rows_at_the_largest_stride(S, N):
    """Every array a slice of rows 2^24 elements apart, the most that is taken without a copy: results are those of packed arrays."""
    gen, rows, ch, b = torch.Generator().manual_seed(N), 60, 20000, [0, 33, 58]               # (so wide that the rows are one chunk, both ways)
    held = torch.empty(rows, 1 << 24, device="cuda")             # 4 GB
    A, D, h0 = -torch.exp(rnd(gen, ch, N)), rnd(gen, ch), rnd(gen, 2, ch, N)
    dy, dh, views, at = rnd(gen, rows, ch), rnd(gen, 2, ch, N), [], 0
    for n in (ch, ch, N, N, ch):
        views.append(held[:, at:at + n].copy_(torch.randn(rows, n, generator=gen)))
        at += n + 1
    runs = []
    for t in (views, [v.contiguous() for v in views]):
        L = [v.detach().requires_grad_() for v in (*t, A, D, h0)]
        u, delta, B, C, z, a, d, h = L
        assert t is not views or B.stride(0) == 1 << 24
        y, f = S.selective_scan(u, delta, a, B, C, d, z, clip_start=starts_of(b), state=h, return_state=True)
        runs.append([y, f, *torch.autograd.grad([y, f], L, [dy, dh])])
        with torch.no_grad():
            s = torch.ones(rows, ch, N, device="cuda")
            runs[-1] += [S.selective_scan_step(u, delta, a, B, C, s, d, z), s]
    for i, (p, q) in enumerate(zip(*runs)):
        assert torch.equal(p, q), i


def test_convolution_and_norm_rows_at_the_largest_stride(S):
    gen, rows, ch, b = torch.Generator().manual_seed(1), 70, 8, [0, 33, 68]
    held = torch.empty(rows, 1 << 24, device="cuda")
    views = [held[:, at:at + ch].copy_(torch.randn(rows, ch, generator=gen)) for at in (0, 8)]
    w, nw, dy = rnd(gen, ch, 4), rnd(gen, ch), rnd(gen, rows, ch)
    runs = []
    for t in (views, [v.contiguous() for v in views]):
        L = [v.detach().requires_grad_() for v in (*t, w, nw)]
        out = [S.causal_conv(L[0], L[2], clip_start=starts_of(b)), *S.rms_norm(L[0], L[3], L[1]), S.rms_norm(L[0], L[3])]
        runs.append([*out, *torch.autograd.grad(out, L, [dy] * 4), *(q.float() for q in S.rms_norm_fp8(t[0], nw, t[1]))])
        runs[-1].append(S.causal_conv_step(t[0], w, torch.ones(rows, 3, ch, device="cuda")))
    for i, (p, q) in enumerate(zip(*runs)):
        assert torch.equal(p, q), i


@pytest.mark.parametrize("rows,taps,N", [(70, 4, 16), (70, 8, 4), (9, 3, 24), (1000, 6, 16), (70, 2, 40)])
@pytest.mark.parametrize("bounds", [[-5, 30, 75], [-3, -1, 70], [0, 30, 200], [5, 2000, 3000], [80, 90], [-9, -4], [-(1 << 31), (1 << 31) - 1], [-7, -7, 20, 20, 5000, 5000],
                                    [20, 10, 40, 5, 90], [60, 0, 70], [69, 3, 2]])
def test_every_entry_is_written_whatever_the_offsets(S, monkeypatch, rows, taps, N, bounds):
    """Outputs, gradients and workspaces come filled with NaN.  Offsets outside the array count as its nearer end, states included; with
    offsets that decrease every row is written all the same."""
    gen, ch, clips = torch.Generator().manual_seed(rows + N), 8, len(bounds) - 1
    allocate, like = torch.Tensor.new_empty, torch.empty_like
    spoil = lambda t: t.fill_(255 if t.dtype == torch.uint8 else float("nan"))
    monkeypatch.setattr(torch.Tensor, "new_empty", lambda self, *a, **k: spoil(allocate(self, *a, **k)))
    monkeypatch.setattr(torch, "empty_like", lambda *a, **k: spoil(like(*a, **k)))
    t = [rnd(gen, rows, n) for n in (ch, ch, N, N, ch)] + [rnd(gen, clips, ch, N), rnd(gen, clips, taps - 1, ch)]
    A, w, dy, dh, dc = -rnd(gen, ch, N).abs(), rnd(gen, ch, taps), rnd(gen, rows, ch), rnd(gen, clips, ch, N), rnd(gen, clips, taps - 1, ch)
    runs = []
    for b in (bounds, [min(max(v, 0), rows) for v in bounds]):
        L = [v.detach().requires_grad_() for v in t]
        y, h = S.selective_scan(L[0], L[1], A, L[2], L[3], None, L[4], clip_start=starts_of(b), state=L[5], return_state=True)
        v, c = S.causal_conv(L[0], w, None, starts_of(b), L[6], return_state=True)
        of_rows = [y, v, *torch.autograd.grad([y, h], L[:5], [dy, dh], retain_graph=True), *torch.autograd.grad([v, c], L[:1], [dy, dc], retain_graph=True)]
        of_clips = [h, c, *torch.autograd.grad([y, h], L[5:6], [dy, dh]), *torch.autograd.grad([v, c], L[6:], [dy, dc])]
        runs.append(of_rows + (of_clips if bounds == sorted(bounds) else []))
    for i, (p, q) in enumerate(zip(*runs)):
        assert bool(torch.isfinite(p).all()), i
        assert torch.equal(p, q), i


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("channels", [5, 64, 1030, 2048, 9000, 33000])
def test_rms_norm_fp8_of_tiny_rows(S, dtype, channels):
    """Rows of numbers around the smallest normal one, 1.2e-38, and far below 1, zeros among them: the nearest values all the same."""
    gen, dt = torch.Generator().manual_seed(channels), DTYPES[dtype]
    size = torch.tensor([1e-20, 1e-30, 1e-35, 1e-36, 3e-37, 1e-37, 3e-38, 1e-38, 1e-39])[:, None]
    x = torch.randn(len(size), channels, generator=gen)
    x = (x / x.abs().amax(1, keepdim=True) * size).to(dt)
    x[:, 1] = 0.0
    w = torch.randn(channels, generator=gen).abs() + 0.5
    w[x[-1].abs().argmax()] = 2.0 ** 5                           # (the last row's scale, 32 x 1e-39 x 1000 / 448 = 7e-38, is a normal number)
    want = R.norm(x, w, None, 1e-6)
    assert float(want["scale"][0].min()) > 1.2e-38
    q, scale = S.rms_norm_fp8(x.cuda(), w.cuda())
    assert torch.equal(q.double().cpu(), want["q"])
    close("scale", scale, want["scale"][0], (channels / 16 + 28) * want["scale"][0])


@pytest.mark.parametrize("rows,channels,N,kind", [(200, 9, 3, "tiles"), (140, 67, 7, "gaps"), (400, 20, 16, "empties"), (70, 5, 16, "singles"), (333, 8, 24, "three"), (131, 18, 64, "tiles"),
                                                  (1300, 65, 4, "one"), (1300, 6, 16, "three")])
def test_scan_of_states_that_forget_at_once(S, rows, channels, N, kind):
    """A of -inf, or so low that its multiple leaves float32, wherever clips and chunks end: exp(s A) = 0.  The restatement, which
    takes finite numbers only, gets -1e9, for which exp(s A) is 0 in 64 bits too."""
    gen, b = torch.Generator().manual_seed(rows + N), bounds_of(kind, rows)
    a = scan_inputs(gen, rows, channels, N, torch.float32, 1 if b is None else len(b) - 1)
    pick = torch.randint(0, 3, (channels, N), generator=gen).cuda()
    pick[0] = 1
    a["A"] = torch.where(pick == 0, a["A"], torch.full_like(a["A"], -1e9))
    dy, df = rnd(gen, rows, channels), torch.randn_like(a["state"])
    want = R.scan(clip_start=b, dy=dy, dfinal=df, **a)
    a["A"] = torch.where(pick == 1, torch.full_like(a["A"], float("-inf")), torch.where(pick == 2, torch.full_like(a["A"], -3e38), a["A"]))
    L = {k: leaf(t) for k, t in a.items()}
    y, f = S.selective_scan(clip_start=starts_of(b), return_state=True, **L)
    close("y", y, *want["y"])
    close("final", f, *want["final"])
    for k, g in zip(L, torch.autograd.grad([y, f], list(L.values()), [dy, df])):
        close("d" + k, g, *want[k])
    with torch.no_grad():
        one = {k: (t if k in ("A", "D", "delta_bias") else t[:1]) for k, t in a.items()}
        want = R.scan(**dict(one, A=one["A"].clamp(min=-1e9)))
        close("y", S.selective_scan_step(**dict(one, state=one["state"].clone())), *want["y"])


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("channels,rows,bounds,bad", [(8, 40, [0, 5, 11, 13, 16, 27, 40], 2), (24, 700, [3, 130, 333, 340, 680, 690], 1),
                                                      (70, 3000, [0, 1000, 1011, 1500, 3000], 1)])
@pytest.mark.parametrize("N", [1, 4, 7, 24, 64])
def test_a_clip_does_not_spoil_its_neighbours_with_any_number_of_states(S, value, channels, rows, bounds, bad, N):
    gen, clips = torch.Generator().manual_seed(rows + N), len(bounds) - 1
    starts, row = starts_of(bounds), torch.arange(rows, device="cuda")
    hit = (row >= bounds[bad]) & (row < bounds[bad + 1])
    others = [i for i in range(clips) if i != bad]
    a, dy, dh = scan_inputs(gen, rows, channels, N, torch.float32, clips), rnd(gen, rows, channels), rnd(gen, clips, channels, N)
    per_row, runs = ("u", "delta", "B", "C", "z"), []
    for spoil in (False, True):
        t, g, f = {k: v.clone() for k, v in a.items()}, dy.clone(), dh.clone()
        if spoil:
            for v in [t[k] for k in per_row] + [g]:
                v[hit] = value
            t["state"][bad], f[bad] = value, value
        L = {k: leaf(v) for k, v in t.items()}
        y, h = S.selective_scan(clip_start=starts, return_state=True, **L)
        *d, dstate = torch.autograd.grad([y, h], [L[k] for k in per_row] + [L["state"]], [g, f])
        runs.append([v[~hit] for v in (y, *d)] + [v[others] for v in (h, dstate)])
    for i, (p, q) in enumerate(zip(*runs)):
        assert torch.equal(p, q), i


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_single_tokens_move_their_states_on(S, dtype):
    """A loop over single tokens, captured once and replayed: states and outputs as those of eager calls, step for step."""
    gen, clips, ch, N, dt = torch.Generator().manual_seed(31), 5, 48, 16, DTYPES[dtype]
    w, nw, a = rnd(gen, ch, 4), rnd(gen, ch) + 1.0, scan_inputs(gen, clips, ch, N, dt, clips)
    h0 = a.pop("state")
    x, conv, scan = a["u"].clone(), rnd(gen, clips, 3, ch, dtype=dt), h0.clone()
    c2, s2 = conv.clone(), scan.clone()

    def once(x, conv, scan):
        with torch.no_grad():
            n, t = S.rms_norm(x, nw, x)
            v = S.causal_conv_step(n, w, conv)
            return S.selective_scan_step(v, a["delta"], a["A"], a["B"], a["C"], scan, a["D"], a["z"], a["delta_bias"]), t, *S.rms_norm_fp8(v, nw)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        once(x, conv.clone(), scan.clone())
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once(x, conv, scan)
    conv.copy_(c2)
    scan.copy_(s2)
    for it in range(6):
        x.copy_(rnd(gen, clips, ch, dtype=dt))
        want = once(x, c2, s2)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip((*out, conv, scan), (*want, c2, s2)):
            assert torch.equal(p.float(), q.float()), it


def test_events_of_a_batch_as_packed_rows(S):
    """Offsets from a batch's index per event: its clips by one call are its clips one by one."""
    from eventad_amd import synthetic
    b = synthetic.make_batch(64, 64, 3000, 3, with_image=False).to("cuda")
    gen = torch.Generator().manual_seed(1)
    clip_start = torch.searchsorted(b.batch, torch.arange(b.num_graphs + 1, device=b.batch.device)).int()
    x = torch.cat([b.x.float().reshape(len(b.batch), -1), b.pos.float()], 1) @ rnd(gen, b.x.float().reshape(len(b.batch), -1).shape[1] + b.pos.shape[1], 24)
    w, A, B, C = rnd(gen, 24, 4), -torch.exp(rnd(gen, 24, 16)), x[:, :16], x[:, 8:]
    v = S.causal_conv(x, w, clip_start=clip_start)
    y = S.selective_scan(v, x, A, B, C, clip_start=clip_start)
    at = clip_start.tolist()
    assert at[-1] == len(b.batch)
    for lo, hi in zip(at, at[1:]):
        assert bool((b.batch[lo:hi] == b.batch[lo]).all())
        one = S.causal_conv(x[lo:hi], w)
        assert torch.equal(v[lo:hi], one)
        alone = S.selective_scan(one, x[lo:hi], A, B[lo:hi], C[lo:hi])
        # other chunks: float32 sums over up to 3000 rows joined elsewhere
        assert float((y[lo:hi] - alone).abs().max()) <= 1e-4 * float(alone.abs().max())


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_block_has_the_same_gradients(S, reentrant):
    """torch.utils.checkpoint forms a block's saved tensors again in the backward pass."""
    from torch.utils.checkpoint import checkpoint
    gen = torch.Generator().manual_seed(41)
    p = {k: leaf(v) for k, v in block_weights(gen, 24, 40, 16, 4, 5).items()}
    x, res, b = rnd(gen, 137, 24), rnd(gen, 137, 24), starts_of([0, 50, 50, 130])
    dy, dr = rnd(gen, 137, 24), rnd(gen, 137, 24)
    results = []
    for again in (False, True):
        L = [leaf(x), leaf(res)]
        f = lambda x, res, *w: block(S, dict(zip(p, w)), x, res, b)[:2]
        out = checkpoint(f, *L, *p.values(), use_reentrant=reentrant) if again else f(*L, *p.values())
        for t in p.values():
            t.grad = None
        torch.autograd.backward(out, [dy, dr])
        results.append([*(o.detach() for o in out), *(t.grad.clone() for t in (*L, *p.values()))])
    for i, (s, t) in enumerate(zip(*results)):
        assert torch.equal(s, t), i


@pytest.mark.parametrize("channels", [40, 2048, 9000])
def test_rms_norm_fp8_scale_of_subnormal_products(S, channels):
    """With a small eps a row of subnormal numbers has a scale in the normal range: it keeps all its bits."""
    gen = torch.Generator().manual_seed(channels)
    size = torch.tensor([1e-38, 1e-39, 1e-41, 1e-43])[:, None]
    x = torch.randn(len(size), channels, generator=gen)
    x = x / x.abs().amax(1, keepdim=True) * size
    w = torch.rand(channels, generator=gen) + 0.5
    want = R.norm(x, w, None, 2.0 ** -100)                       # y = h w 2^50: the squares of h vanish beside eps
    q, scale = S.rms_norm_fp8(x.cuda(), w.cuda(), eps=2.0 ** -100)
    assert torch.equal(q.double().cpu(), want["q"])
    got = scale.double().cpu()
    # the quotient's root, its reciprocal (2 units each) and one rounding
    assert bool(((got - want["scale"][0]).abs() <= 6 * UNIT * want["scale"][0]).all())
