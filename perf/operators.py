"""What the sequence operators of eventad_amd.sequence are measured on: the short causal convolution, the selective
state-space scan and the root-mean-square norm over packed clips, each with its plain form in elementary torch
operations and its definition in 64 bits.

Rows are packed: rows clip_start[s] .. clip_start[s+1]-1 of every [rows, channels] array are clip s, oldest first, and
rows that belong to no clip come out as zeros.  Parameters are float32, activations have the case's type, states of the
scan are float32."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
E4M3_MAX = 448.0


# ---------------------------------------------------------------------------------------------------------------- cases
def _conv(name, mode, rows, channels, clips, taps, dtype, ragged=False, carry=False):
    return {"name": name, "op": "conv", "mode": mode, "rows": rows, "channels": channels, "clips": clips, "taps": taps,
            "dtype": dtype, "ragged": ragged, "carry": carry}


def _scan(name, mode, rows, channels, clips, state, dtype, ragged=False, carry=False, gate=True):
    return {"name": name, "op": "scan", "mode": mode, "rows": rows, "channels": channels, "clips": clips, "state": state,
            "dtype": dtype, "ragged": ragged, "carry": carry, "gate": gate}


def _norm(name, mode, rows, channels, dtype):
    return {"name": name, "op": "norm", "mode": mode, "rows": rows, "channels": channels, "dtype": dtype}


def listed():
    return [
        # one new event per clip of the default batch (6 clips) at the head's width: pure latency
        _conv("conv_step_6x256_f32", "step", 6, 256, 6, 4, "f32"),
        # prompts: clips of up to a pooled level's 2240 nodes, no two of one length, continued from earlier rows
        _conv("conv_prompt_ragged_f16", "forward", 17920, 1024, 8, 4, "f16", ragged=True, carry=True),
        # training over the events of a batch of 8 clips of 50k events at the head's width
        _conv("conv_train_8x50k_f32", "train", 400000, 256, 8, 4, "f32"),
        # one new event per clip of the default batch, through the scan
        _scan("scan_step_6x256_f32", "step", 6, 256, 6, 16, "f32"),
        # serving: single tokens of many clips at once, bound by the states' bytes
        _scan("scan_step_2048x1024_bf16", "step", 2048, 1024, 2048, 16, "bf16"),
        # ragged prompts with states in and out
        _scan("scan_prompt_ragged_bf16", "forward", 16384, 1024, 29, 16, "bf16", ragged=True, carry=True),
        # one clip of 500k events, the longest the bench's configurations have, on the graph branch's 64 channels
        _scan("scan_prompt_500k_f32", "forward", 500000, 64, 1, 16, "f32"),
        # training: the pooled nodes of a batch of 8 clips at the head's width
        _scan("scan_train_8x2240_f32", "train", 17920, 256, 8, 16, "f32"),
        # training at a wide layer, ragged clips
        _scan("scan_train_ragged_bf16", "train", 16001, 1024, 13, 16, "bf16", ragged=True),
        # the norm in front of a single-token step
        _norm("norm_6x256_f32", "forward", 6, 256, "f32"),
        # the norm in front of an 8-bit product
        _norm("norm_8bit_16384x2048_bf16", "eightbit", 16384, 2048, "bf16"),
        # the norm of the training step over a batch's events
        _norm("norm_train_400k_bf16", "train", 400000, 256, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("conv", "scan", "norm"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op == "norm":
        channels = _log_int(rng, 16, 8192)
        return {"op": op, "mode": rng.choice(("forward", "eightbit", "train")), "dtype": dtype, "channels": channels,
                "rows": _log_int(rng, 1, min(400000, 100000000 // channels))}
    mode = rng.choice(("step", "forward", "train"))
    channels = _log_int(rng, 16, 2048)
    if op == "conv":
        case = {"op": op, "mode": mode, "taps": rng.randint(2, 6)}
        most = min(400000, 100000000 // channels)
    else:
        state = rng.choice((4, 8, 16, 16, 16, 24, 32, 64))
        case = {"op": op, "mode": mode, "state": state, "gate": rng.random() < 0.7}
        most = min(400000, 260000000 // (channels * state))
    if mode == "step":
        rows = clips = _log_int(rng, 1, min(4096, 33000000 // (channels * case.get("state", 8))))
        ragged = carry = False
    else:
        rows = _log_int(rng, 1, most)
        clips = min(_log_int(rng, 1, 64), rows)
        ragged = rng.random() < 0.7
        carry = mode == "forward" and rng.random() < 0.5
    case.update({"dtype": dtype, "channels": channels, "rows": rows, "clips": clips, "ragged": ragged, "carry": carry})
    return case


# --------------------------------------------------------------------------------------------------------------- inputs
def _clip_bounds(case, seed):
    """Clip offsets as a list: equal shares, or -- ragged -- cuts anywhere (empty clips and single rows among them) with a
    few rows behind the last clip, as in a batch padded to a bucket."""
    rows, clips = case["rows"], case["clips"]
    if not case["ragged"]:
        return [rows * s // clips for s in range(clips + 1)]
    rng = random.Random(seed * 7919 + 17)
    end = rows - min(rows // 64, 40)
    cuts = sorted(rng.randint(0, end) for _ in range(clips - 1))
    if clips > 3:
        cuts[1] = cuts[0]                       # an empty clip
    return [0] + cuts + [end]


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, D = case["rows"], case["channels"]

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(dtype)

    st = {"case": case}
    train = case["mode"] == "train"
    if case["op"] == "norm":
        st["x"], st["residual"] = normal(rows, D, dtype=dt), normal(rows, D, scale=3.0, dtype=dt)
        st["weight"] = 1.0 + normal(D, scale=0.2)
        if train:
            st["dy"], st["dres"] = normal(rows, D, dtype=dt), normal(rows, D, dtype=dt)
        leaves = ("x", "residual", "weight")
    else:
        bounds = _clip_bounds(case, seed)
        st["clip_start"] = torch.tensor(bounds, dtype=torch.int32, device=dev)
        st["longest"] = max(b - a for a, b in zip(bounds, bounds[1:]))
        if case["op"] == "conv":
            K = case["taps"]
            st["x"] = normal(rows, D, dtype=dt)
            st["weight"], st["bias"] = normal(D, K, scale=K ** -0.5), normal(D, scale=0.1)
            if case["carry"] or case["mode"] == "step":
                st["state"] = normal(case["clips"], K - 1, D, dtype=dt)
            leaves = ("x", "weight", "bias")
        else:
            N = case["state"]
            # a layer's decays: A = -(1 .. N) at first, step sizes spread over 1e-3 .. 1e-1 by the bias, both moved by training
            first = torch.arange(1, N + 1, device=dev, dtype=torch.float32).expand(D, N)
            st["A"] = -first * torch.exp(normal(D, N, scale=0.1))
            step = torch.exp(torch.rand(D, generator=gen, device=dev) * math.log(100.0) + math.log(1e-3))
            st["delta_bias"] = step + torch.log(-torch.expm1(-step))
            st["u"], st["delta"] = normal(rows, D, dtype=dt), normal(rows, D, scale=0.5, dtype=dt)
            st["B"], st["C"] = normal(rows, N, dtype=dt), normal(rows, N, dtype=dt)
            st["D"] = 1.0 + normal(D, scale=0.1)
            st["z"] = normal(rows, D, dtype=dt) if case["gate"] else None
            if case["carry"] or case["mode"] == "step":
                st["state"] = normal(case["clips"], D, N, scale=0.5)
            leaves = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")
        if train:
            st["dy"] = normal(rows, D, dtype=dt)
        if case["mode"] == "step":
            st["state_out"] = torch.empty_like(st["state"])
    if train:
        st["leaves"] = [k for k in leaves if st[k] is not None]
        for k in st["leaves"]:
            st[k].requires_grad_(True)
    return st


# ------------------------------------------------------------------------------------------------- plain forms (32 bits)
def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _silu_slope(x):
    s = 1.0 / (1.0 + torch.exp(-x))
    return s * (1.0 + x * (1.0 - s))


def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-x.abs()))


def _rows_of(st):
    """Per row: its clip, the row its clip starts at, whether it belongs to a clip."""
    start = st["clip_start"].long()
    row = torch.arange(st["case"]["rows"], device=start.device)
    clip = torch.searchsorted(start, row, right=True) - 1
    live = (clip >= 0) & (clip < start.numel() - 1)
    clip = clip.clamp(0, start.numel() - 2)
    return row, clip, start[clip], live


def _conv_taps(st, x):
    """The K inputs of every row, oldest first: rows of the clip, its state's rows before it, or zeros."""
    K = st["case"]["taps"]
    row, clip, first, live = _rows_of(st)
    state = st.get("state")
    taps = []
    for k in range(K):
        pos = row - (K - 1 - k)
        inside = (pos >= first) & live
        v = x[pos.clamp(min=0)] * inside[:, None]
        if state is not None and k < K - 1:
            back = (K - 1 + pos - first).clamp(0, K - 2)
            v = torch.where(inside[:, None], v, state[clip, back].float())
        taps.append(v)
    return taps, live


def _conv_plain(st):
    case, K, dt = st["case"], st["case"]["taps"], DTYPES[st["case"]["dtype"]]
    x, w, bias = st["x"].detach().float(), st["weight"].detach(), st["bias"].detach()
    if case["mode"] == "step":
        window = torch.cat([st["state"].float(), x[:, None]], 1)                     # [S, K, D]
        pre = (window * w.t()[None]).sum(1) + bias
        return {"y": _silu(pre).to(dt), "state": window[:, 1:].to(dt)}
    taps, live = _conv_taps(st, x)
    pre = bias.expand_as(x)
    for k in range(K):
        pre = pre + taps[k] * w[:, k]
    out = {"y": (_silu(pre) * live[:, None]).to(dt)}
    if case["carry"]:
        start = st["clip_start"].long()
        rel = (start[1:] - start[:-1])[:, None] - (K - 1) + torch.arange(K - 1, device=x.device)
        old = torch.gather(st["state"], 1, (rel + K - 1).clamp(0, K - 2)[:, :, None].expand(-1, -1, x.shape[1]))
        new = st["x"][(start[:-1, None] + rel).clamp(0, case["rows"] - 1)]
        out["state"] = torch.where((rel >= 0)[:, :, None], new, old)
    if case["mode"] == "train":
        dpre = st["dy"].float() * _silu_slope(pre) * live[:, None]
        _, clip, _, _ = _rows_of(st)
        dx = torch.zeros_like(x)
        for k in range(K):
            lag = K - 1 - k
            if lag >= x.shape[0]:
                continue
            same = ((clip[lag:] == clip[:x.shape[0] - lag]) & live[lag:])[:, None]
            dx[:x.shape[0] - lag] += dpre[lag:] * same * w[:, k]
        out["x"] = dx.to(dt)
        out["weight"] = torch.stack([torch.sum(dpre * t, 0, dtype=torch.float64) for t in taps], 1).float()
        out["bias"] = torch.sum(dpre, 0, dtype=torch.float64).float()
    return out


def _recurrence(a, b, longest):
    """h_t = a_t h_{t-1} + b_t along the first axis by doubling: after the pass with shift d a row holds the sum of its
    last 2d terms."""
    d = 1
    while d < longest:
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _scan_plain(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    u, delta, B, C = (st[k].detach().float() for k in ("u", "delta", "B", "C"))
    A, skip = st["A"].detach(), st["D"].detach()
    z = None if st["z"] is None else st["z"].detach().float()
    raw = delta + st["delta_bias"].detach()
    step = _softplus(raw)
    if case["mode"] == "step":
        h = torch.exp(step[:, :, None] * A) * st["state"] + (step * u)[:, :, None] * B[:, None, :]
        y = (h * C[:, None, :]).sum(-1) + skip * u
        return {"y": (y if z is None else y * _silu(z)).to(dt), "state": h}
    row, clip, first, live = _rows_of(st)
    step = step * live[:, None]
    a = torch.exp(step[:, :, None] * A)
    b = (step * u)[:, :, None] * B[:, None, :]
    heads = ((row == first) & live).nonzero()[:, 0]
    if case["carry"]:
        b[heads] += a[heads] * st["state"][clip[heads]]
    a[heads] = 0.0
    h = _recurrence(a, b, st["longest"])
    del b
    y = (h * C[:, None, :]).sum(-1) + skip * u
    out = {"y": ((y if z is None else y * _silu(z)) * live[:, None]).to(dt)}
    if case["carry"]:
        start = st["clip_start"].long()
        last = (start[1:] - 1).clamp(min=0)
        out["state"] = torch.where((start[1:] > start[:-1])[:, None, None], h[last], st["state"])
    if case["mode"] != "train":
        return out
    dout = st["dy"].float() * live[:, None]
    dy = dout if z is None else dout * _silu(z)
    back = torch.zeros_like(a)
    back[:-1] = a[1:]
    g = _recurrence(back.flip(0), (dy[:, :, None] * C[:, None, :]).flip(0), st["longest"]).flip(0)
    del back
    dB = torch.sum(g * (step * u)[:, :, None], 1)
    dC = torch.sum(h * dy[:, :, None], 1)
    gB = (g * B[:, None, :]).sum(-1)
    a[1:] *= h[:-1]
    a[0] = 0.0
    a *= g                                                                           # g_t a_t h_{t-1}
    dstep = u * gB + (a * A).sum(-1)
    draw = dstep / (1.0 + torch.exp(-raw)) * live[:, None]
    out["u"] = (skip * dy + step * gB).to(dt)
    out["delta"] = draw.to(dt)
    out["A"] = torch.sum(a * step[:, :, None], 0, dtype=torch.float64).float()
    out["B"], out["C"] = dB.to(dt), dC.to(dt)
    out["D"] = torch.sum(dy * u, 0, dtype=torch.float64).float()
    if z is not None:
        out["z"] = (dout * y * _silu_slope(z)).to(dt)
    out["delta_bias"] = torch.sum(draw, 0, dtype=torch.float64).float()
    return out


def _e4m3(v):
    """The e4m3 value nearest to every float64, ties to even: 3 fraction bits, steps of 2^-9 below 2^-6."""
    exponent = torch.frexp(v)[1].clamp(min=-5) - 1
    grid = torch.ldexp(torch.ones_like(v), exponent - 3)
    return torch.round(v / grid) * grid


def _norm_plain(st):
    """The sum is rounded to the activations' type first: the norm and its gradient are those of the stored sum.  The 8-bit
    form works in 64 bits, because its values lie next to borders of the rounding."""
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    w = st["weight"].detach()
    total = (st["x"].detach().float() + st["residual"].detach().float()).to(dt)
    h = total.double() if case["mode"] == "eightbit" else total.float()
    inv = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    y = h * inv * w
    if case["mode"] == "eightbit":
        top = y.abs().amax(1, keepdim=True)
        scale = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
        return {"values": _e4m3(y / scale).to(torch.bfloat16), "scale": scale[:, 0].float(), "sum": total}
    out = {"y": y.to(dt), "sum": total}
    if case["mode"] == "train":
        dy = st["dy"].float()
        gw = dy * w
        dh = inv * (gw - h * inv * inv * (gw * h).mean(1, keepdim=True)) + st["dres"].float()
        out["x"] = out["residual"] = dh.to(dt)
        out["weight"] = torch.sum(dy * h * inv, 0, dtype=torch.float64).float()
    return out


# ------------------------------------------------------------------------------------------------ the framework's calls
def _with_gradients(st, out, grads):
    """A training step's gradients of `out` (name -> tensor) with respect to the leaves, beside the outputs."""
    got = torch.autograd.grad(list(out.values()), [st[k] for k in st["leaves"]], grads)
    return dict({k: v.detach() for k, v in out.items()}, **dict(zip(st["leaves"], got)))


def _own(st):
    from eventad_amd import sequence
    case, mode = st["case"], st["case"]["mode"]
    if case["op"] == "norm":
        if mode == "eightbit":
            q, scale, total = sequence.rms_norm_fp8(st["x"], st["weight"], residual=st["residual"], eps=EPS)
            return {"values": q.to(torch.bfloat16), "scale": scale, "sum": total}      # every e4m3 value is a bfloat16 value
        y, total = sequence.rms_norm(st["x"], st["weight"], residual=st["residual"], eps=EPS)
        out = {"y": y, "sum": total}
        return _with_gradients(st, out, [st["dy"], st["dres"]]) if mode == "train" else out
    if case["op"] == "conv":
        if mode == "step":
            y = sequence.causal_conv_step(st["x"], st["weight"], st["state"], bias=st["bias"], activation="silu",
                                          state_out=st["state_out"])
            return {"y": y, "state": st["state_out"]}
        r = sequence.causal_conv(st["x"], st["weight"], bias=st["bias"], activation="silu", clip_start=st["clip_start"],
                                 state=st.get("state"), return_state=case["carry"])
    else:
        args = (st["u"], st["delta"], st["A"], st["B"], st["C"])
        more = dict(D=st["D"], z=st["z"], delta_bias=st["delta_bias"], delta_softplus=True)
        if mode == "step":
            y = sequence.selective_scan_step(*args, st["state"], state_out=st["state_out"], **more)
            return {"y": y, "state": st["state_out"]}
        r = sequence.selective_scan(*args, clip_start=st["clip_start"], state=st.get("state"), return_state=case["carry"], **more)
    out = {"y": r[0], "state": r[1]} if case["carry"] else {"y": r}
    return _with_gradients(st, out, [st["dy"]]) if mode == "train" else out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"conv": _conv_plain, "scan": _scan_plain, "norm": _norm_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------ what it costs
def work(case):
    e = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    rows, D, mode = case["rows"], case["channels"], case["mode"]
    cells = rows * D
    if case["op"] == "norm":
        if mode == "eightbit":                       # x, residual in; sum, 8-bit values, scales out
            return {"bytes": cells * (3 * e + 1) + rows * 4 + D * 4, "flops": cells * 9}
        if mode == "forward":
            return {"bytes": cells * 4 * e + D * 4, "flops": cells * 5}
        return {"bytes": cells * 7 * e + D * 8, "flops": cells * 16}                # + dy, dsum in; one gradient for both inputs out
    if case["op"] == "conv":
        K = case["taps"]
        params = D * (K + 1) * 4
        if mode == "train":                          # x, dy in; y, dx out
            return {"bytes": cells * 4 * e + 2 * params, "flops": cells * (6 * K + 16)}
        carried = 2 * case["clips"] * (K - 1) * D * e if (case["carry"] or mode == "step") else 0
        return {"bytes": cells * 2 * e + params + carried, "flops": cells * (2 * K + 4)}
    N = case["state"]
    gate = 1 if case["gate"] else 0
    params = D * (N + 2) * 4
    if mode == "train":                              # u, delta, z, B, C, dout in; out and the gradients of the five out
        return {"bytes": cells * (6 + 2 * gate) * e + rows * N * 4 * e + 2 * params, "flops": cells * (20 * N + 50)}
    carried = 2 * case["clips"] * D * N * 4 if (case["carry"] or mode == "step") else 0
    return {"bytes": cells * (3 + gate) * e + rows * N * 2 * e + params + carried, "flops": cells * (7 * N + 20)}


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def _stepped64(a, b):
    """h_t = a_t h_{t-1} + b_t, row by row inside blocks of about sqrt(rows) rows, then block by block."""
    rows = a.shape[0]
    size = max(1, int(math.isqrt(rows)))
    blocks = -(-rows // size)
    pad = blocks * size - rows
    if pad:
        a = torch.cat([a, torch.ones_like(a[:1]).expand(pad, *a.shape[1:])])
        b = torch.cat([b, torch.zeros_like(b[:1]).expand(pad, *b.shape[1:])])
    a, h = a.reshape(blocks, size, *a.shape[1:]).clone(), b.reshape(blocks, size, *b.shape[1:]).clone()
    for i in range(1, size):
        h[:, i] += a[:, i] * h[:, i - 1]
        a[:, i] *= a[:, i - 1]
    for p in range(1, blocks):
        h[p] += a[p] * h[p - 1, -1]
    return h.reshape(blocks * size, *h.shape[2:])[:rows]


def _exact_conv(st):
    case, K = st["case"], st["case"]["taps"]
    x, w, bias = st["x"].detach().double(), st["weight"].detach().double(), st["bias"].detach().double()
    state = st["state"].double() if "state" in st else torch.zeros(case["clips"], K - 1, x.shape[1], dtype=torch.float64, device=x.device)
    if case["mode"] == "step":
        window = torch.cat([state, x[:, None]], 1)
        pre = torch.einsum("skd,dk->sd", window, w) + bias
        return {"y": pre * torch.sigmoid(pre), "state": window[:, 1:]}
    bounds = st["clip_start"].tolist()
    y, new_state = torch.zeros_like(x), state.clone()
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias)
    for s, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if hi == lo:
            continue
        ext = torch.cat([state[s], x[lo:hi]])
        pre = bias + sum(ext[k:k + hi - lo] * w[:, k] for k in range(K))
        sig = torch.sigmoid(pre)
        y[lo:hi] = pre * sig
        new_state[s] = ext[hi - lo:]
        if case["mode"] == "train":
            dpre = st["dy"][lo:hi].double() * sig * (1 + pre * (1 - sig))
            dext = torch.zeros_like(ext)
            for k in range(K):
                dext[k:k + hi - lo] += dpre * w[:, k]
                dw[:, k] += (dpre * ext[k:k + hi - lo]).sum(0)
            dx[lo:hi] = dext[K - 1:]
            db += dpre.sum(0)
    out = {"y": y}
    if case["carry"]:
        out["state"] = new_state
    if case["mode"] == "train":
        out.update({"x": dx, "weight": dw, "bias": db})
    return out


def _exact_scan(st):
    case = st["case"]
    u, delta, B, C, A, skip, bias = (st[k].detach().double() for k in ("u", "delta", "B", "C", "A", "D", "delta_bias"))
    z = None if st["z"] is None else st["z"].detach().double()
    raw = delta + bias
    step = torch.logaddexp(raw, torch.zeros_like(raw))
    gate = 1.0 if z is None else z * torch.sigmoid(z)
    if case["mode"] == "step":
        h = torch.exp(torch.einsum("sd,dn->sdn", step, A)) * st["state"].double() + torch.einsum("sd,sn->sdn", step * u, B)
        return {"y": (torch.einsum("sdn,sn->sd", h, C) + skip * u) * gate, "state": h}
    bounds = st["clip_start"].tolist()
    alive = torch.zeros(case["rows"], 1, dtype=torch.float64, device=u.device)
    alive[bounds[0]:bounds[-1]] = 1.0
    step = step * alive
    a = torch.exp(step[:, :, None] * A)
    b = (step * u)[:, :, None] * B[:, None, :]
    for s, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if hi > lo:
            if case["carry"]:
                b[lo] += a[lo] * st["state"][s].double()
            a[lo] = 0.0
    h = _stepped64(a, b)
    del b
    y = torch.matmul(h, C[:, :, None])[:, :, 0] + skip * u
    out = {"y": y * gate * alive}
    if case["carry"]:
        out["state"] = torch.stack([h[hi - 1] if hi > lo else st["state"][s].double()
                                    for s, (lo, hi) in enumerate(zip(bounds, bounds[1:]))])
    if case["mode"] != "train":
        return out
    dout = st["dy"].double() * alive
    dy = dout * gate
    later = torch.cat([a[1:], torch.zeros_like(a[:1])])
    g = _stepped64(later.flip(0), (dy[:, :, None] * C[:, None, :]).flip(0)).flip(0)
    del later
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    flow = g * a * before
    del before, a
    into = torch.matmul(g, B[:, :, None])[:, :, 0]
    draw = (u * into + (flow * A).sum(-1)) * torch.sigmoid(raw) * alive
    out["u"], out["delta"] = skip * dy + step * into, draw
    out["A"] = (flow * step[:, :, None]).sum(0)
    out["B"] = (g * (step * u)[:, :, None]).sum(1)
    out["C"] = (h * dy[:, :, None]).sum(1)
    out["D"] = (dy * u).sum(0)
    if z is not None:
        sig = torch.sigmoid(z)
        out["z"] = dout * y * sig * (1 + z * (1 - sig))
    out["delta_bias"] = draw.sum(0)
    return out


def _exact_norm(st):
    case, dt = st["case"], DTYPES[st["case"]["dtype"]]
    w = st["weight"].detach().double()
    total = (st["x"].detach().double() + st["residual"].detach().double()).to(dt)
    h = total.double()
    rms = torch.sqrt(h.pow(2).mean(1, keepdim=True) + EPS)
    unit = h / rms
    y = unit * w
    if case["mode"] == "eightbit":
        top = y.abs().amax(1, keepdim=True)
        scale = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
        levels = torch.arange(127, dtype=torch.uint8, device=h.device).view(torch.float8_e4m3fn).double()   # codes 0 .. 126
        size = (y / scale).abs()
        above = torch.searchsorted(levels, size.contiguous()).clamp(1, 126)
        middle = (levels[above - 1] + levels[above]) / 2
        up = (size > middle) | ((size == middle) & (above % 2 == 0))
        q = torch.where(up, levels[above], levels[above - 1])
        return {"values": torch.copysign(q, y), "scale": scale[:, 0], "sum": h}
    out = {"y": y, "sum": h}
    if case["mode"] == "train":
        gw = st["dy"].double() * w
        dh = (gw - unit * (gw * unit).mean(1, keepdim=True)) / rms + st["dres"].double()
        out.update({"x": dh, "residual": dh, "weight": (st["dy"].double() * unit).sum(0)})
    return out


def exact(case, seed):
    with torch.no_grad():
        return {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm}[case["op"]](prepare(case, seed))
