"""float64 restatement of the sequence operators (eventad_amd/sequence.py) from their formulas, row by row: outputs, final
states and gradients, each with what rounding errors are proportional to -- a magnitude (the same sums over the absolute
values of their terms) or, for the scan, a running error bound.  Test infrastructure only; everything on the CPU."""
import torch


def _d(t):
    return None if t is None else t.detach().double().cpu()


def clips_of(clip_start, rows):
    b = [0, rows] if clip_start is None else [int(v) for v in clip_start]
    return list(zip(b, b[1:]))


def conv(x, w, bias=None, clip_start=None, state=None, silu=True, dy=None, dfinal=None):
    """-> {name: (value, magnitude)} for y, final and -- dy given -- x, weight, bias, state."""
    x, w, bias, state, dy, dfinal = (_d(t) for t in (x, w, bias, state, dy, dfinal))
    rows, D = x.shape
    K = w.shape[1]
    cl = clips_of(clip_start, rows)
    state = torch.zeros(len(cl), K - 1, D, dtype=torch.float64) if state is None else state
    y, ym = torch.zeros_like(x), torch.zeros_like(x)
    final = state.clone()
    g = {k: [torch.zeros_like(t), torch.zeros_like(t)] for k, t in (("x", x), ("weight", w), ("bias", w[:, 0]), ("state", state))}
    for s, (lo, hi) in enumerate(cl):
        n = hi - lo
        ext = torch.cat([state[s], x[lo:hi]])
        final[s] = ext[n:]
        dext, dextm = torch.zeros_like(ext), torch.zeros_like(ext)
        if dfinal is not None:
            dext[n:] += dfinal[s]
            dextm[n:] += dfinal[s].abs()
        for t in range(n):
            terms = ext[t:t + K] * w.t()
            pre = terms.sum(0) + (bias if bias is not None else 0.0)
            mag = terms.abs().sum(0) + (bias.abs() if bias is not None else 0.0)
            sg = torch.sigmoid(pre)
            y[lo + t] = pre * sg if silu else pre
            ym[lo + t] = mag                                     # |silu'| < 1.1
            if dy is not None:
                slope = sg * (1 + pre * (1 - sg)) if silu else torch.ones_like(pre)
                d = dy[lo + t] * slope
                dm = dy[lo + t].abs() * (1 + mag) if silu else dy[lo + t].abs()      # |silu''| <= 1/2: pre's error moves the slope
                dext[t:t + K] += w.t() * d
                dextm[t:t + K] += w.t().abs() * dm
                g["weight"][0] += (ext[t:t + K] * d).t()
                g["weight"][1] += (ext[t:t + K].abs() * dm).t()
                g["bias"][0] += d
                g["bias"][1] += dm
        g["state"][0][s], g["state"][1][s] = dext[:K - 1], dextm[:K - 1]
        g["x"][0][lo:hi], g["x"][1][lo:hi] = dext[K - 1:], dextm[K - 1:]
    out = {"y": (y, ym), "final": (final, final.abs())}
    if dy is not None:
        out.update({k: tuple(v) for k, v in g.items()})
    return out


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=True, clip_start=None, state=None, dy=None, dfinal=None):
    """-> {name: (value, error)} for y, final and -- dy given -- the gradients.  error: a running first-order bound, in units of
    2^-24, of what float32 arithmetic may be off: every quantity is carried as (value v, sum of |terms| m, error e) and a
    product's error is e1 m2 + m1 e2 + m1 m2, a sum's the sum of its parts' plus one unit of m per addition in sequence.
    Functions count the units their float32 forms may lose: softplus 16, exp 2, sigmoid 6; a step's argument delta + bias is
    rounded once, which moves softplus by |raw| relative units and exp(s A) by |s A| times the relative error of s."""
    u, delta, A, B, C, D, z, delta_bias, state, dy, dfinal = (_d(t) for t in (u, delta, A, B, C, D, z, delta_bias, state, dy, dfinal))
    rows, ch = u.shape
    N = A.shape[1]
    cl = clips_of(clip_start, rows)
    state = torch.zeros(len(cl), ch, N, dtype=torch.float64) if state is None else state
    skip = torch.zeros(ch, dtype=torch.float64) if D is None else D
    raw = delta if delta_bias is None else delta + delta_bias
    step = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    # relative error of the step; a step that is a difference of larger numbers loses their rounding (no softplus)
    rs = 16.0 + raw.abs() if softplus else 1.0 + (delta.abs() + (delta_bias.abs() if delta_bias is not None else 0.0)) / step.abs().clamp(min=1e-30)
    # numbers below the smallest normal one, 2^-126 (2^-102 units), count as zero: the step, and below its product with u
    flush = 2.0 ** -102
    rs = rs + flush / step.abs().clamp(min=1e-300)
    gate = torch.ones_like(u) if z is None else z * torch.sigmoid(z)
    rg = 8.0 if z is not None else 0.0
    span = 3.0 + rows / 4.0                                       # joining chunks: exp of a sum of up to rows / 4 steps per lane
    zero = lambda t: [torch.zeros_like(t), torch.zeros_like(t)]
    y, final = zero(u), [state.clone(), torch.zeros_like(state)]
    g = {"u": zero(u), "delta": zero(u), "A": zero(A), "B": zero(B), "C": zero(C), "D": zero(skip), "z": zero(u),
         "delta_bias": zero(skip), "state": zero(state)}
    mags = {"A": torch.zeros_like(A), "D": torch.zeros_like(skip), "delta_bias": torch.zeros_like(skip)}
    dot = 10.0                                                    # additions in sequence of a sum over the states
    for s, (lo, hi) in enumerate(cl):
        hs = [(state[s], state[s].abs(), torch.zeros_like(state[s]))]
        decays = []
        for t in range(lo, hi):
            e = step[t][:, None] * A
            a, ra = torch.exp(e), 3.0 + e.abs() * (rs[t][:, None] + span)
            b = (step[t] * u[t])[:, None] * B[t]
            v, m, err = hs[-1]
            m1 = a * m + b.abs()
            hs.append((a * v + b, m1, a * (err + m * ra) + b.abs() * (rs[t][:, None] + 2.0) + m1))
            decays.append((a, ra))
            v, m, err = hs[-1]
            pre, mag = (v * C[t]).sum(1) + skip * u[t], (m * C[t].abs()).sum(1) + (skip * u[t]).abs()
            off = (err * C[t].abs()).sum(1) + mag * dot
            y[0][t], y[1][t] = pre * gate[t], gate[t].abs() * (off + mag * (rg + 1.0))
            if dy is not None and z is not None:
                sg = torch.sigmoid(z[t])
                slope = sg * (1 + z[t] * (1 - sg))
                width = sg * (1 + z[t].abs() * (1 - sg))
                g["z"][0][t] = dy[t] * pre * slope
                g["z"][1][t] = dy[t].abs() * width * (off + mag * 24.0 * (1.0 + z[t].abs() * sg))
        final[0][s], final[1][s] = hs[-1][0], hs[-1][2]
        if dy is None:
            continue
        q = torch.zeros(ch, N, dtype=torch.float64) if dfinal is None else dfinal[s]
        qm, qe = q.abs(), torch.zeros_like(q)
        for t in range(hi - 1, lo - 1, -1):
            a, ra = decays[t - lo]
            d, x, r = dy[t] * gate[t], step[t] * u[t], rs[t][:, None]
            dm = d.abs()[:, None]
            q, qm = q + d[:, None] * C[t], qm + dm * C[t].abs()
            qe = qe + dm * C[t].abs() * (rg + 2.0) + qm
            (h0, m0, e0), (h1, m1, e1) = hs[t - lo], hs[t - lo + 1]
            deep = 12.0 + ch / 16.0                               # additions in sequence of a sum over the channels
            g["C"][0][t], g["C"][1][t] = (d[:, None] * h1).sum(0), (dm * (e1 + m1 * (rg + 2.0 + deep))).sum(0)
            xm = x.abs()[:, None]
            g["B"][0][t], g["B"][1][t] = (q * x[:, None]).sum(0), (xm * (qe + qm * (r + 2.0 + deep)) + flush * qm).sum(0)
            gb, gbm = (q * B[t]).sum(1), (qm * B[t].abs()).sum(1)
            gbe = (qe * B[t].abs()).sum(1) + gbm * dot
            g["u"][0][t] = skip * d + step[t] * gb
            g["u"][1][t] = (skip * d).abs() * (rg + 3.0) + step[t].abs() * (gbe + gbm * (rs[t] + 3.0))
            f, fm = q * a * h0, qm * a * m0
            fe = a * (qe * m0 + qm * e0 + qm * m0 * (ra + 3.0))
            slope, rsl = (torch.sigmoid(raw[t]), 6.0 + raw[t].abs()) if softplus else (torch.ones(ch, dtype=torch.float64), torch.zeros(ch, dtype=torch.float64))
            dd = (u[t] * gb + (A * f).sum(1)) * slope
            ddm = (u[t].abs() * gbm + (A.abs() * fm).sum(1)) * slope
            dde = (u[t].abs() * gbe + (A.abs() * fe).sum(1)) * slope + ddm * (dot + 4.0 + rsl)
            if softplus:
                dde = dde + flush * (u[t].abs() * gbm + (A.abs() * fm).sum(1))                # the slope
            g["delta"][0][t], g["delta"][1][t] = dd, dde
            sm = step[t].abs()[:, None]
            for k, v, m, err in (("A", step[t][:, None] * f, sm * fm, sm * (fe + fm * (r + 2.0))),
                                 ("D", d * u[t], (d * u[t]).abs(), (d * u[t]).abs() * (rg + 3.0)), ("delta_bias", dd, ddm, dde)):
                g[k][0] += v
                g[k][1] += err
                mags[k] += m
            q, qe, qm = a * q, a * (qe + qm * (ra + 1.0)), a * qm
        g["state"][0][s], g["state"][1][s] = q, qe
    for k, m in mags.items():
        g[k][1] += m * (8.0 + rows)                               # additions in sequence of a sum over the rows
    out = {"y": tuple(y), "final": tuple(final)}
    if dy is not None:
        out.update({k: tuple(v) for k, v in g.items()})
    return out


def norm(x, w, residual=None, eps=1e-6, dy=None, dsum=None):
    """-> {name: (value, magnitude)} for y, sum (rounded to x's type) and -- dy given -- h (the gradient of x and residual) and
    weight; "scale" and "q" of the 8-bit form."""
    total = x if residual is None else (x.detach().double() + residual.detach().double()).to(x.dtype)
    h, w, dy, dsum = _d(total), _d(w), _d(dy), _d(dsum)
    inv = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    y = h * inv * w
    out = {"y": (y, y.abs()), "sum": (h, h.abs())}
    top = y.abs().amax(1, keepdim=True)
    scale = torch.where(top > 0, top / 448.0, torch.ones_like(top))
    grid = torch.ldexp(torch.ones_like(y), torch.frexp(y / scale)[1].clamp(min=-5) - 4)     # 3 fraction bits, subnormal below 2^-6
    out["scale"], out["q"] = (scale[:, 0], scale[:, 0]), torch.round(y / scale / grid) * grid
    if dy is not None:
        e = dy * w
        m = (e * h).mean(1, keepdim=True)
        mm = (e * h).abs().mean(1, keepdim=True)
        extra = 0.0 if dsum is None else dsum
        out["h"] = (inv * (e - h * inv * inv * m) + extra,
                    inv * (e.abs() + h.abs() * inv * inv * mm) + (0.0 if dsum is None else dsum.abs()))
        out["weight"] = ((dy * h * inv).sum(0), (dy * h * inv).abs().sum(0))
    return out
