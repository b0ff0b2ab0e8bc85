"""The causal convolution and the selective scan in 64 bits, token by token, with their gradients written out.

With ``size`` set, every term enters by its absolute value: the result is the sum of the sizes of what is added up, which is what
rounding errors are relative to."""
import torch


def _silu(x):
    return x * torch.sigmoid(x)


def _d_silu(x):
    s = torch.sigmoid(x)
    return s + x * s * (1 - s)


def _f64(*ts):
    return [None if t is None else t.detach().double() for t in ts]


def pieces(n, b, cu):
    """(row, first token, last token + 1) of every sequence"""
    return [(i, 0, n) for i in range(b)] if cu is None else [(0, x, y) for x, y in zip(cu[:-1], cu[1:])]


def conv(x, weight, bias, act, state=None, cu=None, dy=None, dstate=None, size=False):
    """{y, state} and, with dy, {dx, dweight, dbias, dinitial}"""
    x, weight, bias, state, dy, dstate = _f64(x, weight, bias, state, dy, dstate)
    b, n, c = x.shape
    w = weight.shape[1]
    mag = torch.abs if size else (lambda t: t)
    seqs = pieces(n, b, cu)
    out = {"y": torch.zeros_like(x), "state": x.new_zeros(len(seqs), w - 1, c)}
    if dy is not None:
        out.update(dx=torch.zeros_like(x), dweight=torch.zeros_like(weight), dbias=x.new_zeros(c), dinitial=x.new_zeros(len(seqs), w - 1, c))
    for i, (r, lo, hi) in enumerate(seqs):
        before = x.new_zeros(w - 1, c) if state is None else state[i]
        xs = torch.cat([before, x[r, lo:hi]])
        p = x.new_zeros(hi - lo, c) if bias is None else bias.expand(hi - lo, c)
        ps = mag(p)
        for j in range(w):
            p = p + weight[:, j] * xs[j:j + hi - lo]
            ps = ps + mag(weight[:, j] * xs[j:j + hi - lo])
        out["y"][r, lo:hi] = (ps if size else _silu(p)) if act else ps
        out["state"][i] = xs[hi - lo:]
        if dy is None:
            continue
        d = mag(dy[r, lo:hi]) * (mag(_d_silu(p)) + (ps if size else 0) if act else 1)
        dxs = torch.zeros_like(xs)
        for j in range(w):
            dxs[j:j + hi - lo] += mag(weight[:, j]) * d
            out["dweight"][:, j] += (d * mag(xs[j:j + hi - lo])).sum(0)
        if dstate is not None:
            dxs[hi - lo:] += mag(dstate[i])
        out["dbias"] += d.sum(0)
        out["dx"][r, lo:hi] = dxs[w - 1:]
        out["dinitial"][i] = dxs[:w - 1]
    return out


def scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False, state=None, cu=None, dy=None, dstate=None, size=False):
    """{y, state} and, with dy, {du, ddt, dA, dB, dC, dD, dz, ddt_bias, dinitial}.  B, C: (b, n, groups, states)."""
    u, dt, A, B, C, D, z, dt_bias, state, dy, dstate = _f64(u, dt, A, B, C, D, z, dt_bias, state, dy, dstate)
    b, n, c = u.shape
    groups, N = B.shape[2:]
    mag = torch.abs if size else (lambda t: t)
    raw = dt if dt_bias is None else dt + dt_bias
    step = torch.nn.functional.softplus(raw, threshold=1000) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    skip = u.new_zeros(c) if D is None else mag(D)
    u, By, Cy = mag(u), mag(B.repeat_interleave(c // groups, 2)), mag(C.repeat_interleave(c // groups, 2))
    rate = mag(A)
    gate = torch.ones_like(u) if z is None else mag(_silu(z))
    seqs = pieces(n, b, cu)
    out = {"y": torch.zeros_like(u), "state": u.new_zeros(len(seqs), c, N)}
    if dy is not None:
        out.update(du=torch.zeros_like(u), ddt=torch.zeros_like(u), dA=torch.zeros_like(A), dB=torch.zeros_like(B), dC=torch.zeros_like(C),
                   dD=u.new_zeros(c), dz=torch.zeros_like(u), ddt_bias=u.new_zeros(c), dinitial=u.new_zeros(len(seqs), c, N))
    for i, (r, lo, hi) in enumerate(seqs):
        h = u.new_zeros(c, N) if state is None else mag(state[i])
        hs = [h]
        for t in range(lo, hi):
            h = torch.exp(step[r, t][:, None] * A) * h + mag(step[r, t] * u[r, t])[:, None] * By[r, t]
            hs.append(h)
            out["y"][r, t] = ((Cy[r, t] * h).sum(1) + skip * u[r, t])
        out["state"][i] = h
        if dy is not None:
            g = u.new_zeros(c, N) if dstate is None else mag(dstate[i])
            for t in range(hi - 1, lo - 1, -1):
                a = torch.exp(step[r, t][:, None] * A)
                d = mag(dy[r, t])
                if z is not None:
                    out["dz"][r, t] = d * out["y"][r, t] * (mag(_d_silu(z[r, t])) if not size else 1 + z[r, t].abs())
                d = d * gate[r, t]
                now = g + d[:, None] * Cy[r, t]
                hn = hs[t - lo + 1]
                out["dC"][r, t] = (d[:, None] * hn).view(groups, c // groups, N).sum(1)
                out["dB"][r, t] = (now * mag(step[r, t] * u[r, t])[:, None]).view(groups, c // groups, N).sum(1)
                into = (now * By[r, t]).sum(1)
                e = now * a * hs[t - lo]
                out["du"][r, t] = mag(step[r, t]) * into + skip * d
                ddt = (into * u[r, t] + (e * rate).sum(1)) * slope[r, t]
                out["ddt"][r, t] = ddt
                out["ddt_bias"] += ddt
                out["dA"] += e * mag(step[r, t])[:, None]
                out["dD"] += d * u[r, t]
                g = a * now
            out["dinitial"][i] = g
        out["y"][r, lo:hi] *= gate[r, lo:hi]
    return out


def within(got, want, size, steps):
    """Whether got is the rounded want: half a step of its type relative to the value (for fp16, half of its smallest step at
    least), and for the fp32 arithmetic before, `steps` roundings of 2^-22 (two units, as the fast exponential and division have)
    relative to the sizes of what is added up.  Returns the worst excess, at most 1."""
    finfo = torch.finfo(got.dtype)
    room = finfo.eps / 2 * want.abs() + steps * 2.0 ** -22 * size + finfo.smallest_normal * finfo.eps
    return float(((got.double() - want).abs() / room).max()) if got.numel() else 0.0
