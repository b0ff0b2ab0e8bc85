"""What is measured of the recurrent operators: ``causal_conv`` and ``selective_scan`` over prompts and training batches,
``causal_conv_step`` and ``selective_scan_step`` for single tokens.

A case is one call: a forward pass (``op`` "forward"), a forward and a backward pass ("train"), or one token of every row of a
decoding batch ("step").  With ``own`` false the operators are computed from their formulas with elementary torch operations:

    causal_conv      y_t = act(bias + sum_j weight_j x_(t-w+1+j))                       (channel by channel)
    selective_scan   h_t = exp(dt_t A) h_(t-1) + dt_t u_t B_t,   y_t = (<C_t, h_t> + D u_t) silu(z_t),   dt = softplus(dt + dt_bias)

x, u, dt, z are (batch, tokens, channels); B, C are (batch, tokens, groups, states), shared by the channels of a group.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
WIDTH = 4  # taps of the convolution


def _scan(name, op, dtype, b, n, c, states=16, groups=1, lens="", gate=True, softplus=True):
    return _named(name, kind="scan", op=op, dtype=dtype, b=b, n=n, c=c, states=states, groups=groups, lens=lens, gate=gate, softplus=softplus)


def _conv(name, op, dtype, b, n, c, lens="", act=True):
    return _named(name, kind="conv", op=op, dtype=dtype, b=b, n=n, c=c, lens=lens, act=act)


def _named(name, **case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # a short prompt through one narrow layer: launches and latency
        _conv("conv_prompt", "forward", "bf16", 1, 256, 2048),
        # a training batch, the largest of the convolution
        _conv("conv_train", "train", "bf16", 8, 2048, 4096),
        # packed documents, one of them a token long and one empty, at an odd number of channels in fp32
        _conv("conv_train_packed", "train", "fp32", 1, 6003, 1000, lens="2500,1,0,3001,501"),
        # one token of a small decoding batch, and of a large one
        _conv("conv_step", "step", "bf16", 8, 1, 2048),
        _conv("conv_step_batch", "step", "bf16", 256, 1, 4096),
        # a short prompt: the smallest scan
        _scan("scan_prompt", "forward", "bf16", 1, 256, 2048),
        # prefill of a long prompt, the largest
        _scan("scan_prefill", "forward", "bf16", 1, 16384, 4096),
        # an ordinary training layer
        _scan("scan_train", "train", "bf16", 2, 2048, 4096),
        # packed documents, two groups of channels with a B and C of their own, fp16
        _scan("scan_train_packed", "train", "fp16", 1, 6003, 1536, groups=2, lens="2500,1,0,3001,501"),
        # fp32 with more states, step sizes computed by the caller, no gate
        _scan("scan_train_fp32", "train", "fp32", 2, 1000, 1536, states=32, gate=False, softplus=False),
        # one token of a single sequence, and of a large decoding batch
        _scan("scan_step", "step", "bf16", 1, 1, 2048),
        _scan("scan_step_batch", "step", "bf16", 256, 1, 4096),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _channels(rng):
    """Multiples of 64 mostly, any number sometimes."""
    c = _log_uniform(rng, 96, 8192)
    return c if rng.random() < 0.25 else max(64, c // 64 * 64)


def _cut(rng, n):
    """Lengths of packed documents that fill n tokens, some of them empty or one token long."""
    cuts = sorted(rng.randrange(n + 1) for _ in range(rng.randrange(1, 12)))
    if rng.random() < 0.5:
        cuts = sorted(cuts + [cuts[0], min(n, cuts[0] + 1)])
    return ",".join(str(y - x) for x, y in zip([0] + cuts, cuts + [n]))


def draw(rng):
    """The ranges: 1 to 8 batch rows (steps: 1 to 512), 1 to 32768 tokens, 64 to 8192 channels, 8 to 64 states, up to 4 groups;
    packed sometimes; bf16 mostly."""
    kind = rng.choice(["scan", "scan", "conv"])
    op = rng.choices(["train", "forward", "step"], [50, 25, 25])[0]
    dtype = rng.choices(["bf16", "fp16", "fp32"], [60, 20, 20])[0]
    c = _channels(rng)
    states = rng.choices([8, 16, 32, 64, 12], [15, 55, 15, 10, 5])[0]
    groups = rng.choice([1, 1, 2, 4])
    if c % groups:
        groups = 1
    if op == "step":
        b, n, lens = _log_uniform(rng, 1, 512), 1, ""
    else:
        b = rng.choice([1, 1, 1, 2, 2, 3, 4, 8])
        # tokens x channels x states (x 2 with a backward pass) of the largest listed case
        most = (1 << 26) * 16 / (c * b * (states if kind == "scan" else 16)) / (4 if op == "train" else 1)
        n = _log_uniform(rng, 1, max(64, min(32768, most)))
        lens = _cut(rng, n) if b == 1 and rng.random() < 0.5 else ""
    if kind == "conv":
        return _conv(None, op, dtype, b, n, c, lens, rng.random() < 0.8)
    return _scan(None, op, dtype, b, n, c, states, groups, lens, rng.random() < 0.8, rng.random() < 0.8)


def _lens(case):
    return [int(x) for x in case["lens"].split(",")] if case["lens"] else [case["n"]] * case["b"]


def _make(case, seed, device):
    """The inputs as a layer has them: x and z are halves of one projection's output, dt, B and C parts of another's."""
    g = torch.Generator(device=device).manual_seed(int(seed))
    dtype, b, n, c = DTYPES[case["dtype"]], case["b"], case["n"], case["c"]
    step = case["op"] == "step"

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    rows = (b,) if step else (b, n)
    xz = normal(*rows, 2 * c).to(dtype)
    t = {}
    if case["kind"] == "conv":
        t.update(x=xz[..., :c], weight=normal(c, WIDTH) * 0.5, bias=normal(c) * 0.1)
        if step:
            t["state"] = normal(2 * b, WIDTH - 1, c).to(dtype)
    else:
        N, G = case["states"], case["groups"]
        rank = max(1, c // 16)
        proj = normal(*rows, rank + 2 * G * N).to(dtype)
        dt = normal(*rows, c) * 0.5
        bias = torch.expm1(torch.exp(torch.rand(c, generator=g, device=device) * math.log(100.0) + math.log(1e-3))).log()
        if not case["softplus"]:
            dt, bias = torch.nn.functional.softplus(dt + bias), None
        x = normal(*rows, c)
        t.update(u=(x * torch.sigmoid(x)).to(dtype), dt=dt.to(dtype),
                 A=-torch.arange(1, N + 1, device=device, dtype=torch.float32) * torch.exp(0.1 * normal(c, N)),
                 B=proj[..., rank:rank + G * N].unflatten(-1, (G, N)), C=proj[..., rank + G * N:].unflatten(-1, (G, N)),
                 D=1 + 0.1 * normal(c), z=xz[..., c:] if case["gate"] else None, dt_bias=bias)
        if step:
            t["state"] = normal(2 * b, c, N)
    if step:
        t["slots"] = torch.randperm(2 * b, generator=g, device=device)[:b].to(torch.int32)
    if case["lens"]:
        ends = np.concatenate([[0], np.cumsum(_lens(case))]).astype(np.int32)
        t["cu_seqlens"] = torch.from_numpy(ends).to(device)
    if case["op"] == "train":
        t["dy"] = normal(b, n, c).to(dtype)
    return t


WITH_GRADIENT = {"conv": ("x", "weight", "bias"), "scan": ("u", "dt", "A", "B", "C", "D", "z", "dt_bias")}


def prepare(case, seed):
    t = _make(case, seed, torch.device("cuda", torch.cuda.current_device()))
    if case["op"] == "train":
        for name in WITH_GRADIENT[case["kind"]]:
            if t[name] is not None:
                t[name] = t[name].detach().requires_grad_(True)
    return {"case": case, "t": t}


def run(state):
    case, t = state["case"], state["t"]
    if own:
        return _run_own(case, t)
    with torch.no_grad():
        if case["kind"] == "conv":
            return _plain_conv_step(case, t) if case["op"] == "step" else _plain_conv(case, t)
        return _plain_scan_step(case, t) if case["op"] == "step" else _plain_scan(case, t)


def _run_own(case, t):
    import lasp_b200
    op = case["op"]
    if case["kind"] == "conv":
        act = "silu" if case["act"] else None
        if op == "step":
            return {"y": lasp_b200.causal_conv_step(t["state"], t["x"], t["weight"], t["bias"], activation=act, slots=t["slots"]), "state": t["state"]}
        got = lasp_b200.causal_conv(t["x"], t["weight"], t["bias"], activation=act, cu_seqlens=t.get("cu_seqlens"), return_state=op == "forward")
    else:
        args = [t[k] for k in ("u", "dt", "A", "B", "C", "D", "z", "dt_bias")]
        if op == "step":
            return {"y": lasp_b200.selective_scan_step(t["state"], *args, dt_softplus=case["softplus"], slots=t["slots"]), "state": t["state"]}
        got = lasp_b200.selective_scan(*args, dt_softplus=case["softplus"], cu_seqlens=t.get("cu_seqlens"), return_state=op == "forward")
    if op == "forward":
        return {"y": got[0], "state": got[1]}
    names = [k for k in WITH_GRADIENT[case["kind"]] if t[k] is not None]
    return {"y": got.detach(), **dict(zip(names, torch.autograd.grad(got, [t[k] for k in names], t["dy"])))}


# ---- the plain forms: 32 bits, parallel over the tokens ---------------------------------------------------------------------
def _place(t, n):
    """For each token: how many of its sequence lie before it, and how many from it on."""
    at = torch.arange(n, device=t["cu_seqlens"].device) if "cu_seqlens" in t else None
    if at is None:
        return None
    cu = t["cu_seqlens"].long()
    row = torch.searchsorted(cu, at, right=True) - 1   # (of sequences that begin at the same token the last: the others are empty)
    return at - cu[row], cu[row + 1] - at


def _plain_conv(case, t):
    x, weight, bias = t["x"].float(), t["weight"], t["bias"]
    n, w, dtype = case["n"], WIDTH, t["x"].dtype
    pad = torch.nn.functional.pad
    taps = pad(x, (0, 0, w - 1, 0)).unfold(1, w, 1)                                     # (b, n, c, w)
    place = _place(t, n)
    if place:
        inside = place[0][:, None] >= torch.arange(w - 1, -1, -1, device=x.device)      # (n, w)
        taps = taps * inside[None, :, None, :]
    pre = (taps * weight).sum(-1) + bias
    gate = torch.sigmoid(pre) if case["act"] else None
    out = {"y": (pre * gate if case["act"] else pre).to(dtype)}
    if case["op"] == "forward":
        if place:
            cu, back = t["cu_seqlens"].long(), torch.arange(w - 1, 0, -1, device=x.device)
            rows = cu[1:, None] - back                                                  # (sequences, w - 1)
            return {**out, "state": (x[0][rows.clamp(min=0)] * (rows >= cu[:-1, None])[..., None]).to(dtype)}
        return {**out, "state": pad(x, (0, 0, w - 1, 0))[:, n:].to(dtype)}
    d = t["dy"].float()
    if case["act"]:
        d = d * gate * (1 + pre * (1 - gate))
    ahead = pad(d, (0, 0, 0, w - 1)).unfold(1, w, 1)                                    # d of this and the next w - 1 tokens
    if place:
        ahead = ahead * (place[1][:, None] > torch.arange(w, device=x.device))[None, :, None, :]
    return {**out, "x": (ahead * weight.flip(1)).sum(-1).to(dtype), "weight": (taps * d[..., None]).sum((0, 1)), "bias": d.sum((0, 1))}


def _plain_conv_step(case, t):
    slots = t["slots"].long()
    taps = torch.cat([t["state"][slots].float(), t["x"].float()[:, None]], 1)           # (b, w, c)
    pre = (taps * t["weight"].t()).sum(1) + t["bias"]
    t["state"][slots] = taps[:, 1:].to(t["state"].dtype)
    return {"y": (pre * torch.sigmoid(pre) if case["act"] else pre).to(t["x"].dtype), "state": t["state"]}


def _linear_recurrence(a, x):
    """h with h_t = a_t h_(t-1) + x_t along dimension 1, by doubling; a and x are used up."""
    step = 1
    while step < x.shape[1]:
        x[:, step:] += a[:, step:] * x[:, :-step]
        a[:, step:] = a[:, step:] * a[:, :-step]
        step *= 2
    return x


def _step_size(case, t):
    dt = t["dt"].float()
    if t["dt_bias"] is not None:
        dt = dt + t["dt_bias"]
    return torch.clamp(dt, min=0) + torch.log1p(torch.exp(-dt.abs())) if case["softplus"] else dt, dt


def _of_groups(x, c):
    """(..., groups, states) -> (..., channels, states)"""
    return x.float().repeat_interleave(c // x.shape[-2], dim=-2)


def _plain_scan(case, t):
    u, dtype, n, c = t["u"].float(), t["u"].dtype, case["n"], case["c"]
    dt, raw = _step_size(case, t)
    B, C = _of_groups(t["B"], c), _of_groups(t["C"], c)
    a = torch.exp(dt[..., None] * t["A"])                                               # (b, n, c, states)
    place = _place(t, n)
    if place:
        a = a * (place[0] > 0)[None, :, None, None]                                     # nothing enters a sequence
    h = _linear_recurrence(a.clone(), (dt * u)[..., None] * B)
    y0 = (h * C).sum(-1) + t["D"] * u
    gate = None
    if t["z"] is not None:
        z = t["z"].float()
        s = torch.sigmoid(z)
        gate = z * s
    out = {"y": (y0 * gate if gate is not None else y0).to(dtype)}
    if case["op"] == "forward":
        if place:
            cu = t["cu_seqlens"].long()
            return {**out, "state": h[0, (cu[1:] - 1).clamp(min=0)] * (cu[1:] > cu[:-1])[:, None, None]}
        return {**out, "state": h[:, -1].contiguous()}
    d = t["dy"].float()
    if gate is not None:
        out["z"] = (d * y0 * s * (1 + z * (1 - s))).to(dtype)
        d = d * gate
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)                        # g_t = C_t d_t + a_(t+1) g_(t+1)
    g = _linear_recurrence(later.flip(1), (d[..., None] * C).flip(1)).flip(1)
    del later
    per_group = (*u.shape[:2], case["groups"], c // case["groups"], case["states"])
    out["C"] = (d[..., None] * h).reshape(per_group).sum(3).to(dtype)
    out["B"] = (g * (dt * u)[..., None]).reshape(per_group).sum(3).to(dtype)
    through = g * a
    through[:, 1:] *= h[:, :-1]
    through[:, :1] = 0
    gB = (g * B).sum(-1)
    ddt = gB * u + (through * t["A"]).sum(-1)
    out["A"] = (through * dt[..., None]).sum((0, 1))
    out["u"] = (gB * dt + t["D"] * d).to(dtype)
    out["D"] = (d * u).sum((0, 1))
    if case["softplus"]:
        ddt = ddt * torch.sigmoid(raw)
    out["dt"] = ddt.to(dtype)
    if t["dt_bias"] is not None:
        out["dt_bias"] = ddt.sum((0, 1))
    return out


def _plain_scan_step(case, t):
    u, slots, c = t["u"].float(), t["slots"].long(), case["c"]
    dt, _ = _step_size(case, t)
    h = torch.exp(dt[..., None] * t["A"]) * t["state"][slots] + (dt * u)[..., None] * _of_groups(t["B"], c)
    t["state"][slots] = h
    y = (h * _of_groups(t["C"], c)).sum(-1) + t["D"] * u
    if t["z"] is not None:
        z = t["z"].float()
        y = y * z * torch.sigmoid(z)
    return {"y": y.to(t["u"].dtype), "state": t["state"]}


def work(case):
    """Every input read once and every output written once; the arithmetic of the recurrences."""
    b, n, c, size = case["b"], case["n"], case["c"], DTYPES[case["dtype"]].itemsize
    tokens, train, step = b * n, case["op"] == "train", case["op"] == "step"
    sequences = len(_lens(case))
    if case["kind"] == "conv":
        elements = tokens * c
        moved = elements * size * (4 if train else 2) + c * (WIDTH + 1) * 4 * (2 if train else 1)   # x, y; dy, dx
        if step:
            moved += 2 * b * (WIDTH - 1) * c * size + 4 * b
        elif not train:
            moved += sequences * (WIDTH - 1) * c * size
        return {"bytes": moved, "flops": elements * (2 * WIDTH + 6) * (3 if train else 1)}
    N, G = case["states"], case["groups"]
    wide = 3 + (1 if case["gate"] else 0)                                                # u, dt, y, z
    moved = tokens * size * (wide * c + 2 * G * N) + c * (N + 2) * 4
    if train:                                                                            # dy read; du, ddt, dz, dB, dC written
        moved += tokens * size * (wide * c + 2 * G * N) + c * (N + 2) * 4
    elif step:
        moved += 2 * b * c * N * 4 + 4 * b
    else:
        moved += sequences * c * N * 4
    # dt A, exp, (dt u) B, a h + x, C h; and for the gradients g, dC, dB, g a h, and their sums into du, ddt, dA
    return {"bytes": moved, "flops": tokens * c * (7 * N + 10 + ((17 * N + 20) if train else 0))}


# ---- the definition, token by token in 64 bits --------------------------------------------------------------------------------
def exact(case, seed):
    t = _make(case, seed, torch.device("cuda", torch.cuda.current_device()))
    t = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in t.items()}
    if case["op"] == "step":
        return (_exact_conv_step if case["kind"] == "conv" else _exact_scan_step)(case, t)
    parts, begin = [], 0
    for length in _lens(case) if case["lens"] else [case["n"]]:   # one packed sequence at a time
        rows = slice(begin, begin + length)
        one = {k: v[:, rows] if v is not None and v.dim() >= 3 else v for k, v in t.items()}
        parts.append((_exact_conv if case["kind"] == "conv" else _exact_scan)(case, one, length))
        begin += length
    out = {}
    for name in parts[0]:
        pieces = [p[name] for p in parts]
        if name in ("weight", "bias", "A", "D", "dt_bias"):
            out[name] = sum(pieces)
        else:
            out[name] = torch.cat(pieces, 1 if case["lens"] and name != "state" else 0)
    return out


def _d_silu(x):
    s = 1 / (1 + torch.exp(-x))
    return s + x * s * (1 - s)


def _exact_conv(case, t, n):
    x, weight, c = t["x"], t["weight"], case["c"]
    before = torch.cat([torch.zeros(x.shape[0], WIDTH - 1, c, dtype=x.dtype, device=x.device), x], 1)
    pre = t["bias"].expand(x.shape)
    for j in range(WIDTH):
        pre = pre + weight[:, j] * before[:, j:j + n]
    out = {"y": pre / (1 + torch.exp(-pre)) if case["act"] else pre}
    if case["op"] == "forward":
        return {**out, "state": before[:, n:]}
    d = t["dy"] * _d_silu(pre) if case["act"] else t["dy"]
    dx = torch.zeros_like(before)
    dw = torch.zeros_like(weight)
    for j in range(WIDTH):
        dx[:, j:j + n] += weight[:, j] * d
        dw[:, j] = (d * before[:, j:j + n]).sum((0, 1))
    return {**out, "x": dx[:, WIDTH - 1:], "weight": dw, "bias": d.sum((0, 1))}


def _exact_conv_step(case, t):
    slots, state = t["slots"].tolist(), t["state"].clone()
    y = torch.empty_like(t["x"])
    for i, s in enumerate(slots):
        taps = torch.cat([state[s], t["x"][i:i + 1]])
        y[i] = t["bias"] + torch.einsum("wc,cw->c", taps, t["weight"])
        state[s] = taps[1:]
    return {"y": y / (1 + torch.exp(-y)) if case["act"] else y, "state": state}


def _wide(x, c):
    rows, G, N = x.shape
    return x[:, :, None].expand(rows, G, c // G, N).reshape(rows, c, N)


def _exact_dt(case, t):
    v = t["dt"] if t["dt_bias"] is None else t["dt"] + t["dt_bias"]
    return torch.logaddexp(v, torch.zeros_like(v)) if case["softplus"] else v


def _exact_scan(case, t, n):
    u, A, D, c, N, rows = t["u"], t["A"], t["D"], case["c"], case["states"], t["u"].shape[0]
    dt = _exact_dt(case, t)
    h = torch.zeros(rows, c, N, dtype=A.dtype, device=A.device)
    kept, y0 = [], torch.zeros_like(u)
    for i in range(n):
        h = torch.exp(dt[:, i, :, None] * A) * h + (dt[:, i] * u[:, i])[..., None] * _wide(t["B"][:, i], c)
        y0[:, i] = torch.einsum("bcn,bcn->bc", h, _wide(t["C"][:, i], c)) + D * u[:, i]
        if case["op"] == "train":
            kept.append(h)
    y = y0 if t["z"] is None else y0 * t["z"] / (1 + torch.exp(-t["z"]))
    if case["op"] == "forward":
        return {"y": y, "state": h}
    out = {"y": y}
    d = t["dy"]
    if t["z"] is not None:
        out["z"] = d * y0 * _d_silu(t["z"])
        d = d * t["z"] / (1 + torch.exp(-t["z"]))
    du, ddt, dB, dC = (torch.zeros_like(t[k]) for k in ("u", "dt", "B", "C"))
    dA, carry, groups = torch.zeros_like(A), torch.zeros_like(h), (rows, case["groups"], c // case["groups"], N)
    for i in range(n - 1, -1, -1):
        a = torch.exp(dt[:, i, :, None] * A)
        g = carry + d[:, i, :, None] * _wide(t["C"][:, i], c)
        dC[:, i] = (kept[i] * d[:, i, :, None]).view(groups).sum(2)
        dB[:, i] = (g * (dt[:, i] * u[:, i])[..., None]).view(groups).sum(2)
        into = (g * _wide(t["B"][:, i], c)).sum(-1)
        du[:, i] = into * dt[:, i] + D * d[:, i]
        ddt[:, i] = into * u[:, i]
        if i:
            da = g * a * kept[i - 1]
            dA += (da * dt[:, i, :, None]).sum(0)
            ddt[:, i] += (da * A).sum(-1)
        carry = g * a
    if case["softplus"]:
        v = t["dt"] if t["dt_bias"] is None else t["dt"] + t["dt_bias"]
        ddt = ddt / (1 + torch.exp(-v))
    out.update(u=du, dt=ddt, A=dA, B=dB, C=dC, D=(d * t["u"]).sum((0, 1)))
    if t["dt_bias"] is not None:
        out["dt_bias"] = ddt.sum((0, 1))
    return out


def _exact_scan_step(case, t):
    c, state, dt = case["c"], t["state"].clone(), _exact_dt(case, t)
    y = torch.empty_like(t["u"])
    for i, s in enumerate(t["slots"].tolist()):
        h = torch.exp(dt[i][:, None] * t["A"]) * state[s] + (dt[i] * t["u"][i])[:, None] * _wide(t["B"][i:i + 1], c)[0]
        state[s] = h
        y[i] = (h * _wide(t["C"][i:i + 1], c)[0]).sum(1) + t["D"] * t["u"][i]
    return {"y": y if t["z"] is None else y * t["z"] / (1 + torch.exp(-t["z"])), "state": state}
