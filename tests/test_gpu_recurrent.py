"""causal_conv, selective_scan and their single-token steps against the formulas in 64 bits."""
import pytest
import torch

from tests import recurrent_formulas as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _cu(cu, dtype=torch.int32):
    return None if cu is None else torch.tensor(cu, dtype=dtype, device=DEV)


def _close(got, want, size, steps, names=None):
    for name in names or got:
        if got[name] is not None:
            assert got[name].shape == want[name].shape, (name, got[name].shape, want[name].shape)
            off = F.within(got[name], want[name], size[name], steps)
            assert off <= 1.0, (name, off)


# ---- convolution -------------------------------------------------------------------------------------------------------------
def conv_inputs(seed, dtype, b, n, c, width, sequences, ptype=F32, strided=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = _normal(g, b, n, 2 * c if strided else c).to(dtype)
    return dict(x=x[..., c:] if strided else x, weight=(_normal(g, c, width) * 0.5).to(ptype), bias=_normal(g, c).to(ptype),
                state=_normal(g, sequences, width - 1, c).to(dtype), dy=_normal(g, b, n, c).to(dtype), dstate=_normal(g, sequences, width - 1, c).to(dtype))


CONV = [
    # b, n, c, width, cu, dtype, parameters' type, strided
    (2, 37, 64, 4, None, BF16, F32, False),
    (2, 37, 64, 4, None, BF16, BF16, True),
    (1, 1, 8, 4, None, F32, F32, False),
    (3, 2, 24, 3, None, F16, F32, True),
    (1, 130, 257, 4, None, BF16, F32, False),         # an odd number of channels
    (2, 1000, 8, 2, None, F32, F32, False),
    (1, 600, 300, 4, None, F16, F16, True),
    (1, 100, 40, 4, [0, 0, 1, 2, 4, 33, 33, 100], F32, F32, False),
    (1, 100, 40, 3, [3, 10, 64, 90], BF16, F32, True),   # tokens in no sequence on both sides
    (1, 700, 9, 4, [0, 350, 351, 351, 699], BF16, F32, False),
]


@pytest.mark.parametrize("b,n,c,width,cu,dtype,ptype,strided", CONV)
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("full", [True, False])
def test_convolution(b, n, c, width, cu, dtype, ptype, strided, act, full):
    from lasp_b200 import causal_conv
    t = conv_inputs(n + c, dtype, b, n, c, width, len(cu) - 1 if cu else b, ptype, strided)
    names = ["x", "weight"] + (["bias", "state"] if full else [])
    leaf = {k: t[k].detach().requires_grad_(True) for k in names}
    y, last = causal_conv(leaf["x"], leaf["weight"], leaf.get("bias"), activation=act, initial_state=leaf.get("state"), cu_seqlens=_cu(cu), return_state=True)
    grads = torch.autograd.grad([y, last] if full else [y], list(leaf.values()), [t["dy"], t["dstate"]] if full else [t["dy"]])
    got = {"y": y.detach(), "state": last.detach(), **dict(zip(["dx", "dweight", "dbias", "dinitial"], grads))}
    args = (t["x"], t["weight"], t["bias"] if full else None, act == "silu", t["state"] if full else None, cu, t["dy"], t["dstate"] if full else None)
    _close(got, F.conv(*args), F.conv(*args, size=True), 40)   # 5 products, sigmoid and its derivative; sums of a run in fp32
    with torch.no_grad():
        alone = causal_conv(t["x"], leaf["weight"], leaf.get("bias"), activation=act, initial_state=leaf.get("state"), cu_seqlens=_cu(cu, torch.int64))
    assert torch.equal(alone, y)


# ---- scan --------------------------------------------------------------------------------------------------------------------------
def scan_inputs(seed, dtype, b, n, c, N, groups, sequences, gate=True, softplus=True, ptype=F32, strided=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rank = 3 if strided else 0
    proj = _normal(g, b, n, rank + 2 * groups * N).to(dtype)
    xz = _normal(g, b, n, 2 * c).to(dtype)
    t = dict(u=_normal(g, b, n, c).to(dtype), dt=(_normal(g, b, n, c) * 0.5 if softplus else torch.rand(b, n, c, generator=g, device=DEV) * 0.2).to(dtype),
             A=-torch.exp(_normal(g, c, N)), B=proj[..., rank:rank + groups * N].unflatten(-1, (groups, N)),
             C=proj[..., rank + groups * N:].unflatten(-1, (groups, N)), D=_normal(g, c).to(ptype), z=xz[..., c:] if gate else None,
             dt_bias=(_normal(g, c) - 2).to(ptype) if softplus else None, state=_normal(g, sequences, c, N),
             dy=_normal(g, b, n, c).to(dtype), dstate=_normal(g, sequences, c, N))
    return t if strided else {k: v if v is None else v.contiguous() for k, v in t.items()}


SCAN = [
    # b, n, c, states, groups, cu, dtype, parameters' type, gate, softplus, strided
    (2, 70, 64, 16, 1, None, BF16, F32, True, True, True),
    (1, 1, 16, 16, 1, None, F32, F32, True, True, False),
    (3, 2, 48, 16, 2, None, F16, F16, True, True, False),
    (1, 200, 37, 16, 1, None, F32, F32, False, False, False),    # channels that fill no tile
    (2, 65, 34, 5, 2, None, BF16, F32, True, True, True),         # few states, groups of 17
    (1, 129, 40, 32, 1, None, F32, F32, True, True, True),
    (1, 90, 20, 64, 4, None, F16, F32, True, False, True),
    (1, 63, 24, 33, 1, None, BF16, BF16, False, True, False),
    (1, 64, 8, 1, 1, None, F32, F32, True, True, False),
    (1, 150, 32, 16, 1, [0, 0, 1, 2, 66, 66, 130, 150], F32, F32, True, True, False),
    (1, 150, 32, 16, 2, [5, 70, 140], BF16, F32, True, True, True),
    (1, 300, 96, 12, 1, [0, 128, 299, 300, 300], F16, F32, False, True, False),
    (1, 150, 16, 64, 1, [0, 64, 128, 150], F32, F32, True, True, False),
]
GRADIENTS = dict(u="du", dt="ddt", A="dA", B="dB", C="dC", D="dD", z="dz", dt_bias="ddt_bias", state="dinitial")


def scan_args(t, names=("u", "dt", "A", "B", "C", "D", "z", "dt_bias")):
    return [t.get(k) for k in names]


@pytest.mark.parametrize("b,n,c,N,groups,cu,dtype,ptype,gate,softplus,strided", SCAN)
@pytest.mark.parametrize("full", [True, False])
def test_scan(b, n, c, N, groups, cu, dtype, ptype, gate, softplus, strided, full):
    from lasp_b200 import selective_scan
    t = scan_inputs(n + c, dtype, b, n, c, N, groups, len(cu) - 1 if cu else b, gate, softplus, ptype, strided)
    if not full:
        t.update(D=None, state=None, dstate=None)
    leaf = {k: t[k].detach().requires_grad_(True) for k in GRADIENTS if t[k] is not None}
    y, last = selective_scan(*scan_args(leaf), dt_softplus=softplus, initial_state=leaf.get("state"), cu_seqlens=_cu(cu), return_state=True)
    grads = torch.autograd.grad([y, last] if full else [y], list(leaf.values()), [t["dy"], t["dstate"]] if full else [t["dy"]])
    got = {"y": y.detach(), "state": last.detach(), **dict(zip([GRADIENTS[k] for k in leaf], grads))}
    args = dict(softplus=softplus, cu=cu, **{k: v for k, v in t.items()})
    # a decay's two units for each token that a value has come through, and 20 of the rest
    _close(got, F.scan(**args), F.scan(**args, size=True), 2 * n + 20)
    with torch.no_grad():
        alone = selective_scan(*scan_args(t), dt_softplus=softplus, initial_state=t["state"], cu_seqlens=_cu(cu, torch.int64))
    assert torch.equal(alone, y)


SEGMENTS = [   # few channels and many tokens: sequences are cut into segments (of 256 tokens and more), some of whose lengths are odd
    (1, 1301, 20, 16, 1, None, F32, F32, True, True, True),
    (2, 1025, 40, 32, 1, None, BF16, F32, True, True, False),
    (1, 777, 9, 64, 1, None, F16, F32, False, True, True),
    (1, 2113, 36, 16, 2, [3, 3, 903, 904, 1416, 2100], F32, F32, True, True, True),
    (1, 2049, 16, 24, 1, [0, 1, 258, 2049, 2049], BF16, F32, True, False, False),
]


@pytest.mark.parametrize("b,n,c,N,groups,cu,dtype,ptype,gate,softplus,strided", SEGMENTS)
@pytest.mark.parametrize("full", [True, False])
def test_scan_in_segments(b, n, c, N, groups, cu, dtype, ptype, gate, softplus, strided, full):
    test_scan(b, n, c, N, groups, cu, dtype, ptype, gate, softplus, strided, full)


def test_a_state_of_zero_stays_so_where_rates_grow():
    """A above zero: the decay of a whole segment is beyond fp32, that of a token is not."""
    from lasp_b200 import selective_scan
    n, c, N = 1400, 8, 16
    u, dt = torch.zeros(1, n, c, device=DEV), torch.ones(1, n, c, device=DEV)
    B, C = torch.ones(1, n, N, device=DEV), torch.ones(1, n, N, device=DEV)
    leaf = u.requires_grad_(True)
    y, last = selective_scan(leaf, dt, torch.full((c, N), 0.5, device=DEV), B, C, return_state=True)
    assert not y.any() and not last.any()
    assert not torch.autograd.grad(y, leaf, torch.zeros_like(y))[0].any()


# ---- single tokens -------------------------------------------------------------------------------------------------------------------
STEP = [
    # rows, slots, channels, states, groups, dtype, parameters' type, gate, softplus
    (1, 1, 64, 16, 1, BF16, F32, True, True),
    (5, 9, 100, 16, 2, F32, F32, True, True),
    (7, 7, 33, 5, 1, F16, F16, False, True),
    (3, 4, 40, 32, 1, BF16, BF16, True, False),
    (40, 64, 24, 64, 4, F32, F32, True, True),
    (2, 3, 9, 1, 1, F32, F32, True, True),
]


def _step_order(slots, count):
    """(row, slot) in the order in which tokens are taken"""
    return [(r, s) for r, s in enumerate(slots) if 0 <= s < count]


def _slots(seed, rows, count, kind):
    g = torch.Generator().manual_seed(seed)
    if kind == "none":
        return None
    slots = torch.randperm(count, generator=g)[:rows].tolist()
    if kind == "padded":
        slots[::2] = [-1 if i % 4 else count for i in range(0, rows, 2)]
    if kind == "repeated":
        slots = [slots[min(i // 2, rows // 2 - 1) if rows > 1 else 0] for i in range(rows)]
    return slots


@pytest.mark.parametrize("rows,count,c,N,groups,dtype,ptype,gate,softplus", STEP)
@pytest.mark.parametrize("kind", ["none", "some", "padded", "repeated"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_scan_step(rows, count, c, N, groups, dtype, ptype, gate, softplus, kind, index):
    from lasp_b200 import selective_scan_step
    slots = _slots(c, rows, count, kind)
    count = rows if slots is None else count
    t = scan_inputs(c, dtype, rows, 1, c, N, groups, count, gate, softplus, ptype, strided=True)
    state = t["state"].clone()
    one = {k: v[:, 0] if k in ("u", "dt", "B", "C", "z") and v is not None else v for k, v in t.items()}
    y = selective_scan_step(state, *scan_args(one), dt_softplus=softplus, slots=None if slots is None else torch.tensor(slots, dtype=index, device=DEV))
    want, size = t["state"].double(), t["state"].double().abs()
    ys, ysize = torch.zeros(rows, c, dtype=torch.float64, device=DEV), torch.zeros(rows, c, dtype=torch.float64, device=DEV)
    for r, s in _step_order(list(range(rows)) if slots is None else slots, count):
        args = {k: t[k][r:r + 1] if t[k] is not None else None for k in ("u", "dt", "B", "C", "z")}
        args.update({k: t[k] for k in ("A", "D", "dt_bias")}, softplus=softplus)
        for out, at, sz in ((want, ys, False), (size, ysize, True)):
            o = F.scan(**args, state=out[s:s + 1].clone(), size=sz)
            at[r], out[s] = o["y"][0, 0], o["state"][0]
    _close({"y": y, "state": state}, {"y": ys, "state": want}, {"y": ysize, "state": size}, 4 * rows + 20)
    untouched = [s for s in range(count) if s not in (range(rows) if slots is None else slots)]
    assert torch.equal(state[untouched], t["state"][untouched])


@pytest.mark.parametrize("rows,count,c,width,dtype,ptype", [(1, 1, 64, 4, BF16, F32), (6, 11, 100, 4, F32, F32), (5, 5, 33, 3, F16, F16), (33, 40, 2056, 2, BF16, BF16)])
@pytest.mark.parametrize("kind", ["none", "some", "padded", "repeated"])
@pytest.mark.parametrize("act", [None, "silu"])
def test_conv_step(rows, count, c, width, dtype, ptype, kind, act):
    from lasp_b200 import causal_conv_step
    slots = _slots(c, rows, count, kind)
    count = rows if slots is None else count
    t = conv_inputs(c, dtype, rows, 1, c, width, count, ptype, strided=True)
    state = t["state"].clone()
    y = causal_conv_step(state, t["x"][:, 0], t["weight"], t["bias"], activation=act, slots=None if slots is None else torch.tensor(slots, device=DEV))
    want = t["state"].double()
    ys, ysize = torch.zeros(rows, c, dtype=torch.float64, device=DEV), torch.zeros(rows, c, dtype=torch.float64, device=DEV)
    for r, s in _step_order(list(range(rows)) if slots is None else slots, count):
        for at, sz in ((ysize, True), (ys, False)):
            o = F.conv(t["x"][r:r + 1], t["weight"], t["bias"], act == "silu", want[s:s + 1], size=sz)
            at[r] = o["y"][0, 0]
        want[s] = o["state"][0]
    _close({"y": y}, {"y": ys}, {"y": ysize}, 40)
    assert torch.equal(state.double(), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("packed", [False, True])
def test_a_layer_from_prompt_to_tokens(dtype, packed):
    """Convolution and scan over a prompt, cut in two calls that hand their states on, then token by token: the outputs of one
    call over all tokens.  Steps and scans add in different orders: what separates them is counted as in the other tests."""
    from lasp_b200 import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    n, cut, prompt, c, N = 90, 40, 80, 48, 16
    lens = [n] * (3 if packed else 2)
    g = torch.Generator(device=DEV).manual_seed(5)
    b = len(lens)
    x, z = (_normal(g, b, n, c).to(dtype) for _ in range(2))
    w, bias, A, D = _normal(g, c, 4) * 0.5, _normal(g, c), -torch.exp(_normal(g, c, N)), _normal(g, c)
    dt, dt_bias = (_normal(g, b, n, c) * 0.5).to(dtype), _normal(g, c) - 2
    B, C = (_normal(g, b, n, N).to(dtype) for _ in range(2))
    conv = dict(activation="silu")
    whole = causal_conv(x, w, bias, **conv)
    want = selective_scan(whole, dt, A, B, C, D, z, dt_bias, dt_softplus=True)

    def over(lo, hi, states):
        piece = [t[:, lo:hi] for t in (x, dt, B, C, z)]
        cu = None
        if packed:
            piece = [t.reshape(1, -1, t.shape[-1]) for t in piece]
            cu = torch.arange(b + 1, device=DEV, dtype=torch.int32) * (hi - lo)
        xs, dts, Bs, Cs, zs = piece
        u, cs = causal_conv(xs, w, bias, initial_state=states[0], cu_seqlens=cu, return_state=True, **conv)
        y, ss = selective_scan(u, dts, A, Bs, Cs, D, zs, dt_bias, dt_softplus=True, initial_state=states[1], cu_seqlens=cu, return_state=True)
        return u.view(b, hi - lo, c), y.view(b, hi - lo, c), (cs, ss)

    u0, y0, states = over(0, cut, (None, None))
    u1, y1, states = over(cut, prompt, states)
    us, ys = [u0, u1], [y0, y1]
    for t in range(prompt, n):
        u = causal_conv_step(states[0], x[:, t], w, bias, **conv)
        ys.append(selective_scan_step(states[1], u, dt[:, t], A, B[:, t], C[:, t], D, z[:, t], dt_bias, dt_softplus=True)[:, None])
        us.append(u[:, None])
    assert torch.equal(torch.cat(us, 1), whole)
    got = torch.cat(ys, 1)
    args = dict(u=whole, dt=dt, A=A, B=B[:, :, None], C=C[:, :, None], D=D, z=z, dt_bias=dt_bias, softplus=True)
    ref, size = F.scan(**args), F.scan(**args, size=True)
    _close({"y": got}, ref, size, 2 * n + 20)
    _close({"y": want}, ref, size, 2 * n + 20)
    _close({"state": states[1]}, ref, size, 2 * n + 20)


@pytest.mark.parametrize("packed", [False, True])
def test_nothing_to_do(packed):
    """No tokens, no rows: states go through, gradients of the parameters are zero."""
    from lasp_b200 import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    for b, n in ((1, 0), (0, 4)) if not packed else ((1, 0),):
        cu = torch.zeros(4, dtype=torch.int32, device=DEV) if packed else None
        s = 3 if packed else b
        t = scan_inputs(1, BF16, b, n, 24, 16, 1, s)
        leaf = {k: t[k].detach().requires_grad_(True) for k in GRADIENTS}
        y, last = selective_scan(*scan_args(leaf), dt_softplus=True, initial_state=leaf["state"], cu_seqlens=cu, return_state=True)
        grads = dict(zip(leaf, torch.autograd.grad([y, last], list(leaf.values()), [t["dy"], t["dstate"]])))
        assert y.shape == (b, n, 24) and torch.equal(last, t["state"]) and torch.equal(grads["state"], t["dstate"])
        assert all(not grads[k].any() for k in ("A", "D", "dt_bias")) and grads["u"].shape == y.shape
        t = conv_inputs(2, F32, b, n, 24, 4, s)
        leaf = {k: t[k].detach().requires_grad_(True) for k in ("x", "weight", "bias", "state")}
        y, last = causal_conv(leaf["x"], leaf["weight"], leaf["bias"], initial_state=leaf["state"], cu_seqlens=cu, return_state=True)
        grads = torch.autograd.grad([y, last], list(leaf.values()), [t["dy"], t["dstate"]])
        assert torch.equal(last, t["state"]) and torch.equal(grads[3], t["dstate"]) and not grads[1].any() and not grads[2].any()
    t = scan_inputs(1, BF16, 0, 1, 24, 16, 1, 2)
    one = {k: v[:, 0] if k in ("u", "dt", "B", "C", "z") else v for k, v in t.items()}
    before = t["state"].clone()
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    assert selective_scan_step(t["state"], *scan_args(one), slots=none).shape == (0, 24) and torch.equal(t["state"], before)
    assert causal_conv_step(torch.zeros(2, 3, 24, device=DEV), torch.zeros(0, 24, device=DEV), torch.zeros(24, 4, device=DEV), slots=none).shape == (0, 24)
