"""causal_conv, selective_scan and their steps at the limits: large values, long rows, many rows, more than 2^31 numbers."""
import pytest
import torch

from tests import recurrent_formulas as F
from tests.test_gpu_recurrent import BF16, DEV, F16, F32, _cu, _normal, conv_inputs, scan_args, scan_inputs

pytestmark = pytest.mark.gpu


# ---- large values --------------------------------------------------------------------------------------------------------------
LARGE = [0.0, 1.0, 4.0, 15.0, 30.0, 88.0, 1e4, 2.0 ** 24 - 1, 2.0 ** 24 + 2, 2.0 ** 24 + 4, 2.0 ** 25, 1e9, 1e30]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("c_odd", [False, True])
@pytest.mark.parametrize("n", [1, 64])
def test_silu_derivative_of_large_inputs(dtype, c_odd, n):
    """The derivative s (1 + p (1 - s)) is one for every large p and zero for every large -p.  With one tap of 1 in a row of equal
    inputs p is the input, so that dx, and of a single token every gradient, is the derivative itself."""
    from lasp_b200 import causal_conv
    p = torch.tensor([s * v for v in LARGE for s in (1, -1) if v <= torch.finfo(dtype).max] + [2.0] * c_odd, device=DEV).to(dtype)
    c, width = p.numel(), 4
    x = p.expand(1, n, c).contiguous().requires_grad_(True)
    weight = torch.zeros(c, width, device=DEV)
    weight[:, -1] = 1
    if n == 1:   # (behind a state of zeros the other taps count for the gradients alone)
        weight[:] = 1
    weight.requires_grad_(True)
    bias, state = torch.zeros(c, device=DEV, requires_grad=True), torch.zeros(1, width - 1, c, dtype=dtype, device=DEV, requires_grad=True)
    y = causal_conv(x, weight, bias, activation="silu", initial_state=state)
    dx, dw, db, ds = torch.autograd.grad(y, [x, weight, bias, state], torch.ones_like(y))
    v = p.double()
    s = torch.sigmoid(v)
    want = s * (1 + v * (1 - s))
    # s is off by 2^-22 and by |p| 2^-23 of itself (the exponent's rounding), 1 - s by 2^-22 until it is exact, from 18 on
    room = (4 + 3 * v.abs().clamp(max=18)) * 2.0 ** -22
    half = torch.finfo(dtype).eps / 2
    assert ((dx[0].double() - want).abs() <= room + half * want.abs()).all(), (dx[0].double() - want).abs().max()
    assert ((db.double() / n - want).abs() <= room + n * 2.0 ** -24).all()
    if n == 1:
        assert ((dw[:, -1].double() - v * want).abs() <= v.abs() * (room + 2.0 ** -24)).all() and not dw[:, :-1].any()
        assert ((ds[0].double() - want).abs() <= room + half * want.abs()).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_infinite_weights_and_tokens_outside_the_sequences(dtype):
    """Tokens that lie in no sequence get zeros, whatever the weights are."""
    from lasp_b200 import causal_conv
    t = conv_inputs(9, dtype, 1, 60, 24, 4, 2)
    weight = t["weight"].clone()
    weight[::2] = float("inf")
    leaf = [v.requires_grad_(True) for v in (t["x"].clone(), weight, t["bias"].clone())]
    y = causal_conv(*leaf, cu_seqlens=_cu([7, 30, 41]))
    dx = torch.autograd.grad(y, leaf, t["dy"])[0]
    for v in (y, dx):
        assert not v[:, :7].any() and not v[:, 41:].any()
        assert v[:, 7:41, 1::2].isfinite().all()


def test_a_state_of_zero_stays_so_where_a_part_grows_beyond_fp32():
    """The decay of 32 tokens is e^256, its root e^128: neither is an fp32 number; a token's, e^8, is."""
    from lasp_b200 import selective_scan
    n, c, N = 1400, 8, 16
    u, dt = torch.zeros(1, n, c, device=DEV), torch.ones(1, n, c, device=DEV)
    B, C = torch.ones(1, n, N, device=DEV), torch.ones(1, n, N, device=DEV)
    leaf = u.requires_grad_(True)
    y, last = selective_scan(leaf, dt, torch.full((c, N), 8.0, device=DEV), B, C, return_state=True)
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(last, torch.zeros_like(last))
    du = torch.autograd.grad(y, leaf, torch.zeros_like(y))[0]
    assert torch.equal(du, torch.zeros_like(du))


# ---- long rows -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("b,n,c", [(1, 2000, 64), (2, 1000, 4800)])   # in segments, and whole
def test_long_rows_lose_no_bits(b, n, c):
    """Decays between a half and one, states with a hundred tokens' memory.  Relative errors in the norm: some 100 roundings of 2^-25 on
    average each for decays and for states, in no order, are 10 x 2.4e-8 each, and the sums of a result as much again, 4e-7 together; a decay that
    is 2e-8 low on average, as the hardware's exponential is, makes 100 x 2e-8 of it, sums with less than 22 bits more than that.  dA is a sum
    of products of a state and a gradient that have each come through such a row: twice of either."""
    from lasp_b200 import selective_scan
    g = torch.Generator(device=DEV).manual_seed(n)
    N = 16
    t = dict(u=_normal(g, b, n, c), dt=torch.rand(b, n, c, generator=g, device=DEV) * 0.02 + 0.001, A=-(0.5 + torch.rand(c, N, generator=g, device=DEV)),
             B=_normal(g, b, n, 1, N), C=_normal(g, b, n, 1, N), dy=_normal(g, b, n, c), state=_normal(g, b, c, N), dstate=_normal(g, b, c, N))
    leaf = {k: t[k].requires_grad_(True) for k in ("u", "dt", "A", "B", "C", "state")}
    y, last = selective_scan(*scan_args(t, ("u", "dt", "A", "B", "C")), initial_state=t["state"], return_state=True)
    grads = torch.autograd.grad([y, last], list(leaf.values()), [t["dy"], t["dstate"]])
    got = {"y": y.detach(), "state": last.detach(), **dict(zip(("du", "ddt", "dA", "dB", "dC", "dinitial"), grads))}
    want = F.scan(**t)
    off = {k: float((got[k].double() - want[k]).norm() / want[k].norm()) for k in got}
    assert all(v < (2e-6 if k == "dA" else 1e-6) for k, v in off.items()), off


# ---- blocks of several rows ----------------------------------------------------------------------------------------------------
ROWS = 301


def _slots_of(kind, count):
    g = torch.Generator().manual_seed(4)
    slots = torch.randperm(count, generator=g)[:ROWS].tolist()
    if kind in ("padded", "mixed"):
        for r in [0, 1, 4, 13, 14, 15, 16, 40, 41, 42, 150, 299, 300]:
            slots[r] = -1 if r % 3 else count
    if kind in ("repeated", "mixed"):   # within a block, across blocks, in the first and the last row
        for r, other in [(2, 5), (2, 7), (3, 8), (9, 10), (9, 12), (20, 25), (20, 200), (25, 299), (60, 61), (60, 62), (60, 63), (100, 297), (101, 298), (11, 300)]:
            slots[other] = slots[r]
    return slots


def _blocks_take_several_rows(tiles, resident):
    blocks = resident * torch.cuda.get_device_properties(0).multi_processor_count // tiles   # for the rows
    assert ROWS > 2 * blocks, "every block has one or two rows: the test needs more of them"


@pytest.mark.parametrize("kind", ["unique", "padded", "repeated", "mixed"])
@pytest.mark.parametrize("c,N,dtype", [(4096, 16, BF16), (4098, 12, F32)])   # whole vectors of channels and states, and parts of them
def test_scan_step_of_many_rows(kind, c, N, dtype):
    from lasp_b200 import selective_scan_step
    _blocks_take_several_rows(c // 128, 5)
    count = ROWS + 9
    t = scan_inputs(3, dtype, ROWS, 1, c, N, 1, count, strided=True)
    tok = {k: t[k][:, 0] if k in ("u", "dt", "B", "C", "z") else t[k] for k in t if t[k] is not None}
    slots = torch.tensor(_slots_of(kind, count), device=DEV)
    got, want = t["state"].clone(), t["state"].clone()
    y = selective_scan_step(got, *scan_args(tok), dt_softplus=True, slots=slots)
    for r in range(ROWS):
        one = {k: v[r:r + 1] if k in ("u", "dt", "B", "C", "z") else v for k, v in tok.items()}
        assert torch.equal(y[r:r + 1], selective_scan_step(want, *scan_args(one), dt_softplus=True, slots=slots[r:r + 1])), r
    assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["unique", "padded", "repeated", "mixed"])
@pytest.mark.parametrize("c,dtype", [(4096, BF16), (4097, F32)])
def test_conv_step_of_many_rows(kind, c, dtype):
    from lasp_b200 import causal_conv_step
    _blocks_take_several_rows(c // 512 if c % 4 == 0 else c // 128, 8)
    count = ROWS + 9
    t = conv_inputs(3, dtype, ROWS, 1, c, 4, count, strided=True)
    x, slots = t["x"][:, 0], torch.tensor(_slots_of(kind, count), device=DEV)
    got, want = t["state"].clone(), t["state"].clone()
    y = causal_conv_step(got, x, t["weight"], t["bias"], activation="silu", slots=slots)
    for r in range(ROWS):
        assert torch.equal(y[r:r + 1], causal_conv_step(want, x[r:r + 1], t["weight"], t["bias"], activation="silu", slots=slots[r:r + 1])), r
    assert torch.equal(got, want)


# ---- more than 2^31 numbers ----------------------------------------------------------------------------------------------------
def _long_row(g, n, c):
    x = torch.empty(1, n, c, dtype=BF16, device=DEV)
    x[:, :200], x[:, 200:-200], x[:, -200:] = _normal(g, 1, 200, c).to(BF16), 0.25, _normal(g, 1, 200, c).to(BF16)
    return x


def test_gradients_of_convolutions_beyond_32_bits():
    from lasp_b200 import causal_conv
    n, c, cut = 526000, 4104, 525900
    g = torch.Generator(device=DEV).manual_seed(0)
    x, dy, w = _long_row(g, n, c).requires_grad_(True), _long_row(g, n, c), _normal(g, c, 4).requires_grad_(True)
    dx, dw = torch.autograd.grad(causal_conv(x, w, activation="silu"), [x, w], dy)
    x, w = x.detach(), w.detach()
    tail, before = x[:, cut:].requires_grad_(True), x[:, cut - 3:cut].contiguous().requires_grad_(True)
    dtail, dbefore = torch.autograd.grad(causal_conv(tail, w, activation="silu", initial_state=before), [tail, before], dy[:, cut:])
    assert torch.equal(dx[:, cut:], dtail)
    # the head: what the tail hands back is a gradient of the state behind it
    head, wh = x[:, :cut].requires_grad_(True), w.clone().requires_grad_(True)
    y, last = causal_conv(head, wh, activation="silu", return_state=True)
    dhead = torch.autograd.grad([y, last], head, [dy[:, :cut], dbefore])[0]
    assert torch.equal(dx[:, :cut - 3], dhead[:, :cut - 3])
    # (the state's gradient has been rounded: two roundings more for the last three tokens; terms of up to a few units)
    torch.testing.assert_close(dx[:, cut - 3:cut].float(), dhead[:, cut - 3:].float(), rtol=2 ** -7, atol=2 ** -5)
    assert dw.isfinite().all()


def test_gradients_of_scans_beyond_32_bits():
    from lasp_b200 import selective_scan
    n, c, N, cut = 263024, 8200, 16, 262928
    assert n * c > 2 ** 31 and cut % 16 == 0
    g = torch.Generator(device=DEV).manual_seed(0)
    u, dy = _long_row(g, n, c), _long_row(g, n, c)
    A, B, C = -torch.exp(_normal(g, c, N)), _normal(g, 1, n, N).to(BF16), _normal(g, 1, n, N).to(BF16)

    def grads(lo, hi, state, dstate):
        leaf = [v.requires_grad_(True) for v in (u.detach()[:, lo:hi], B.detach()[:, lo:hi], C.detach()[:, lo:hi])] + [state]
        leaf = [v for v in leaf if v is not None]
        y, last = selective_scan(leaf[0], u.detach()[:, lo:hi], A, leaf[1], leaf[2], dt_softplus=True, initial_state=state, return_state=True)
        outs = ([y, last], [dy[:, lo:hi], dstate]) if dstate is not None else ([y], [dy[:, lo:hi]])
        return last.detach(), torch.autograd.grad(outs[0], leaf, outs[1])

    whole = grads(0, n, None, None)[1]
    with torch.no_grad():
        middle = selective_scan(u[:, :cut], u[:, :cut], A, B[:, :cut], C[:, :cut], dt_softplus=True, return_state=True)[1]
    tail = grads(cut, n, middle.requires_grad_(True), None)[1]
    assert all(torch.equal(a[:, cut:], b) for a, b in zip(whole, tail))
    head = grads(0, cut, None, tail[3])[1]
    assert all(torch.equal(a[:, :cut], b) for a, b in zip(whole, head))


def test_weights_beyond_32_bits():
    """Taps and a bias of more than 2^31 numbers together."""
    from lasp_b200 import causal_conv
    c = 429_500_000
    assert 5 * c >= 2 ** 31
    x = torch.ones(1, 1, c, dtype=BF16, device=DEV)
    x[..., -1000:] = _normal(torch.Generator(device=DEV).manual_seed(0), 1000).to(BF16)
    w = torch.zeros(c, 4, dtype=BF16, device=DEV).requires_grad_(True)
    bias = torch.zeros(c, dtype=BF16, device=DEV).requires_grad_(True)
    dw, db = torch.autograd.grad(causal_conv(x, w, bias), [w, bias], x)
    assert torch.equal(db, x[0, 0]) and not dw[:, :3].any()
    assert torch.equal(dw[:, 3], (x[0, 0].float() ** 2).to(BF16))
