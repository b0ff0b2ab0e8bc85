"""causal_conv, selective_scan and their steps at the limits."""
import pytest
import torch

from tests.test_gpu_recurrent import BF16, DEV, F16, F32, _cu, _normal, conv_inputs

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


# ---- more than 2^31 numbers ----------------------------------------------------------------------------------------------------
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
