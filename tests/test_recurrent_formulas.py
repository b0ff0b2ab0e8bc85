"""The written-out gradients of the 64-bit formulas against differences of their values."""
import pytest
import torch

from tests import recurrent_formulas as F


def _value(out, dy, dstate):
    return float((out["y"] * dy).sum() + (out["state"] * dstate).sum())


def _check(f, inputs, names, dy, dstate, seed):
    g = torch.Generator().manual_seed(seed)
    grads = f(dy=dy, dstate=dstate, **inputs)
    for name, grad in names.items():
        if inputs.get(name) is None:
            continue
        way = torch.randn(inputs[name].shape, generator=g, dtype=torch.float64)
        h = 1e-6
        up, down = (_value(f(**{**inputs, name: inputs[name] + s * h * way}), dy, dstate) for s in (1, -1))
        want, got = (up - down) / (2 * h), float((grads[grad] * way).sum())
        # central differences: h^2 of the third derivative, and 2^-52 / h of the value
        assert abs(got - want) < 1e-6 * max(1.0, abs(got)), (name, got, want)


@pytest.mark.parametrize("cu", [None, [0, 0, 3, 4, 9], [1, 2, 2, 8]])
@pytest.mark.parametrize("act", [False, True])
@pytest.mark.parametrize("width", [2, 4])
def test_convolution(cu, act, width):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    b, n, c = (1 if cu else 2), 9, 3
    s = len(cu) - 1 if cu else b
    inputs = dict(x=r(b, n, c), weight=r(c, width), bias=r(c), act=act, state=r(s, width - 1, c), cu=cu)
    _check(F.conv, inputs, dict(x="dx", weight="dweight", bias="dbias", state="dinitial"), r(b, n, c), r(s, width - 1, c), 2)


@pytest.mark.parametrize("cu", [None, [0, 0, 3, 4, 9], [1, 2, 2, 8]])
@pytest.mark.parametrize("softplus,gate,groups", [(True, True, 2), (False, False, 1)])
def test_scan(cu, softplus, gate, groups):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    b, n, c, N = (1 if cu else 2), 9, 4, 3
    s = len(cu) - 1 if cu else b
    inputs = dict(u=r(b, n, c), dt=r(b, n, c) * 0.3, A=-torch.rand(c, N, generator=g, dtype=torch.float64) - 0.2, B=r(b, n, groups, N),
                  C=r(b, n, groups, N), D=r(c), z=r(b, n, c) if gate else None, dt_bias=r(c) * 0.3 if softplus else None, softplus=softplus,
                  state=r(s, c, N), cu=cu)
    names = dict(u="du", dt="ddt", A="dA", B="dB", C="dC", D="dD", z="dz", dt_bias="ddt_bias", state="dinitial")
    _check(F.scan, inputs, names, r(b, n, c), r(s, c, N), 4)
