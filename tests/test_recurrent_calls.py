"""What causal_conv, selective_scan and their steps refuse, as far as they look before they need a GPU; the C ABI's checks."""
import ctypes as C

import pytest
import torch

from lasp_b200 import _cabi, causal_conv, causal_conv_step, selective_scan, selective_scan_step


def scan(drop=(), **change):
    b, n, c, N = 2, 6, 8, 4
    t = dict(u=torch.zeros(b, n, c), dt=torch.zeros(b, n, c), A=torch.zeros(c, N), B=torch.zeros(b, n, N), C=torch.zeros(b, n, N), D=torch.zeros(c),
             z=torch.zeros(b, n, c), dt_bias=torch.zeros(c))
    t.update(change)
    return selective_scan(**t)


def conv(**change):
    t = dict(x=torch.zeros(2, 6, 8), weight=torch.zeros(8, 4), bias=torch.zeros(8))
    t.update(change)
    return causal_conv(**t)


def test_cpu_tensors_are_refused():
    for call in (scan, conv, lambda: causal_conv_step(torch.zeros(2, 3, 8), torch.zeros(2, 8), torch.zeros(8, 4)),
                 lambda: selective_scan_step(torch.zeros(2, 8, 4), torch.zeros(2, 8), torch.zeros(2, 8), torch.zeros(8, 4), torch.zeros(2, 4), torch.zeros(2, 4))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("change", [
    dict(u=torch.zeros(6, 8)), dict(u=torch.zeros(2, 6, 0)), ])
def test_scan_shapes(change):
    with pytest.raises(ValueError):
        scan(**change)


def test_conv_shapes():
    for change in (dict(x=torch.zeros(6, 8)), dict(x=torch.zeros(2, 6, 0)), dict(weight=torch.zeros(8, 5)), dict(weight=torch.zeros(8, 1)), dict(weight=torch.zeros(7, 4)),
                   dict(weight=torch.zeros(8))):
        with pytest.raises(ValueError):
            conv(**change)
    with pytest.raises(ValueError, match="activation"):
        conv(activation="gelu")
    for kind in (torch.float64, torch.int32):
        with pytest.raises(TypeError):
            conv(x=torch.zeros(2, 6, 8, dtype=kind))


def test_arguments_that_are_no_tensors():
    with pytest.raises(TypeError):
        conv(x=None)
    with pytest.raises(TypeError):
        conv(bias=3.0)
    with pytest.raises(TypeError):
        scan(B=None)
    with pytest.raises(TypeError):
        scan(cu_seqlens=[0, 6])


def test_a_tangent_is_refused():
    import torch.autograd.forward_ad as fa
    with fa.dual_level():
        x = fa.make_dual(torch.ones(2, 6, 8), torch.ones(2, 6, 8))
        with pytest.raises(NotImplementedError):
            conv(x=x)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            scan(u=x)


P = 4096   # an address that nothing is done with


def tokens(p=P):
    return _cabi.Tokens(p, 64, 8, 0)


def conv_args(**kw):
    a = _cabi.ConvArgs(rows=1, tokens=8, channels=8, width=4, dtype=_cabi.BF16, param_dtype=_cabi.F32, x=tokens(), y=tokens(), dy=tokens(), dx=tokens(),
                       weight=P, dweight=P, ws=P, ws_bytes=1 << 30)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def scan_args(**kw):
    a = _cabi.ScanArgs(rows=1, tokens=8, channels=8, states=16, groups=1, dtype=_cabi.BF16, param_dtype=_cabi.F32, A=P, kept=P, kept_bytes=1 << 30, ws=P,
                       ws_bytes=1 << 30, **{k: tokens() for k in ("u", "dt", "B", "C", "y", "dy", "du", "ddt", "dB", "dC")})
    for k, v in kw.items():
        setattr(a, k, v)
    return a


SHAPES = [dict(rows=0), dict(tokens=-1), dict(channels=0), dict(sequences=2, offsets=P, index_bits=32, rows=2), dict(sequences=2, offsets=P, index_bits=16),
          dict(sequences=-1)]


@pytest.mark.parametrize("kw,status", [(x, -2) for x in SHAPES + [dict(width=5), dict(width=1), dict(activation=7)]] + [
    (dict(dtype=9), -3), (dict(param_dtype=_cabi.F16), -3), (dict(weight=None), -1), (dict(x=tokens(None)), -1), (dict(sequences=2, index_bits=32), -1),
    (dict(rows=65536), -9), (dict(tokens=2**31 - 1), -9), (dict(sequences=(1 << 17) + 1, index_bits=32, offsets=P), -9)])
def test_conv_c_checks(kw, status):
    lib = _cabi.load()
    for f in (lib.lasp_b200_conv_forward, lib.lasp_b200_conv_backward):
        assert f(C.byref(conv_args(**kw)), None) == status
    assert lib.lasp_b200_conv_forward(None, None) == -1 and lib.lasp_b200_conv_backward(None, None) == -1


def test_conv_c_checks_of_one_pass():
    lib = _cabi.load()
    assert lib.lasp_b200_conv_forward(C.byref(conv_args(y=tokens(None))), None) == -1
    for kw, status in ((dict(dx=tokens(None)), -1), (dict(dy=tokens(None)), -1), (dict(ws=None), -1), (dict(ws=P + 4), -4), (dict(ws_bytes=8), -5)):
        assert lib.lasp_b200_conv_backward(C.byref(conv_args(**kw)), None) == status


@pytest.mark.parametrize("kw,status", [(x, -2) for x in SHAPES + [dict(states=0), dict(states=65), dict(groups=0), dict(groups=3)]] + [
    (dict(dtype=9), -3), (dict(param_dtype=_cabi.F16), -3), (dict(A=None), -1), (dict(B=tokens(None)), -1), (dict(sequences=2, index_bits=32), -1),
    (dict(tokens=2**31 - 1), -9), (dict(rows=2**30, tokens=0), -9)])
def test_scan_c_checks(kw, status):
    lib = _cabi.load()
    for f in (lib.lasp_b200_scan_forward, lib.lasp_b200_scan_backward):
        assert f(C.byref(scan_args(**kw)), None) == status
    assert lib.lasp_b200_scan_workspace_bytes(C.byref(scan_args(**kw))) == 0 and lib.lasp_b200_scan_kept_bytes(C.byref(scan_args(**kw))) == 0
    assert lib.lasp_b200_scan_forward(None, None) == -1 and lib.lasp_b200_scan_backward(None, None) == -1


def test_scan_c_checks_of_one_pass():
    lib = _cabi.load()
    for kw, status in ((dict(y=tokens(None)), -1), (dict(kept=P + 8), -4), (dict(kept_bytes=8), -5)):
        assert lib.lasp_b200_scan_forward(C.byref(scan_args(**kw)), None) == status
    for kw, status in ((dict(dy=tokens(None)), -1), (dict(dB=tokens(None)), -1), (dict(z=tokens()), -1), (dict(ws=None), -1), (dict(kept=None), -1),
                       (dict(ws=P + 4), -4), (dict(kept=P + 8), -4), (dict(ws_bytes=8), -5), (dict(kept_bytes=8), -5)):
        assert lib.lasp_b200_scan_backward(C.byref(scan_args(**kw)), None) == status


def test_scan_c_checks_of_the_forward_workspace():
    """A long sequence of few channels is cut into segments, which takes a workspace; a short one takes none."""
    lib = _cabi.load()
    need = lambda **kw: lib.lasp_b200_scan_forward_workspace_bytes(C.byref(scan_args(**kw)))   # noqa: E731
    assert need(rows=1, tokens=4096) > 0 and need(rows=1, tokens=100) == 0 and need(rows=1, tokens=4096, states=0) == 0 and need(rows=1, tokens=0) == 0
    for kw, status in ((dict(ws=None), -1), (dict(ws=P + 4), -4), (dict(ws_bytes=8), -5)):
        kw = {**dict(rows=1, tokens=4096, kept=None, ws=P, ws_bytes=need(rows=1, tokens=4096)), **kw}
        assert lib.lasp_b200_scan_forward(C.byref(scan_args(**kw)), None) == status


def test_step_c_checks():
    lib = _cabi.load()

    def conv_step(**kw):
        a = _cabi.ConvStepArgs(rows=2, channels=8, width=4, dtype=_cabi.BF16, slot_count=2, x=tokens(), y=tokens(), weight=P, state=P)
        [setattr(a, k, v) for k, v in kw.items()]
        return lib.lasp_b200_conv_step(C.byref(a), None)

    def scan_step(**kw):
        a = _cabi.ScanStepArgs(rows=2, channels=8, states=16, groups=1, dtype=_cabi.BF16, slot_count=2, A=P, state=P,
                               **{k: tokens() for k in ("u", "dt", "B", "C", "y")})
        [setattr(a, k, v) for k, v in kw.items()]
        return lib.lasp_b200_scan_step(C.byref(a), None)

    for step, more in ((conv_step, [(dict(width=5), -2), (dict(weight=None), -1), (dict(x=tokens(None)), -1), (dict(activation=3), -2)]),
                       (scan_step, [(dict(states=65), -2), (dict(groups=3), -2), (dict(A=None), -1), (dict(C=tokens(None)), -1)])):
        for kw, status in more + [(dict(rows=0), -2), (dict(channels=0), -2), (dict(slot_count=-1), -2), (dict(slots=P, index_bits=8), -2), (dict(dtype=5), -3),
                                  (dict(param_dtype=_cabi.F16), -3), (dict(rows=65536), -9), (dict(state=None), -1), (dict(y=tokens(None)), -1)]:
            assert step(**kw) == status, kw
    assert lib.lasp_b200_conv_step(None, None) == -1 and lib.lasp_b200_scan_step(None, None) == -1
