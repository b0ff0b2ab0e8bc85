"""causal_conv, selective_scan and their steps as programs use them: streams, graphs, autograd, layouts, masked tokens, large tensors."""
import pytest
import torch

from tests import recurrent_formulas as F
from tests.test_gpu_recurrent import BF16, DEV, F32, GRADIENTS, _close, _cu, _normal, conv_inputs, scan_args, scan_inputs

pytestmark = pytest.mark.gpu


def scan_grads(t, cu=None, names=("u", "dt", "A", "B", "C", "D", "z", "dt_bias"), dy=None):
    from lasp_b200 import selective_scan
    leaf = {k: t[k].detach().requires_grad_(True) for k in names if t[k] is not None}
    y = selective_scan(*scan_args({**t, **leaf}), dt_softplus=True, cu_seqlens=t["cu"] if "cu" in t else _cu(cu))
    return [y.detach(), *torch.autograd.grad(y, list(leaf.values()), t["dy"] if dy is None else dy)]


def conv_grads(t, cu=None, dy=None):
    from lasp_b200 import causal_conv
    leaf = [t[k].detach().requires_grad_(True) for k in ("x", "weight", "bias")]
    y = causal_conv(*leaf, activation="silu", cu_seqlens=t["cu"] if "cu" in t else _cu(cu))
    return [y.detach(), *torch.autograd.grad(y, leaf, t["dy"] if dy is None else dy)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


CALLS = {"scan": (scan_grads, lambda s: scan_inputs(s, BF16, 2, 700, 40, 16, 1, 2)),   # (in segments)
         "packed scan": (scan_grads, lambda s: {**scan_inputs(s, F32, 1, 700, 40, 16, 1, 4), "cu": _cu([0, 3, 3, 690, 700])}),
         "conv": (conv_grads, lambda s: conv_inputs(s, BF16, 2, 700, 40, 4, 2)),
         "packed conv": (conv_grads, lambda s: {**conv_inputs(s, F32, 1, 700, 40, 4, 4), "cu": _cu([0, 3, 3, 690, 700])})}


@pytest.mark.parametrize("call", CALLS)
def test_the_same_bits_each_time_and_on_two_streams_at_once(call):
    run, make = CALLS[call]
    inputs = [make(s) for s in (1, 2)]
    want = [run(t) for t in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run(inputs[i])
        torch.cuda.synchronize()
        assert same(got[0], want[0]) and same(got[1], want[1])


@pytest.mark.parametrize("call", CALLS)
def test_two_graphs_of_forward_and_backward(call):
    run, make = CALLS[call]
    inputs, fresh = [make(s) for s in (1, 2)], [make(s) for s in (3, 4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(inputs[0])
    torch.cuda.synchronize()
    graphs, got = [], []
    for t in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got.append(run(t))
        graphs.append(graph)
    for t, f in zip(inputs, fresh):
        for k in t:
            if t[k] is not None:
                t[k].copy_(f[k])
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(same(g, run(f)) for g, f in zip(got, fresh))


def test_steps_in_a_graph():
    from lasp_b200 import causal_conv_step, selective_scan_step
    c, N, rows, count = 72, 16, 6, 9
    t = scan_inputs(7, BF16, rows, 1, c, N, 1, count)
    v = conv_inputs(7, BF16, rows, 1, c, 4, count)
    tok = {k: t[k][:, 0] if k in ("u", "dt", "B", "C", "z") else t[k] for k in t if t[k] is not None}
    slots = torch.tensor([3, 0, 8, 3, -1, 20], device=DEV)

    def step(cs, ss):
        u = causal_conv_step(cs, v["x"][:, 0], v["weight"], v["bias"], activation="silu", slots=slots)
        return selective_scan_step(ss, u, *scan_args(tok)[1:], dt_softplus=True, slots=slots)

    states = [v["state"].clone(), t["state"].clone()]
    wants = [v["state"].clone(), t["state"].clone()]
    side = torch.cuda.Stream()
    step(v["state"].clone(), t["state"].clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = step(*states)
    for i in range(4):
        v["x"].copy_(_normal(torch.Generator(device=DEV).manual_seed(i), *v["x"].shape))
        slots.copy_(torch.tensor([[3, 0, 8, 3, -1, 20], [1, 1, 1, 1, 1, 1], [0, 1, 2, 3, 4, 5], [-1, -1, 9, 7, 7, 0]][i], device=DEV))
        graph.replay()
        assert torch.equal(y, step(*wants)) and same(states, wants)


def test_gradients_of_some_inputs_only():
    from lasp_b200 import causal_conv, selective_scan
    t = scan_inputs(11, F32, 2, 40, 24, 16, 1, 2)
    want = dict(zip(GRADIENTS, scan_grads(t)[1:]))
    for name in ("A", "B", "z", "dt_bias"):
        assert torch.equal(scan_grads(t, names=(name,))[1], want[name])
    v = conv_inputs(11, F32, 2, 40, 24, 4, 2)
    x, weight, bias = conv_grads(v)[1:]
    w = v["weight"].detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(causal_conv(v["x"], w, v["bias"], activation="silu"), w, v["dy"])[0], weight)
    # of the states alone: the outputs have no gradient
    leaf = {k: t[k].detach().requires_grad_(True) for k in GRADIENTS}
    last = selective_scan(*scan_args(leaf), dt_softplus=True, initial_state=leaf["state"], return_state=True)[1]
    got = torch.autograd.grad(last, list(leaf.values()), t["dstate"], allow_unused=True)
    args = dict(softplus=True, cu=None, **{**t, "dy": torch.zeros_like(t["dy"])})
    got = {GRADIENTS[k]: g for k, g in zip(leaf, got)}
    _close(got, F.scan(**args), F.scan(**args, size=True), 2 * 40 + 20)


def test_broadcast_transposed_and_unaligned_inputs():
    """B and C shared by all rows, a gradient that is one number, tokens innermost, and tensors that begin in the middle of a vector."""
    t = scan_inputs(5, F32, 2, 33, 24, 16, 1, 2)
    for k in ("B", "C"):
        t[k] = t[k][:1].expand_as(t[k])
    for k in ("u", "dt"):
        t[k] = t[k].transpose(1, 2).contiguous().transpose(1, 2)
    for k in ("z", "dy"):
        t[k] = torch.cat([t[k].new_zeros(1), t[k].flatten()])[1:].view(t[k].shape)
    for k in ("A", "D", "dt_bias"):
        t[k] = torch.cat([t[k].new_zeros(1), t[k].flatten()])[1:].view(t[k].shape)
    plain = {k: None if v is None else v.contiguous().clone() for k, v in t.items()}
    assert same(scan_grads(t), scan_grads(plain))
    one = torch.ones((), device=DEV).expand_as(t["dy"])
    assert same(scan_grads(t, dy=one), scan_grads(plain, dy=one.contiguous()))
    # the gradient of what was broadcast is the sum
    shared = t["B"][:1].detach().requires_grad_(True)
    from lasp_b200 import selective_scan
    y = selective_scan(t["u"], t["dt"], t["A"], shared.expand_as(t["B"]), t["C"], t["D"], t["z"], t["dt_bias"], dt_softplus=True)
    assert torch.equal(torch.autograd.grad(y, shared, t["dy"])[0], scan_grads(plain)[4].sum(0, keepdim=True))
    v = conv_inputs(5, BF16, 2, 33, 24, 4, 2)
    odd = dict(v, x=torch.cat([v["x"].new_zeros(1), v["x"].flatten()])[1:].view(v["x"].shape), weight=v["weight"].t().contiguous().t(),
               dy=v["dy"].transpose(0, 1).contiguous().transpose(0, 1))
    assert same(conv_grads(odd), conv_grads(v))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_tokens_outside_the_sequences_are_not_looked_at(bad):
    cu, n = [5, 70, 70, 140], 150
    t, v = scan_inputs(3, F32, 1, n, 24, 16, 1, 3), conv_inputs(3, F32, 1, n, 24, 4, 3)
    want, vwant = scan_grads(t, cu), conv_grads(v, cu)
    for x in (t, v):
        for k in ("u", "dt", "B", "C", "z", "dy", "x"):
            if x.get(k) is not None:
                x[k] = x[k].clone()
                x[k][:, :5], x[k][:, 140:] = bad, bad
    got, vgot = scan_grads(t, cu), conv_grads(v, cu)
    assert same(got, want) and same(vgot, vwant)
    for g in (got[0], got[1], got[2], got[4], got[5], got[7], vgot[0], vgot[1]):
        assert not g[:, :5].any() and not g[:, 140:].any()


def test_a_bad_token_stays_in_its_sequence():
    cu, n = [0, 300, 1400, 1500], 1500   # (in segments)
    t = scan_inputs(3, F32, 1, n, 8, 16, 1, 3)
    want = scan_grads(t, cu)
    t["u"] = t["u"].clone()
    t["u"][0, 600, 2] = float("nan")
    got = scan_grads(t, cu)
    assert torch.equal(got[0][0, :600], want[0][0, :600]) and torch.equal(got[0][0, 1400:], want[0][0, 1400:]) and got[0][0, 600:1400, 2].isnan().all()
    assert torch.equal(got[0][0, 600:1400, 3:], want[0][0, 600:1400, 3:])


def test_infinite_rates():
    """A of minus infinity forgets at every step but those of zero."""
    from lasp_b200 import selective_scan, selective_scan_step
    n, c, N = 20, 8, 4
    g = torch.Generator(device=DEV).manual_seed(0)
    u, dt, B, C = _normal(g, 1, n, c), torch.rand(1, n, c, generator=g, device=DEV) + 0.1, _normal(g, 1, n, N), _normal(g, 1, n, N)
    dt[:, 5:8] = 0
    A = torch.full((c, N), float("-inf"), device=DEV)
    y, last = selective_scan(u, dt, A, B, C, return_state=True)
    put = (dt * u)[0, :, :, None] * B[0, :, None, :]
    put[5:8] = put[4]
    torch.testing.assert_close(y[0], (put * C[0, :, None, :]).sum(-1), rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(last[0], put[-1], rtol=1e-6, atol=0)
    state = torch.zeros(1, c, N, device=DEV)
    for i in range(n):
        ys = selective_scan_step(state, u[:, i], dt[:, i], A, B[:, i], C[:, i])
        torch.testing.assert_close(ys, y[:, i], rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("cu", [[0, 900, 100, 1400], [-7, 500, 2000, 1 << 30], [1400, 700, 0, 0]])
def test_offsets_that_are_no_offsets_do_no_harm(cu):
    """Offsets are read on the device and kept within the row: the results are whatever they are, and the next call is right."""
    t, v = scan_inputs(3, F32, 1, 1400, 8, 16, 1, 3), conv_inputs(3, F32, 1, 1400, 8, 4, 3)
    want, vwant = scan_grads(t, [0, 3, 700, 1400]), conv_grads(v, [0, 3, 700, 1400])
    scan_grads(t, cu), conv_grads(v, cu)
    torch.cuda.synchronize()
    assert same(scan_grads(t, [0, 3, 700, 1400]), want) and same(conv_grads(v, [0, 3, 700, 1400]), vwant)


def test_inference_mode_hooks_and_versions():
    from lasp_b200 import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    t, v = scan_inputs(2, F32, 1, 30, 16, 16, 1, 1), conv_inputs(2, F32, 1, 30, 16, 4, 1)
    want, vwant = scan_grads(t), conv_grads(v)
    with torch.inference_mode():
        assert torch.equal(selective_scan(*scan_args(t), dt_softplus=True), want[0])
        assert torch.equal(causal_conv(v["x"], v["weight"], v["bias"], activation="silu"), vwant[0])
    with torch.autograd.graph.save_on_cpu():
        assert same(scan_grads(t), want) and same(conv_grads(v), vwant)
    leaf = t["u"].detach().requires_grad_(True)
    B = t["B"].clone()
    y = selective_scan(leaf, t["dt"], t["A"], B, t["C"])
    B.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    state, cstate = t["state"].clone(), v["state"].clone()
    before = state._version, cstate._version
    selective_scan_step(state, *[a[:, 0] for a in (t["u"], t["dt"])], t["A"], t["B"][:, 0], t["C"][:, 0])
    causal_conv_step(cstate, v["x"][:, 0], v["weight"])
    assert state._version > before[0] and cstate._version > before[1]


def test_second_derivatives_are_refused():
    from lasp_b200 import causal_conv, selective_scan
    t, v = scan_inputs(2, F32, 1, 9, 8, 16, 1, 1), conv_inputs(2, F32, 1, 9, 8, 4, 1)
    u, x = t["u"].detach().requires_grad_(True), v["x"].detach().requires_grad_(True)
    for y, leaf in ((selective_scan(u, t["dt"], t["A"], t["B"], t["C"]), u), (causal_conv(x, v["weight"]), x)):
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)


def test_refusals():
    from lasp_b200 import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    t, v = scan_inputs(2, F32, 2, 9, 8, 16, 2, 2), conv_inputs(2, F32, 2, 9, 8, 4, 2)
    good = dict(zip(("u", "dt", "A", "B", "C", "D", "z", "dt_bias"), scan_args(t)))
    for error, change in [(ValueError, dict(dt=t["dt"][:, :8])), (TypeError, dict(z=t["z"].to(BF16))), (ValueError, dict(B=t["B"][..., :7])),
                          (ValueError, dict(C=t["C"][:, :, :1])), (TypeError, dict(A=t["A"].double())), (ValueError, dict(A=t["A"][:7])),
                          (TypeError, dict(D=t["D"].long())), (ValueError, dict(dt_bias=t["dt_bias"][:3])), (RuntimeError, dict(B=t["B"].cpu())),
                          (ValueError, dict(initial_state=t["state"][:1])), (TypeError, dict(initial_state=t["state"].to(BF16))),
                          (ValueError, dict(cu_seqlens=_cu([0, 9]))), (TypeError, dict(cu_seqlens=torch.zeros(2, device=DEV)))]:
        with pytest.raises(error):
            selective_scan(**{**good, **change})
    for error, change in [(ValueError, dict(bias=v["bias"][:3])), (TypeError, dict(weight=v["weight"].long())), (ValueError, dict(initial_state=v["state"][:, :2])),
                          (TypeError, dict(initial_state=v["state"].to(BF16))), (RuntimeError, dict(x=v["x"].cpu()))]:
        with pytest.raises(error):
            causal_conv(**{**dict(x=v["x"], weight=v["weight"], bias=v["bias"]), **change})
    x, state = v["x"][:, 0], v["state"]
    for error, args, change in [(ValueError, (state.transpose(1, 2).contiguous().transpose(1, 2), x), {}), (ValueError, (state[:1], x), {}), (TypeError, (state.to(BF16), x), {}),
                                (ValueError, (state, v["x"]), {}), (ValueError, (state, x), dict(slots=_cu([0]))), (TypeError, (state, x), dict(slots=torch.zeros(2, device=DEV))),
                                (RuntimeError, (state.clone().requires_grad_(True), x), {}), (RuntimeError, (state, x.clone().requires_grad_(True)), {})]:
        with pytest.raises(error):
            causal_conv_step(*args, v["weight"], **change)
    tok = [a[:, 0] for a in (t["u"], t["dt"])] + [t["A"], t["B"][:, 0], t["C"][:, 0]]
    for error, state, change in [(ValueError, t["state"].transpose(0, 1), {}), (ValueError, t["state"][..., :3].contiguous(), {}), (TypeError, t["state"].to(BF16), {}),
                                 (ValueError, t["state"], dict(slots=_cu([0, 1, 1]))), (RuntimeError, t["state"].clone().requires_grad_(True), {})]:
        with pytest.raises(error):
            selective_scan_step(state, *tok, **change)


@pytest.mark.parametrize("b,n,c,N", [(1, 5, 1, 1), (2, 1, 3, 2), (1, 17, 2, 3), (1, 1030, 1, 1)])
def test_the_smallest(b, n, c, N):
    t, v = scan_inputs(n, F32, b, n, c, N, 1, b), conv_inputs(n, F32, b, n, c, 2, b)
    t.update(state=None, dstate=None)
    names = ["y", *[GRADIENTS[k] for k in ("u", "dt", "A", "B", "C", "D", "z", "dt_bias")]]
    args = dict(softplus=True, cu=None, **t)
    _close(dict(zip(names, scan_grads(t))), F.scan(**args), F.scan(**args, size=True), 2 * n + 20)
    args = (v["x"], v["weight"], v["bias"], True, None, None, v["dy"])
    _close(dict(zip(("y", "dx", "dweight", "dbias"), conv_grads(v))), F.conv(*args), F.conv(*args, size=True), 40)


def test_a_batch_that_is_mostly_padding():
    """600 rows, most of which stand for no sequence and two of which share one."""
    from lasp_b200 import causal_conv_step, selective_scan_step
    rows, c, N = 600, 40, 16
    t, v = scan_inputs(1, F32, rows, 1, c, N, 1, 7), conv_inputs(1, F32, rows, 1, c, 4, 7)
    tok = {k: t[k][:, 0] if k in ("u", "dt", "B", "C", "z") else t[k] for k in t if t[k] is not None}
    slots = torch.full((rows,), -1, device=DEV)
    real = torch.tensor([3, 77, 78, 400, 599], device=DEV)
    slots[real] = torch.tensor([6, 0, 4, 6, 2], device=DEV)
    for step, state, args, kw in ((selective_scan_step, t["state"], scan_args(tok), dict(dt_softplus=True)),
                                  (causal_conv_step, v["state"], (v["x"][:, 0], v["weight"], v["bias"]), dict(activation="silu"))):
        got, want = state.clone(), state.clone()
        y = step(got, *args, slots=slots, **kw)
        small = [a if a is None or a.shape[:1] != (rows,) else a[real] for a in args]
        assert torch.equal(y[real], step(want, *small, slots=slots[real], **kw)) and torch.equal(got, want)
        assert not y[slots < 0].any() and torch.equal(got[[1, 3, 5]], state[[1, 3, 5]])


def test_traced():
    """torch.jit.trace: the graph holds the operators themselves."""
    from lasp_b200 import causal_conv, selective_scan
    t, v = scan_inputs(2, F32, 1, 30, 16, 16, 1, 1), conv_inputs(2, F32, 1, 30, 16, 4, 1)

    def f(x, dt):
        u = causal_conv(x, v["weight"], v["bias"], activation="silu")
        return selective_scan(u, dt, t["A"], t["B"], t["C"], t["D"], t["z"], t["dt_bias"], dt_softplus=True)

    traced = torch.jit.trace(f, (torch.zeros_like(v["x"]), torch.zeros_like(t["dt"])), check_trace=False)
    assert {"lasp_b200::causal_conv", "lasp_b200::selective_scan"} <= {n.kind() for n in traced.graph.nodes()}
    assert torch.equal(traced(v["x"], t["dt"]), f(v["x"], t["dt"]))


def test_transforms_are_refused():
    from lasp_b200 import causal_conv, selective_scan
    t, v = scan_inputs(2, F32, 3, 9, 8, 16, 1, 3), conv_inputs(2, F32, 3, 9, 8, 4, 3)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(lambda x: causal_conv(x[None], v["weight"]))(v["x"])
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(lambda u, dt, B, C: selective_scan(u[None], dt[None], t["A"], B[None], C[None]))(t["u"], t["dt"], t["B"], t["C"])
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.grad(lambda x: causal_conv(x, v["weight"]).sum())(v["x"])


def test_beyond_32_bits():
    """More than 2^31 numbers: the last tokens of a long row, and the last slots of a large cache."""
    from lasp_b200 import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    n, c, N, cut = 526000, 4104, 16, 525900
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.empty(1, n, c, dtype=BF16, device=DEV)
    x[:, :100], x[:, 100:cut], x[:, cut - 100:] = _normal(g, 1, 100, c).to(BF16), 0.5, _normal(g, 1, n - cut + 100, c).to(BF16)
    w, A, B, C = _normal(g, c, 4), -torch.exp(_normal(g, c, N)), _normal(g, 1, n, N).to(BF16), _normal(g, 1, n, N).to(BF16)
    with torch.no_grad():
        y, last = causal_conv(x, w, return_state=True)
        tail = causal_conv(x[:, cut:], w, initial_state=x[:, cut - 3:cut].contiguous())
        assert torch.equal(y[:, cut:], tail) and torch.equal(last, x[:, -3:])
        del y
        y, last = selective_scan(x, x, A, B, C, dt_softplus=True, return_state=True)
        head = selective_scan(x[:, :cut], x[:, :cut], A, B[:, :cut], C[:, :cut], dt_softplus=True, return_state=True)[1]
        tail, end = selective_scan(x[:, cut:], x[:, cut:], A, B[:, cut:], C[:, cut:], dt_softplus=True, initial_state=head, return_state=True)
        # (a row of 100 tokens is not cut into segments, nor is one of this many channels: the sums are the same)
        assert torch.equal(y[:, cut:], tail) and torch.equal(last, end)
    del x, y, tail
    count = 2 ** 31 // (4096 * N) + 5
    state = torch.zeros(count, 4096, N, device=DEV)
    slots = torch.tensor([count - 1, count - 3], device=DEV)
    u, Bs, Cs = _normal(g, 2, 4096), _normal(g, 2, N), _normal(g, 2, N)
    small = torch.zeros(2, 4096, N, device=DEV)
    want = selective_scan_step(small, u, u, A[:4096].contiguous(), Bs, Cs, dt_softplus=True)
    assert torch.equal(selective_scan_step(state, u, u, A[:4096].contiguous(), Bs, Cs, dt_softplus=True, slots=slots), want)
    assert torch.equal(state[slots], small) and not state[:count - 3].any()
    del state
    count = 2 ** 31 // (4096 * 3) + 5
    state = torch.zeros(count, 3, 4096, dtype=BF16, device=DEV)
    u, small = u.to(BF16), torch.zeros(2, 3, 4096, dtype=BF16, device=DEV)
    slots = torch.tensor([count - 1, count - 3], device=DEV)
    want = causal_conv_step(small, u, w[:4096])
    assert torch.equal(causal_conv_step(state, u, w[:4096], slots=slots), want) and torch.equal(state[slots], small)
