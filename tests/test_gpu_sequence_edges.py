"""Sequence operators at the edges of their ranges: saturated gates, float32 results of bf16 calls, infinities, views that negate, calls that have to
be refused.  Each case is one that the ordinary sizes of test_gpu_sequence.py do not reach."""
import pytest
import torch

import horizonnet_amd as hn
from oracle import sequence_ref as ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("name,M,K,F", [("f32", 60, 16, 81), ("f32", 60, 128, 81), ("bf16", 60, 16, 81), ("bf16", 300, 64, 200), ("bf16", 8192, 128, 768)])
def test_sigmoid_gate_saturated(name, M, K, F):
    """Gates from -20 to 20: the slope s (1 - s) of a sigmoid is a bare factor of dg, so it has to be right relative to itself, however small.
    (The sizes take the small tiles, the kept projections and the large bf16 tiles.)  Everything that is summed here is positive, so the bounds are
    relative: the slope is off by its exponential (|g| 2 u of the short one), a reciprocal and two products, by its argument's error (its relative
    slope is at most 1) -- (K + 2) u of the sum's terms and u |g| --, u by its own sum's; then half a step where dg is rounded and where the result is."""
    g = torch.Generator().manual_seed(K + F)
    dt = DT[name]
    some = lambda *s, low, high: (torch.rand(*s, generator=g) * (high - low) + low).to(dt)  # noqa: E731
    x, dy = some(M, K, low=0.5, high=1.5), some(M, F, low=0.5, high=1.5)
    wg, wu = some(F, K, low=0.0, high=0.5 / K), some(F, K, low=0.0, high=0.5 / K)
    bg, bu = torch.linspace(-20, 20, F).to(dt), torch.ones(F, dtype=dt)
    xd, wgd, wud = x.double().to(DEV), wg.double().to(DEV), wu.double().to(DEV)
    gate, up = xd @ wgd.t() + bg.double().to(DEV), xd @ wud.t() + 1.0
    slope = torch.sigmoid(gate) * torch.sigmoid(-gate)
    dg = dy.double().to(DEV) * up * slope
    want = {"dbg": dg.sum(0), "dwg": dg.t() @ xd}
    half, u = ref.rounding(dt), ref.U
    # |g| <= 21, the sums' terms add up to at most 0.75 + 1
    r = (2 * 21 + 16) * u + (K + 2) * u * 1.75 * 2 + 21 * u + (M + 2) * u
    room = {"dbg": r + half, "dwg": (1 + r) * (1 + half) ** 2 - 1 if name == "bf16" else r + half}
    args = [t.to(DEV).requires_grad_(True) for t in (x, wg, wu, bg, bu)]
    y = hn.gated_linear(*args, activation="sigmoid")
    grads = torch.autograd.grad(y, [args[3], args[1]], dy.to(DEV))
    for n, t in zip(("dbg", "dwg"), grads):
        off = ((t.double() - want[n]).abs() / want[n]).max()
        assert float(off) <= room[n] * 1.0001, (n, float(off), room[n])


def test_float32_results_of_bf16_recurrence():
    """The states and dh0 of a bf16 call are float32 and have to be right to float32's last bits: with v = 0 they are products of gates alone.  One
    gate is off by 2 u for the exponential, 0.9 u for what its constant leaves out, u for the sum that adds it, u for 1 + e, u for its reciprocal (in
    [1/2, 1]) and u for the product: 6.9 u, and u more for the product with the state; a gate of the output in dh0 adds 6.9 u and the product u (the order in
    which steps are joined adds u a step)."""
    u = ref.U
    g = torch.Generator().manual_seed(3)
    for T, B, C in ((1, 7, 130), (1, 300, 512), (2, 5, 64)):
        f = (-80 + 72 * torch.rand(T, B, C, generator=g) if T == 1 else -40 + 32 * torch.rand(T, B, C, generator=g)).bfloat16()
        o = (-80 + 160 * torch.rand(T, B, C, generator=g)).bfloat16()
        v, h0 = torch.zeros(T, B, C, dtype=torch.bfloat16), 1 + torch.rand(B, C, generator=g)
        a = torch.sigmoid(f.double()).prod(0)
        want = a * h0.double()
        for direction in ("forward", "both"):
            leaves = [f.to(DEV).requires_grad_(True), v.to(DEV), o.to(DEV), h0.to(DEV).requires_grad_(True)]
            y, last = hn.gated_recurrence(leaves[0], leaves[1], out_gate=leaves[2], h0=leaves[3], direction=direction)
            assert float(((last.detach().cpu().double() - want) / want).abs().max()) <= 8 * T * u
            with torch.no_grad():
                assert torch.equal(hn.gated_recurrence(leaves[0], leaves[1], h0=leaves[3], direction=direction)[1], last)
            dlast = 1 + torch.rand(B, C, generator=g)
            dh0, = torch.autograd.grad(last, [leaves[3]], dlast.to(DEV), retain_graph=True)
            w = a * dlast.double()
            assert float(((dh0.cpu().double() - w) / w).abs().max()) <= 8 * T * u
            if T == 1:
                dy = (1 + torch.rand(T, B, C, generator=g)).bfloat16()
                few = o.clamp(min=-5)                                        # (the product of the two gates stays a normal number)
                y, last = hn.gated_recurrence(leaves[0], leaves[1], out_gate=few.to(DEV), h0=leaves[3], direction=direction)
                dh0, = torch.autograd.grad(y, [leaves[3]], dy.to(DEV))
                w = (torch.sigmoid(f.double()) * torch.sigmoid(few.double()) * dy.double())[0]
                assert float(((dh0.cpu().double() - w) / w).abs().max()) <= 16 * u
        if T == 1:
            state = h0.to(DEV)
            hn.gated_recurrence_step(f[0].to(DEV), v[0].to(DEV), state)
            assert float(((state.cpu().double() - want) / want).abs().max()) <= 8 * u
    steps = (-30 + 60 * torch.rand(1, 1, 4096, generator=g)).bfloat16()      # the other side: 1 - a of a nearly closed gate, and gates at infinity
    one = torch.ones(1, 1, 4096, dtype=torch.bfloat16)
    want = torch.sigmoid(-steps.double())[0]
    assert float(((hn.gated_recurrence(steps.to(DEV), one.to(DEV))[1].cpu().double() - want) / want).abs().max()) <= 8 * u
    ends = torch.tensor([float("inf"), -float("inf"), 3e38, -3e38, 200.0, -200.0, float("nan")]).bfloat16().view(1, 1, -1).to(DEV)
    for got in (hn.gated_recurrence(ends, torch.full_like(ends, 2.0), h0=torch.full((1, 7), 9.0, device=DEV))[1][0].tolist(),):
        assert got[:6] == [9.0, 2.0, 9.0, 2.0, 9.0, 2.0] and got[6] != got[6]


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("direction", ["forward", "reverse", "both"])
@pytest.mark.parametrize("T,B,C", [(30, 2, 6), (60, 3, 40), (120, 2, 64), (120, 40, 520), (300, 2, 36), (1500, 1, 64), (1500, 9, 330)])
def test_infinite_state_stays(T, B, C, direction, name):
    """An infinite value makes the state infinite from its step on: a gate above 0 passes it on however many steps follow, also where the product of
    their gates is no float32 number any more.  The gradient of a state flows back the same way."""
    g = torch.Generator().manual_seed(T + B)
    f = (torch.randn(T, B, C, generator=g) * 1.5 - 3).to(DT[name])           # (gates of about 1/20: 30 of them are 1e-39)
    f[:, :, 1] = -30                                                         # (and in one channel 2 of them)
    v, h0 = torch.randn(T, B, C, generator=g).to(DT[name]), torch.randn(B, C, generator=g)
    at, sign = T // 3, torch.where(torch.rand(C, generator=g) < 0.5, -1.0, 1.0)
    hit = torch.arange(C) % 4 == 1
    v[at, :, hit] = (float("inf") * sign[hit]).to(DT[name])
    back = torch.zeros(C, dtype=torch.bool)                                  # channels that run from the last step
    back[C // 2 if direction == "both" else 0 if direction == "reverse" else C:] = True
    step = torch.arange(T)[:, None]
    gone = torch.where(back, step <= at, step >= at) & hit                   # [T, C]: steps whose state is infinite
    fd, vd, hd = (t.to(DEV).requires_grad_(True) for t in (f, v, h0))
    y, last = hn.gated_recurrence(fd, vd, h0=hd, direction=direction)
    got = y.detach().cpu().float()
    assert bool((got[gone[:, None].expand(T, B, C)] == (sign * float("inf")).expand(T, B, C)[gone[:, None].expand(T, B, C)]).all())
    assert bool(torch.isfinite(got[~gone[:, None].expand(T, B, C)]).all())
    assert bool((last.detach().cpu()[:, hit] == (sign * float("inf"))[hit]).all()) and bool(torch.isfinite(last[:, ~hit.to(DEV)]).all())
    # the gradient of an infinite dy at step `at` is infinite at every step in front of it, and at h0
    v, dy = torch.randn(T, B, C, generator=g).to(DT[name]), torch.randn(T, B, C, generator=g).to(DT[name])
    dy[at, :, hit] = (float("inf") * sign[hit]).to(DT[name])
    gone = torch.where(back, step >= at, step <= at) & hit
    vd = v.to(DEV).requires_grad_(True)
    y, last = hn.gated_recurrence(fd, vd, h0=hd, direction=direction)
    dv, dh0 = torch.autograd.grad(y, [vd, hd], dy.to(DEV))
    got, full = dv.cpu().float(), gone[:, None].expand(T, B, C)
    assert bool((got[full] == (sign * float("inf")).expand(T, B, C)[full]).all()) and bool(torch.isfinite(got[~full]).all())
    assert bool((dh0.cpu()[:, hit] == (sign * float("inf"))[hit]).all()) and bool(torch.isfinite(dh0[:, ~hit.to(DEV)]).all())


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_closed_gate_forgets_exactly(name):
    """A gate that is 0 leaves nothing of a finite state, on whichever side of a join it lies."""
    T, C = 1500, 64
    f, v = torch.full((T, 1, C), 2.0, dtype=DT[name], device=DEV), torch.zeros(T, 1, C, dtype=DT[name], device=DEV)
    f[700] = -float("inf")
    y, last = hn.gated_recurrence(f, v, h0=torch.full((1, C), 1e30, device=DEV))
    assert bool((y[700:] == 0).all()) and bool((last == 0).all()) and bool((y[0] > 1e29).all())


@pytest.mark.parametrize("name,M,K,F", [("f32", 40, 24, 9), ("f32", 40, 136, 9), ("bf16", 40, 24, 9), ("bf16", 300, 64, 203), ("bf16", 8192, 128, 767)])
def test_infinite_row_with_odd_hidden_units(name, M, K, F):
    """x of one row infinite, weights positive, relu: dx of that row is +inf as the formula says and not NaN, also where the rows of dg | du are padded
    to whole vectors; the other rows are what they are without it."""
    g = torch.Generator().manual_seed(F)
    dt = DT[name]
    x, dy = (torch.rand(M, K, generator=g) + 0.5).to(dt), (torch.rand(M, F, generator=g) + 0.5).to(dt)
    wg, wu = ((torch.rand(F, K, generator=g) + 0.5) / K for _ in range(2))
    x[7, 3] = float("inf")
    xd = x.to(DEV).requires_grad_(True)
    wgd, wud = wg.to(dt).to(DEV), wu.to(dt).to(DEV)
    y = hn.gated_linear(xd, wgd, wud, activation="relu")
    dx, = torch.autograd.grad(y, [xd], dy.to(DEV))
    assert bool(torch.isposinf(y[7]).all()) and bool(torch.isposinf(dx[7]).all())
    tame = torch.where(torch.isinf(x), torch.ones((), dtype=dt), x).to(DEV).requires_grad_(True)
    want, = torch.autograd.grad(hn.gated_linear(tame, wgd, wud, activation="relu"), [tame], dy.to(DEV))
    rest = torch.arange(M) != 7
    assert torch.equal(dx[rest], want[rest])


def _calls(x):
    """The four operators on x [4, 2, 8]."""
    w = torch.ones(3, 8, device=DEV)
    other = torch.zeros(4, 2, 8, device=DEV)
    return [lambda: hn.gated_recurrence(x, other), lambda: hn.gated_recurrence(other, x), lambda: hn.gated_recurrence(other, other, out_gate=x),
            lambda: hn.gated_recurrence(other, other, h0=x[0]), lambda: hn.gated_linear(x, w, w), lambda: hn.gated_linear(other, x[:, 0, :], w[:1].expand(4, 8)),
            lambda: hn.dropout(x, 0.5, 1), lambda: hn.dropout(other, 0.5, 1, residual=x),
            lambda: hn.gated_recurrence_step(x[0], other[0], torch.zeros(2, 8, device=DEV)),
            lambda: hn.gated_recurrence_step(other[0], other[0], torch.zeros(2, 8, device=DEV), out_gate=x[0])]


def test_forward_mode_is_refused():
    """A tangent would be dropped: refused, with and without requires_grad, with and without grad mode."""
    with torch.autograd.forward_ad.dual_level():
        for primal in (torch.randn(4, 2, 8, device=DEV), torch.randn(4, 2, 8, device=DEV, requires_grad=True)):
            dual = torch.autograd.forward_ad.make_dual(primal, torch.ones(4, 2, 8, device=DEV))
            for call in _calls(dual):
                with pytest.raises(RuntimeError):
                    call()
                with torch.no_grad(), pytest.raises(RuntimeError):
                    call()
    x = torch.randn(4, 2, 8, device=DEV)
    for transform in (lambda fn: torch.func.jvp(fn, (x,), (x,)), lambda fn: torch.func.vmap(fn)(x[None]), lambda fn: torch.func.grad(lambda t: fn(t).sum())(x)):
        with pytest.raises(RuntimeError):
            transform(lambda t: hn.dropout(t, 0.5, 1))
        with pytest.raises(RuntimeError):
            transform(lambda t: hn.gated_recurrence(t, t)[0])


def test_tracing_is_refused():
    """A trace sees the outputs' memory and nothing that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.randn(4, 2, 8, device=DEV)
    for k in range(len(_calls(x))):
        def fn(t):
            y = _calls(t)[k]()
            return y[0] if isinstance(y, tuple) else y
        for grad in (False, True):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                torch.jit.trace(fn, (x,), check_trace=False)
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                make_fx(fn)(x)


def test_backward_is_seen_too():
    """The same in a backward pass whose forward pass ran outside: an incoming gradient with a tangent, a trace of the backward pass alone."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x, w = torch.randn(4, 2, 8, device=DEV, requires_grad=True), torch.randn(8, 8, device=DEV)
    dy = torch.randn(4, 2, 8, device=DEV)
    for call in (lambda: hn.gated_recurrence(x, x)[0], lambda: hn.gated_linear(x, w, w), lambda: hn.dropout(x, 0.5, 1)):
        y = call()
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(y, x, torch.autograd.forward_ad.make_dual(dy, dy), retain_graph=True)
        for trace in (lambda fn: torch.jit.trace(fn, (dy,), check_trace=False), lambda fn: make_fx(fn)(dy)):
            with pytest.raises(RuntimeError):
                trace(lambda d: torch.autograd.grad(y, x, d, retain_graph=True)[0])
        assert torch.autograd.grad(y, x, dy)[0].shape == x.shape
    last = hn.gated_recurrence(x, x)[1]
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.autograd.grad(last, x, torch.autograd.forward_ad.make_dual(dy[0], dy[0]))


def _behind(kind):
    """A leaf on the device and the operator's output through a node of torch between them."""
    other, weight = torch.randn(4, 2, 64, device=DEV), torch.randn(32, 64, device=DEV)
    if kind == "batch":                                       # x is reshaped to a matrix
        leaf = torch.randn(4, 2, 64, device=DEV, requires_grad=True)
        return leaf, lambda: hn.gated_linear(leaf, weight, weight)
    if kind == "weight":                                      # rows of a transposed weight are copied
        leaf = torch.randn(64, 32, device=DEV, requires_grad=True)
        return leaf, lambda: hn.gated_linear(other, leaf.t(), weight)
    if kind == "cast":
        leaf = torch.randn(32, 64, device=DEV, requires_grad=True)
        return leaf, lambda: hn.gated_linear(other.bfloat16(), leaf.bfloat16(), weight.bfloat16())
    leaf = torch.randn(64, 4, 2, device=DEV).permute(1, 2, 0).requires_grad_(True)      # channels apart
    assert leaf.is_leaf and leaf.stride(-1) != 1
    return leaf, {"forget": lambda: hn.gated_recurrence(leaf, other)[0], "value": lambda: hn.gated_recurrence(other, leaf)[0],
                  "out_gate": lambda: hn.gated_recurrence(other, other, out_gate=leaf)[0], "h0": lambda: hn.gated_recurrence(other, other, h0=leaf[0])[0],
                  "x": lambda: hn.gated_linear(leaf, weight, weight), "dropout": lambda: hn.dropout(leaf, 0.5, 1),
                  "residual": lambda: hn.dropout(other, 0.5, 1, residual=leaf)}[kind]


@pytest.mark.parametrize("kind", ["batch", "weight", "cast", "forget", "value", "out_gate", "h0", "x", "dropout", "residual"])
def test_captured_backward_of_leaves_behind_a_view(kind):
    """A leaf that an eager graph on the default stream holds is refused also where a node of torch stands between it and the operator; once that graph is
    gone the capture works."""
    leaf, call = _behind(kind)
    held = call()
    dy = torch.randn_like(held)
    want = torch.autograd.grad(held, leaf, dy, retain_graph=True)[0]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="being captured while a graph"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(call(), leaf, dy)
    torch.cuda.synchronize()
    assert torch.equal(torch.autograd.grad(held, leaf, dy)[0], want)
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call(), leaf, dy)[0]
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_step_refuses_a_state_that_overlaps_an_input():
    """The state is written while other elements' inputs are read: an input that lies over it in part is refused; one that is the state itself, or lies beside
    or between its rows, is taken."""
    buf = torch.randn(64, device=DEV)
    state = buf[16:32].view(2, 8)
    far = torch.randn(2, 8, device=DEV)
    over = [buf[8:24].view(2, 8), buf[24:40].view(2, 8), buf[17:33].view(2, 8), buf.as_strided((2, 8), (24, 1), 0), buf.as_strided((2, 8), (20, 1), 4),
            buf.as_strided((2, 8), (0, 1), 20), buf.as_strided((2, 8), (16, 1), 16), buf.as_strided((2, 8), (31, 1), 0)]
    before = buf.clone()
    for t in over:
        for call in (lambda: hn.gated_recurrence_step(t, far, state), lambda: hn.gated_recurrence_step(far, t, state),
                     lambda: hn.gated_recurrence_step(far, far, state, out_gate=t)):
            with pytest.raises(RuntimeError, match="shares memory"):
                call()
    half = torch.randn(2, 8, device=DEV).bfloat16()
    with pytest.raises(RuntimeError, match="shares memory"):
        hn.gated_recurrence_step(buf.view(torch.bfloat16)[32:48].view(2, 8), half, state)
    assert torch.equal(buf, before)
    beside = [buf[:16].view(2, 8), buf[32:48].view(2, 8), buf.as_strided((2, 8), (24, 1), 8), buf.as_strided((2, 8), (0, 1), 8), state]
    for t in beside + [state[:, [3, 1, 2, 0, 5, 6, 7, 4]], buf.as_strided((2, 8), (8, 2), 12)]:            # (copies: channels apart)
        want = state.clone()
        y = hn.gated_recurrence_step(t.clone(), far, want)
        with torch.no_grad():
            keep = state.clone()
            assert torch.equal(hn.gated_recurrence_step(t, far, state), y) and torch.equal(state, want)
            state.copy_(keep)


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_negated_views(name):
    """A view whose sign is pending (torch's imaginary part of a conjugate) is read with its sign."""
    g = torch.Generator().manual_seed(17)
    n = lambda *s: torch.randn(*s, generator=g).to(DT[name]).to(DEV)  # noqa: E731
    neg = torch._neg_view
    f, v, o, h0, w, b = n(5, 3, 8), n(5, 3, 8), n(5, 3, 8), torch.randn(3, 8, generator=g).to(DEV), n(4, 8), n(4)
    for a, c in zip(hn.gated_recurrence(neg(f), neg(v), out_gate=neg(o), h0=neg(h0)), hn.gated_recurrence(-f, -v, out_gate=-o, h0=-h0)):
        assert torch.equal(a, c)
    assert torch.equal(hn.gated_linear(neg(f), neg(w), neg(w), neg(b), neg(b)), hn.gated_linear(-f, -w, -w, -b, -b))
    assert torch.equal(hn.dropout(neg(f), 0.5, 3, residual=neg(v)), hn.dropout(-f, 0.5, 3, residual=-v))
    s1, s2 = h0.clone(), h0.clone()
    assert torch.equal(hn.gated_recurrence_step(neg(f[0]), neg(v[0]), s1, out_gate=neg(o[0])), hn.gated_recurrence_step(-f[0], -v[0], s2, out_gate=-o[0]))
    assert torch.equal(s1, s2)
    with pytest.raises(ValueError):
        hn.gated_recurrence_step(f[0], v[0], neg(s1))
    # gradients that arrive negated
    leaf = [t.detach().clone().requires_grad_(True) for t in (f, v, h0)]
    y, last = hn.gated_recurrence(leaf[0], leaf[1], h0=leaf[2])
    dy, dl = n(5, 3, 8), torch.randn(3, 8, generator=g).to(DEV)
    for a, c in zip(torch.autograd.grad((y, last), leaf, (neg(dy), neg(dl)), retain_graph=True), torch.autograd.grad((y, last), leaf, (-dy, -dl))):
        assert torch.equal(a, c)
    x = f.detach().clone().requires_grad_(True)
    z = hn.gated_linear(x, w, w)
    d = n(5, 3, 4)
    assert torch.equal(torch.autograd.grad(z, x, neg(d), retain_graph=True)[0], torch.autograd.grad(z, x, -d)[0])
    z = hn.dropout(x, 0.5, 1, residual=x)
    assert torch.equal(torch.autograd.grad(z, x, neg(dy), retain_graph=True)[0], torch.autograd.grad(z, x, -dy)[0])


def test_imaginary_part():
    """One hidden unit as the imaginary part of a number that is conjugated later: its gradient arrives as such a view."""
    g = torch.Generator().manual_seed(18)
    x, w = torch.randn(6, 16, generator=g).to(DEV).requires_grad_(True), torch.randn(1, 16, generator=g).to(DEV)
    factor = torch.randn(6, 1, generator=g).to(DEV)
    y = hn.gated_linear(x, w, w)
    got, = torch.autograd.grad((torch.complex(torch.zeros_like(y), y).conj() * torch.complex(torch.zeros_like(factor), factor)).real.sum(), x)
    y = hn.gated_linear(x, w, w)
    want, = torch.autograd.grad((y * factor).sum(), x)
    assert torch.equal(got, want)
