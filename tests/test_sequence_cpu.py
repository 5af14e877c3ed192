"""Sequence operators without a GPU: the oracle's gradients against differences, the generator's statistics, and the refusals that the
host makes before any launch."""
import ctypes

import pytest
import torch

import horizonnet_amd as hn
from horizonnet_amd import _lib
from oracle import sequence_ref as ref


def _differences(fn, args, grads, names, eps=1e-6):
    """Central differences of the scalar fn along one random direction per argument, in float64: truncation eps^2, rounding 2^-53 / eps."""
    g = torch.Generator().manual_seed(5)
    for i, name in enumerate(names):
        d = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        at = lambda s: fn(*[a + s * eps * d if j == i else a for j, a in enumerate(args)])  # noqa: E731
        want = float((grads[name] * d).sum())
        assert abs(float(at(1) - at(-1)) / (2 * eps) - want) < 1e-7 * (1 + float((grads[name] * d).abs().sum())), name


@pytest.mark.parametrize("direction", ["forward", "reverse", "both"])
@pytest.mark.parametrize("ragged", [False, True])
def test_recurrence_gradient_against_differences(direction, ragged):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    T, B, C = 9, 3, 4
    f, v, o, h0, dy, dlast = r(T, B, C), r(T, B, C), r(T, B, C), r(B, C), r(T, B, C), r(B, C)
    lengths = torch.tensor([9, 4, 0]) if ragged else None

    def value(f, v, o, h0):
        got, _ = ref.recurrence(f, v, o, h0, lengths, direction)
        return (got["y"] * dy).sum() + (got["last"] * dlast).sum()

    got, _ = ref.recurrence(f, v, o, h0, lengths, direction, dy, dlast)
    _differences(value, [f, v, o, h0], got, ["df", "dv", "do", "dh0"])


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "relu"])
def test_linear_gradient_against_differences(act):
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, wg, wu, bg, bu, dy = r(5, 7), r(6, 7), r(6, 7), r(6), r(6), r(5, 6)
    got, _ = ref.linear(x, wg, wu, bg, bu, act, dy)
    _differences(lambda *a: (ref.linear(*a, act)[0]["y"] * dy).sum(), [x, wg, wu, bg, bu], got, ["dx", "dwg", "dwu", "dbg", "dbu"])


def test_dropout_generator_statistics():
    """The kept share is that of n independent draws: within 5 standard deviations, for near-by seeds and for one seed's parts."""
    n = 1 << 18
    for p in (0.1, 0.5, 0.9):
        for seed in (0, 1, 2, 2 ** 63):
            k = ref.dropout_keep(n, p, seed).double()
            assert abs(float(k.mean()) - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5
        a, b = ref.dropout_keep(n, p, 7).double(), ref.dropout_keep(n, p, 8).double()
        assert abs(float((a * b).mean()) - (1 - p) ** 2) < 5 * 0.5 / n ** 0.5
    assert bool(ref.dropout_keep(1000, 0.0, 3).all())


def test_no_cpu_fallback():
    x = torch.zeros(4, 2, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hn.gated_recurrence(x, x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hn.gated_recurrence_step(x[0], x[0], x[0])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hn.gated_linear(x, torch.zeros(3, 8), torch.zeros(3, 8))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        hn.dropout(x, 0.5, 1)
    with pytest.raises(TypeError):
        hn.dropout([1.0], 0.5, 1)


def _fails(rc, text):
    assert rc != 0 and text in _lib.load().hn_last_error().decode()


def test_library_refusals():
    """Every refusal is made by the host before anything is enqueued (so it needs no device)."""
    lib, one = _lib.load(), ctypes.c_void_p(256)              # an address that is never read

    def rec(T=4, B=2, C=8, dtype=0, direction=0, y=one, last=one, ws=None, n=0):
        return lib.hn_gated_recurrence(one, 16, 8, one, 16, 8, None, 0, 0, None, None, y, last, None, ws, n, T, B, C, dtype, direction, None)

    _fails(rec(dtype=2), "dtype")
    _fails(rec(direction=3), "direction")
    _fails(rec(C=7, direction=2), "even number of channels")
    _fails(rec(T=-1), "bad sizes")
    _fails(rec(C=1 << 31), "bad sizes")
    _fails(rec(y=None), "null pointer")
    _fails(rec(last=None), "null pointer")
    _fails(rec(T=5000), "workspace too small")
    _fails(rec(T=5000, n=1 << 20), "workspace too small")     # a size without an address
    assert rec(B=0, y=None, last=None) == 0
    _fails(lib.hn_gated_recurrence_bwd(one, 16, 8, one, 16, 8, None, 0, 0, one, 16, 8, None, None, None, one, one, None, None, None, 0, 4, 2, 8, 0, 0, None),
           "null pointer")
    _fails(lib.hn_gated_recurrence_bwd(one, 16, 8, one, 16, 8, one, 16, 8, one, 16, 8, None, None, one, one, one, None, None, None, 0, 4, 2, 8, 0, 0, None),
           "null pointer")
    _fails(lib.hn_gated_recurrence_step(one, 8, one, 8, None, 0, None, one, 2, 8, 0, None), "null pointer")
    _fails(lib.hn_gated_recurrence_step(one, 8, one, 8, None, 0, one, one, 2, 8, 7, None), "dtype")

    def lin(M=4, K=8, F=8, dtype=0, act=0, y=one, ld=8, kept=None):
        return lib.hn_gated_linear(one, ld, one, 8, one, 8, None, None, y, kept, None, 0, M, K, F, dtype, act, None)

    _fails(lin(dtype=-1), "dtype")
    _fails(lin(act=4), "activation")
    _fails(lin(y=None), "null pointer")
    _fails(lin(ld=-8), "negative row stride")
    _fails(lin(K=1 << 20), "bad sizes")
    _fails(lin(F=1 << 20), "bad sizes")
    _fails(lin(kept=one), "kept")                             # K < 128: nothing is kept
    _fails(lib.hn_gated_linear_bwd(one, 8, one, 8, one, 8, None, None, one, 8, None, one, one, one, None, None, None, 0, 4, 8, 8, 0, 0, None), "workspace too small")
    assert lib.hn_gated_linear_kept(4, 128, 12, 0) == 4 * 2 * 16 and lib.hn_gated_linear_kept(4, 128, 12, 1) == 0
    assert lin(M=0, y=None) == 0

    for p in (1.0, -0.1, float("nan")):
        _fails(lib.hn_dropout(one, None, one, 4, 0, p, 1, None, None), "p=")
    _fails(lib.hn_dropout(one, None, None, 4, 0, 0.5, 1, None, None), "null pointer")
    _fails(lib.hn_dropout(one, None, one, 4, 3, 0.5, 1, None, None), "dtype")
    _fails(lib.hn_dropout(one, None, one, -1, 0, 0.5, 1, None, None), "n=-1")
    assert lib.hn_dropout(None, None, None, 0, 0, 0.5, 1, None, None) == 0


def test_workspace_of_refused_sizes():
    """The size functions answer 0 for what the calls refuse (one channel in both directions and steps past 2^31 divided by zero)."""
    lib = _lib.load()
    for T, B, C, direction in ((1000, 1, 1, 2), (1000, 3, 7, 2), (1 << 46, 1, 8, 0), (1000, 1 << 33, 8, 0), (1000, 1, 1 << 40, 1), (0, 1, 8, 0), (-5, 1, 8, 0)):
        assert lib.hn_gated_recurrence_workspace(T, B, C, direction) == 0
    assert lib.hn_gated_recurrence_workspace(5000, 2, 8, 0) > 0
    for M, K, F, dtype in ((1 << 31, 8, 8, 0), (4, 1 << 20, 8, 0), (4, 8, 1 << 20, 1), (-1, 8, 8, 0), (4, 8, 8, 2)):
        assert lib.hn_gated_linear_workspace(256, 8, 256, 8, 256, 8, M, K, F, dtype, 1) == 0
        assert lib.hn_gated_linear_kept(M, K, F, dtype) == 0
