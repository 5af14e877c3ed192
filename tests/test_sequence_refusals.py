"""Calls of the sequence operators that the host has to refuse, without a GPU: each check comes before any launch."""
import ctypes

import pytest
import torch

import horizonnet_amd as hn
from horizonnet_amd import _lib


def _calls(x):
    """The four operators on x [4, 2, 8], in each place that takes a gradient."""
    w, other, state = torch.ones(3, 8), torch.zeros(4, 2, 8), torch.zeros(2, 8)
    return [lambda: hn.gated_recurrence(x, other), lambda: hn.gated_recurrence(other, x), lambda: hn.gated_recurrence(other, other, out_gate=x),
            lambda: hn.gated_recurrence(other, other, h0=x[0]), lambda: hn.gated_linear(x, w, w), lambda: hn.gated_linear(other, x[:3, 0], w),
            lambda: hn.gated_linear(other, w, x[:3, 0]), lambda: hn.gated_linear(other, w, w, b_gate=x[:3, 0, 0]), lambda: hn.gated_linear(other, w, w, b_up=x[:3, 0, 0]),
            lambda: hn.dropout(x, 0.5, 1), lambda: hn.dropout(other, 0.5, 1, residual=x), lambda: hn.gated_recurrence_step(x[0], other[0], state),
            lambda: hn.gated_recurrence_step(other[0], x[0], state), lambda: hn.gated_recurrence_step(other[0], other[0], state, out_gate=x[0]),
            lambda: hn.gated_recurrence_step(other[0], other[0], x[0])]


def test_forward_mode_is_refused():
    """A tangent would be dropped, which counts as zero."""
    with torch.autograd.forward_ad.dual_level():
        for primal in (torch.randn(4, 2, 8), torch.randn(4, 2, 8, requires_grad=True)):
            dual = torch.autograd.forward_ad.make_dual(primal, torch.ones(4, 2, 8))
            for call in _calls(dual):
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call()
                with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call()
            with pytest.raises(RuntimeError, match="no CPU fallback"):       # what carries no tangent goes on
                hn.dropout(primal, 0.5, 1)


def test_tracing_is_refused():
    """A trace would keep the outputs' memory and nothing that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.randn(4, 2, 8)
    for k in range(len(_calls(x))):
        for trace in (lambda fn: torch.jit.trace(fn, (x,), check_trace=False), lambda fn: make_fx(fn)(x)):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                trace(lambda t: _calls(t)[k]())


@torch.library.custom_op("horizonnet_tests::dropped", mutates_args=())
def _dropped(x: torch.Tensor) -> torch.Tensor:
    return hn.dropout(x, 0.5, 1)


def test_registered_operators_may_be_traced():
    """Inside the kernel of an operator that a program has registered, the trace records that operator: the call goes on (here to the missing device)."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.randn(4, 2, 8)
    for trace in (lambda fn: torch.jit.trace(fn, (x,), check_trace=False), lambda fn: make_fx(fn)(x)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            trace(lambda t: _dropped(t))


def _fails(rc, text):
    assert rc != 0 and text in _lib.load().hn_last_error().decode()


def test_launches_past_2_32_threads_are_refused():
    """Sizes inside each argument's own range whose launch would hold 2^32 threads or more (a step of 2^32 sequences, rows of one hidden unit, ...)."""
    lib, one = _lib.load(), ctypes.c_void_p(256)              # an address that is never read
    for T, B, C, direction in ((1, 1 << 26, 1, 0), (1, 1 << 26, 3, 1), (50, 1 << 25, 1, 0), (100, 1 << 24, 2, 2), (1, (1 << 31) - 1, 1 << 20, 0)):
        for dtype in (0, 1):
            n = lib.hn_gated_recurrence_workspace(T, B, C, direction)
            assert n == 0
            _fails(lib.hn_gated_recurrence(one, C, C, one, C, C, None, 0, 0, None, None, one, one, None, None, 0, T, B, C, dtype, direction, None), "2^32 threads")
            _fails(lib.hn_gated_recurrence_bwd(one, C, C, one, C, C, None, 0, 0, one, C, C, None, None, one, one, one, None, None, None, 0, T, B, C, dtype, direction,
                                               None), "2^32 threads")
    for B, C in (((1 << 31) - 1, 3), ((1 << 31) - 1, 8), (1 << 20, 1 << 14)):
        _fails(lib.hn_gated_recurrence_step(one, C, one, C, None, 0, one, one, B, C, 0, None), "2^32 threads")
    for dtype in (0, 1):
        _fails(lib.hn_gated_linear(one, 8, one, 8, one, 8, None, None, one, None, None, 0, (1 << 31) - 1, 8, 1, dtype, 0, None), "2^32 threads")
        need = lib.hn_gated_linear_workspace(one, 8, one, 8, one, 8, (1 << 31) - 1, 8, 1, dtype, 1)
        _fails(lib.hn_gated_linear_bwd(one, 8, one, 8, one, 8, None, None, one, 1, None, one, one, one, None, None, one, need, (1 << 31) - 1, 8, 1, dtype, 0, None),
               "2^32 threads")
