"""Calls of the sequence operators that the host has to refuse, without a GPU: each check comes before any launch."""
import pytest
import torch

import horizonnet_amd as hn


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
