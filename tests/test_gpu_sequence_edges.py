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
