"""Sequence operators on the device: the pieces of a recurrent block over the 256 columns of a panorama, next to the LSTM layers the
engine itself runs (reference ``model.py:222-227,263-266``: bi-LSTM, dropout, linear).

* ``gated_recurrence`` / ``gated_recurrence_step`` -- a gated linear recurrence, parallel over time (``hn_gated_recurrence*``)
* ``gated_linear``                                 -- both projections, activation and product in one kernel (``hn_gated_linear*``)
* ``dropout``                                      -- counter-based, its mask never stored, with the residual sum (``hn_dropout``)

All take ROCm tensors in float32 or bfloat16 (one type per call; float32 states), run on the current stream, are differentiable
(once) and give the same bits every time.  There is no CPU fallback.
"""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_DIRECTIONS = {"forward": 0, "reverse": 1, "both": 2}
_ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2, "relu": 3}


class _Here:
    """The current device is the tensors' own: nothing to switch."""

    def __enter__(self):
        return None

    def __exit__(self, *a):
        return False


_HERE = _Here()
# The public torch.cuda.current_device() / current_stream() cost 3 and 7 us in a call that is not in a tight loop, as much as a launch; these
# are what they ask in turn.
_device_now = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on(device):
    return _HERE if _device_now() == device.index else torch.cuda.device(device)


def _addr(t):
    return None if t is None else t.data_ptr()


def _check_main(who, name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s: %s must be a tensor" % (who, name))
    if not t.is_cuda:
        raise RuntimeError("%s needs cuda/ROCm tensors (no CPU fallback): %s is on %s" % (who, name, t.device))
    if t.dtype not in _DTYPES:
        raise ValueError("%s: %s is %s; float32 and bfloat16 are supported" % (who, name, t.dtype))


def _check_like(who, name, t, shape, dtype, device):
    if isinstance(t, torch.Tensor) and t.shape == shape and t.dtype == dtype and t.device == device:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s: %s must be a tensor" % (who, name))
    if t.device != device:
        raise RuntimeError("%s: %s is on %s, expected %s" % (who, name, t.device, device))
    if t.dtype != dtype:
        raise ValueError("%s: %s is %s, expected %s" % (who, name, t.dtype, dtype))
    raise ValueError("%s: %s has shape %s, expected %s" % (who, name, tuple(t.shape), tuple(shape)))


def _rows(t):
    """Channels next to each other; the other axes as they are."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _tb(t):
    return (None, 0, 0) if t is None else (t.data_ptr(), t.stride(0), t.stride(1))


# ---- gated linear recurrence ----
def _recurrence_forward(f, v, o, h0, lengths, direction, keep):
    dev, (T, B, C) = f.device, f.shape
    lib = _lib.load()
    y = torch.empty((T, B, C), dtype=f.dtype, device=dev)
    last = torch.empty((B, C), dtype=torch.float32, device=dev)
    n = lib.hn_gated_recurrence_workspace(T, B, C, direction)
    ws = torch.empty(n, dtype=torch.float32, device=dev) if n else None
    states = torch.empty(lib.hn_gated_recurrence_states(T, B, C), dtype=torch.float32, device=dev) if keep else None
    with _on(dev):
        _lib.check(lib.hn_gated_recurrence(*_tb(f), *_tb(v), *_tb(o), _addr(h0), _addr(lengths), y.data_ptr(), last.data_ptr(), _addr(states), _addr(ws), n,
                                           T, B, C, _DTYPES[f.dtype], direction, _raw_stream(dev.index)), "hn_gated_recurrence")
    return y, last, states


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, f, v, o, h0, lengths, direction):
        y, last, states = _recurrence_forward(f, v, o, h0, lengths, direction, True)
        ctx.save_for_backward(f, v, o, lengths, states)
        ctx.direction, ctx.has_h0 = direction, h0 is not None
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        f, v, o, lengths, states = ctx.saved_tensors
        dev, (T, B, C) = f.device, f.shape
        lib = _lib.load()
        dy = torch.zeros((T, B, C), dtype=f.dtype, device=dev) if dy is None else _rows(dy)
        dlast = None if dlast is None else dlast.contiguous()
        grads = torch.empty((2 if o is None else 3, T, B, C), dtype=f.dtype, device=dev)      # one allocation: an allocation costs as much as a launch
        df, dv, d_o = grads[0], grads[1], None if o is None else grads[2]
        dh0 = torch.empty((B, C), dtype=torch.float32, device=dev) if ctx.has_h0 else None
        n = lib.hn_gated_recurrence_workspace(T, B, C, ctx.direction)
        ws = torch.empty(n, dtype=torch.float32, device=dev) if n else None
        with _on(dev):
            _lib.check(lib.hn_gated_recurrence_bwd(*_tb(f), *_tb(v), *_tb(o), *_tb(dy), _addr(dlast), _addr(lengths), states.data_ptr(), df.data_ptr(),
                                                   dv.data_ptr(), _addr(d_o), _addr(dh0), _addr(ws), n, T, B, C, _DTYPES[f.dtype], ctx.direction,
                                                   _raw_stream(dev.index)), "hn_gated_recurrence_bwd")
        return df, dv, d_o, dh0, None, None


def gated_recurrence(forget, value, out_gate=None, h0=None, lengths=None, direction="forward"):
    """``a = sigmoid(forget)``, ``h_t = a_t h_{t-1} + (1 - a_t) value_t``, ``y_t = sigmoid(out_gate_t) h_t`` -> ``(y, h_last)``.

    forget, value, out_gate (None: y = h): ``[T, B, C]`` like ``nn.LSTM``'s input, any strides (channels that are not next to each other are
    copied), so the parts of one projection's output or a batch-first tensor's transpose are taken as they are.  h0: float32 ``[B, C]`` or None
    (zeros).  direction: "forward", "reverse" (from the last step), or "both": the first ``C / 2`` channels run forward and the others in reverse,
    the layout of a bidirectional LSTM's output.  lengths: int32 / int64 tensor ``[B]`` on the same device: a sequence's steps at or past its
    length are not read, their y (and gradients) are 0, and the state passes; values outside ``0 .. T`` count as the nearest bound.

    y has the inputs' type; the state runs in float32 and h_last ``[B, C]`` is float32: the state behind the last step taken."""
    who = "gated_recurrence"
    _check_main(who, "forget", forget)
    if forget.dim() != 3:
        raise ValueError("%s: forget must be [T, B, C], got shape %s" % (who, tuple(forget.shape)))
    if direction not in _DIRECTIONS:
        raise ValueError("%s: direction must be one of %s, got %r" % (who, sorted(_DIRECTIONS), direction))
    T, B, C = forget.shape
    dev = forget.device
    _check_like(who, "value", value, forget.shape, forget.dtype, dev)
    if out_gate is not None:
        _check_like(who, "out_gate", out_gate, forget.shape, forget.dtype, dev)
    if h0 is not None:
        _check_like(who, "h0", h0, (B, C), torch.float32, dev)
        h0 = h0.contiguous()
    if direction == "both" and C % 2:
        raise ValueError("%s: direction 'both' needs an even number of channels, got %d" % (who, C))
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError("%s: lengths must be an int32 or int64 tensor" % who)
        _check_like(who, "lengths", lengths, (B,), lengths.dtype, dev)
        lengths = lengths.contiguous() if lengths.dtype == torch.int32 else lengths.clamp(0, T).to(torch.int32)
    f, v, o = _rows(forget), _rows(value), None if out_gate is None else _rows(out_gate)
    if torch.is_grad_enabled() and (f.requires_grad or v.requires_grad or (o is not None and o.requires_grad) or (h0 is not None and h0.requires_grad)):
        return _GatedRecurrence.apply(f, v, o, h0, lengths, _DIRECTIONS[direction])
    return _recurrence_forward(f, v, o, h0, lengths, _DIRECTIONS[direction], False)[:2]


def gated_recurrence_step(forget, value, state, out_gate=None):
    """One step of ``gated_recurrence`` for a serving loop: forget, value, out_gate ``[B, C]``; state float32 ``[B, C]``, contiguous, is updated
    IN PLACE; returns y ``[B, C]``.  Not differentiable."""
    who = "gated_recurrence_step"
    _check_main(who, "forget", forget)
    if forget.dim() != 2:
        raise ValueError("%s: forget must be [B, C], got shape %s" % (who, tuple(forget.shape)))
    B, C = forget.shape
    dev = forget.device
    _check_like(who, "value", value, forget.shape, forget.dtype, dev)
    if out_gate is not None:
        _check_like(who, "out_gate", out_gate, forget.shape, forget.dtype, dev)
    _check_like(who, "state", state, forget.shape, torch.float32, dev)
    if not state.is_contiguous():
        raise ValueError("%s: state is updated in place and must be contiguous" % who)
    f, v, o = _rows(forget), _rows(value), None if out_gate is None else _rows(out_gate)
    y = torch.empty((B, C), dtype=f.dtype, device=dev)
    with _on(dev):
        _lib.check(_lib.load().hn_gated_recurrence_step(f.data_ptr(), f.stride(0), v.data_ptr(), v.stride(0), _addr(o), 0 if o is None else o.stride(0),
                                                        state.data_ptr(), y.data_ptr(), B, C, _DTYPES[f.dtype], _raw_stream(dev.index)), "hn_gated_recurrence_step")
    torch.autograd.graph.increment_version(state)      # written behind torch's back: a graph that saved it must notice
    return y


# ---- gated linear block ----
def _linear_forward(x, wg, wu, bg, bu, act):
    dev, (M, K), F = x.device, x.shape, wg.shape[0]
    lib, dt = _lib.load(), _DTYPES[x.dtype]
    y = torch.empty((M, F), dtype=x.dtype, device=dev)
    mats = (x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0))
    n = lib.hn_gated_linear_workspace(*mats, M, K, F, dt, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    with _on(dev):
        _lib.check(lib.hn_gated_linear(*mats, _addr(bg), _addr(bu), y.data_ptr(),
                                       _addr(ws), n, M, K, F, dt, act, _raw_stream(dev.index)), "hn_gated_linear")
    return y


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, bg, bu, act):
        ctx.save_for_backward(x, wg, wu, bg, bu)
        ctx.act = act
        return _linear_forward(x, wg, wu, bg, bu, act)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, wg, wu, bg, bu = ctx.saved_tensors
        dev, (M, K), F = x.device, x.shape, wg.shape[0]
        lib, dt = _lib.load(), _DTYPES[x.dtype]
        dy = _rows(dy)
        need = ctx.needs_input_grad
        new = lambda i, *shape: torch.empty(shape, dtype=x.dtype, device=dev) if need[i] else None  # noqa: E731
        dx = new(0, M, K)
        if need[1] and need[2] and F * K % 8 == 0:
            dwg, dwu = torch.empty((2, F, K), dtype=x.dtype, device=dev)      # one allocation for two results on 16 bytes
        else:
            dwg, dwu = new(1, F, K), new(2, F, K)
        dbg, dbu = None if bg is None else new(3, F), None if bu is None else new(4, F)
        mats = (x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0))
        n = lib.hn_gated_linear_workspace(*mats, M, K, F, dt, 1)
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        with _on(dev):
            _lib.check(lib.hn_gated_linear_bwd(*mats, _addr(bg), _addr(bu), dy.data_ptr(), dy.stride(0), _addr(dx), _addr(dwg), _addr(dwu), _addr(dbg), _addr(dbu), _addr(ws), n, M, K, F, dt,
                                               ctx.act, _raw_stream(dev.index)), "hn_gated_linear_bwd")
        return dx, dwg, dwu, dbg, dbu, None


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    """``act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)`` in one kernel.  x ``[..., K]``, weights ``[F, K]`` (the layout of
    ``nn.Linear.weight``), biases ``[F]`` or None, each by itself; activation "silu", "gelu" (error function), "sigmoid" or "relu".  Products and
    activations run in float32 and the result ``[..., F]`` is rounded once to the inputs' type.  The backward pass forms the projections again
    instead of keeping them: only the inputs stay in memory between the passes."""
    who = "gated_linear"
    _check_main(who, "x", x)
    if x.dim() < 1:
        raise ValueError("%s: x must be [..., K]" % who)
    if activation not in _ACTIVATIONS:
        raise ValueError("%s: activation must be one of %s, got %r" % (who, sorted(_ACTIVATIONS), activation))
    dev, K = x.device, x.shape[-1]
    if not isinstance(w_gate, torch.Tensor) or w_gate.dim() != 2:
        raise ValueError("%s: w_gate must be a tensor [F, K]" % who)
    F = w_gate.shape[0]
    _check_like(who, "w_gate", w_gate, (F, K), x.dtype, dev)
    _check_like(who, "w_up", w_up, (F, K), x.dtype, dev)
    for name, b in (("b_gate", b_gate), ("b_up", b_up)):
        if b is not None:
            _check_like(who, name, b, (F,), x.dtype, dev)
    x2 = _rows(x if x.dim() == 2 else x.reshape(-1, K) if K else x.new_empty((x.shape[:-1].numel(), 0)))
    wg, wu = _rows(w_gate), _rows(w_up)
    bg, bu = None if b_gate is None else b_gate.contiguous(), None if b_up is None else b_up.contiguous()
    act = _ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x2, wg, wu, bg, bu)):
        y = _GatedLinear.apply(x2, wg, wu, bg, bu, act)
    else:
        y = _linear_forward(x2, wg, wu, bg, bu, act)
    return y if x.dim() == 2 else y.view(x.shape[:-1] + (F,))


# ---- dropout ----
def _drop(x, residual, p, seed):
    dev = x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    number, tensor = (0, seed) if isinstance(seed, torch.Tensor) else (seed, None)
    with _on(dev):
        _lib.check(_lib.load().hn_dropout(x.data_ptr(), _addr(residual), y.data_ptr(), x.numel(), _DTYPES[x.dtype], p, number, _addr(tensor), _raw_stream(dev.index)),
                   "hn_dropout")
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed):
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)
            ctx.seed = None
        else:
            ctx.seed = seed
        ctx.p = p
        return _drop(x, residual, p, seed)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            dx = _drop(dy.contiguous(), None, ctx.p, ctx.saved_tensors[0] if ctx.seed is None else ctx.seed)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None


def dropout(x, p, seed, residual=None):
    """``x`` with each element dropped with probability p and the kept ones divided by ``1 - p``; plus ``residual`` (same shape and type) if
    given, in the same pass.  The mask is never stored: it is a function of (seed, position in x read row by row), the same one in the
    backward pass, and the one the training step of ``HorizonNet`` draws from its own seeds.  seed: an int in ``0 .. 2**64 - 1``, or an int64
    tensor with one element on x's device, which the kernel reads: a captured step that changes it draws a new mask on every replay (it must
    not be changed between a forward pass and its backward pass; autograd refuses that).  A dropped element is 0 whatever x holds there."""
    who = "dropout"
    _check_main(who, "x", x)
    p = float(p)
    if not 0.0 <= p < 1.0 or ctypes.c_float(p).value >= 1.0:
        raise ValueError("%s: p must be in [0, 1), got %r" % (who, p))
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
            raise ValueError("%s: a seed tensor must be one int64 on %s, got %s %s on %s" % (who, x.device, tuple(seed.shape), seed.dtype, seed.device))
    elif isinstance(seed, bool) or not isinstance(seed, int) or not 0 <= seed < 1 << 64:
        raise ValueError("%s: seed must be an int in 0 .. 2**64 - 1 or an int64 tensor, got %r" % (who, seed))
    if residual is not None:
        _check_like(who, "residual", residual, x.shape, x.dtype, x.device)
        residual = residual.contiguous()
    x = x.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, p, seed)
    return _drop(x, residual, p, seed)
