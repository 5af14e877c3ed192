"""Sequence operators on the device: the pieces of a recurrent block over the 256 columns of a panorama, next to the LSTM layers the
engine itself runs (reference ``model.py:222-227,263-266``: bi-LSTM, dropout, linear).

* ``gated_recurrence`` / ``gated_recurrence_step`` -- a gated linear recurrence, parallel over time (``hn_gated_recurrence*``)
* ``gated_linear``                                 -- both projections, activation and product in one kernel (``hn_gated_linear*``)
* ``dropout``                                      -- counter-based, its mask never stored, with the residual sum (``hn_dropout``)

All take ROCm tensors in float32 or bfloat16 (one type per call; float32 states), run on the current stream, are differentiable
(once) and give the same bits every time.  There is no CPU fallback.  Argument checks and autograd nodes are native
(``csrc/sequence_torch.cpp``): a small call is bound by its host time.  Forward-mode derivatives and tracing (``torch.jit.trace``, ``make_fx``) are
refused: both would lose what the kernels do.

Calls may be captured into graphs, the first ones too.  A captured backward pass is refused while an eager graph made on the default stream
still holds one of the operator's leaf inputs, or a leaf that the pass reaches behind it: drop that graph first.
"""
_native = None


def _load():
    global _native
    if _native is None:
        import torch  # noqa: F401  (the extension links against it)
        try:
            from . import _sequence_torch
        except ImportError as e:
            raise ImportError("horizonnet_amd/_sequence_torch.so is missing or does not load (%s) -- build it with horizonnet_amd/csrc/build.sh "
                              "(python -c 'import __graft_entry__ as g; g.build()'); there is no fallback path." % e) from e
        _native = _sequence_torch
    return _native


def gated_recurrence(forget, value, out_gate=None, h0=None, lengths=None, direction="forward"):
    """``a = sigmoid(forget)``, ``h_t = a_t h_{t-1} + (1 - a_t) value_t``, ``y_t = sigmoid(out_gate_t) h_t`` -> ``(y, h_last)``.

    forget, value, out_gate (None: y = h): ``[T, B, C]`` like ``nn.LSTM``'s input, any strides (channels that are not next to each other are
    copied), so the parts of one projection's output or a batch-first tensor's transpose are taken as they are.  h0: float32 ``[B, C]`` or None
    (zeros).  direction: "forward", "reverse" (from the last step), or "both": the first ``C / 2`` channels run forward and the others in reverse,
    the layout of a bidirectional LSTM's output.  lengths: int32 / int64 tensor ``[B]`` on the same device: a sequence's steps at or past its
    length are not read, their y (and gradients) are 0, and the state passes; values outside ``0 .. T`` count as the nearest bound.

    y has the inputs' type; the state runs in float32 and h_last ``[B, C]`` is float32: the state behind the last step taken.  An infinite state stays
    infinite until a gate of 0 (in bfloat16, one below 2**-126), which makes NaN of it as the formula does."""
    return (_native or _load()).gated_recurrence(forget, value, out_gate, h0, lengths, direction)


def gated_recurrence_step(forget, value, state, out_gate=None):
    """One step of ``gated_recurrence`` for a serving loop: forget, value, out_gate ``[B, C]``; state float32 ``[B, C]``, contiguous, is updated
    IN PLACE and overlaps no input in part (an input may be the state itself); returns y ``[B, C]``.  Not differentiable: refuses inputs that ask
    for gradients."""
    return (_native or _load()).gated_recurrence_step(forget, value, state, out_gate)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    """``act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)`` in one kernel.  x ``[..., K]``, weights ``[F, K]`` (the layout of
    ``nn.Linear.weight``), biases ``[F]`` or None, each by itself; activation "silu", "gelu" (error function), "sigmoid" or "relu".  Products and
    activations run in float32 and the result ``[..., F]`` is rounded once to the inputs' type.  In bfloat16 the backward pass forms the
    projections again and only the inputs stay in memory between the passes; in float32 (K >= 128) both projections are kept.  The projections' gradients
    are rounded to the inputs' type in front of the products for dx and the weights' gradients, which in bfloat16 makes those 1.4 times as far off as one
    rounding would; the biases' gradients are sums of the unrounded ones."""
    return (_native or _load()).gated_linear(x, w_gate, w_up, b_gate, b_up, activation)


def dropout(x, p, seed, residual=None):
    """``x`` with each element dropped with probability p and the kept ones divided by ``1 - p``; plus ``residual`` (same shape and type) if
    given, in the same pass.  The mask is never stored: it is a function of (seed, position in x read row by row), the same one in the
    backward pass, and the one the training step of ``HorizonNet`` draws from its own seeds.  seed: an int in ``0 .. 2**64 - 1``, or an int64
    tensor with one element on x's device, which the kernel reads: a captured step that changes it draws a new mask on every replay (it must
    not be changed between a forward pass and its backward pass; autograd refuses that).  A dropped element is 0 whatever x holds there."""
    return (_native or _load()).dropout(x, p, seed, residual)
