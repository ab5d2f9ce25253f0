"""Operators along a sequence: a short causal convolution, the selective state space scan, and the
norm of heads with the rotation by position. Each is one operation of the engine with kernels of
its own, forward and backward (first derivatives; differentiating a gradient again is refused with
GRAD_UNSUPPORTED). They take prompts and single tokens alike: what a sequence leaves behind is
returned as a state, and a call on the next tokens takes it. The reference has no counterpart.

Values are float32 or float64, one dtype a call; lengths and positions are int32.
"""

from ._native import _rg  # noqa: F401  (the engine has to be there before an operator is traced)
from .ops import _as_index, arange
from .tensor import TRACES, Tracer, caller_source, error, first_dtype, lift

# The operand and variant flags of include/rg_plan.h.
_CONV_BIAS, _CONV_STATE, _CONV_LENGTHS, _CONV_SILU = 1, 2, 4, 8
_SCAN_SKIP, _SCAN_GATE, _SCAN_STATE, _SCAN_LENGTHS, _SCAN_SOFTPLUS, _SCAN_JOINED, _SCAN_BIAS, _SCAN_LOG = 1, 2, 4, 8, 16, 64, 128, 256
_ROTARY_GAIN = 1


def _traced(name, operands, attrs):
    """The node of operator `name` over `operands` in the innermost trace, its graph and source."""
    g, where = TRACES.graph, caller_source()
    dtype = first_dtype(operands)
    return g, where, g.op(name, [lift(g, v, dtype) for v in operands], attrs, where)


def _eagerly(fn, operands):
    from .program import compile
    return compile(fn, tuple(operands), validate="none")(*operands)


def _present(required, optional, flags):
    """The operands given, in order, and the flags that say which optional ones are among them."""
    values, mask = list(required), 0
    for value, flag in zip(optional, flags):
        if value is not None:
            values.append(value)
            mask |= flag
    return values, mask


def _with_results(name, operands, attrs, count):
    """The first `count` results of an operator, traced or computed at once."""
    if not TRACES.active:
        return _eagerly(lambda *v: _with_results(name, v, attrs, count), operands)
    g, where, node = _traced(name, operands, attrs)
    return tuple(Tracer(g, g.result(node, k, where)) for k in range(count))


def causal_conv(x, w, bias=None, state=None, lengths=None, activation=None):
    """A depthwise causal convolution along a sequence: `x` (batch, length, width) and `w` (taps,
    width), two to eight taps, give `(y, new state)` with

        y[:, t] = act(bias + sum_k w[k] * past[:, t + k]),   past = state, then x.

    `state` (batch, taps - 1, width) holds the inputs before `x` (zeros without it), and the new
    state those that end the sequence, for the call on what follows. `activation` is None or
    "silu". With `lengths` (batch,), a padded batch: y is 0 from lengths[b] on, what x holds there
    is not read, and the new state ends at lengths[b]."""
    if activation not in (None, "silu"):
        raise error("INVALID_ARGUMENT", {"activation": repr(activation)}, "activation_must_be_none_or_silu")
    if lengths is not None:
        lengths = _as_index(lengths)
    operands, flags = _present((x, w), (bias, state, lengths), (_CONV_BIAS, _CONV_STATE, _CONV_LENGTHS))
    return _with_results("causal_conv", operands, {"flags": flags | (_CONV_SILU if activation else 0)}, 2)


def selective_scan(x, dt, a, b, c=None, d=None, z=None, state=None, lengths=None, softplus=False, dt_bias=None, log_rates=False):
    """The selective state space scan: every channel of `x` (batch, length, width) drives `states`
    linear recurrences whose step `dt` (as `x`) and maps `b`, `c` change from position to position,

        h[t] = exp(dt[t] a) h[t-1] + dt[t] x[t] b[t],   y[t] = (sum_n c[t] h[t] + d x[t]) silu(z[t]).

    `a` is (width, states), at most 64 of them; `b` and `c` are (batch, length, groups, states),
    each group serving width / groups neighbouring channels, or (batch, length, states) for one;
    without `c`, `b` holds both, (batch, length, 2 * groups, states), as one projection makes them.
    `d` (width,) and the gate `z` (as `x`) may be left out. `state` (batch, width, states) is h
    before the first position (zeros without it). `dt_bias` (width,) is added to `dt`, and with
    `softplus` the sum taken through log(1 + e^dt) first. With `log_rates`, `a` holds the logarithms
    of the rates at which states decay: -e^a takes its place. Returns `(y, final state)`. With `lengths` (batch,), a padded batch: y is 0
    from lengths[b] on, nothing is read there, and the final state is that at lengths[b]."""
    if lengths is not None:
        lengths = _as_index(lengths)
    if c is not None and b.ndim == 3 and c.ndim == 3:
        b, c = (v.reshape(v.shape[0], v.shape[1], 1, v.shape[2]) for v in (b, c))
    maps, joined = ((b,), _SCAN_JOINED) if c is None else ((b, c), 0)
    operands, flags = _present((x, dt, a, *maps), (d, z, state, lengths, dt_bias),
                               (_SCAN_SKIP, _SCAN_GATE, _SCAN_STATE, _SCAN_LENGTHS, _SCAN_BIAS))
    flags |= joined | (_SCAN_SOFTPLUS if softplus else 0) | (_SCAN_LOG if log_rates else 0)
    return _with_results("selective_scan", operands, {"flags": flags}, 2)


def rotary_norm(x, gain=None, positions=None, sections=None, rotary_dims=None, base=10000.0, eps=1e-6):
    """The norm of each head and its rotation by position in one pass over `x` (batch, length,
    heads, head). `sections` counts the heads of each section, in order (one of all heads without
    it); the heads of section s are divided by their root mean square (over the head, `eps` added
    to the mean square: 0 or a number that the dtype holds) and multiplied by `gain[s]`, and heads
    past the sections pass unchanged: queries, keys and values of a fused projection are sections
    (heads, heads) of 3 * heads. Without `gain` heads are only rotated. The first `rotary_dims`
    values of a head (all of them by default, 0 for none) are turned in pairs (i, i + rotary_dims /
    2) by the angle position * base^(-2 i / rotary_dims), formed in 64 bits. `positions` is int32:
    (length,), (batch, length), or (batch, 1) for the first of each sequence, the others following
    it; 0, 1, ... without it."""
    if x.ndim != 4:
        raise error("SHAPE_MISMATCH", {"input_shapes": [x.shape]}, "x_must_be_batch_length_heads_head")
    if gain is not None and gain.ndim == 1:
        gain = gain.reshape(1, gain.shape[0])
    counts = [x.shape[2]] if sections is None else [int(n) for n in sections]
    turn = x.shape[3] if rotary_dims is None else int(rotary_dims)
    if turn < 0 or any(n < 1 for n in counts):
        raise error("INVALID_ARGUMENT", {"sections": counts, "rotary_dims": turn}, "sections_and_rotary_dims_must_not_be_negative")
    positions = arange(x.shape[1]) if positions is None else _as_index(positions)
    operands, flags = _present((x, positions), (gain,), (_ROTARY_GAIN,))
    attrs = {"flags": flags, "sections": counts, "rotary_dims": turn, "base": float(base), "eps": float(eps)}

    def call(*values):
        g, _where, node = _traced("rotary_norm", values, attrs)
        return Tracer(g, node)

    return call(*operands) if TRACES.active else _eagerly(call, operands)
