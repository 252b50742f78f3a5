"""Operators of sequence models on lazy arrays: root-mean-square norm, short causal convolution,
selective state space scan and sampling -- what stands between the projections (``matvec``) of a
recurrent model's forward pass.

Activations are float16, float32 or float64.  Sums, statistics and states are float32 (float64 for
float64 activations), and every result is rounded once.  Operands are whole arrays; views are copied
first, as for ``matvec``, and host data is converted to the type an operand needs.  On several GPUs
every rank works on the rows (sequences) that it owns.
"""
import numbers

import numpy as np

from . import wire
from .frontend import _ArrayOps, _Op, _is_scalar_like, _new_array, _normalize_dtype, _record, _whole, asarray

_ACTIVATIONS = (np.dtype("float16"), np.dtype("float32"), np.dtype("float64"))
_F32, _F64, _I32, _I8 = (np.dtype(t) for t in ("float32", "float64", "int32", "int8"))
MAX_CONV_WIDTH = 8
MAX_SCAN_STATES = 256
MAX_VOCABULARY = 1 << 24


def _activations(x, what, dims):
    x = _whole(asarray(x))
    if x.dtype not in _ACTIVATIONS:
        raise TypeError(f"{what} must be float16, float32 or float64, got {x.dtype}")
    if x.ndims not in dims:
        raise ValueError(f"{what} must have {' or '.join(str(d) for d in dims)} dimensions, got {x.ndims}")
    return x


def _acc(x):
    return _F64 if x.dtype == _F64 else _F32


def _operand(v, what, dtypes, shape):
    """An operand of a required type and shape, or None; host data is converted to the first type."""
    if v is None:
        return None
    if not isinstance(v, _ArrayOps):
        host = np.asarray(v)
        if host.dtype not in dtypes:
            with np.errstate(invalid="ignore"):
                v = host.astype(dtypes[0])
            if dtypes[0].kind == "i" and not np.array_equal(v, host):
                raise ValueError(f"{what} must be whole numbers that {dtypes[0]} holds")
            host = v
        v = asarray(host)
    if v.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(d.name for d in dtypes)}, got {v.dtype}")
    if shape is not None and tuple(v.shape) != tuple(shape):
        raise ValueError(f"{what} must have shape {tuple(shape)}, got {tuple(v.shape)}")
    return _whole(v)


def _apply(opcode, operands, results):
    infos = [r._info for r in results]
    _record(_Op("seq", opcode, infos[0], [o._operand() if isinstance(o, _ArrayOps) else o for o in operands], payload=infos))


def rms_norm(x, weight=None, *, residual=None, eps=1e-6, bits=None, group=None):
    """Root-mean-square norm over the last dimension: ``h / sqrt(mean(h^2) + eps) * weight`` with
    ``h = x + residual``.

    Returns ``y``, or ``(y, h)`` with a residual.  With ``bits=8`` the result is held as int8 codes and
    one scale for every ``group`` columns (default: the whole row): ``(codes, scale)``, or
    ``(codes, scale, h)``; ``dequantize`` gives the values.  With ``v = h * weight`` and a group's largest
    ``|v|``, a, codes are ``rint(v * (1 / a * 127))``, whatever the row's norm.  A group that is all zero (or
    so small that 1 / a overflows) has codes and scale 0, one with an infinity or a NaN codes 0 and
    scale NaN.  Squares are summed in float32 (float64 for float64): float32 rows with values beyond 1.8e19 are 0.
    """
    x = _activations(x, "x", (1, 2, 3))
    n = x.shape[-1]
    if n < 1:
        raise ValueError("rms_norm needs at least one column")
    weight = _operand(weight, "weight", (x.dtype,), (n,))
    residual = _operand(residual, "residual", (x.dtype,), x.shape)
    if not float(eps) >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if bits not in (None, 8):
        raise ValueError(f"bits must be None or 8, got {bits}")
    if group is not None:
        if bits is None:
            raise ValueError("group is for the 8-bit output: give bits=8 too")
        if not isinstance(group, numbers.Integral) or not 1 <= group <= n:
            raise ValueError(f"group must be 1 to {n} columns, got {group}")
    group = 0 if bits is None else n if group is None else int(group)
    results = [_new_array(x.shape, _I8 if bits else x.dtype)]
    if bits:
        results.append(_new_array(tuple(x.shape[:-1]) + (-(-n // group),), _acc(x)))
        results[1]._info.set_group(group)  # so that dequantize need not be told
    if residual is not None:
        results.append(_new_array(x.shape, x.dtype))
    _apply(wire.OP_RMS_NORM, [x, weight, residual, float(eps), group], results)
    return results[0] if len(results) == 1 else tuple(results)


def dequantize(codes, scale, *, group=None, dtype=None):
    """The values that int8 codes stand for, ``code * scale`` with one scale for every ``group`` columns
    of the last dimension, in ``dtype`` (default: that of the scales).  ``group`` may be left out for scales
    that ``rms_norm`` returned, their copies, conversions, rows and what is computed from them value by value.
    Scales from elsewhere are taken to have as many columns each as divide evenly: give the group of others (30 of
    100 columns make four scales, as 25 do)."""
    codes = _operand(codes, "codes", (_I8,), None)
    scale = _operand(scale, "scale", (_F32, _F64), None)
    dtype = scale.dtype if dtype is None else _normalize_dtype(dtype)
    if dtype not in _ACTIVATIONS:
        raise TypeError(f"dequantize makes float16, float32 or float64 values, not {dtype}")
    n = codes.shape[-1]
    if scale.ndims != codes.ndims or tuple(scale.shape[:-1]) != tuple(codes.shape[:-1]):
        raise ValueError(f"scales of shape {tuple(scale.shape)} do not go with codes of shape {tuple(codes.shape)}")
    groups = scale.shape[-1]
    if group is None:
        group = scale._info.group
        if group == 0 and groups > 1:
            raise ValueError("give the group: the scales were assigned to, from others that may have another one")
        if not group:
            if not groups or n % groups:
                raise ValueError(f"give the group: {n} columns do not divide evenly among {groups} scales")
            group = n // groups
    if not isinstance(group, numbers.Integral) or group < 1 or -(-n // group) != groups:
        raise ValueError(f"{groups} scales do not belong to {n} columns in groups of {group}")
    out = _new_array(codes.shape, dtype)
    _apply(wire.OP_CONVERT, [codes, scale, min(int(group), max(n, 1))], [out])
    return out


def _sequences(x, lengths):
    return _operand(lengths, "lengths", (_I32,), (x.shape[0],))


def _state_result(given, state, inplace, others, shape, dtype):
    if not inplace:
        return _new_array(shape, dtype)
    if state is None or state is not given:
        raise ValueError("inplace needs the state as a whole array")
    if any(o is not None and o._info is state._info for o in others):
        raise ValueError("a state that is updated in place cannot be another operand too")
    return state


def causal_conv(x, weight, bias=None, *, state=None, lengths=None, activation=None, inplace=False):
    """Convolution along time, one filter of width k = 2 to 8 per channel, that looks back only:
    ``y[b, t, c] = bias[c] + sum_j weight[c, j] * X[b, t - k + 1 + j, c]``, through ``x * sigmoid(x)`` with
    ``activation="silu"``.

    ``x`` is (sequences, time, channels), ``weight`` (channels, k), ``bias`` (channels).  ``state``,
    (sequences, k - 1, channels), holds the inputs before the first (default: zeros).  ``lengths`` (int32,
    one per sequence, clipped to the time) ends sequences early: behind its end ``y`` is 0.  Returns
    ``(y, state)`` with the state after each sequence's last input; a prompt and a single token are the
    same call.  With ``inplace`` the given state array is brought up to date itself.
    """
    x = _activations(x, "x", (3,))
    b, _, d = x.shape
    weight = _operand(weight, "weight", (x.dtype,), None)
    if weight.ndims != 2 or weight.shape[0] != d:
        raise ValueError(f"weight must be ({d}, width), got {tuple(weight.shape)}")
    k = weight.shape[1]
    if not 2 <= k <= MAX_CONV_WIDTH:
        raise NotImplementedError(f"causal_conv has widths of 2 to {MAX_CONV_WIDTH}, got {k}")
    bias = _operand(bias, "bias", (x.dtype,), (d,))
    given = state
    state = _operand(state, "state", (x.dtype,), (b, k - 1, d))
    lengths = _sequences(x, lengths)
    if activation not in (None, "silu"):
        raise ValueError(f'activation must be None or "silu", got {activation!r}')
    after = _state_result(given, state, inplace, (x, weight, bias, lengths), (b, k - 1, d), x.dtype)
    y = _new_array(x.shape, x.dtype)
    _apply(wire.OP_CAUSAL_CONV, [x, weight, bias, state, lengths, 1 if activation else 0], [y, after])
    return y, after


def selective_scan(x, delta, A, B, C, *, D=None, z=None, delta_bias=None, softplus=True, state=None, lengths=None, inplace=False):
    """Selective state space scan.  With ``dt = softplus(delta + delta_bias)`` (or the sum itself),

        h[b, c, n] <- exp(dt A[c, n]) h[b, c, n] + dt B[b, t, n] x[b, t, c]
        y[b, t, c]  = (sum_n C[b, t, n] h[b, c, n] + D[c] x[b, t, c]) * z * sigmoid(z)

    ``x``, ``delta`` and ``z`` are (sequences, time, channels), ``A`` (channels, n) with up to 256 states,
    ``B`` and ``C`` (sequences, time, groups * n): the channels are divided evenly among the groups, in
    order.  ``A``, ``D``, ``delta_bias`` and ``state`` (sequences, channels, n) are float32 (float64 for
    float64 activations); the state's default is zeros.  ``lengths`` (int32) ends sequences early:
    behind its end ``y`` is 0 and the state stays.  Returns ``(y, state)``; a prompt and a single token are
    the same call.  With ``inplace`` the given state array is brought up to date itself.
    """
    x = _activations(x, "x", (3,))
    b, t, d = x.shape
    acc = _acc(x)
    delta = _operand(delta, "delta", (x.dtype,), x.shape)
    A = _operand(A, "A", (acc,), None)
    if A.ndims != 2 or A.shape[0] != d:
        raise ValueError(f"A must be ({d}, states), got {tuple(A.shape)}")
    n = A.shape[1]
    if not 1 <= n <= MAX_SCAN_STATES:
        raise NotImplementedError(f"selective_scan has 1 to {MAX_SCAN_STATES} states per channel, got {n}")
    B = _operand(B, "B", (x.dtype,), None)
    if B.ndims != 3 or tuple(B.shape[:2]) != (b, t) or B.shape[2] < n or B.shape[2] % n:
        raise ValueError(f"B must be ({b}, {t}, groups * {n}), got {tuple(B.shape)}")
    if d % (B.shape[2] // n):
        raise ValueError(f"{d} channels do not divide into {B.shape[2] // n} groups")
    C = _operand(C, "C", (x.dtype,), B.shape)
    D = _operand(D, "D", (acc,), (d,))
    z = _operand(z, "z", (x.dtype,), x.shape)
    delta_bias = _operand(delta_bias, "delta_bias", (acc,), (d,))
    given = state
    state = _operand(state, "state", (acc,), (b, d, n))
    lengths = _sequences(x, lengths)
    after = _state_result(given, state, inplace, (x, delta, A, B, C, D, z, delta_bias, lengths), (b, d, n), acc)
    y = _new_array(x.shape, x.dtype)
    _apply(wire.OP_SELECTIVE_SCAN, [x, delta, A, B, C, D, z, delta_bias, state, lengths, 1 if softplus else 0], [y, after])
    return y, after


def sample(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token for each row of ``logits`` (rows, vocabulary), or of one row (vocabulary), from given
    random numbers ``u`` in [0, 1) (rows), float32 or float64.

    With ``e = exp((logits - max) / temperature)`` the filters apply one after the other: ``top_k`` keeps the
    largest logits (0: all of them; ties: the lowest index), ``top_p`` the shortest prefix of these in
    descending order whose share of the sum of e reaches it (1: all), ``min_p`` those with e of at least it.
    The token is the first in index order whose running sum of kept e exceeds ``u`` times their total.
    A temperature of 0 takes the largest logit.  NaN counts as -infinity; a row with nothing above
    -infinity has the token -1.  Each parameter is a number, or an array with one for every row.

    Returns ``(token, logp)``: int32, and the token's log probability among the kept ones.
    """
    logits = _activations(logits, "logits", (1, 2))
    v = logits.shape[-1]
    if not 1 <= v <= MAX_VOCABULARY:
        raise ValueError(f"sample takes vocabularies of 1 to {MAX_VOCABULARY}, got {v}")
    rows = logits.shape[0] if logits.ndims == 2 else 1
    u = _operand(np.atleast_1d(u) if _is_scalar_like(u) else u, "u", (_F32, _F64), (rows,))

    def parameter(value, what, low, high, integer=False):
        if not _is_scalar_like(value):
            return _operand(value, what, (_I32,) if integer else (_F32, _F64), (rows,))
        value = value.item() if isinstance(value, (np.ndarray, np.generic)) else value
        if integer and value != int(value):
            raise ValueError(f"{what} must be a whole number, got {value}")
        if not low <= value <= high:
            raise ValueError(f"{what} must be {low} to {high}, got {value}")
        return float(value)

    parameters = [parameter(temperature, "temperature", 0, float("inf")), parameter(top_k, "top_k", 0, 2 ** 31 - 1, integer=True),
                  parameter(top_p, "top_p", 0, 1), parameter(min_p, "min_p", 0, 1)]
    token, logp = _new_array((rows,), _I32), _new_array((rows,), _acc(logits))
    _apply(wire.OP_SAMPLE, [logits, u] + parameters, [token, logp])
    return token, logp
