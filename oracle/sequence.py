"""CPU oracle of the sequence model operators: the formulas in 64 bits, one rounding at the end.

Every function takes the operands of its DAG node in order (a plain number in the place of an operand
that was left out, and for literals) and returns the list of results.
"""
import numpy as np


def _given(v):
    return isinstance(v, np.ndarray)


def _wide(v):
    return v.astype(np.float64)


def _acc(dtype):
    return np.float64 if dtype == np.float64 else np.float32


def silu(v):
    with np.errstate(over="ignore"):
        return v / (1.0 + np.exp(-v))


def rms_norm(x, weight, residual, eps, group, to=None):
    h = _wide(x) + (_wide(residual) if _given(residual) else 0.0)
    w = _wide(weight) if _given(weight) else np.ones(x.shape[-1])
    with np.errstate(all="ignore"):
        r = 1.0 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
        if not group:
            results = [(h * r * w).astype(x.dtype)]
        else:
            # the products of the codes are single rounded operations of the accumulator's type
            acc, n, g = _acc(x.dtype), x.shape[-1], int(group)
            ha = x.astype(acc) + (residual.astype(acc) if _given(residual) else acc(0))
            v = ha * weight.astype(acc) if _given(weight) else ha
            codes, scales = np.zeros(x.shape, np.int8), []
            for i in range(0, n, g):
                part = v[..., i:i + g]
                most = np.abs(part).max(-1, keepdims=True)
                fine = np.isfinite(most)
                factor = (acc(1) / most * acc(127)).astype(acc)
                factor = np.where(fine & (most > 0) & np.isfinite(factor), factor, acc(0))
                codes[..., i:i + g] = np.where(factor > 0, np.rint(part * factor), 0).astype(np.int8)
                scales.append(np.where(fine, np.where(factor > 0, _wide(most) * r / 127.0, 0.0), np.nan))
            results = [codes, np.concatenate(scales, -1).astype(acc)]
    return results + ([h.astype(x.dtype)] if _given(residual) else [])


def _ends(lengths, b, t):
    return np.clip(lengths, 0, t) if _given(lengths) else np.full(b, t)


def causal_conv(x, weight, bias, state, lengths, activation, to=None):
    b, t, d = x.shape
    k = weight.shape[1]
    old = state if _given(state) else np.zeros((b, k - 1, d), x.dtype)
    y, new = np.zeros(x.shape, np.float64), np.empty_like(old)
    for i, end in enumerate(_ends(lengths, b, t)):
        row = np.concatenate([old[i], x[i, :end]])
        s = np.zeros((end, d)) + (_wide(bias) if _given(bias) else 0.0)
        for j in range(k):
            s = s + _wide(weight[:, j]) * _wide(row[j:j + end])
        y[i, :end] = silu(s) if activation else s
        new[i] = row[end:]
    return [y.astype(x.dtype), new]


def scan_step_sizes(delta, delta_bias, softplus):
    dt = _wide(delta) + (_wide(delta_bias) if _given(delta_bias) else 0.0)
    return np.logaddexp(0.0, dt) if softplus else dt


def selective_scan(x, delta, A, B, C, D, z, delta_bias, state, lengths, softplus, to=None):
    b, t, d = x.shape
    n = A.shape[1]
    dt = scan_step_sizes(delta, delta_bias, softplus)
    h = _wide(state) if _given(state) else np.zeros((b, d, n))
    groups = B.shape[2] // n
    per = lambda v, i: np.repeat(_wide(v[:, i]).reshape(b, groups, n), d // groups, axis=1)  # noqa: E731
    y = np.zeros(x.shape, np.float64)
    ends = _ends(lengths, b, t)
    for i in range(t):
        on = i < ends
        xi = _wide(x[:, i])
        new = np.exp(dt[:, i, :, None] * _wide(A)) * h + (dt[:, i] * xi)[:, :, None] * per(B, i)
        out = (per(C, i) * new).sum(2) + (_wide(D) * xi if _given(D) else 0.0)
        if _given(z):
            out = out * silu(_wide(z[:, i]))
        h = np.where(on[:, None, None], new, h)
        y[:, i] = np.where(on[:, None], out, 0.0)
    return [y.astype(x.dtype), h.astype(A.dtype)]


def sample_row(x, u, temperature, top_k, top_p, min_p):
    """(token, log probability) of one row of logits in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x)
    most = x.max()
    if most == -np.inf:
        return -1, -np.inf
    if not temperature > 0:
        return int(x.argmax()), 0.0
    with np.errstate(invalid="ignore"):
        z = np.where(x == most, 0.0, np.where((x == -np.inf) | (most == np.inf), -np.inf, (x * 0.5 - most * 0.5) / temperature * 2.0))  # halves: no overflow
    e = np.exp(z)
    keep = np.argsort(-x, kind="stable")
    if 1 <= top_k < len(x):
        keep = keep[:int(top_k)]
    if top_p < 1:
        sums = np.cumsum(e[keep])
        keep = keep[np.concatenate([[True], sums[:-1] < top_p * sums[-1]])]
    keep = np.sort(keep[e[keep] >= min_p])
    sums = np.cumsum(e[keep])
    at = min(int(np.searchsorted(sums, max(u, 0.0) * sums[-1], side="right")), np.flatnonzero(e[keep])[-1])
    return int(keep[at]), z[keep[at]] - np.log(sums[-1])


def sample(logits, u, temperature, top_k, top_p, min_p, to=None):
    rows = _wide(np.atleast_2d(logits))
    each = [np.broadcast_to(np.asarray(v, np.float64), (len(rows),)) for v in (u, temperature, top_k, top_p, min_p)]
    drawn = [sample_row(row, *(float(v[i]) for v in each)) for i, row in enumerate(rows)]
    return [np.array([t for t, _ in drawn], np.int32), np.array([p for _, p in drawn]).astype(_acc(logits.dtype))]


def convert(x, scale, group, to):
    with np.errstate(all="ignore"):
        if _given(scale):
            factor = np.repeat(_wide(scale), int(group), -1)[..., :x.shape[-1]]
            return [(_wide(x) * factor).astype(to)]
        return [x.astype(to)]


OPERATORS = {15: rms_norm, 16: causal_conv, 17: selective_scan, 18: sample, 19: convert}
