"""GPU tests of the sequence model operators against the CPU oracle, which runs the formulas in 64 bits
on the same DAG.

Tolerances.  u is half a step of the accumulator's type (2^-24, or 2^-53), e half a step of the output's
(f16 2^-11, f32 2^-24, f64 2^-53; below 2^-14 f16 steps are 2^-24 apart: 2^-25 absolute).  Every bound is
a count of roundings: library functions are allowed 4u (exp and log1p are specified within 2 ulp, the
fast 2^x within 2 ulp and its argument's rounding).
"""
import numpy as np
import pytest

import charmnumeric_b200 as cnp
from oracle import sequence as S
from tests.helpers import run_both

pytestmark = pytest.mark.gpu

TYPES = ["float16", "float32", "float64"]
HALF_STEP = {"float16": 2.0 ** -11, "float32": 2.0 ** -24, "float64": 2.0 ** -53}


def unit(dtype):
    return 2.0 ** -53 if dtype == "float64" else 2.0 ** -24


def acc(dtype):
    return "float64" if dtype == "float64" else "float32"


def check(got, want, bound, dtype, what=""):
    """|got - want| <= bound + both sides' rounding to the output type."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    np.testing.assert_array_equal(got[~fine], want[~fine], err_msg=what)
    allowed = np.broadcast_to(bound, want.shape) + 2 * (HALF_STEP[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "float16" else 1e-300))
    off = np.where(fine, np.abs(got - want), 0.0)
    assert (off <= allowed)[fine].all(), (what, float((off / allowed)[fine].max()), int((off > allowed).sum()))


def bits(gpu, cpu):
    assert gpu.dtype == cpu.dtype and gpu.shape == cpu.shape
    np.testing.assert_array_equal(gpu.view(np.uint8), cpu.view(np.uint8))


# ---- rms_norm ---------------------------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (3, 2), (5, 31), (4, 64), (7, 127), (2, 128), (9, 1000), (2, 3, 513), (1, 2048), (300, 96),
               (3, 5003), (2, 8192), (2, 16385), (1, 70001), (1025,), (1, 300000)]


def norm_bound(n, eps_, h, y, dtype):
    # a sum of n squares, at most n / 32 of them one after the other and 32 partial sums in trees,
    # halved by the root; the mean, eps, the root, its reciprocal, two products; h's own rounding
    u = unit(dtype)
    return ((n / 32 + 24) / 2 + 10) * u * np.abs(y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_rms_norm(interface, shape, dtype):
    rng = np.random.default_rng(sum(shape))
    x, r = (rng.standard_normal(shape).astype(dtype) for _ in range(2))
    w = (1 + 0.2 * rng.standard_normal(shape[-1])).astype(dtype)
    def program():
        y, h = cnp.rms_norm(cnp.asarray(x), cnp.asarray(w), residual=cnp.asarray(r), eps=1e-5)
        plain = cnp.rms_norm(cnp.asarray(x))
        return {"y": y, "h": h, "plain": plain}
    gpu, cpu = run_both(interface, program)
    hs = x.astype(np.float64) + r.astype(np.float64)
    check(gpu["h"], cpu["h"], unit(dtype) * np.abs(hs), dtype)
    exact = hs / np.sqrt((hs * hs).mean(-1, keepdims=True) + 1e-5) * w.astype(np.float64)
    # f16: both sides round an exact 11-bit product once, from sums that differ by the bound
    check(gpu["y"], exact, norm_bound(shape[-1], 1e-5, hs, exact, dtype), dtype)
    xs = x.astype(np.float64)
    exact = xs / np.sqrt((xs * xs).mean(-1, keepdims=True) + 1e-6)
    check(gpu["plain"], exact, norm_bound(shape[-1], 1e-6, xs, exact, dtype), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,group", [((1, 1), 1), ((5, 31), None), ((7, 127), 32), ((9, 1000), 128), ((2, 3, 513), 100),
                                         ((2, 4096), 128), ((2, 4096), 64), ((3, 5003), 128), ((2, 8192), None), ((2, 16385), 4096),
                                         ((1025,), 16), ((4, 2048), 32), ((1, 70001), 70000)], ids=str)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_8_bits(interface, shape, group, residual, dtype):
    rng = np.random.default_rng(sum(shape) + 1)
    x, r = (rng.standard_normal(shape).astype(dtype) for _ in range(2))
    w = (1 + 0.2 * rng.standard_normal(shape[-1])).astype(dtype)
    def program():
        q, s, *h = cnp.rms_norm(cnp.asarray(x), cnp.asarray(w), residual=cnp.asarray(r) if residual else None, bits=8, group=group)
        out = {"q": q, "s": s, "v": cnp.dequantize(q, s), "v16": cnp.dequantize(q, s, dtype="float16")}
        return dict(out, h=h[0]) if residual else out
    gpu, cpu = run_both(interface, program)
    bits(gpu["q"], cpu["q"])          # the codes do not depend on the order of any sum
    n = shape[-1]
    check(gpu["s"], cpu["s"], ((n / 32 + 24) / 2 + 12) * unit(dtype) * np.abs(cpu["s"]), acc(dtype))
    scale = np.repeat(gpu["s"].astype(np.float64), group or n, -1)[..., :n]
    check(gpu["v"], gpu["q"] * scale, 0.0, acc(dtype))
    check(gpu["v16"], gpu["q"] * scale, 2.0 ** -24 * np.abs(gpu["q"] * scale), "float16")
    if residual:
        check(gpu["h"], cpu["h"], unit(dtype) * np.abs(x.astype(np.float64) + r.astype(np.float64)), dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_rms_norm_rows_of_zeros_infinities_and_nan(interface, dtype):
    x = np.ones((6, 200), dtype)
    x[0] = 0
    x[1, 7] = np.inf
    x[2, 190] = np.nan
    x[3, :64] = 0
    x[4, 3] = -np.inf
    def program():
        a = cnp.asarray(x)
        q, s = cnp.rms_norm(a, bits=8, group=64, eps=0.0)
        return {"y": cnp.rms_norm(a, eps=1e-6), "y0": cnp.rms_norm(a, eps=0.0), "q": q, "s": s, "v": cnp.dequantize(q, s)}
    gpu, cpu = run_both(interface, program)
    for name in ("y", "y0"):
        np.testing.assert_array_equal(np.isnan(gpu[name]), np.isnan(cpu[name]))
        fine = np.isfinite(cpu[name])
        np.testing.assert_allclose(gpu[name][fine], cpu[name][fine], rtol=30 * HALF_STEP[dtype])
    bits(gpu["q"], cpu["q"])
    fine = ~np.isnan(cpu["s"])
    # row 0 has r = 1 / sqrt(0): its scale is 0 * inf
    np.testing.assert_array_equal(np.isnan(gpu["s"]), ~fine)
    np.testing.assert_allclose(gpu["s"][fine], cpu["s"][fine], rtol=30 * unit(dtype))


def test_rms_norm_large_and_tiny_values(interface):
    """f16 rows whose squares lie beyond f16's range, and f16 subnormals."""
    x = np.stack([np.full(500, 60000.0), np.full(500, 6e-8), np.full(500, 3e-5)]).astype("float16")
    gpu, cpu = run_both(interface, lambda: {"y": cnp.rms_norm(cnp.asarray(x), eps=0.0)})
    np.testing.assert_allclose(gpu["y"].astype(float), 1.0, rtol=2.0 ** -10)


# ---- causal_conv --------------------------------------------------------------------------------------------

def conv_bound(x, w, bias, state, dtype, silu):
    k = w.shape[1]
    mag = S.causal_conv(np.abs(x).astype(float), np.abs(w).astype(float), np.abs(bias).astype(float),
                        np.abs(state).astype(float), None, 0)[0]
    # k products and sums; the logistic's exp, sum and quotient.  |silu'| <= 1.1
    return unit(dtype) * mag * ((k + 2) * 1.1 + (10 if silu else 0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,d,k", [(1, 1, 1, 2), (2, 1, 5, 3), (3, 1, 256, 4), (1, 2, 33, 4), (2, 7, 64, 8), (3, 65, 130, 4),
                                     (1, 1000, 96, 4), (2, 300, 1025, 2), (4, 33, 2048, 4), (1, 129, 24, 5), (130, 1, 40, 4),
                                     (70000, 1, 2, 2), (2, 5000, 8, 6)])
def test_causal_conv(interface, b, t, d, k, dtype):
    rng = np.random.default_rng(b + t + d + k)
    x, state = rng.standard_normal((b, t, d)).astype(dtype), rng.standard_normal((b, k - 1, d)).astype(dtype)
    w, bias = (rng.standard_normal((d, k)) * 0.5).astype(dtype), rng.standard_normal(d).astype(dtype)
    lengths = rng.integers(-1, t + 3, b).astype(np.int32)
    def program():
        ax, aw, ab, ast = (cnp.asarray(v) for v in (x, w, bias, state))
        y1, s1 = cnp.causal_conv(ax, aw, ab, state=ast, activation="silu")
        y2, s2 = cnp.causal_conv(ax, aw, lengths=lengths)
        y3, s3 = cnp.causal_conv(ax, aw, ab, state=ast, lengths=lengths, activation="silu")
        inner = cnp.array(ast)
        y4, s4 = cnp.causal_conv(ax, aw, ab, state=inner, lengths=lengths, inplace=True)
        assert s4 is inner
        return {"y1": y1, "s1": s1, "y2": y2, "s2": s2, "y3": y3, "s3": s3, "y4": y4, "s4": s4}
    gpu, cpu = run_both(interface, program)
    zero = np.zeros_like(state)
    for i, (bb, st, ln, act) in {1: (bias, state, None, 1), 2: (np.zeros(d), zero, lengths, 0), 3: (bias, state, lengths, 1),
                                 4: (bias, state, lengths, 0)}.items():
        exact = S.causal_conv(x.astype(float), w.astype(float), bb.astype(float), st.astype(float), ln, act)[0]
        check(gpu[f"y{i}"], exact, conv_bound(x, w, bb, st, dtype, act), dtype, f"y{i}")
        bits(gpu[f"s{i}"], cpu[f"s{i}"])


@pytest.mark.parametrize("dtype", TYPES)
def test_causal_conv_token_by_token_is_the_prompt(interface, dtype):
    """A prompt cut into pieces of any length gives the same bits: every output is the same sum."""
    rng = np.random.default_rng(5)
    x, w = rng.standard_normal((2, 11, 70)).astype(dtype), rng.standard_normal((70, 4)).astype(dtype)
    cuts = [0, 1, 2, 5, 6, 11]
    def program():
        whole, last = cnp.causal_conv(cnp.asarray(x), cnp.asarray(w), activation="silu")
        state, out = None, {"whole": whole, "last": last}
        for i, (a, b) in enumerate(zip(cuts, cuts[1:])):
            out[f"y{i}"], state = cnp.causal_conv(cnp.asarray(np.ascontiguousarray(x[:, a:b])), cnp.asarray(w), state=state, activation="silu")
        return dict(out, state=state)
    gpu, _ = run_both(interface, program)
    bits(np.concatenate([gpu[f"y{i}"] for i in range(len(cuts) - 1)], 1), gpu["whole"])
    bits(gpu["state"], gpu["last"])


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_causal_conv_reads_nothing_behind_the_end(interface, dtype):
    x = np.ones((3, 40, 64), dtype)
    lengths = np.array([0, 13, 39], np.int32)
    for i, n in enumerate(lengths):
        x[i, n:] = np.nan
    w = np.ones((64, 4), dtype)
    gpu, cpu = run_both(interface, lambda: dict(zip("ys", cnp.causal_conv(cnp.asarray(x), cnp.asarray(w), lengths=lengths))))
    bits(gpu["y"], cpu["y"])
    bits(gpu["s"], cpu["s"])


# ---- selective_scan --------------------------------------------------------------------------------------------

def scan_inputs(rng, b, t, d, n, dtype, groups=1):
    f = acc(dtype)
    step = np.exp(rng.uniform(np.log(1e-3), np.log(0.1), d))
    return {"x": rng.standard_normal((b, t, d)).astype(dtype), "delta": (0.5 * rng.standard_normal((b, t, d))).astype(dtype),
            "A": (-np.arange(1, n + 1) * np.exp(0.1 * rng.standard_normal((d, n)))).astype(f),
            "B": rng.standard_normal((b, t, groups * n)).astype(dtype), "C": rng.standard_normal((b, t, groups * n)).astype(dtype),
            "D": (1 + 0.1 * rng.standard_normal(d)).astype(f), "z": rng.standard_normal((b, t, d)).astype(dtype),
            "delta_bias": np.log(np.expm1(step)).astype(f), "state": rng.standard_normal((b, d, n)).astype(f)}


def scan_exact(a, lengths=None, softplus=1):
    """Values, and how far a result may be: the recurrence run on magnitudes with each step's roundings."""
    x, dtype = a["x"].astype(float), a["x"].dtype.name
    u = unit(dtype)
    b, t, d = x.shape
    n = a["A"].shape[1]
    groups = a["B"].shape[2] // n
    wide = lambda k: None if a.get(k) is None else a[k].astype(float)  # noqa: E731
    A, B, C, D, z, db = (wide(k) for k in ("A", "B", "C", "D", "z", "delta_bias"))
    raw = a["delta"].astype(float) + (db if db is not None else 0.0)
    dt = np.logaddexp(0.0, raw) if softplus else raw
    # delta + bias rounds once; softplus' error: its own functions' and the argument's (slope <= 1)
    ddt = u * (np.abs(raw) + 12 * np.abs(dt) + (4 if softplus else 0) * np.minimum(np.abs(dt), 1.0))
    h = np.zeros((b, d, n)) if a.get("state") is None else a["state"].astype(float)
    off = np.zeros_like(h)
    ys, yo = np.zeros((b, t, d)), np.zeros((b, t, d))
    ends = np.clip(lengths, 0, t) if lengths is not None else np.full(b, t)
    for i in range(t):
        on = (i < ends)[:, None]
        per = lambda v: np.repeat(v[:, i].reshape(b, groups, n), d // groups, axis=1)  # noqa: E731
        dti, xi = dt[:, i, :, None], x[:, i, :, None]
        arg = dti * A
        a_ = np.exp(arg)
        term = dti * xi * per(B)
        da = np.abs(A) * ddt[:, i, :, None] + u * (6 + 3 * np.abs(arg))      # relative error of the decay
        new = a_ * h + term
        noff = a_ * off + np.abs(a_ * h) * (da + 2 * u) + np.abs(term) * 6 * u + np.abs(xi * per(B)) * ddt[:, i, :, None] + u * np.abs(new)
        # pieces of the time axis are joined by one more product and sum each
        noff = noff + 2 * u * np.abs(new)
        h, off = np.where(on[:, :, None], new, h), np.where(on[:, :, None], noff, off)
        y = (per(C) * h).sum(2) + (D * x[:, i] if D is not None else 0.0)
        o = (np.abs(per(C)) * off).sum(2) + (n + 4) * u * ((np.abs(per(C) * h)).sum(2) + (np.abs(D * x[:, i]) if D is not None else 0.0))
        if z is not None:
            g = S.silu(z[:, i])
            y, o = y * g, o * np.abs(g) + 12 * u * np.abs(y * g) + 4 * u * np.abs(y) * np.abs(z[:, i])
        ys[:, i], yo[:, i] = np.where(on, y, 0.0), np.where(on, o, 0.0)
    return ys, yo, h, off


def run_scan(a, lengths=None, **kw):
    arrays = {k: cnp.asarray(v) for k, v in a.items()}
    first = [arrays.pop(k) for k in ("x", "delta", "A", "B", "C")]
    return cnp.selective_scan(*first, lengths=lengths, **arrays, **kw)


SCANS = [(1, 1, 1, 1, 1), (2, 1, 5, 3, 1), (3, 1, 256, 16, 1), (1, 2, 33, 4, 1), (2, 7, 64, 8, 2), (3, 65, 130, 16, 1),
         (1, 1000, 24, 16, 1), (2, 129, 64, 64, 4), (1, 40, 12, 256, 1), (2, 33, 100, 5, 1), (5, 300, 36, 12, 3),
         (1, 2049, 8, 2, 1), (130, 1, 40, 16, 1), (1, 63, 515, 16, 5), (2, 500, 40, 32, 1), (70000, 1, 1, 2, 1), (1, 20, 7, 33, 7)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,d,n,groups", SCANS)
def test_selective_scan(interface, b, t, d, n, groups, dtype):
    rng = np.random.default_rng(b + t + d + n)
    a = scan_inputs(rng, b, t, d, n, dtype, groups)
    lengths = rng.integers(-1, t + 3, b).astype(np.int32)
    few = {k: a[k] for k in ("x", "delta", "A", "B", "C")}
    def program():
        out = {}
        out["y1"], out["s1"] = run_scan(a)
        out["y2"], out["s2"] = run_scan(dict(few, delta=np.abs(few["delta"]) * np.asarray(0.1, dtype)), softplus=False)
        out["y3"], out["s3"] = run_scan(a, lengths=lengths)
        arrays = {k: cnp.asarray(v) for k, v in a.items()}
        first = [arrays.pop(k) for k in ("x", "delta", "A", "B", "C")]
        out["y4"], out["s4"] = cnp.selective_scan(*first, lengths=lengths, inplace=True, **arrays)
        assert out["s4"] is arrays["state"]
        return out
    gpu, _ = run_both(interface, program)
    cases = {1: (a, None, 1), 2: (dict(few, delta=np.abs(few["delta"]) * np.asarray(0.1, dtype)), None, 0), 3: (a, lengths, 1)}
    for i, (inputs, ln, sp) in cases.items():
        y, yo, h, ho = scan_exact(inputs, ln, sp)
        check(gpu[f"s{i}"], h, ho, acc(dtype), f"s{i}")
        check(gpu[f"y{i}"], y, yo, dtype, f"y{i}")
    bits(gpu["y4"], gpu["y3"])
    bits(gpu["s4"], gpu["s3"])


@pytest.mark.parametrize("dtype", TYPES)
def test_selective_scan_in_pieces(interface, dtype):
    rng = np.random.default_rng(9)
    a = scan_inputs(rng, 2, 90, 48, 16, dtype)
    cuts = [0, 1, 2, 40, 41, 90]
    def program():
        out, state = {}, cnp.asarray(a["state"])
        for i, (lo, hi) in enumerate(zip(cuts, cuts[1:])):
            piece = {k: np.ascontiguousarray(v[:, lo:hi]) if k in ("x", "delta", "B", "C", "z") else v for k, v in a.items() if k != "state"}
            arrays = {k: cnp.asarray(v) for k, v in piece.items()}
            first = [arrays.pop(k) for k in ("x", "delta", "A", "B", "C")]
            out[f"y{i}"], state = cnp.selective_scan(*first, state=state, **arrays)
        return dict(out, state=state)
    gpu, _ = run_both(interface, program)
    y, yo, h, ho = scan_exact(a)
    check(gpu["state"], h, ho, acc(dtype))
    check(np.concatenate([gpu[f"y{i}"] for i in range(len(cuts) - 1)], 1), y, yo, dtype)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("t", [1, 40, 700])
def test_selective_scan_reads_nothing_behind_the_end(interface, t, dtype):
    rng = np.random.default_rng(3)
    a = scan_inputs(rng, 3, t, 64, 16, dtype)
    lengths = np.array([0, t // 2, max(0, t - 1)], np.int32)
    for i, n in enumerate(lengths):
        for k in ("x", "delta", "B", "C", "z"):
            a[k][i, n:] = np.nan
    gpu, _ = run_both(interface, lambda: dict(zip("ys", run_scan(a, lengths=lengths))))
    for k in ("x", "delta", "B", "C", "z"):
        a[k] = np.nan_to_num(a[k])
    y, yo, h, ho = scan_exact(a, lengths)
    check(gpu["y"], y, yo, dtype)
    check(gpu["s"], h, ho, acc(dtype))
    assert (gpu["y"][0] == 0).all() and (gpu["s"][0] == a["state"][0]).all()


def test_selective_scan_extreme_step_sizes(interface):
    """Step sizes whose decay is exactly 0 or 1, and softplus far from 0 on both sides."""
    rng = np.random.default_rng(4)
    a = scan_inputs(rng, 1, 64, 32, 16, "float32")
    a["delta"][0, ::3] = 60.0
    a["delta"][0, 1::3] = -80.0
    gpu, _ = run_both(interface, lambda: dict(zip("ys", run_scan(a))))
    y, yo, h, ho = scan_exact(a)
    check(gpu["y"], y, yo, "float32")
    check(gpu["s"], h, ho, "float32")


# ---- sample ------------------------------------------------------------------------------------------------------

def logp_bound(x, temperature, dtype):
    """Errors of a weight: its argument's rounding and the exponential's (relative)."""
    most = x.max()
    with np.errstate(all="ignore"):
        z = np.where(x == most, 0.0, np.where(np.isfinite(most), np.maximum((x * 0.5 - most * 0.5) / max(temperature, 1e-30) * 2.0, -700.0), -700.0))
    e = np.exp(z)
    return unit(dtype) * float((e * (3 * np.abs(z) + 8)).sum() / e.sum()) * 2 + 2.0 ** -36


def check_samples(x, token, logp, u, temperature, top_k, top_p, min_p):
    """The token is the oracle's, or the oracle's for borders moved by no more than the sums' error."""
    dtype = x.dtype.name
    each = [np.broadcast_to(np.asarray(v, float), (len(x),)) for v in (u, temperature, top_k, top_p, min_p)]
    for i, row in enumerate(x.astype(float)):
        p = [float(v[i]) for v in each]
        want, lp = S.sample_row(row, *p)
        slack = logp_bound(np.where(np.isnan(row), -np.inf, row), p[1], dtype) if want >= 0 and p[1] > 0 else 0.0
        if token[i] != want:
            near = [S.sample_row(row, p[0] + a * slack, p[1], p[2], p[3] + b * slack if p[3] < 1 else 1.0, p[4] * (1 + c * 16 * unit(dtype) * (1 + abs(np.log(p[4] or 1)))))
                    for a in (-1, 0, 1) for b in (-1, 0, 1) for c in (-1, 0, 1)]
            got = [q for q in near if q[0] == token[i]]
            assert got, (i, token[i], want, p)
            lp = got[0][1]
        if np.isfinite(lp):
            # a border that moves by the sums' error moves the total by as much and by one more token
            z = max(abs(lp), 1.0)
            assert abs(logp[i] - lp) <= 4 * slack + 8 * unit(dtype) * z + 1e-5 * (token[i] != want) + (0 if p[3] >= 1 else edge_weight(row, p, slack)), (i, logp[i], lp)
        else:
            assert logp[i] == lp


def edge_weight(row, p, slack):
    """Share of a token that top-p keeps or drops when its border moves by `slack`."""
    totals = [np.exp(-S.sample_row(row, 0.0, p[1], p[2], min(max(p[3] + s, 0.0), 1.0 - 1e-16), p[4])[1]) if p[1] > 0 else 1.0 for s in (-slack, slack)]
    first = [S.sample_row(row, 0.0, p[1], p[2], min(max(p[3] + s, 0.0), 1.0 - 1e-16), p[4])[0] for s in (-slack, slack)]
    return abs(np.log(totals[0] / totals[1])) if first[0] == first[1] else 1e-5


VOCABULARIES = [1, 2, 5, 31, 32, 33, 1000, 1024, 4097, 8192, 20000, 32768, 50021, 65536, 100003, 131072, 200000, 262144]
FILTERS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.3, 0, 0.98, 0.0), (0.8, 0, 0.5, 0.05), (1.0, 7, 1.0, 0.0), (1.0, 0, 1.0, 0.1),
           (0.0, 0, 1.0, 0.0), (2.0, 1000, 0.999, 0.001), (1.0, 1, 0.3, 0.0), (0.9, 0, 0.0, 0.0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", VOCABULARIES)
def test_sample(interface, v, dtype):
    rng = np.random.default_rng(v)
    rows = 6 if v > 1000 else 40
    x = (rng.standard_normal((rows, v)) * 2.5 + rng.standard_normal((rows, 1)) * 3).astype(dtype)
    u = rng.random(rows).astype("float64" if dtype == "float64" else "float32")
    u[0], u[1 % rows] = 0.0, 1.0 - 2.0 ** -24
    def program():
        out, ax, au = {}, cnp.asarray(x), cnp.asarray(u)
        for i, (t, k, p, m) in enumerate(FILTERS):
            out[f"t{i}"], out[f"p{i}"] = cnp.random.sample(ax, au, temperature=t, top_k=k, top_p=p, min_p=m)
        return out
    gpu, _ = run_both(interface, program)
    for i, f in enumerate(FILTERS):
        check_samples(x, gpu[f"t{i}"], gpu[f"p{i}"], u, *f)


@pytest.mark.parametrize("v", [100, 5000, 70000])
def test_sample_parameters_per_row(interface, v):
    rng = np.random.default_rng(v)
    rows = 24
    x = (rng.standard_normal((rows, v)) * 3).astype("float32")
    u = rng.random(rows)
    t = rng.choice([0.0, 0.5, 1.0, 2.0], rows).astype("float32")
    k = rng.choice([0, 1, 3, 40, v, v + 5, -2], rows).astype("int32")
    p, m = rng.choice([0.1, 0.8, 1.0, 1.5], rows), rng.choice([0.0, 0.02, 1.0], rows).astype("float32")
    gpu, _ = run_both(interface, lambda: dict(zip("tp", cnp.random.sample(cnp.asarray(x), cnp.asarray(u), temperature=t, top_k=k, top_p=p, min_p=m))))
    check_samples(x, gpu["t"], gpu["p"], u, t, k, p, m)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [64, 3000, 40000])
def test_sample_masks_ties_and_infinities(interface, v, dtype):
    low = np.finfo(dtype).min
    x = np.zeros((12, v), dtype)
    x[0] = -np.inf                                   # nothing left
    x[1] = np.nan
    x[2] = -np.inf; x[2, v // 2] = -3                # one left  # noqa: E702
    x[3] = low                                       # all at the type's lowest value
    x[4] = low; x[4, 5:9] = 1                        # noqa: E702
    x[5, 7] = np.inf; x[5, v - 1] = np.inf           # two infinities  # noqa: E702
    x[6, 3] = np.nan
    x[7, ::2] = -0.0
    x[8] = np.linspace(-1, 1, v)
    x[9, : v // 2] = -np.inf
    x[10] = np.where(np.arange(v) % 3 == 0, 1, 0)
    x[11, v - 1] = 9
    u = np.tile(np.array([0.0, 0.2, 0.4999, 0.7, 0.95, 0.999999]), 2).astype("float32")
    sets = [(1.0, 0, 1.0, 0.0), (1.0, 5, 1.0, 0.0), (1.0, 0, 0.4, 0.0), (0.5, 20, 0.7, 0.1), (0.0, 3, 0.5, 0.0), (1.0, v - 1, 0.99, 0.0)]
    def program():
        out, ax, au = {}, cnp.asarray(x), cnp.asarray(u)
        for i, (t, k, p, m) in enumerate(sets):
            out[f"t{i}"], out[f"p{i}"] = cnp.random.sample(ax, au, temperature=t, top_k=k, top_p=p, min_p=m)
        return out
    gpu, _ = run_both(interface, program)
    for i, f in enumerate(sets):
        check_samples(x, gpu[f"t{i}"], gpu[f"p{i}"], u, *f)
        assert gpu[f"t{i}"][0] == -1 and gpu[f"t{i}"][1] == -1


@pytest.mark.parametrize("dtype,v", [("float16", 600000), ("float32", 262145), ("float32", 1000003), ("float64", 300000)])
def test_sample_vocabularies_beyond_shared_memory(interface, dtype, v):
    rng = np.random.default_rng(v)
    x = (rng.standard_normal((2, v)) * 2).astype(dtype)
    u = np.array([0.3, 0.999], "float64" if dtype == "float64" else "float32")
    sets = [(1.0, 0, 1.0, 0.0), (0.8, 300, 0.9, 0.0), (1.5, 0, 0.97, 0.001)]
    def program():
        out, ax, au = {}, cnp.asarray(x), cnp.asarray(u)
        for i, (t, k, p, m) in enumerate(sets):
            out[f"t{i}"], out[f"p{i}"] = cnp.random.sample(ax, au, temperature=t, top_k=k, top_p=p, min_p=m)
        return out
    gpu, _ = run_both(interface, program)
    for i, f in enumerate(sets):
        check_samples(x, gpu[f"t{i}"], gpu[f"p{i}"], u, *f)


def test_sample_one_dimension_and_given_numbers(interface):
    rng = np.random.default_rng(1)
    x = rng.standard_normal(3000)
    def program():
        u = cnp.random.uniform((1,), seed=11)
        t, p = cnp.random.sample(cnp.asarray(x), u, top_k=20)
        return {"u": u, "t": t, "p": p}
    gpu, cpu = run_both(interface, program)
    check_samples(x[None], gpu["t"], gpu["p"], gpu["u"], 1.0, 20, 1.0, 0.0)


def test_sample_frequencies(interface):
    """Many rows of one distribution: the counts follow the probabilities (5 standard deviations)."""
    p = np.array([0.5, 0.25, 0.125, 0.0625, 0.0625])
    rows = 20000
    x = np.tile(np.log(p), (rows, 1)).astype("float32")
    gpu, _ = run_both(interface, lambda: {"t": cnp.random.sample(cnp.asarray(x), cnp.random.uniform((rows,), seed=3))[0]})
    counts = np.bincount(gpu["t"], minlength=5)
    assert (np.abs(counts - rows * p) <= 5 * np.sqrt(rows * p * (1 - p))).all(), counts


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_extreme_temperatures_and_spans(interface, dtype):
    """Weights that are all alike, all but one nothing, and logits at both ends of the type."""
    rng = np.random.default_rng(21)
    big = float(np.finfo(dtype).max)
    v = 9000
    x = np.stack([rng.standard_normal(v), np.linspace(-big, big, v), np.where(np.arange(v) % 7, -big, big * 0.5),
                  rng.standard_normal(v) * 1e-3, 20 + rng.standard_normal(v) * 1e-2, np.where(np.arange(v) == 4000, 60.0, rng.standard_normal(v))]).astype(dtype)
    u = np.array([0.1, 0.3, 0.5, 0.7, 0.9, 0.99999], "float32")
    sets = [(t, k, p, 0.0) for t in (1e-30, 1e-3, 1.0, 1e4, 1e30, float("inf")) for k, p in ((0, 0.7), (100, 1.0), (4500, 0.5))]
    def program():
        out, ax, au = {}, cnp.asarray(x), cnp.asarray(u)
        for i, (t, k, p, m) in enumerate(sets):
            out[f"t{i}"], out[f"p{i}"] = cnp.random.sample(ax, au, temperature=t, top_k=k, top_p=p, min_p=m)
        return out
    gpu, _ = run_both(interface, program)
    for i, f in enumerate(sets):
        check_samples(x, gpu[f"t{i}"], gpu[f"p{i}"], u, *f)


# ---- conversions, storage types, steps ----------------------------------------------------------------------------

@pytest.mark.parametrize("source", ["float16", "float32", "float64", "int32", "int64", "int8"])
@pytest.mark.parametrize("target", ["float16", "float32", "float64", "int32", "int64", "int8"])
def test_astype(interface, source, target):
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((37, 19)) * 30).astype(source)
    gpu, cpu = run_both(interface, lambda: {"a": cnp.asarray(x).astype(target)})
    assert gpu["a"].dtype == np.dtype(target)
    bits(gpu["a"], x.astype(target))
    bits(gpu["a"], cpu["a"])


@pytest.mark.parametrize("dtype", ["float16", "int8"])
def test_storage_types_are_made_filled_copied_and_moved(interface, dtype):
    rng = np.random.default_rng(8)
    x = (rng.standard_normal((6, 10)) * 20).astype(dtype)
    def program():
        a = cnp.asarray(x)
        view = a[1:5, 2:9:3].copy()
        z = cnp.zeros((6, 10), dtype=dtype)
        z[2:4, 1:] = a[0:2, :9]
        z[5, :] = 3
        row = cnp.zeros((10,), dtype=dtype)
        row[...] = a[3, :]
        return {"a": a, "view": view, "z": z, "row": row, "full": cnp.full((3, 3), 2, dtype=dtype), "tile": cnp.tile(a, (2, 1))}
    gpu, cpu = run_both(interface, program)
    for k in cpu:
        bits(gpu[k], cpu[k])
    bits(gpu["view"], np.ascontiguousarray(x[1:5, 2:9:3]))


def test_views_are_copied_for_the_operators(interface):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((8, 100)).astype("float16")
    gpu, cpu = run_both(interface, lambda: {"y": cnp.rms_norm(cnp.asarray(x)[1:7:2, 10:90])})
    np.testing.assert_allclose(gpu["y"].astype(float), cpu["y"].astype(float), rtol=2.0 ** -10)


def test_backend_refuses_arithmetic_on_storage_types(interface):
    """Also where a caller of the C ABI asks for it."""
    from charmnumeric_b200 import wire
    from charmnumeric_b200._lib import CnError
    ctx = interface.context
    ctx.put(880001, np.ones(64, "float16"))
    leaf = lambda: wire.leaf(880001, (64,), wire.F16)  # noqa: E731
    for root in (wire.Ast(880002, wire.OP_ADD, shape=(64,), dtype=wire.F16, operands=[(leaf(), None), (leaf(), None)]),
                 wire.Ast(880002, wire.OP_ADD, shape=(64,), dtype=wire.F32, operands=[(leaf(), None), (leaf(), None)]),
                 wire.Ast(880002, wire.OP_SUM, shape=(1,), dtype=wire.F16, operands=[(leaf(), None)]),
                 wire.Ast(880002, wire.OP_REDUCE, shape=(1,), dtype=wire.F16, operands=[(leaf(), None), (leaf(), None)]),
                 wire.Ast(880002, wire.OP_RANDU, shape=(64,), dtype=wire.F16, operands=[(wire.scalar(v), None) for v in (1, 0, 1)])):
        with pytest.raises(CnError) as e:
            ctx.run([wire.Node(0, [root], fusible=root.opcode == wire.OP_ADD)])
        assert e.value.status == 7
    ctx.delete_array(880001)


def test_recorded_step_follows_its_inputs(interface):
    x, w = cnp.asarray(np.arange(12.0).reshape(3, 4)), cnp.asarray(np.ones(4))
    step = cnp.record(lambda: cnp.rms_norm(x, w))
    first = step.run(interface).get(interface)
    x[...] = x * -1.0
    again = step.run(interface).get(interface)
    np.testing.assert_array_equal(again, -first)
    del x, w                                          # the step keeps what it uses
    cnp.execute(interface)
    np.testing.assert_array_equal(step.run(interface).get(interface), -first)


def test_device_memory_of_another_library(interface):
    import torch
    t = torch.randn(5, 300, device="cuda").half()
    a = cnp.from_device(interface, t)
    np.testing.assert_array_equal(a.get(interface), t.cpu().numpy())
    y = cnp.rms_norm(a)
    view = torch.as_tensor(y.device_view(interface), device="cuda")
    interface.context.synchronize()
    np.testing.assert_array_equal(view.cpu().numpy(), y.get(interface))
    with pytest.raises(ValueError):
        cnp.from_device(interface, t.t())
    with pytest.raises(TypeError):
        cnp.from_device(interface, np.zeros(3))
    empty = cnp.from_device(interface, torch.zeros(0, 4, device="cuda"))
    assert empty.get(interface).shape == (0, 4)


def test_empty_arrays(interface):
    def program():
        y = cnp.rms_norm(cnp.zeros((0, 7), dtype="float16"))
        c, s = cnp.causal_conv(cnp.zeros((2, 0, 5)), np.ones((5, 3)), state=np.ones((2, 2, 5)))
        a = {"x": np.zeros((2, 0, 4)), "delta": np.zeros((2, 0, 4)), "A": -np.ones((4, 3)), "B": np.zeros((2, 0, 3)),
             "C": np.zeros((2, 0, 3)), "state": np.full((2, 4, 3), 7.0)}
        z, h = run_scan(a)
        t, p = cnp.random.sample(cnp.zeros((0, 9)), cnp.zeros((0,)))
        return {"y": y, "c": c, "s": s, "z": z, "h": h, "t": t, "p": p}
    gpu, cpu = run_both(interface, program)
    for k in cpu:
        bits(gpu[k], cpu[k])
    assert (gpu["h"] == 7).all() and (gpu["s"] == 1).all()


def test_a_model_step(interface):
    """The operators together, as a recurrent model's decoding step uses them between matvecs: norm,
    projection, convolution, scan, gate, projection back, residual, norm, logits, token."""
    rng = np.random.default_rng(12)
    width, inner, n, v = 48, 96, 8, 500
    par = {"in": rng.standard_normal((2 * inner, width)) * 0.2, "out": rng.standard_normal((width, inner)) * 0.2,
           "bc": rng.standard_normal((2 * n, inner)) * 0.2, "delta": rng.standard_normal((inner, inner)) * 0.05,
           "head": rng.standard_normal((v, width)), "conv": rng.standard_normal((inner, 4)) * 0.5,
           "A": -np.abs(rng.standard_normal((inner, n))), "D": np.ones(inner), "norm": np.ones(width), "bias": np.full(inner, -2.0)}
    token_in = rng.standard_normal(width)

    def program():
        p = {k: cnp.asarray(a) for k, a in par.items()}
        h, out = cnp.asarray(token_in), {}
        conv = cnp.zeros((1, 3, inner))
        ssm = cnp.zeros((1, inner, n))
        r = cnp.zeros((width,))
        for i in range(3):
            y, r = cnp.rms_norm(h, p["norm"], residual=r)
            xz = p["in"] @ y
            x, z = cnp.zeros((1, 1, inner)), cnp.zeros((1, 1, inner))
            x[0, 0, :] = xz[:inner]
            z[0, 0, :] = xz[inner:]
            x, conv = cnp.causal_conv(x, p["conv"], state=conv, activation="silu")
            flat = cnp.zeros((inner,))
            flat[...] = x[0, 0, :]
            bc = p["bc"] @ flat
            B, C, delta = cnp.zeros((1, 1, n)), cnp.zeros((1, 1, n)), cnp.zeros((1, 1, inner))
            B[0, 0, :] = bc[:n]
            C[0, 0, :] = bc[n:]
            delta[0, 0, :] = p["delta"] @ flat
            y, ssm = cnp.selective_scan(x, delta, p["A"], B, C, D=p["D"], z=z, delta_bias=p["bias"], state=ssm)
            flat = cnp.zeros((inner,))
            flat[...] = y[0, 0, :]
            h = p["out"] @ flat
            last, _ = cnp.rms_norm(h, p["norm"], residual=r)
            out[f"t{i}"], out[f"p{i}"] = cnp.random.sample(p["head"] @ last, cnp.random.uniform((1,), seed=i), temperature=0.9, top_k=40, top_p=0.95)
        return dict(out, h=h, ssm=ssm, conv=conv)
    gpu, cpu = run_both(interface, program)
    for k in cpu:
        np.testing.assert_allclose(gpu[k], cpu[k], rtol=1e-9, atol=1e-12, err_msg=k)


# ---- what the backend itself refuses -------------------------------------------------------------------------------

def _leaf(ctx, name, array):
    from charmnumeric_b200 import wire
    from charmnumeric_b200.context import WIRE_DTYPES
    ctx.put(name, array)
    return wire.leaf(name, array.shape, WIRE_DTYPES[array.dtype])


def _cases():
    from charmnumeric_b200 import wire
    f = np.float32
    none = wire.scalar(0.0)
    x2, x3 = np.ones((3, 8), f), np.ones((2, 5, 4), f)
    scan = [x3, x3, -np.ones((4, 3), f), np.ones((2, 5, 3), f), np.ones((2, 5, 3), f), none, none, none, none, none, wire.scalar(1)]
    def put(i, v, base):
        return base[:i] + [v] + base[i + 1:]
    norm, conv = [x2, none, none, wire.scalar(1e-5), wire.scalar(0)], [x3, np.ones((4, 3), f), none, none, none, wire.scalar(0)]
    draw = [x2, np.ones(3, f), wire.scalar(1), wire.scalar(0), wire.scalar(1), wire.scalar(0)]
    return [
        (wire.OP_RMS_NORM, put(0, x2.astype("int32"), norm), 1, 7), (wire.OP_RMS_NORM, put(1, np.ones(7, f), norm), 1, 4),
        (wire.OP_RMS_NORM, put(2, np.ones((3, 9), f), norm), 2, 4), (wire.OP_RMS_NORM, put(2, x2.astype("float16"), norm), 2, 7),
        (wire.OP_RMS_NORM, put(3, wire.scalar(float("nan")), norm), 1, 1), (wire.OP_RMS_NORM, put(4, wire.scalar(9), norm), 2, 1),
        (wire.OP_RMS_NORM, put(4, wire.scalar(1.5), norm), 2, 1), (wire.OP_RMS_NORM, norm, 2, 2), (wire.OP_RMS_NORM, norm[:4], 1, 2),
        (wire.OP_RMS_NORM, put(0, none, norm), 1, 2),
        (wire.OP_CAUSAL_CONV, put(0, x2, conv), 2, 4), (wire.OP_CAUSAL_CONV, put(1, np.ones((5, 3), f), conv), 2, 4),
        (wire.OP_CAUSAL_CONV, put(1, np.ones((4, 9), f), conv), 2, 5), (wire.OP_CAUSAL_CONV, put(3, np.ones((2, 3, 4), f), conv), 2, 4),
        (wire.OP_CAUSAL_CONV, put(4, np.ones(2, f), conv), 2, 7), (wire.OP_CAUSAL_CONV, put(4, np.ones(3, "int32"), conv), 2, 4),
        (wire.OP_CAUSAL_CONV, put(5, wire.scalar(2), conv), 2, 1), (wire.OP_CAUSAL_CONV, conv, 1, 2),
        (wire.OP_SELECTIVE_SCAN, put(1, x3[:1], scan), 2, 4), (wire.OP_SELECTIVE_SCAN, put(2, -np.ones((4, 257), f), scan), 2, 5),
        (wire.OP_SELECTIVE_SCAN, put(2, -np.ones((4, 3)), scan), 2, 7), (wire.OP_SELECTIVE_SCAN, put(3, np.ones((2, 5, 4), f), scan), 2, 4),
        (wire.OP_SELECTIVE_SCAN, put(4, np.ones((2, 5, 6), f), scan), 2, 4), (wire.OP_SELECTIVE_SCAN, put(8, np.ones((2, 4, 2), f), scan), 2, 4),
        (wire.OP_SELECTIVE_SCAN, put(7, np.ones(5, f), scan), 2, 4), (wire.OP_SELECTIVE_SCAN, scan[:10], 2, 2),
        (wire.OP_SAMPLE, put(1, np.ones(2, f), draw), 2, 4), (wire.OP_SAMPLE, put(1, np.ones(3, "int32"), draw), 2, 7),
        (wire.OP_SAMPLE, put(3, np.ones(3, f), draw), 2, 7), (wire.OP_SAMPLE, put(4, np.ones(4, f), draw), 2, 4),
        (wire.OP_SAMPLE, put(0, x3, draw), 2, 4), (wire.OP_SAMPLE, draw, 1, 2),
        (wire.OP_CONVERT, [x2, np.ones((3, 1), f), wire.scalar(8)], 1, 7),
        (wire.OP_CONVERT, [x2.astype("int8"), np.ones((3, 2), f), wire.scalar(8)], 1, 4),
        (wire.OP_CONVERT, [x2.astype("int8"), np.ones((3, 1), f), wire.scalar(0)], 1, 1),
        (99, [x2], 1, 6),
    ]


@pytest.mark.parametrize("case", range(36))
def test_backend_refusals(interface, case):
    from charmnumeric_b200 import wire
    from charmnumeric_b200._lib import CnError
    ctx = interface.context
    opcode, operands, results, status = _cases()[case]
    leaves = [(_leaf(ctx, 880100 + i, v) if isinstance(v, np.ndarray) else v, None) for i, v in enumerate(operands)]
    roots = [wire.Ast(880200, opcode, shape=(1,), dtype=wire.F32, operands=leaves)]
    roots += [wire.Ast(880200 + i, wire.OP_NOOP, shape=(1,), dtype=wire.F32) for i in range(1, results)]
    before = ctx.stats()["kernel_launches"]
    with pytest.raises(CnError) as e:
        ctx.run([wire.Node(0, roots, fusible=False)])
    assert e.value.status == status, e.value
    assert ctx.stats()["kernel_launches"] == before
    ctx.synchronize()                                  # the context stays usable
    for i, v in enumerate(operands):
        if isinstance(v, np.ndarray):
            ctx.delete_array(880100 + i)


def test_backend_refuses_results_that_are_operands(interface):
    from charmnumeric_b200 import wire
    from charmnumeric_b200._lib import CnError
    ctx = interface.context
    x = _leaf(ctx, 880300, np.ones((2, 1, 4), np.float32))
    w = _leaf(ctx, 880301, np.ones((4, 2), np.float32))
    none, noop = wire.scalar(0.0), lambda n: wire.Ast(n, wire.OP_NOOP, shape=(1,), dtype=wire.F32)  # noqa: E731
    def conv(y, state, operand=none):
        return [wire.Ast(y, wire.OP_CAUSAL_CONV, shape=(1,), dtype=wire.F32, operands=[(v, None) for v in (x, w, none, operand, none, none)]), noop(state)]
    for roots in (conv(880300, 880310), conv(880310, 880301), conv(880310, 880310), conv(880310, 880300, x)):
        with pytest.raises(CnError) as e:
            ctx.run([wire.Node(0, roots, fusible=False)])
        assert e.value.status == 11
    np.testing.assert_array_equal(ctx.get(880300), 1)
    for name in (880300, 880301):
        ctx.delete_array(name)


def test_host_memory_is_no_device_array(interface):
    from charmnumeric_b200._lib import CnError
    host = np.zeros(16, np.float32)
    class Fake:
        __cuda_array_interface__ = {"shape": (16,), "typestr": "<f4", "data": (host.ctypes.data, False), "version": 3}
    with pytest.raises(CnError) as e:
        cnp.from_device(interface, Fake())
    assert e.value.status == 1


def test_two_contexts_at_once(interface):
    """Two interfaces on one GPU, each with its own arrays and stream, interleaved."""
    rng = np.random.default_rng(3)
    other = cnp.CharmNumericInterface(device=0)
    try:
        x = [rng.standard_normal((40, 30000)).astype("float32") for _ in range(2)]
        u = rng.random(40).astype("float32")
        steps = []
        for itf, v in zip((interface, other), x):
            a, b = cnp.asarray(v), cnp.asarray(u)
            cnp.execute(itf)
            steps.append((itf, cnp.record(lambda: cnp.random.sample(a, b, top_k=30, top_p=0.9))))
        for _ in range(20):
            for itf, step in steps:
                step.run(itf)
        for (itf, step), v in zip(steps, x):
            check_samples(v, step.results[0].get(itf), step.results[1].get(itf), u, 1.0, 30, 0.9, 0.0)
    finally:
        del steps
        other.close()


def test_a_long_decoding_loop_in_place(interface):
    """A recorded step that brings its states up to date itself, against the prompt's scan."""
    rng = np.random.default_rng(31)
    b, t, d, n = 4, 24, 64, 16
    a = scan_inputs(rng, b, t, d, n, "float32")
    x, delta, B, C, zz = (cnp.zeros((b, 1, v.shape[2]), dtype="float32") for v in (a["x"], a["delta"], a["B"], a["C"], a["z"]))
    state = cnp.asarray(a["state"])
    fixed = {k: cnp.asarray(a[k]) for k in ("A", "D", "delta_bias")}
    cnp.execute(interface)
    step = cnp.record(lambda: cnp.selective_scan(x, delta, fixed["A"], B, C, D=fixed["D"], z=zz, delta_bias=fixed["delta_bias"], state=state, inplace=True))
    ys = []
    for i in range(t):
        for to, k in ((x, "x"), (delta, "delta"), (B, "B"), (C, "C"), (zz, "z")):
            interface.context.put(to.name, np.ascontiguousarray(a[k][:, i:i + 1]))
        ys.append(step.run(interface)[0].get(interface))
    y, yo, h, ho = scan_exact(a)
    check(np.concatenate(ys, 1), y, yo, "float32")
    check(state.get(interface), h, ho, "float32")


@pytest.mark.parametrize("t", [1, 50])
@pytest.mark.parametrize("dtype", TYPES)
def test_selective_scan_steps_of_no_size_change_nothing(interface, t, dtype):
    rng = np.random.default_rng(17)
    a = scan_inputs(rng, 5, t, 256, 16, dtype)
    a["delta"][...] = -1200.0 if dtype == "float64" else -300.0     # softplus is exactly 0
    gpu, _ = run_both(interface, lambda: dict(zip("ys", run_scan(a))))
    bits(gpu["s"], a["state"])


@pytest.mark.parametrize("dtype", ["float16", "int8"])
def test_storage_types_in_three_dimensions(interface, dtype):
    """Steps in every dimension, diagonals and repeats."""
    rng = np.random.default_rng(18)
    x = (rng.standard_normal((7, 9, 11)) * 20).astype(dtype)
    def program():
        a = cnp.asarray(x)
        part = a[1::2, ::3, 2:10:2].copy()
        b = cnp.zeros((9, 10, 13), dtype=dtype)
        b[2:9:3, 1:10:3, 5:9] = part
        b[::4, 9, :] = 7
        return {"part": part, "b": b, "tile": cnp.tile(a, (2, 1, 3)), "diag": cnp.diag(cnp.asarray(x[0]))}
    gpu, cpu = run_both(interface, program)
    for k in cpu:
        bits(gpu[k], cpu[k])
    bits(gpu["part"], np.ascontiguousarray(x[1::2, ::3, 2:10:2]))
    bits(gpu["tile"], np.tile(x, (2, 1, 3)))
    bits(gpu["diag"], np.diag(x[0]).copy())


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_temperatures_without_an_inverse(interface, dtype):
    """So small that 1 / temperature is infinite (in 32 bits): the largest logit, as at 0.  Neighbours of the
    largest whose difference from it is next to nothing have no weight either."""
    x = np.random.default_rng(22).standard_normal((3, 5000)).astype(dtype)
    x[1] *= np.asarray(1e-3, dtype)
    x[2] = np.where(np.arange(5000) % 2, x[2], 4).astype(dtype)       # 2500 equal ones: the draw is among them
    u = np.array([0.2, 0.5, 0.9], "float32")
    def program():
        ax, au, out = cnp.asarray(x), cnp.asarray(u), {}
        for i, (k, p) in enumerate([(0, 1.0), (50, 1.0), (0, 0.9), (4000, 0.5)]):
            out[f"t{i}"], out[f"p{i}"] = cnp.random.sample(ax, au, temperature=1e-42, top_k=k, top_p=p)
        return out
    gpu, _ = run_both(interface, program)
    for i, (k, p) in enumerate([(0, 1.0), (50, 1.0), (0, 0.9), (4000, 0.5)]):
        check_samples(x, gpu[f"t{i}"], gpu[f"p{i}"], u, 1e-42, k, p, 0.0)
