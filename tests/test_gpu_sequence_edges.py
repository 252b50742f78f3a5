"""GPU tests of the sequence model operators where values are infinite or NaN, against the CPU oracle."""
import numpy as np
import pytest

import charmnumeric_b200 as cnp
from oracle import sequence as S
from tests.helpers import run_both
from tests.test_gpu_sequence import TYPES, acc, bits, check_samples, run_scan, scan_exact

pytestmark = pytest.mark.gpu


# ---- causal_conv --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [24, 6, 5])
@pytest.mark.parametrize("k", range(2, 9))
def test_causal_conv_infinities_reach_as_far_as_the_filter(interface, k, d, dtype):
    """One infinity or NaN in the inputs or the state shows in k outputs, across the borders of runs too, and in
    no other.  Small whole numbers: every sum is exact."""
    rng = np.random.default_rng(k + d)
    x = rng.integers(-3, 4, (3, 100, d)).astype(dtype)
    state = rng.integers(-3, 4, (3, k - 1, d)).astype(dtype)
    w = rng.choice([-3, -2, -1, 1, 2, 3], (d, k)).astype(dtype)
    for at, c, v in ((3, 1, np.inf), (31, 2, np.nan), (70, 3, -np.inf), (63, d - 1, np.inf), (99, 0, np.nan)):
        x[0, at, c] = v
    state[1, 0, 0], state[1, k - 2, d - 1], state[2, :, 1] = np.inf, np.nan, -np.inf
    lengths = np.array([100, 40, 7], np.int32)

    def program():
        ax, aw, ast = (cnp.asarray(v) for v in (x, w, state))
        y1, s1 = cnp.causal_conv(ax, aw, state=ast)
        y2, s2 = cnp.causal_conv(ax, aw, state=ast, lengths=lengths)
        y3, s3 = cnp.causal_conv(cnp.asarray(x[:, 3:4].copy()), aw, state=ast)
        return {"y1": y1, "s1": s1, "y2": y2, "s2": s2, "y3": y3, "s3": s3}
    gpu, _ = run_both(interface, program)
    with np.errstate(invalid="ignore"):
        want = {"1": S.causal_conv(x, w, None, state, None, 0), "2": S.causal_conv(x, w, None, state, lengths, 0),
                "3": S.causal_conv(x[:, 3:4], w, None, state, None, 0)}
    for i, (y, s) in want.items():
        np.testing.assert_array_equal(gpu["y" + i], y)
        np.testing.assert_array_equal(gpu["s" + i], s)


# ---- selective_scan -----------------------------------------------------------------------------------------

def flat_inputs(b, t, d, n, dtype, **more):
    """Every value 1 and every decay e^-dt: all sums have one sign, so that an infinity meets no other."""
    f = acc(dtype)
    a = {"x": np.ones((b, t, d), dtype), "delta": np.zeros((b, t, d), dtype), "A": -np.ones((d, n), f),
         "B": np.ones((b, t, n), dtype), "C": np.ones((b, t, n), dtype)}
    return dict(a, **more)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [1, 40, 700])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 12, 16, 20, 31, 40, 64, 100, 128, 200, 256])
def test_selective_scan_infinities(interface, n, t, dtype):
    """Infinite inputs and step sizes: infinite from there on in their channel, whatever the number of states is
    filled up to, with D and without, gated and not."""
    f = acc(dtype)
    a = flat_inputs(2, t, 9, n, dtype)
    a["x"][0, t // 2, 3] = np.inf
    a["x"][1, t - 1, 8] = np.inf
    a["delta"][1, t // 3, 5] = np.inf
    with_d, gated = dict(a, D=np.ones(9, f)), dict(a, z=np.ones_like(a["x"]))

    def program():
        return {k + i: v for i, inputs in (("0", a), ("1", with_d), ("2", gated)) for k, v in zip("ys", run_scan(inputs))}
    gpu, cpu = run_both(interface, program)
    for i in "012":
        for k in "ys":
            np.testing.assert_array_equal(np.isinf(gpu[k + i]), np.isinf(cpu[k + i]), err_msg=k + i)
            assert not np.isnan(gpu[k + i]).any()
        assert np.isinf(cpu["y" + i][0, t // 2:, 3]).all() and np.isinf(cpu["y" + i]).sum() == (t - t // 2) + 1 + (t - t // 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_selective_scan_decays_beyond_the_range_of_a_type(interface, dtype):
    """Few channels and many steps, which are walked in pieces: what a piece multiplies an earlier state by may
    leave the type's range on either side while the product does not."""
    f = acc(dtype)
    much = 800.0 if dtype == "float64" else 100.0          # beyond e^88 and e^709
    b, t, d, n = 1, 640, 4, 3
    a = flat_inputs(b, t, d, n, dtype)
    a["delta"] = np.zeros((b, t, d), dtype)
    a["delta"][0, :64] = 1
    a["delta"][0, 576:] = 2.0 ** -10
    a["x"][0, :64] = 0
    a["A"] = (np.array([[1.0], [-1.0], [1.0], [-1.0]]) * [1.0, 0.5, 0.25] * much / 64).astype(f)
    a["A"][3] *= 20                                        # 64 steps leave nothing, one of them something
    large = 1e300 if dtype == "float64" else 1e36
    a["state"] = np.array([[[0.0] * 3, [large, 1.0, 0.0], [1 / large] * 3, [np.inf, -np.inf, 1.0]]], f)
    gpu, _ = run_both(interface, lambda: dict(zip("ys", run_scan(dict(a), softplus=False))))
    with np.errstate(all="ignore"):
        y, yo, h, ho = scan_exact(dict(a), None, 0)
    fine = np.isfinite(h)
    np.testing.assert_array_equal(gpu["s"][~fine], h.astype(f)[~fine])
    off = np.abs(gpu["s"].astype(float) - np.where(fine, h, 0))
    assert fine[0, :3].all() and (off <= ho + 2.0 ** -23 * np.abs(np.where(fine, h, 0)))[fine].all()


@pytest.mark.parametrize("t,launches", [(1, 1), (100, 1), (640, 2)])
def test_selective_scan_counts_its_launches(interface, t, launches):
    """Few channels: long sequences are walked in pieces, by two kernels."""
    arrays = {k: cnp.asarray(v) for k, v in flat_inputs(1, t, 4, 3, "float32").items()}
    cnp.execute(interface)
    before = interface.context.stats()["kernel_launches"]
    y, s = cnp.selective_scan(*arrays.values())
    cnp.execute(interface)
    assert interface.context.stats()["kernel_launches"] - before == launches


# ---- conversions ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("scales", ["float32", "float64"])
@pytest.mark.parametrize("target", TYPES)
@pytest.mark.parametrize("n,group", [(2048, 64), (2047, 2047), (2050, 3)])
def test_dequantize_rounds_once(interface, n, group, target, scales):
    rng = np.random.default_rng(n)
    q = rng.integers(-127, 128, (257, n)).astype(np.int8)
    s = np.exp(rng.uniform(-22, 3, (257, -(-n // group)))).astype(scales)
    s[0, 0], s[1, 0], s[2, 0], s[3, 0] = 0, np.inf, np.nan, np.finfo(scales).max
    gpu, _ = run_both(interface, lambda: {"v": cnp.dequantize(cnp.asarray(q), cnp.asarray(s), group=group, dtype=target)})
    with np.errstate(all="ignore"):
        # 8 bits times 53 fit the 64 of a long double; to 16 bits through the neighbouring double whose last bit
        # is 1 where it is not exact, which lies on the same side of every border as the product
        exact = q.astype(np.longdouble) * np.repeat(s.astype(np.longdouble), group, -1)[:, :n]
        if target == "float16":
            near = exact.astype(np.float64)
            odd = near.view(np.uint64) & np.uint64(1) == 1
            other = np.nextafter(near, np.where(exact > near, np.inf, -np.inf))
            exact = np.where((near == exact) | ~np.isfinite(near) | odd, near, other)
        exact = exact.astype(target)
    assert np.finfo(np.longdouble).nmant >= 63
    np.testing.assert_array_equal(gpu["v"], exact)


# ---- refusals -------------------------------------------------------------------------------------------------

def test_a_refused_node_leaves_its_results_alone(interface):
    """The second result is an operand, or the first: the first one, an array of another shape, is as it was."""
    from charmnumeric_b200 import wire
    from charmnumeric_b200._lib import CnError
    ctx = interface.context
    keep = np.arange(5.0, dtype=np.float32)
    ctx.put(880400, np.ones((2, 3, 4), np.float32))
    ctx.put(880401, np.ones((4, 2), np.float32))
    ctx.put(880402, keep)
    x, w, none = (wire.leaf(880400, (2, 3, 4), wire.F32), None), (wire.leaf(880401, (4, 2), wire.F32), None), (wire.scalar(0.0), None)
    flat = (wire.leaf(880402, (5,), wire.F32), None)
    noop = lambda name: wire.Ast(name, wire.OP_NOOP, shape=(1,), dtype=wire.F32)  # noqa: E731
    conv = wire.Ast(880402, wire.OP_CAUSAL_CONV, shape=(1,), dtype=wire.F32, operands=[x, w, none, none, none, none])
    norm = wire.Ast(880402, wire.OP_RMS_NORM, shape=(1,), dtype=wire.I8, operands=[x, none, none, none, (wire.scalar(4.0), None)])
    draw = wire.Ast(880403, wire.OP_SAMPLE, shape=(1,), dtype=wire.I32, operands=[flat, (wire.leaf(880404, (1,), wire.F32), None)] + [none] * 4)
    ctx.put(880404, np.zeros(1, np.float32))
    for roots in ([conv, noop(880401)], [conv, noop(880402)], [norm, noop(880400)], [draw, noop(880402)]):
        with pytest.raises(CnError) as e:
            ctx.run([wire.Node(0, roots, fusible=False)])
        assert e.value.status == 11
        bits(ctx.get(880402), keep)
    for name in (880400, 880401, 880402, 880404):
        ctx.delete_array(name)


# ---- a rank's part --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n", [1, 2, 7, 1000, 4099])
def test_a_rank_converts_its_part_of_a_vector(n):
    """Each of two ranks' contexts alone: converting needs nothing of the other."""
    from charmnumeric_b200 import wire
    x = np.arange(n) * 0.37 - 5
    parts = []
    for rank in range(2):
        ctx = cnp.Context(device=0, rank=rank, nranks=2)
        try:
            ctx.put(1, x)
            for name, code in ((2, wire.F16), (3, wire.I32)):
                ctx.run([wire.Node(0, [wire.Ast(name, wire.OP_CONVERT, shape=(n,), dtype=code,
                                                operands=[(wire.leaf(1, (n,), wire.F64), None), (wire.scalar(0.0), None), (wire.scalar(0.0), None)])],
                                   fusible=False)])
            ctx.synchronize()
            (begin, end), half = ctx.get_local(2)
            _, whole = ctx.get_local(3)
            bits(half, x[begin:end].astype(np.float16))
            bits(whole, x[begin:end].astype(np.int32))
            parts.append(half)
        finally:
            ctx.close()
    if n > 1:
        bits(np.concatenate(parts), x.astype(np.float16))


@pytest.mark.parametrize("rows", [2, 5, 8])
def test_a_rank_works_on_its_rows(rows):
    """The operators on two ranks' contexts without parameters to gather: each has its rows of the results."""
    from charmnumeric_b200 import wire
    rng = np.random.default_rng(rows)
    x, u = rng.standard_normal((rows, 300)).astype(np.float32), rng.random(rows).astype(np.float32)
    whole = S.rms_norm(x, None, None, 1e-6, 0)[0]
    token = S.sample(x, u, 1.0, 5, 1.0, 0.0)[0]
    q, s = S.rms_norm(x, None, None, 1e-6, 100)
    for rank in range(2):
        ctx = cnp.Context(device=0, rank=rank, nranks=2)
        try:
            ctx.put(1, x)
            ctx.put(2, u)
            none, lit = (wire.scalar(0.0), None), lambda v: (wire.scalar(v), None)  # noqa: E731
            ax, au = (wire.leaf(1, x.shape, wire.F32), None), (wire.leaf(2, u.shape, wire.F32), None)
            noop = lambda name, shape, code: wire.Ast(name, wire.OP_NOOP, shape=shape, dtype=code)  # noqa: E731
            nodes = [wire.Node(0, [wire.Ast(3, wire.OP_RMS_NORM, shape=x.shape, dtype=wire.F32, operands=[ax, none, none, lit(1e-6), none])], fusible=False),
                     wire.Node(1, [wire.Ast(4, wire.OP_SAMPLE, shape=(rows,), dtype=wire.I32, operands=[ax, au, lit(1.0), lit(5.0), lit(1.0), none]),
                                   noop(5, (rows,), wire.F32)], fusible=False),
                     wire.Node(2, [wire.Ast(6, wire.OP_RMS_NORM, shape=x.shape, dtype=wire.I8, operands=[ax, none, none, lit(1e-6), lit(100.0)]),
                                   noop(7, (rows, 3), wire.F32)], fusible=False),
                     wire.Node(3, [wire.Ast(8, wire.OP_CONVERT, shape=x.shape, dtype=wire.F32, operands=[
                         (wire.leaf(6, x.shape, wire.I8), None), (wire.leaf(7, (rows, 3), wire.F32), None), lit(100.0)])], fusible=False)]
            ctx.run(nodes)
            ctx.synchronize()
            (b, e), y = ctx.get_local(3)
            np.testing.assert_allclose(y, whole[b:e], rtol=30 * 2.0 ** -24)
            np.testing.assert_array_equal(ctx.get_local(4)[1], token[b:e])
            bits(ctx.get_local(6)[1], q[b:e])
            got = ctx.get_local(7)[1]
            np.testing.assert_allclose(got, s[b:e], rtol=30 * 2.0 ** -24)
            np.testing.assert_array_equal(ctx.get_local(8)[1], ctx.get_local(6)[1] * np.repeat(got, 100, -1))
        finally:
            ctx.close()


# ---- steps and other libraries' memory ------------------------------------------------------------------------

def test_a_step_built_by_a_helper(interface):
    """Its operands are results that nothing has computed yet when the helper returns."""
    rng = np.random.default_rng(5)
    x, w = rng.standard_normal((3, 40)), rng.standard_normal((40,))

    def helper():
        h, s = cnp.asarray(x) * 2.0 + 1.0, cnp.exp(cnp.asarray(w))
        return cnp.record(lambda: cnp.rms_norm(h, s))
    step = helper()
    want = S.rms_norm(x * 2.0 + 1.0, np.exp(w), None, 1e-6, 0)[0]
    for _ in range(3):
        np.testing.assert_allclose(step.run(interface).get(interface), want, rtol=1e-13)


def test_a_step_that_lets_go_of_its_input(interface):
    x = np.random.default_rng(6).standard_normal((3, 40))
    h = cnp.asarray(x)
    cnp.execute(interface)

    def fn():
        nonlocal h
        h = cnp.rms_norm(h)
        return h
    step = cnp.record(fn)
    want = S.rms_norm(x, None, None, 1e-6, 0)[0]
    for _ in range(3):
        np.testing.assert_allclose(step.run(interface).get(interface), want, rtol=1e-13)


def test_scales_keep_their_group(interface):
    """Groups of 30 of 100 columns make as many scales as groups of 25."""
    x = np.random.default_rng(7).standard_normal((5, 100)).astype("float32")

    def program():
        q, s = cnp.rms_norm(cnp.asarray(x), bits=8, group=30)
        return {"q": q, "s": s, "v": cnp.dequantize(q, s), "copy": cnp.dequantize(q, s.copy()),
                "view": cnp.dequantize(q, s[:]), "wide": cnp.dequantize(q, s.astype("float64"), dtype="float32")}
    gpu, _ = run_both(interface, program)
    want = gpu["q"] * np.repeat(gpu["s"], 30, -1)[:, :100]
    for k in ("v", "copy", "view", "wide"):
        np.testing.assert_array_equal(gpu[k], want, err_msg=k)


@pytest.mark.parametrize("named", ["argument", "interface"])
def test_device_memory_made_on_another_stream(interface, named):
    import torch
    side = torch.cuda.Stream()
    t = torch.zeros(1 << 22, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)                # some 25 ms
        t += 3
        if named == "argument":
            a = cnp.from_device(interface, t, stream=side.cuda_stream)
        else:
            class Named:
                __cuda_array_interface__ = dict(t.__cuda_array_interface__, version=3, stream=side.cuda_stream)
            a = cnp.from_device(interface, Named())
        t.zero_()                                      # behind the copy
    assert (a.get(interface) == 3).all()
    side.synchronize()


# ---- sample -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float32", "float64"])
def test_sample_logits_and_temperatures_at_the_end_of_a_type(interface, dtype):
    """Logits as large as the type's values over temperatures as large: a few powers of e from end to end, which
    in the units of the logits leave the type's range."""
    most = float(np.finfo(dtype).max)
    rng = np.random.default_rng(23)
    v = 6000
    span = np.linspace(-1, 1, v)
    x = (most * np.stack([span, rng.permutation(span), rng.uniform(-1, 1, v), rng.uniform(-1, 0.25, v)])).astype(dtype)
    u = np.array([0.2, 0.99, 0.9999, 0.5], dtype)
    sets = [(most / over, k, p, 0.0) for over in (1.0, 3.4, 10.0, 30.0) for k, p in ((0, 0.9), (0, 0.999), (0, 0.9999), (3000, 1.0), (5500, 0.9999))]

    def program():
        out, ax, au = {}, cnp.asarray(x), cnp.asarray(u)
        for i, (t, k, p, m) in enumerate(sets):
            out[f"t{i}"], out[f"p{i}"] = cnp.random.sample(ax, au, temperature=t, top_k=k, top_p=p, min_p=m)
        return out
    gpu, _ = run_both(interface, program)
    for i, f in enumerate(sets):
        check_samples(x, gpu[f"t{i}"], gpu[f"p{i}"], u, *f)
