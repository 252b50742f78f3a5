"""CPU tests of the sequence model operators' frontend: refusals, what is recorded, and the oracle
behind the same programs."""
import numpy as np
import pytest

import charmnumeric_b200 as cnp
from charmnumeric_b200 import frontend as F, wire
from tests.helpers import run_oracle


def z(*shape, dtype="float32"):
    return cnp.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call,error", [
    (lambda: cnp.rms_norm(z(3, 4, dtype="int32")), TypeError),
    (lambda: cnp.rms_norm(z(3, 4, dtype="int8")), TypeError),
    (lambda: cnp.rms_norm(z(3, 0)), ValueError),
    (lambda: cnp.rms_norm(z(3, 4), z(5)), ValueError),
    (lambda: cnp.rms_norm(z(3, 4), z(4, dtype="float64")), TypeError),
    (lambda: cnp.rms_norm(z(3, 4), residual=z(3, 5)), ValueError),
    (lambda: cnp.rms_norm(z(3, 4), residual=z(3, 4, dtype="float16")), TypeError),
    (lambda: cnp.rms_norm(z(3, 4), eps=-1.0), ValueError),
    (lambda: cnp.rms_norm(z(3, 4), eps=float("nan")), ValueError),
    (lambda: cnp.rms_norm(z(3, 4), bits=4), ValueError),
    (lambda: cnp.rms_norm(z(3, 4), group=2), ValueError),
    (lambda: cnp.rms_norm(z(3, 4), bits=8, group=0), ValueError),
    (lambda: cnp.rms_norm(z(3, 4), bits=8, group=5), ValueError),
    (lambda: cnp.rms_norm(z(3, 4), bits=8, group=2.0), ValueError),
    (lambda: cnp.dequantize(z(3, 4), z(3, 1)), TypeError),
    (lambda: cnp.dequantize(z(3, 4, dtype="int8"), z(3, 3)), ValueError),
    (lambda: cnp.dequantize(z(3, 4, dtype="int8"), z(2, 1)), ValueError),
    (lambda: cnp.dequantize(z(3, 4, dtype="int8"), z(3, 2), group=4), ValueError),
    (lambda: cnp.dequantize(z(3, 4, dtype="int8"), z(3, 2), dtype="int32"), TypeError),
    (lambda: cnp.causal_conv(z(3, 4), z(4, 2)), ValueError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(5, 2)), ValueError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(4, 1)), NotImplementedError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(4, 9)), NotImplementedError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(4, 3, dtype="float64")), TypeError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(4, 3), z(3)), ValueError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(4, 3), state=z(2, 3, 4)), ValueError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(4, 3), lengths=z(2)), TypeError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(4, 3), lengths=[1, 2, 3]), ValueError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(4, 3), activation="tanh"), ValueError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(4, 3), inplace=True), ValueError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(4, 3), state=z(2, 2, 8)[:, :, ::2], inplace=True), ValueError),
    (lambda: cnp.causal_conv(z(2, 3, 4), z(4, 3), state=np.zeros((2, 2, 4)), inplace=True), ValueError),
    (lambda: cnp.selective_scan(z(2, 3), z(2, 3), z(3, 2), z(2, 2), z(2, 2)), ValueError),
    (lambda: cnp.selective_scan(z(2, 3, 4), z(2, 3, 5), z(4, 2), z(2, 3, 2), z(2, 3, 2)), ValueError),
    (lambda: cnp.selective_scan(z(2, 3, 4), z(2, 3, 4), z(5, 2), z(2, 3, 2), z(2, 3, 2)), ValueError),
    (lambda: cnp.selective_scan(z(2, 3, 4), z(2, 3, 4), z(4, 2), z(2, 3, 3), z(2, 3, 3)), ValueError),
    (lambda: cnp.selective_scan(z(2, 3, 4), z(2, 3, 4), z(4, 2), z(2, 3, 6), z(2, 3, 6)), ValueError),
    (lambda: cnp.selective_scan(z(2, 3, 4), z(2, 3, 4), z(4, 2), z(2, 3, 2), z(2, 3, 4)), ValueError),
    (lambda: cnp.selective_scan(z(2, 3, 4), z(2, 3, 4), z(4, 257), z(2, 3, 257), z(2, 3, 257)), NotImplementedError),
    (lambda: cnp.selective_scan(*[z(2, 3, 4, dtype="float16")] * 2, z(4, 2, dtype="float64"), *[z(2, 3, 2, dtype="float16")] * 2), TypeError),
    (lambda: cnp.selective_scan(*[z(2, 3, 4)] * 2, z(4, 2), *[z(2, 3, 2)] * 2, state=z(2, 4, 3)), ValueError),
    (lambda: cnp.selective_scan(*[z(2, 3, 4)] * 2, z(4, 2), *[z(2, 3, 2)] * 2, inplace=True), ValueError),
    (lambda: cnp.random.sample(z(2, 3, 4), z(2)), ValueError),
    (lambda: cnp.random.sample(z(2, 4, dtype="int32"), z(2)), TypeError),
    (lambda: cnp.random.sample(z(2, 0), z(2)), ValueError),
    (lambda: cnp.random.sample(z(2, 4), z(3)), ValueError),
    (lambda: cnp.random.sample(z(2, 4), z(2, dtype="int32")), TypeError),
    (lambda: cnp.random.sample(z(2, 4), z(2), temperature=-1.0), ValueError),
    (lambda: cnp.random.sample(z(2, 4), z(2), temperature=float("nan")), ValueError),
    (lambda: cnp.random.sample(z(2, 4), z(2), top_k=-1), ValueError),
    (lambda: cnp.random.sample(z(2, 4), z(2), top_k=1.5), ValueError),
    (lambda: cnp.random.sample(z(2, 4), z(2), top_k=z(2)), TypeError),
    (lambda: cnp.random.sample(z(2, 4), z(2), top_p=1.5), ValueError),
    (lambda: cnp.random.sample(z(2, 4), z(2), min_p=-0.5), ValueError),
    (lambda: cnp.random.sample(z(2, 4), z(2), min_p=z(3)), ValueError),
    (lambda: z(3, dtype="float16") + 1, TypeError),
    (lambda: 2.0 * z(3, dtype="int8"), TypeError),
    (lambda: cnp.exp(z(3, dtype="float16")), TypeError),
    (lambda: cnp.sum(z(3, dtype="float16")), TypeError),
    (lambda: z(3, dtype="float16") @ z(3, dtype="float16"), TypeError),
    (lambda: z(3, 3, dtype="float16") @ z(3), TypeError),
    (lambda: cnp.random.uniform((3,), dtype="float16"), TypeError),
    (lambda: z(3).__setitem__(slice(None), z(3, dtype="float16")), TypeError),
    (lambda: z(3, dtype="float16").__setitem__(slice(None), z(2, dtype="float16")), ValueError),
    (lambda: cnp.zeros((3,), dtype="uint8"), TypeError),
    (lambda: cnp.from_device(None, np.zeros(3)), TypeError),
    (lambda: cnp.record(lambda: cnp.asarray([1.0, 2.0]) + 1), ValueError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def test_node_layout():
    """One root with the operands in order, a literal for each that is left out, then the results."""
    x, w = z(3, 40, dtype="float16"), z(40, dtype="float16")
    F._state.pending = []
    q, s, h = cnp.rms_norm(x, w, residual=x, bits=8, group=16, eps=0.25)
    (kind, node), = F.build_nodes(F._state.pending)
    assert kind == "node" and not node.fusible
    main, scale, total = node.roots
    assert (main.opcode, main.dtype, main.shape) == (wire.OP_RMS_NORM, wire.I8, (3, 40))
    assert [o.is_scalar for o, _ in main.operands] == [False, False, False, True, True]
    assert [o.scalar for o, _ in main.operands[3:]] == [0.25, 16.0]
    assert (scale.opcode, scale.dtype, scale.shape, scale.result_name) == (wire.OP_NOOP, wire.F32, (3, 3), s.name)
    assert (total.dtype, total.shape, total.result_name) == (wire.F16, (3, 40), h.name)
    assert cnp.dag_check(wire.dag_blob([node])) == (1, 3)


def test_the_longest_operand_list_parses_and_a_longer_one_does_not():
    F._state.pending = []
    cnp.selective_scan(z(2, 3, 4), z(2, 3, 4), z(4, 2), z(2, 3, 2), z(2, 3, 2), D=z(4), z=z(2, 3, 4), delta_bias=z(4),
                       state=z(2, 4, 2), lengths=z(2, dtype="int32"))
    nodes = [n for _, n in F.build_nodes(F._state.pending)]
    assert cnp.dag_check(wire.dag_blob(nodes))[0] == len(nodes)
    nodes[-1].roots[0].operands *= 2
    with pytest.raises(cnp._lib.CnError):
        cnp.dag_check(wire.dag_blob(nodes))


def test_programs_on_the_oracle():
    """The four operators through the frontend against independent arithmetic, in 64 bits."""
    rng = np.random.default_rng(0)
    x, r, w = rng.standard_normal((3, 20)), rng.standard_normal((3, 20)), rng.standard_normal(20)
    got = run_oracle(lambda: dict(zip("yh", cnp.rms_norm(cnp.asarray(x), cnp.asarray(w), residual=cnp.asarray(r), eps=0.0))))
    h = x + r
    np.testing.assert_allclose(got["y"], h / np.linalg.norm(h, axis=1, keepdims=True) * np.sqrt(20) * w, rtol=1e-13)
    np.testing.assert_array_equal(got["h"], h)

    seq, filt = rng.standard_normal((1, 9, 2)), rng.standard_normal((2, 4))
    got = run_oracle(lambda: dict(zip("ys", cnp.causal_conv(cnp.asarray(seq), cnp.asarray(filt)))))
    for c in range(2):
        np.testing.assert_allclose(got["y"][0, :, c], np.convolve(seq[0, :, c], filt[c, ::-1])[:9], rtol=1e-12)
    np.testing.assert_array_equal(got["s"], seq[:, 6:])

    # constant coefficients: a geometric series
    ones = np.ones((1, 6, 1))
    got = run_oracle(lambda: dict(zip("ys", cnp.selective_scan(*(cnp.asarray(v) for v in (ones, ones * 0.5, np.array([[-1.0]]), ones, ones)), softplus=False))))
    q = np.exp(-0.5)
    np.testing.assert_allclose(got["y"].ravel(), [0.5 * (1 - q ** (i + 1)) / (1 - q) for i in range(6)], rtol=1e-13)

    p = np.array([0.1, 0.4, 0.2, 0.3])
    for u, kw, want in [(0.05, {}, 0), (0.3, {}, 1), (0.65, {}, 2), (0.95, {}, 3), (0.05, {"top_k": 2}, 1), (0.6, {"top_k": 2}, 3),
                        (0.5, {"top_p": 0.35}, 1), (0.9, {"top_p": 0.6}, 3), (0.4, {"min_p": 0.6}, 1), (0.99, {"temperature": 0}, 1)]:
        got = run_oracle(lambda: dict(zip("tp", cnp.random.sample(cnp.asarray(np.log(p)), u, **kw))))
        assert got["t"][0] == want, (u, kw)


def test_astype_between_types():
    x = np.array([[1.5, -2.25], [1e-8, 70000.0]])
    with np.errstate(over="ignore"):
        got = run_oracle(lambda: {"h": cnp.asarray(x).astype("float16"), "back": cnp.asarray(x).astype("float16").astype("float64")})
        np.testing.assert_array_equal(got["h"], x.astype("float16"))
    np.testing.assert_array_equal(got["back"], x.astype("float16").astype("float64"))


def test_scan_is_linear_in_its_input_matrix():
    rng = np.random.default_rng(7)
    a = [rng.standard_normal(s) for s in ((1, 5, 2), (1, 5, 2))] + [-np.abs(rng.standard_normal((2, 3)))] + [rng.standard_normal((1, 5, 3)) for _ in range(2)]
    y = lambda v: run_oracle(lambda: {"y": cnp.selective_scan(*(cnp.asarray(t) for t in v))[0]})["y"]  # noqa: E731
    twice = y(a[:3] + [2 * a[3], a[4]])
    np.testing.assert_allclose(twice, 2 * y(a), rtol=1e-12)


def test_storage_arrays_never_join_a_fused_group():
    F._state.pending = []
    a, h = z(8), z(8, dtype="float16")
    b = a + 1.0
    h[...] = 2
    c = b * 2.0
    nodes = [n for _, n in F.build_nodes(F._state.pending)]
    for n in nodes:
        kinds = {r.dtype for r in n.roots}
        assert len(kinds) == 1, kinds
    assert c.dtype == np.float32


def test_a_state_in_place_is_no_other_operand():
    s = z(2, 1, 4)
    with pytest.raises(ValueError):
        cnp.causal_conv(s, z(4, 2), state=s, inplace=True)
    w = z(2, 4, 4)
    with pytest.raises(ValueError):
        cnp.selective_scan(w, z(2, 4, 4), z(4, 4), z(2, 4, 4), z(2, 4, 4), state=w, inplace=True)


def test_a_recorded_step_keeps_what_it_uses():
    """Arrays of a step are released when both the program and the step have let go of them."""
    import gc
    x = z(3, 4)
    F._state.pending, F._state.dead = [], []
    x._info.materialised = True
    step = cnp.record(lambda: cnp.rms_norm(x))
    names = {x.name, step.results.name}
    del x
    gc.collect()
    assert not names & set(F._state.dead)
    step.results = None
    gc.collect()
    assert not names & set(F._state.dead)
    del step
    gc.collect()
    assert names <= set(F._state.dead)
    F._state.dead = []


def test_a_step_executes_nothing_while_it_is_recorded():
    class Nowhere:
        context = None
    F._state.pending = []
    x = z(3, 4)
    with pytest.raises(RuntimeError):
        cnp.record(lambda: cnp.execute(Nowhere()))
    with pytest.raises(RuntimeError):
        cnp.record(lambda: cnp.rms_norm(x).get(Nowhere()))
    assert not F._state.recording and len(F._state.pending) == 1    # x is still to be made
    inner = []
    outer = cnp.record(lambda: (inner.append(cnp.record(lambda: cnp.rms_norm(x))), cnp.rms_norm(x))[1])
    assert outer.results.name != inner[0].results.name and not F._state.recording
    F._state.pending, F._state.dead = [], []


def test_the_profiled_kernels_built_ahead_of_time_are_the_ones_in_the_tree():
    """A DRAM traffic capture counts for the source that it was taken from only."""
    import hashlib
    import json
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    csrc = root / "charmnumeric_b200" / "csrc"
    now = hashlib.sha256((csrc / "kernels.cu").read_bytes() + (csrc / "kernels.hpp").read_bytes()).hexdigest()[:8]
    entries = json.loads((root / "profiles" / "dram_traffic.json").read_text())["kernels"]
    assert [e["code"] for e in entries if "matvec" in e["match"]] == ["#" + now]


@pytest.mark.parametrize("value", [128, -129, 300.5, float("nan"), float("inf")])
def test_int8_arrays_are_not_filled_with_what_they_cannot_hold(value):
    with pytest.raises(OverflowError):
        cnp.full((2,), value, dtype="int8")
    a = z(2, dtype="int8")
    with pytest.raises(OverflowError):
        a[:1] = value
    a[:1] = -128
    a[1:] = 127
