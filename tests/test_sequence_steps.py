"""CPU tests of recorded steps: what a step uses exists when it runs, and is released with it."""
import gc

import pytest

import charmnumeric_b200 as cnp
from charmnumeric_b200 import frontend as F, wire


def leaves(node):
    return {leaf.result_name for root in node.roots for leaf, _ in root.operands if isinstance(leaf, wire.Ast) and not leaf.is_scalar}


class Backend:
    """An interface and its context that keep the names of the arrays a backend would have."""

    def __init__(self):
        self.context = self
        self.arrays, self.steps = set(), 0

    def run(self, nodes, deletes=()):
        for node in nodes:
            assert leaves(node) <= self.arrays
            self.arrays |= {r.result_name for r in node.roots if not r.is_temp and r.opcode != wire.OP_SET_REGION}
        self.arrays -= set(deletes)

    def put(self, name, host):
        self.arrays.add(name)

    def receive_dag(self, blob):
        self.steps += 1


def record(fn, monkeypatch):
    """cnp.record, and the names of the arrays that the step reads and does not make."""
    nodes, build = [], F.build_nodes

    def watch(ops):
        items = build(ops)
        nodes.extend(node for _, node in items)
        return items
    with monkeypatch.context() as m:
        m.setattr(F, "build_nodes", watch)
        step = cnp.record(fn)
    made = {r.result_name for node in nodes for r in node.roots}
    return step, set().union(*(leaves(node) for node in nodes)) - made


def test_a_step_keeps_results_that_are_not_made_yet(monkeypatch):
    """The operands of a step that a helper returns: pending elementwise results without a handle."""
    backend = Backend()

    def helper():
        x, w = cnp.asarray([[1.0, 2.0], [3.0, 4.0]]) * 2.0 + 1.0, cnp.exp(cnp.ones((2,)))
        return record(lambda: cnp.rms_norm(x, w), monkeypatch)
    step, used = helper()
    gc.collect()
    assert len(used) == 2
    for _ in range(2):
        step.run(backend)
        assert used <= backend.arrays
    assert backend.steps == 2
    del step
    gc.collect()
    cnp.execute(backend)
    assert not used & backend.arrays


def test_a_step_keeps_what_its_function_lets_go_of(monkeypatch):
    """`h = rms_norm(h)` inside: the last handle on the operand goes while the step is recorded."""
    backend = Backend()
    h = cnp.asarray([[1.0, 2.0], [3.0, 4.0]])
    cnp.execute(backend)

    def fn():
        nonlocal h
        h = cnp.rms_norm(h)
        gc.collect()
        return h
    step, used = record(fn, monkeypatch)
    assert len(used) == 1
    for _ in range(2):
        step.run(backend)
        assert used <= backend.arrays
    del step
    gc.collect()
    cnp.execute(backend)
    assert not used & backend.arrays


def test_a_step_does_not_run_while_another_is_recorded():
    """It would run once, then and there, and not be part of the recorded step."""
    backend = Backend()
    x = cnp.asarray([[1.0, 2.0], [3.0, 4.0]])
    inner = cnp.record(lambda: cnp.rms_norm(x))
    cnp.execute(backend)
    with pytest.raises(RuntimeError):
        cnp.record(lambda: inner.run(backend))
    assert backend.steps == 0 and not F._state.recording
    inner.run(backend)
    assert backend.steps == 1
