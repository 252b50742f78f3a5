"""Recorded steps: a piece of a program that is built once and run many times.

``record(fn)`` calls ``fn``, keeps what it recorded instead of executing it, and returns a ``Step``.
Each ``Step.run`` submits the same DAG bytes again, which the backend recognises (no parsing, no
lowering, no new arrays): the cheap path of a time-step or decoding loop.  What a step reads it reads
anew each time, and its results are the same arrays each time.
"""
import weakref

from . import wire
from . import frontend as F


def _unpin(infos):
    for info in infos:
        info.pins -= 1
        if not info.pins and not info.alive and info.materialised:
            F._state.dead.append(info.name)


class Step:
    """A recorded step.  ``results`` is what the recorded function returned."""

    def __init__(self, nodes, infos, results):
        self.results = results
        self._blob = wire.dag_blob(nodes)
        for info in infos:
            info.pins += 1
        # one that the recorded function let go of waits to be released: _unpin does that now
        kept = {info.name for info in infos}
        F._state.dead[:] = [name for name in F._state.dead if name not in kept]
        weakref.finalize(self, _unpin, infos)

    def run(self, interface):
        """Run the step once (asynchronously), after everything recorded before."""
        if F._state.pending or F._state.dead or F._state.recording:    # which execute refuses
            F.execute(interface)
        interface.context.receive_dag(self._blob)
        return self.results


def record(fn):
    """The operations that ``fn()`` records, as a ``Step``.  It must not upload host data,
    and nothing can be executed or fetched inside, nor another step run."""
    outer, F._state.pending = F._state.pending, []
    flush, F._state.auto_flush = F._state.auto_flush, None
    within, F._state.recording = F._state.recording, True
    try:
        results = fn()
        ops = F._state.pending
    finally:
        F._state.pending, F._state.auto_flush, F._state.recording = outer, flush, within
    if any(op.kind == "put" for op in ops):
        raise ValueError("a recorded step uploads host data: make its arrays before")
    infos = {}
    for op in ops:
        used = [info for info, _ in F._op_views(op)] + list(op.payload if op.kind == "seq" else [op.result])
        infos.update((info.name, info) for info in used if info is not None)
    nodes = [item for _, item in F.build_nodes(ops)]
    return Step(nodes, list(infos.values()), results)
