"""Calls captured into a HIP graph: norms, dropout and joints whose results need no workspace, replayed on new inputs with
eager work between the replays.  The dropout draws its capture's mask at every replay.  A backward that needs a workspace is
refused and leaves the capture as it was.

The context's stream joins a capture by waiting for an event of the capturing stream (orca_hip_event_wait), and that stream
waits for an event of the context's (orca_hip_event_record) before the capture ends."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from orcaml_amd import _lib
from tests.test_gpu_norm import Joint, Matrix, params, stream

pytestmark = pytest.mark.gpu

THREAD_LOCAL, DISABLE_TIMING = 1, 2  # hipStreamCaptureModeThreadLocal, hipEventDisableTiming


class Capture:
    """A stream of the HIP runtime that the library runs on, and a graph captured from it."""

    def __init__(self, ctx):
        _lib.load()
        path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
        self.ctx, self.hip, self.graph, self.exec = ctx, ctypes.CDLL(path), ctypes.c_void_p(), ctypes.c_void_p()
        self.stream, self.event = ctypes.c_void_p(), ctypes.c_void_p()
        self.call("hipStreamCreateWithFlags", ctypes.byref(self.stream), 1)  # non-blocking
        self.call("hipEventCreateWithFlags", ctypes.byref(self.event), DISABLE_TIMING)

    def call(self, name, *args):
        rc = getattr(self.hip, name)(*args)
        assert rc == 0, (name, rc)

    def __enter__(self):
        self.ctx.sync()
        self.call("hipStreamBeginCapture", self.stream, THREAD_LOCAL)
        self.call("hipEventRecord", self.event, self.stream)
        self.ctx.event_wait(self.event.value)
        return self

    def __exit__(self, *exc):
        mark = self.ctx.event_record()
        self.call("hipStreamWaitEvent", self.stream, ctypes.c_void_p(mark), 0)
        self.call("hipStreamEndCapture", self.stream, ctypes.byref(self.graph))
        self.ctx.event_release(mark)
        self.call("hipGraphInstantiate", ctypes.byref(self.exec), self.graph, None, None, ctypes.c_size_t(0))

    def replay(self):
        self.ctx.sync()  # the inputs are there
        self.call("hipGraphLaunch", self.exec, self.stream)
        self.call("hipStreamSynchronize", self.stream)

    def close(self):
        self.call("hipGraphExecDestroy", self.exec)
        self.call("hipGraphDestroy", self.graph)
        self.call("hipEventDestroy", self.event)
        self.call("hipStreamDestroy", self.stream)


@pytest.fixture
def own():
    from orcaml_amd.device import Context
    c = Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("n", [300, 1003, 2600, 9000])
def test_forwards_and_a_short_backward(own, n):
    print(f"capture {n}", flush=True)
    ctx, rng = own, np.random.default_rng(n)
    j = Joint(ctx, n, 6, n, "rms", "layer", 1, 0.3)
    short = n <= 1024  # up to 8 rows in one block, without partial sums
    d, p = j.dev, params("layer", None, None)
    x = d["x"]

    def calls(o):
        """The same work into other results; the backward's without gradients that need partial sums."""
        _lib.call("orca_hip_residual_norm", ctx.handle, 6, n, x.ptr, n, d["f"].ptr, n, ctypes.byref(j.block), o["y"].ptr, n,
                  o["u"].ptr, n, None)
        _lib.call("orca_hip_dropout", ctx.handle, 6, n, x.ptr, n, 0.3, j.seed, j.offset, o["drop"].ptr, n)
        _lib.call("orca_hip_norm", ctx.handle, 6, n, o["y"].ptr, n, ctypes.byref(p), o["norm"].ptr, n, None)
        if short:
            _lib.call("orca_hip_norm_backward", ctx.handle, 6, n, d["dy"].ptr, n, x.ptr, n, ctypes.byref(p), d["du"].ptr, n,
                      o["dx"].ptr, n, o["dw"].ptr, None)

    def results():
        return {k: j.matrix(rows=1 if k == "dw" else 6) for k in ("y", "u", "drop", "norm", "dx", "dw")}

    captured, eager = results(), results()
    calls(eager)  # what is loaded at a first call is
    many = Matrix(ctx, 3000, 64, stream(rng, 3000, 64))
    dw = ctx.alloc(4 * 64)
    graph = Capture(ctx)
    with graph:
        calls(captured)
        with pytest.raises(_lib.OrcaHipError, match="captured graph"):
            _lib.call("orca_hip_norm_backward", ctx.handle, 3000, 64, many.ptr, 64, many.ptr, 64, ctypes.byref(p), None, 0,
                      None, 0, dw.ptr, None)
    masks = []
    for _ in range(4):
        x.buf.upload(stream(rng, 6, n, 9.0).reshape(-1))  # no zeros among them
        calls(eager)
        want = {k: m.buf.download() for k, m in eager.items()}
        graph.replay()
        for k, m in captured.items():
            np.testing.assert_array_equal(m.buf.download(), want[k], err_msg=k)
        masks.append(captured["drop"].read() == 0)
        _lib.call("orca_hip_norm_backward", ctx.handle, 3000, 64, many.ptr, 64, many.ptr, 64, ctypes.byref(p), None, 0, None,
                  0, dw.ptr, None)  # eager work with a workspace between the replays
    assert masks[0].any() and not masks[0].all() and all((m == masks[0]).all() for m in masks)
    graph.close()
