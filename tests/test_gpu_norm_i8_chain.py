"""The GroupNorm and 8-bit operators run together on the GPU through sdvk_amd.ops (tests/norm_i8_chain.py): against 64 bits; on streams
of their own, two at once; captured into graphs that share a workspace and are replayed between eager runs."""
import numpy as np
import pytest

import norm_i8_chain
from norm_i8_chain import Chain
from sdvk_amd import ops
from sdvk_amd.hip import Graph, Stream, synchronize
from test_gpu_bwd import Backend

pytestmark = pytest.mark.gpu

SIZES = [dict(), dict(B=2, P=1024, C=640, F=2560, N=640), dict(B=1, P=333, C=320, F=1280, N=328)]


@pytest.fixture
def backend(gpu):
    ops.tuning_reset()
    return Backend(gpu)


def put(handle, arr):
    handle.b.upload(np.ascontiguousarray(arr))


def same(a, b):
    return [n for n in a if not np.array_equal(a[n].view(np.uint8), b[n].view(np.uint8))] == []


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_chain(backend, size):
    print(size, flush=True)
    norm_i8_chain.chain(backend, **size)


def test_streams(backend):
    """Two runs at once, each on a stream and with a workspace of its own, give the bits that each gives alone."""
    runs = [Chain(backend, ops, seed=s, **size) for s, size in ((21, SIZES[2]), (22, dict(B=2, P=256, C=640, F=640, N=320)))]
    alone = []
    for c in runs:
        c.reset(put)
        c.run()
        alone.append(c.results())
        c.check(alone[-1])
        c.reset(put)
    streams = [Stream() for _ in runs]
    synchronize()
    for c, st in zip(runs, streams):
        c.run(stream=st)
    for st in streams:
        st.synchronize()
    for c, first in zip(runs, alone):
        assert same(c.results(), first)


def test_graphs(backend):
    """Two graphs that share one workspace and one stream, replayed in turn, with eager runs in between: every replay gives the eager
    run's bits, also after the inputs have changed in place."""
    st = Stream()
    runs = [Chain(backend, ops, seed=s, **size) for s, size in ((31, dict(B=1, P=300, C=320, F=320, N=64)), (32, dict()))]
    big = max(runs, key=lambda c: c.ws.nbytes).ws
    eager, graphs = [], []
    for c in runs:
        c.ws = big
        c.reset(put)
        c.run(stream=st)
        st.synchronize()
        eager.append(c.results())
        c.check(eager[-1])
        g = Graph(st)
        g.begin()
        c.run(stream=st)
        g.end()
        graphs.append(g)
    for _ in range(3):
        for c, g, first in zip(runs, graphs, eager):
            c.reset(put)
            g.launch()
            st.synchronize()
            assert same(c.results(), first)
            c.reset(put)
            c.run(stream=st)  # eager work between the replays
            st.synchronize()
            assert same(c.results(), first)
    for c, g in zip(runs, graphs):
        c.x, c.x16 = c.x[:, ::-1].copy(), -c.x16
        put(c.dev["x"], c.x.reshape(-1))
        put(c.dev["x16"], c.x16.reshape(-1))
        c.reset(put)
        g.launch()
        st.synchronize()
        got = c.results()
        c.check(got)
        c.reset(put)
        c.run(stream=st)
        st.synchronize()
        assert same(c.results(), got)
