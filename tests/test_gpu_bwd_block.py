"""A transformer block's backward pass on the GPU through sdvk_amd.ops (tests/bwd_block.py): against 64 bits and against
differences; on streams of its own, two at once; captured into graphs that are replayed between eager passes."""
import numpy as np
import pytest

import bwd_block
from bwd_block import RESULTS, Block, Device
from sdvk_amd import ops
from sdvk_amd.hip import Graph, Stream, synchronize
from test_gpu_bwd import Backend

pytestmark = pytest.mark.gpu


@pytest.fixture
def backend(gpu):
    ops.tuning_reset()
    return Backend(gpu)


@pytest.mark.parametrize("op", list(bwd_block.OPS))
def test_block(backend, op):
    print(op, flush=True)
    bwd_block.OPS[op](backend)


def device(backend, seed):
    blk = Block(seed)
    stages = blk.forward(blk.x, blk.ctx)
    return blk, Device(backend, ops, blk, stages), blk.backward(stages, blk.dy.astype(np.float64))


def clear(dev):
    for k in RESULTS + bwd_block.INNER:
        dev.out[k].b.upload(np.full(dev.n[k], np.nan, np.float32))
    dev.ws.handle.b.upload(np.full(dev.ws.nbytes, 0xff, np.uint8))


def same(a, b):
    return all(np.array_equal(a[k].view(np.uint32), b[k].view(np.uint32)) for k in RESULTS)


def test_streams(backend):
    """Two passes at once, each on a stream and with a workspace of its own, give the bits that each gives alone."""
    runs = [device(backend, s) for s in (21, 22)]
    alone = []
    for blk, dev, want in runs:
        dev.backward()
        alone.append(dev.results())
        bwd_block.check_block(blk, alone[-1], want)
        clear(dev)
    streams = [Stream() for _ in runs]
    synchronize()
    for (_, dev, _), st in zip(runs, streams):
        dev.backward(stream=st)
    for st in streams:
        st.synchronize()
    for (_, dev, _), first in zip(runs, alone):
        assert same(dev.results(), first)


def test_graphs(backend):
    """Two graphs that share one workspace and one stream, replayed in turn, with eager passes in between: every replay
    gives the eager pass's bits, also after the inputs have changed in place."""
    st = Stream()
    runs = [device(backend, s) for s in (31, 32)]
    big = max((d for _, d, _ in runs), key=lambda d: d.ws.nbytes).ws
    eager, graphs = [], []
    for blk, dev, want in runs:
        dev.ws = big
        dev.backward(stream=st)
        st.synchronize()
        eager.append(dev.results())
        bwd_block.check_block(blk, eager[-1], want)
        g = Graph(st)
        g.begin()
        dev.backward(stream=st)
        g.end()
        graphs.append(g)
    for _ in range(3):
        for (_, dev, _), g, first in zip(runs, graphs, eager):
            clear(dev)
            g.launch()
            st.synchronize()
            assert same(dev.results(), first)
            dev.backward(stream=st)  # eager work between the replays
            st.synchronize()
            assert same(dev.results(), first)
    for (blk, dev, _), g in zip(runs, graphs):
        blk.dy = -2 * blk.dy  # exact: every gradient follows
        dev.dy.b.upload(blk.dy.reshape(-1))
        g.launch()
        st.synchronize()
        got = dev.results()
        dev.backward(stream=st)
        st.synchronize()
        assert same(dev.results(), got)
    for (_, dev, _), first in zip(runs, eager):
        got = dev.results()
        assert all(np.allclose(got[k], -2 * first[k], rtol=1e-3, atol=1e-3 * np.abs(first[k]).max()) for k in RESULTS)
