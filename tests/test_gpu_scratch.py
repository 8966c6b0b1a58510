"""The scratch of ae_matmul_i8 and ae_linear_i8 (rows quantized or laid out ahead of the product): who uses it, and until
when. Every result is compared bit for bit with the same call's on its own, which test_gpu_linear_i8.py checks."""
import time

import numpy as np
import pytest
import torch

from arctic_embed_s_int8 import AeError, Engine
from conftest import rng

pytestmark = pytest.mark.gpu

N, K = 192, 1003  # contiguous rows that TMA cannot read where they are


@pytest.fixture
def eng():
    e = Engine(0)
    yield e
    e.close()


class Call:
    """A linear_i8 or, with `ints`, a matmul_i8 of M tokens, its output, and the wanted one (by an engine of its own)."""

    def __init__(self, M, seed, ints=False):
        r = rng(seed)
        self.w = torch.from_numpy(r.integers(-127, 128, (N, K), dtype=np.int8)).cuda()
        self.w_scale = torch.from_numpy(r.uniform(1e-4, 1e-3, N).astype(np.float32)).cuda()
        self.x = torch.from_numpy(r.integers(-127, 128, (M, K), dtype=np.int8) if ints else
                                  r.normal(0, 1, (M, K)).astype(np.float32)).cuda()
        self.scale = torch.from_numpy(r.uniform(1e-3, 1e-2, M).astype(np.float32)).cuda() if ints else None
        self.out = torch.empty(M, N, device="cuda")
        alone = Engine(0)
        self.run(alone)
        alone.sync()
        alone.close()
        self.want = self.out.clone()
        self.out.fill_(float("nan"))
        torch.cuda.synchronize()

    def run(self, eng):
        if self.scale is None:
            eng.linear_i8(self.x, self.w, self.w_scale, self.out)
        else:
            eng.matmul_i8(self.x, self.scale, self.w, self.w_scale, self.out)

    def right(self):
        same = torch.equal(self.out, self.want)
        self.out.fill_(float("nan"))
        return same


def captured(eng, stream, calls):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        eng.set_stream(stream)
        with torch.cuda.graph(g, stream=stream):
            for c in calls:
                c.run(eng)
    return g


def test_replay_after_larger_calls(eng):
    """A graph's replays use scratch that later calls on its stream neither free nor write."""
    s = torch.cuda.Stream()
    small, ints, large = Call(64, 1), Call(40, 2, ints=True), Call(700, 3)
    eng.set_stream(s)
    with torch.cuda.stream(s):
        small.run(eng)
        s.synchronize()
        assert small.right()
        g = captured(eng, s, [small, ints])
        for _ in range(3):
            large.run(eng)
            s.synchronize()
            assert large.right()
            taken = [torch.full((2 ** 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(8)]
            g.replay()
            large.run(eng)
            s.synchronize()
            assert small.right() and ints.right() and large.right()
            assert all((t == 7).all() for t in taken)


def test_first_call_is_the_captured_one(eng):
    """No scratch has to be there before a capture, and a capture may ask for more on its way."""
    s, calls = torch.cuda.Stream(), [Call(40, 4), Call(300, 5), Call(120, 6, ints=True)]
    torch.cuda.synchronize()
    g = captured(eng, s, calls)
    with torch.cuda.stream(s):
        for _ in range(2):
            g.replay()
            s.synchronize()
            assert all(c.right() for c in calls)


def test_graphs_of_one_stream_on_two(eng):
    """Two graphs captured on one stream replay side by side on two others."""
    s, calls = torch.cuda.Stream(), [Call(600, 7), Call(600, 8)]
    torch.cuda.synchronize()
    graphs = [captured(eng, s, [c] * 8) for c in calls]
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, t in zip(graphs, streams):
            with torch.cuda.stream(t):
                g.replay()
        torch.cuda.synchronize()
        assert all(c.right() for c in calls)


def test_release(eng):
    """A stream's block, and that of a graph once it is gone, go back to the device; the next calls take new ones."""
    s, c = torch.cuda.Stream(), Call(100000, 9)
    size = 100000 * 1008

    def free():
        torch.cuda.synchronize()
        torch.cuda.empty_cache()  # what torch keeps for itself is not meant
        return torch.cuda.mem_get_info()[0]

    eng.set_stream(s)
    c.run(eng)
    before = free()
    eng.release_scratch()
    assert free() >= before + size
    eng.release_scratch()  # nothing left
    c.run(eng)
    s.synchronize()
    assert c.right()
    eng.release_scratch()

    g = captured(eng, s, [c])
    held = free()
    eng.release_scratch()
    assert free() < held + size
    with torch.cuda.stream(s):
        g.replay()
    s.synchronize()
    assert c.right()
    del g
    for _ in range(100):  # the driver gives the block back in its own time
        eng.release_scratch()
        if free() >= held + size:
            break
        time.sleep(0.05)
    assert free() >= held + size


def test_release_is_refused_in_a_capture(eng):
    s, c = torch.cuda.Stream(), Call(64, 10)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    eng.set_stream(s)
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        c.run(eng)
        with pytest.raises(AeError) as e:
            eng.release_scratch()
        c.run(eng)
    assert e.value.code == -1 and "captured" in str(e.value)
    with torch.cuda.stream(s):
        g.replay()
    s.synchronize()
    assert c.right()


def test_graph_outlives_the_engine():
    """Destroyed, not replayed, after the engine."""
    s, c, e = torch.cuda.Stream(), Call(64, 11), Engine(0)
    torch.cuda.synchronize()
    g = captured(e, s, [c])
    with torch.cuda.stream(s):
        g.replay()
    s.synchronize()
    assert c.right()
    e.close()
    del g
    torch.cuda.synchronize()
