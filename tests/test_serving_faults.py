"""The replay's executor stage when functions decode, without a GPU: engines that only plan stand in for the real ones, the calls
that would run kernels are counted and take time on a clock of the test's own."""
import numpy as np
import pytest

from torpor_b200 import kv_cache, serving
from torpor_b200 import workloads as W
from torpor_b200.memory_manager import MemoryManager, repo_reset

ARCH, STEPS = "llama_tiny", 50


class World:
    def __init__(self, swap_s):
        self.now, self.call_s, self.swap_s, self.calls, self.status = 100.0, 1e-4, swap_s, 0, 0
        self.ready = {}

    def clock(self):
        self.now += 1e-6
        return self.now


@pytest.fixture()
def world(built, monkeypatch):
    import torch
    repo_reset()
    w = World(swap_s=3e-3)

    class Engine(MemoryManager):
        def __init__(self, cap, device=0, **kw):
            super().__init__(cap, device=-1, **kw)

        def swap_in(self, func, src=-1):
            w.ready[id(self), func] = w.now + w.swap_s
            return super().swap_in(func, src)

        def poll_ready(self, func):
            return 0 if w.now >= w.ready.get((id(self), func), 0.0) else 1

        def kv_append(self, func, args, stream=0):
            w.calls += 1
            w.now += w.call_s

        prefix_attention = kv_append

        def cudaMemcpyAsyncBackendHtoD(self, *a):
            return 0

    class Stream:
        cuda_stream = 0

        def __init__(self, device=None):
            pass

        def synchronize(self):
            pass

    class Event:
        def record(self, stream):
            self.at = w.now + 2e-3

        def query(self):
            return w.now >= self.at

    def kv_status(device=0, stream=0, clear=False):
        word = w.status
        if clear:
            w.status = 0
        return word

    monkeypatch.setattr(serving, "MemoryManager", Engine)
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(kv_cache, "kv_status", kv_status)
    monkeypatch.setattr(serving.time, "perf_counter", w.clock)
    yield w
    repo_reset()


def server(n_gpus=1, functions=3, cap=200 << 20):
    srv = serving.SwapServer(n_gpus, cap, devices=[0] * n_gpus, decode_tokens=STEPS, prompt_tokens=40)
    for i in range(functions):
        srv.cold_start(f"fn{i}", ARCH, i, tensor_data=lambda k: np.zeros(srv.weight_set(ARCH).tensors[k].nbytes, dtype=np.uint8))
    return srv


def finish(srv):
    for _ in range(200000):
        if not srv.busy():
            return
        srv.poll()
    raise AssertionError("requests that never end")


def test_a_decode_that_reported_something_is_not_a_completed_one(world):
    srv = server()
    for i, status in enumerate([0, kv_cache.WAIT_GAVE_UP, 0, kv_cache.BAD_PAGE | kv_cache.BAD_LENGTH, 0]):
        srv.submit(f"fn{i % 3}", world.now)
        world.status = status
        finish(srv)
    assert srv.completed == srv.decoded == 3
    assert [(f["func"], f["status"]) for f in srv.faults] == [("fn1", kv_cache.WAIT_GAVE_UP), ("fn0", kv_cache.BAD_PAGE | kv_cache.BAD_LENGTH)]
    assert world.status == 0
    srv.close()


def test_functions_that_do_not_decode_are_not_asked(world, monkeypatch):
    monkeypatch.setattr(kv_cache, "kv_status", lambda *a, **kw: pytest.fail("asked"))
    srv = serving.SwapServer(1, 300 << 20, devices=[0], decode_tokens=STEPS, prompt_tokens=40)
    srv.cold_start("r", "resnet50", 1, tensor_data=lambda k: np.zeros(W.weight_set("resnet50").tensors[k].nbytes, dtype=np.uint8))
    srv.submit("r", world.now)
    finish(srv)
    assert srv.completed == 1 and srv.decoded == 0 and not srv.faults
    srv.close()


def test_the_time_of_a_swap_does_not_hold_the_enqueueing_of_its_decode(world):
    """A request is 2 layers of 2 calls a step, 100 us of host time each: 20 ms, behind swaps of 3 ms."""
    srv = server()
    layers = W.ATTENTION[ARCH].layers
    for i in range(6):
        srv.submit(f"fn{i % 3}", world.now)
        finish(srv)
    assert srv.completed == 6 and world.calls == 6 * STEPS * layers * 2
    assert len(srv.swaps) >= 3
    slice_ms = 2 * world.call_s * 1e3
    for s in srv.swaps:
        assert world.swap_s * 1e3 <= s["ms"] <= world.swap_s * 1e3 + slice_ms + 0.1, s
    srv.close()


def test_a_decode_on_one_gpu_does_not_hold_up_the_look_at_another(world):
    srv = server(n_gpus=3, functions=9, cap=150 << 20)
    for i in range(18):
        srv.submit(f"fn{i % 9}", world.now)
        for _ in range(7):
            srv.poll()
    finish(srv)
    assert srv.completed == srv.decoded == 18 and len(srv.swaps) >= 6
    slice_ms = 2 * world.call_s * 1e3
    for s in srv.swaps:                       # each GPU's slice lies between two looks at the same one
        assert s["ms"] <= world.swap_s * 1e3 + 3 * slice_ms + 0.1, s
    srv.close()


def test_a_stream_of_unknown_architectures_has_made_no_engine(built, monkeypatch):
    made = []
    monkeypatch.setattr(serving, "MemoryManager", lambda *a, **kw: made.append(a))
    with pytest.raises(KeyError):
        serving.run_stream(n_gpus=1, n_models=2, rate=10.0, duration_s=0.1, cap_bytes=1 << 28, archs=("no_such_set",), devices=[-1])
    assert not made
