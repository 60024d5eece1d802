"""Calls of two host threads on one stream share the stream's scratch: the launches of one call are not
interleaved with those of another.  The native library is a stand-in that records who uses the scratch."""
import threading
import time
import types
from collections import Counter
from contextlib import nullcontext

import pytest
import torch

from rns_llm_b200 import _native as N
from rns_llm_b200.arena import StreamArena
from rns_llm_b200.backends import cuda_backend, kv_cache


class Arena(StreamArena):
    """One stream's scratch in host memory."""

    def __init__(self):
        super().__init__()
        self.bytes = torch.empty(1 << 16, dtype=torch.uint8)

    def buffer(self, index, stream, nbytes):
        return self.bytes

    def block(self, device, nbytes):
        return self.bytes.data_ptr(), 7


class Library:
    def __init__(self):
        self.owner, self.mixed, self.calls = None, 0, 0

    def first(self):
        self.owner = threading.get_ident()
        time.sleep(0.002)                        # a foreign call lets other threads run
        return N.OK

    def last(self):
        self.calls += 1
        self.mixed += self.owner != threading.get_ident()
        return N.OK

    # attention over the cache: two kernels in one foreign call
    def rns_kv_attention_workspace(self, cache, args):
        return 4096

    def rns_kv_attention(self, cache, args, stream):
        return self.first() or self.last()

    # a linear of few tokens: two foreign calls
    def rns_linear_small_supported(self, *a):
        return 0

    def rns_linear_stream_supported(self, *a):
        return 1

    def rns_quantize_activations_tiled(self, *a):
        return self.first()

    def rns_linear_stream(self, *a):
        return self.last()


@pytest.fixture
def backend(monkeypatch):
    monkeypatch.setattr(torch.cuda, "device", lambda *_: nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(kv_cache, "_on", lambda device: nullcontext())
    monkeypatch.setattr(kv_cache, "_stream", lambda device: 7)
    own = object.__new__(cuda_backend.CudaRNSBackend)
    own._lib, own.arena, own._stats, own._moduli_arrays = Library(), Arena(), Counter(), {}
    own._state = lambda device: types.SimpleNamespace(status=torch.zeros(1, dtype=torch.int32))
    return own


def attention(backend):
    device = torch.device("cpu")
    cache = types.SimpleNamespace(device=device, kv_heads=2, head_dim=16, _args=N.KVCacheArgs())
    q, ints = torch.zeros(1, 2, 16, dtype=torch.float16), lambda *v: torch.tensor(v, dtype=torch.int32)
    return lambda: backend.kv_cache_attention(q, cache, ints(0).view(1, 1), ints(1), ints(0, 1))


def linear(backend):
    prepared = types.SimpleNamespace(kernel="tcgen05", moduli=(127, 126, 125, 121), k=64, n=16,
                                     weight_packed=torch.zeros(64, dtype=torch.int8))
    x, scale = torch.zeros(4, 64, dtype=torch.float16), torch.ones(16)
    return lambda: backend.linear_forward(x, prepared, scale, None)


@pytest.mark.parametrize("calls", [(attention, attention), (linear, linear), (attention, linear)])
def test_launches_of_one_call_stay_together(backend, calls):
    started = threading.Barrier(2)
    failed = []

    def work(call):
        started.wait()
        try:
            for _ in range(20):
                call()
        except Exception as exc:                 # shown by the assertion below
            failed.append(exc)

    threads = [threading.Thread(target=work, args=(make(backend),)) for make in calls]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failed and backend._lib.calls == 40 and backend._lib.mixed == 0
