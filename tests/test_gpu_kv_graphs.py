"""Captured calls of the quantised cache on the GPU, first calls and status, and calls of several host threads."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def ints_like(tensor, values):
    """An int32 tensor made inside a capture, without a copy from the host."""
    out = torch.zeros_like(tensor)
    if values:
        out[1:] = values[1]
    return out


@pytest.mark.parametrize("new", [1, 70])
def test_first_calls_in_a_graph(new):
    """Nothing has to run before the capture on a cache that the backend made; an index that goes out of range in
    one replay is still reported after the next."""
    from rns_llm_b200.backends import CudaRNSBackend

    backend = CudaRNSBackend()
    cache = backend.create_kv_cache(pages=8, kv_heads=2, head_dim=64, page_tokens=32)
    table, lens, starts = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8), ints(100), ints(0, new)
    x = torch.randn(new, 2, 64, device="cuda").half()
    q = torch.randn(new, 4, 64, device="cuda").half()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        backend.kv_cache_write(cache, x, x, table, lens, starts)
        out = backend.kv_cache_attention(q, cache, table, lens, starts)
        k, v = backend.kv_cache_read(cache, table, ints_like(lens, 0), ints_like(starts, (0, 100)), rows=100)
    graph.replay()
    backend.check_status()
    again = CudaRNSBackend()
    twin = again.create_kv_cache(pages=8, kv_heads=2, head_dim=64, page_tokens=32)
    again.kv_cache_write(twin, x, x, table, lens, starts)
    assert torch.equal(out, again.kv_cache_attention(q, twin, table, lens, starts))
    lens.fill_(1000)
    graph.replay()
    lens.fill_(100)
    graph.replay()
    with pytest.raises(RuntimeError, match="out of range"):
        backend.check_status()
    graph.replay()
    backend.check_status()


def test_first_call_of_a_backend_is_not_captured():
    """Its status words would belong to the graph, which clears them in every replay."""
    from rns_llm_b200.backends import CudaRNSBackend

    maker, backend = CudaRNSBackend(), CudaRNSBackend()
    cache = maker.create_kv_cache(pages=2, kv_heads=1, head_dim=16, page_tokens=16)
    x = torch.zeros(1, 1, 16, dtype=torch.float16, device="cuda")
    args = (ints(0, 1).view(1, 2), ints(1), ints(0, 1))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            backend.kv_cache_write(cache, x, x, *args)
    torch.cuda.synchronize()
    backend.kv_cache_write(cache, x, x, *args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        backend.kv_cache_write(cache, x, x, *args)
    graph.replay()
    backend.check_status()


def test_host_threads_on_one_stream():
    """Attention whose keys are split among CTAs, of two kernels in turn, beside a linear that uses the same scratch:
    every result is that of a call alone."""
    from rns_llm_b200.backends import CudaRNSBackend
    from rns_llm_b200.layers import RNSLinear

    backend = CudaRNSBackend()
    gen = torch.Generator(device="cuda").manual_seed(1)

    def attention(new, length):
        cache = backend.create_kv_cache(pages=64, kv_heads=2, head_dim=64, page_tokens=64)
        table, lens, starts = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 64), ints(length), ints(0, length)
        x = torch.randn(length, 2, 64, generator=gen, device="cuda").half()
        backend.kv_cache_write(cache, x, x, table, lens, starts)
        q = torch.randn(new, 4, 64, generator=gen, device="cuda").half()
        return lambda: backend.kv_cache_attention(q, cache, table, lens, ints_like(starts, (0, new)))

    linear = RNSLinear.from_linear(torch.nn.Linear(2048, 512, device="cuda", dtype=torch.float16), backend=backend,
                                   mode="rns", fused=True, moduli=(127, 126, 125, 121)).eval()
    rows = torch.randn(64, 2048, generator=gen, device="cuda").half()
    calls = [attention(1, 4000), attention(70, 3500), attention(3, 4096), lambda: linear(rows)]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    outs, started = [[] for _ in calls], threading.Barrier(len(calls))

    def work(i):
        started.wait()
        with torch.no_grad():
            for _ in range(60):
                outs[i].append(calls[i]())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    for got, alone in zip(outs, want):
        assert len(got) == 60 and all(torch.equal(out, alone) for out in got)
    backend.check_status()
