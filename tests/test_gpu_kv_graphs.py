"""Captured calls of the quantised cache on the GPU: first calls and status."""
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
