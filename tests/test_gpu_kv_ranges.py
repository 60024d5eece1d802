"""The quantised key/value cache at the ends of its ranges, on the GPU: windows near 2^31 first.
"""
import numpy as np
import pytest
import torch

from test_gpu_kv_cache import Setup, check_attention, starts_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    from rns_llm_b200.backends import CudaRNSBackend
    return CudaRNSBackend()


def queries(s, tokens, heads, dim, dtype=torch.float16):
    return torch.from_numpy(s.rng.standard_normal((tokens, heads, dim)).astype(np.float32)).to(dtype)


# ---------------------------------------------------------------------------------------
# windows
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("window", [2 ** 40, 2 ** 31 - 1, 2 ** 31 - 8])
@pytest.mark.parametrize("lens,new,heads", [
    ([5], [10], 2), ([40, 7], [12, 10], 4),                      # rows kernel: positions from -5, -3
    ([5, 200], [60, 150], 2), ([100, 7], [300, 270], 6),         # prompt kernel: from -55, -200
])
def test_wide_window_with_more_queries_than_tokens(backend, lens, new, heads, window):
    """Positions before the first, less a window near 2^31, do not fit 32 bits."""
    s = Setup(backend, lens, kv_heads=2, dim=64, page=16, seed=31)
    q = queries(s, sum(new), heads, 64)
    got, lse = backend.kv_cache_attention(q.cuda(), s.cache, s.d_table, s.ints(lens), s.ints(starts_of(new)),
                                          max_query_len=max(new), window=window, return_lse=True)
    check_attention(s, q, new, got, lse, scale=0.125, window=window, dtype=torch.float16)
    plain, plain_lse = backend.kv_cache_attention(q.cuda(), s.cache, s.d_table, s.ints(lens), s.ints(starts_of(new)),
                                                  max_query_len=max(new), return_lse=True)
    assert torch.equal(got, plain) and torch.equal(lse, plain_lse)
    backend.check_status()
