"""Host side of the paged 8-bit key/value cache: refusals of the C entries and the addressing of
lengths, starts and pages (the source the kernels run), without a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

ONE = 1 << 20      # a 16-byte aligned stand-in for a device pointer that no check dereferences


def cache_args(native, **change):
    values = dict(d_k=ONE, d_v=ONE, d_k_scale=ONE, d_v_scale=ONE, pages=8, page_tokens=16, kv_heads=2, head_dim=64,
                  format=native.KV_INT8, d_page_table=ONE, table_stride=4, table_pages=4, sequences=2, d_status=None)
    values.update(change)
    return native.KVCacheArgs(**values)


def attention_args(native, **change):
    values = dict(d_q=ONE, type=native.F16, heads=4, tokens=2, q_token_stride=256, q_head_stride=64, d_seq_lens=ONE,
                  d_query_starts=ONE, max_new=1, causal=1, window=0, softmax_scale=0.125, d_out=ONE,
                  out_token_stride=256, out_head_stride=64, d_lse=None, d_workspace=None, workspace_bytes=0)
    values.update(change)
    return native.KVAttentionArgs(**values)


BAD_CACHES = [
    (dict(d_k=None), "ERR_INVALID_ARGUMENT"), (dict(d_v_scale=None), "ERR_INVALID_ARGUMENT"),
    (dict(d_k=ONE + 8), "ERR_INVALID_ARGUMENT"), (dict(format=2), "ERR_INVALID_ARGUMENT"),
    (dict(page_tokens=48), "ERR_UNSUPPORTED"), (dict(page_tokens=256), "ERR_UNSUPPORTED"),
    (dict(head_dim=72), "ERR_UNSUPPORTED"), (dict(head_dim=0), "ERR_UNSUPPORTED"), (dict(head_dim=272), "ERR_UNSUPPORTED"),
    (dict(kv_heads=0), "ERR_INVALID_ARGUMENT"), (dict(pages=0), "ERR_INVALID_ARGUMENT"),
    (dict(pages=1 << 31), "ERR_INVALID_ARGUMENT"), (dict(sequences=-1), "ERR_INVALID_ARGUMENT"),
    (dict(sequences=65536), "ERR_INVALID_ARGUMENT"), (dict(table_stride=3), "ERR_INVALID_ARGUMENT"),
    (dict(d_page_table=None), "ERR_INVALID_ARGUMENT"),
    (dict(table_pages=1 << 27, table_stride=1 << 27), "ERR_UNSUPPORTED"),
]


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_bad_caches_are_refused(native, change, code):
    lib, cache, want = native.load(), cache_args(native, **change), getattr(native, code)
    assert lib.rns_kv_write(C.byref(cache), ONE, ONE, native.F16, 2, 128, 64, 128, 64, ONE, ONE, 1, None) == want
    assert lib.rns_kv_read(C.byref(cache), ONE, ONE, 2, 1, ONE, ONE, native.F16, None) == want
    assert lib.rns_kv_attention_workspace(C.byref(cache), C.byref(attention_args(native))) == -want
    assert lib.rns_kv_attention(C.byref(cache), C.byref(attention_args(native)), None) == want
    assert native.last_error()


def test_bad_calls_are_refused(native):
    lib, cache = native.load(), cache_args(native)
    ref = C.byref(cache)
    bad, unsupported = native.ERR_INVALID_ARGUMENT, native.ERR_UNSUPPORTED
    assert lib.rns_kv_write(None, ONE, ONE, native.F16, 2, 128, 64, 128, 64, ONE, ONE, 1, None) == bad
    assert lib.rns_kv_write(ref, None, ONE, native.F16, 2, 128, 64, 128, 64, ONE, ONE, 1, None) == bad
    assert lib.rns_kv_write(ref, ONE, ONE, 7, 2, 128, 64, 128, 64, ONE, ONE, 1, None) == bad
    assert lib.rns_kv_write(ref, ONE, ONE, native.F16, -1, 128, 64, 128, 64, ONE, ONE, 1, None) == bad
    assert lib.rns_kv_write(ref, ONE, ONE, native.F16, 2, 128, 64, 128, 64, None, ONE, 1, None) == bad
    assert lib.rns_kv_read(ref, ONE, ONE, 2, 1, ONE, ONE + 8, native.F16, None) == bad
    assert lib.rns_kv_read(ref, ONE, ONE, 2, -1, ONE, ONE, native.F16, None) == bad
    assert lib.rns_kv_read(ref, ONE, None, 2, 1, ONE, ONE, native.F16, None) == bad
    for change, want in [(dict(type=native.F32), unsupported), (dict(heads=3), bad), (dict(heads=0), bad),
                         (dict(tokens=-1), bad), (dict(max_new=-1), bad), (dict(window=-1), bad),
                         (dict(window=4, causal=0), bad), (dict(softmax_scale=float("nan")), bad),
                         (dict(softmax_scale=float("inf")), bad), (dict(d_q=None), bad), (dict(d_out=None), bad),
                         (dict(d_seq_lens=None), bad)]:
        assert lib.rns_kv_attention(ref, C.byref(attention_args(native, **change)), None) == want, change
    assert lib.rns_kv_attention(ref, None, None) == bad


def test_calls_without_work_return_at_once(native):
    lib = native.load()
    none = C.byref(cache_args(native, sequences=0, table_pages=0, d_page_table=None))
    assert lib.rns_kv_write(none, ONE, ONE, native.F16, 2, 128, 64, 128, 64, ONE, ONE, 1, None) == native.OK
    assert lib.rns_kv_read(none, ONE, ONE, 2, 1, ONE, ONE, native.F16, None) == native.OK
    assert lib.rns_kv_attention(none, C.byref(attention_args(native)), None) == native.OK
    some = C.byref(cache_args(native))
    assert lib.rns_kv_write(some, None, None, native.F16, 0, 128, 64, 128, 64, None, None, 0, None) == native.OK
    assert lib.rns_kv_read(some, None, None, 0, 0, None, None, native.F16, None) == native.OK
    empty = attention_args(native, tokens=0, d_q=None, d_out=None)
    assert lib.rns_kv_attention(some, C.byref(empty), None) == native.OK


def rows(native, table, lens, starts, tokens, pages=8, page_tokens=16):
    table, lens, starts = (np.ascontiguousarray(x, dtype=np.int32) for x in (table, lens, starts))
    status, out = np.zeros(1, np.int32), np.full(tokens, -7, np.int64)
    cache = cache_args(native, pages=pages, page_tokens=page_tokens, d_page_table=table.ctypes.data,
                       table_stride=table.shape[1], table_pages=table.shape[1], sequences=table.shape[0],
                       d_status=status.ctypes.data)
    native.check(native.load().rns_host_kv_rows(C.byref(cache), lens.ctypes.data, starts.ctypes.data, tokens,
                                                out.ctypes.data))
    return out.tolist(), int(status[0])


def test_rows_of_new_tokens(native):
    block, row = 2 * 16 * 64, 64
    got, status = rows(native, [[3, 5, 0, 0], [1, 7, 2, 0]], [17, 33], [0, 3, 5], 6)
    assert status == native.OK
    # positions 14, 15, 16 of the first sequence, 31, 32 of the second; row 5 belongs to none
    assert got == [3 * block + 14 * row, 3 * block + 15 * row, 5 * block, 7 * block + 15 * row, 2 * block, -1]


@pytest.mark.parametrize("lens,starts", [
    ([-1, 4], [0, 1, 2]), ([65, 4], [0, 1, 2]), ([2 ** 31 - 1, 4], [0, 1, 2]),   # beyond the table's four pages
    ([4, 4], [0, 2, 1]), ([4, 4], [-1, 1, 2]), ([4, 4], [0, 1, 3]),              # not ascending inside the tokens
])
def test_bad_lengths_and_starts_are_flagged(native, lens, starts):
    got, status = rows(native, [[0, 1, 2, 3], [4, 5, 6, 7]], lens, starts, 2)
    assert status == native.ERR_BAD_INDEX
    assert all(-1 <= g < 8 * 2 * 16 * 64 for g in got)


@pytest.mark.parametrize("page", [-1, 8, 2 ** 31 - 1, -2 ** 31])
def test_bad_pages_are_flagged(native, page):
    got, status = rows(native, [[0, page, 2, 3]], [20], [0, 6], 6)
    assert status == native.ERR_BAD_INDEX and got[:2] == [14 * 64, 15 * 64] and got[2:] == [-1] * 4
    # an entry behind the sequence's length is not read
    got, status = rows(native, [[0, page, 2, 3]], [16], [0, 2], 2)
    assert status == native.OK and got == [14 * 64, 15 * 64]


def test_tokens_before_the_first_position_are_dropped(native):
    got, status = rows(native, [[2, 0, 0, 0], [0, 0, 0, 0]], [2, 0], [0, 4, 5], 5)
    assert status == native.OK and got == [-1, -1, 2 * 2048, 2 * 2048 + 64, -1]


def test_cache_tensors_are_checked():
    from rns_llm_b200.backends import QuantizedKVCache

    def make(k=(4, 2, 16, 64), v=None, scale=(4, 2), dtype=torch.int8, scale_dtype=torch.float32):
        return QuantizedKVCache(k=torch.zeros(k, dtype=dtype), v=torch.zeros(v or k, dtype=dtype),
                                k_scale=torch.zeros(scale, dtype=scale_dtype), v_scale=torch.zeros(scale))

    with pytest.raises(ValueError, match="one 8-bit type"):
        make(dtype=torch.uint8)
    with pytest.raises(ValueError, match="one 8-bit type"):
        make(v=(4, 2, 16, 80))
    with pytest.raises(ValueError, match="one 8-bit type"):
        make(k=(4, 2, 64), scale=(4, 2))
    with pytest.raises(ValueError, match="k_scale and v_scale"):
        make(scale=(4, 3))
    with pytest.raises(ValueError, match="k_scale and v_scale"):
        make(scale_dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA tensors"):
        make()
