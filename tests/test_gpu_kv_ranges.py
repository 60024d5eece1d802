"""The quantised key/value cache at the ends of its ranges, on the GPU: windows, scales of very different
size, values that are not finite, bounds and positions at their limits.

Attention is compared with float64 element by element.  Its bound is that of test_gpu_kv_cache.py but for the
weights below fp16's normal range: a weight is rounded in units of 2^M, where 2^M is at most twice the largest
p_j * scale_j over the keys that THE ROW SEES (p_j: its softmax weight, scale_j: the value scale of the key's
page), by up to half of fp16's smallest step, 2^-25.  It meets a byte of at most Q (127 or 448) there, so a row
of n keys is off by n * 2^-24 * max_j (p_j * scale_j * Q), whatever pages it does not see or heed hold.
"""
import numpy as np
import pytest
import torch

import kv_oracle as O
from test_gpu_kv_cache import ATTENTION, HALF_STEP, Setup, check_attention, starts_of

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


# ---------------------------------------------------------------------------------------
# value scales
# ---------------------------------------------------------------------------------------
SMALLEST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}      # of the output types


def check_rows(s, q, new, got, lse, *, scale, dtype, causal=True, window=0, telling=None):
    """Outputs and lse against float64 by the bound above; `telling`: the share of outputs that the bound must
    be able to tell from zero ten times over."""
    starts, (_, heads, dim) = starts_of(new), q.shape
    got = got.float().cpu().numpy().astype(np.float64)
    lse = lse.cpu().numpy().astype(np.float64)
    told = []
    for b, n in enumerate(new):
        keys, values = s.values(b, 0), s.values(b, 1)
        rows = slice(starts[b], starts[b + 1])
        x = q[rows].float().numpy()
        want, want_lse, spread, loud = O.attention(x, keys, values, s.lens[b], scale=scale, causal=causal, window=window)
        group = heads // keys.shape[1]
        holds = np.stack([s.scale[1][s.table[b][t // s.page]] for t in range(s.lens[b])]) if s.lens[b] else None
        most = np.zeros((n, heads))                              # n_keys * max_j p_j scale_j Q of each row
        for i in range(n):
            position = s.lens[b] - n + i
            if position < 0:
                continue
            first, last = max(0, position - window + 1) if window else 0, position + 1 if causal else s.lens[b]
            for h in range(heads):
                t = keys[first:last, h // group].astype(np.float64) @ x[i, h].astype(np.float64) * scale
                p = np.exp(t - want_lse[i, h])
                most[i, h] = (last - first) * (p * holds[first:last, h // group]).max() * float(O.LARGEST[s.fmt])
        score = (dim + 8) * 2.0 ** -22 * loud[:, :, None]
        bound = (HALF_STEP[dtype] * np.abs(want) + (2.0 ** -11 + 2.0 ** -20 + 2 * score) * spread * 1.01 +
                 2.0 ** -24 * 1.01 * most[:, :, None] + SMALLEST[dtype])
        error = np.abs(got[rows] - want)
        assert np.isfinite(got[rows]).all()
        assert (error <= bound).all(), (b, float((error / bound).max()))
        told.append((bound * 10 < np.abs(want)).ravel())
        slack = (dim + 8) * 2.0 ** -22 * loud + 2.0 ** -20 * (1 + np.abs(np.where(np.isinf(want_lse), 0, want_lse)))
        seen = ~np.isneginf(want_lse)
        assert np.array_equal(np.isneginf(lse[rows]), ~seen)
        assert (np.abs(lse[rows][seen] - want_lse[seen]) <= slack[seen]).all()
    if telling is not None:
        assert np.concatenate(told).mean() >= telling, np.concatenate(told).mean()


def attend(backend, s, q, new, **kw):
    return backend.kv_cache_attention(q.cuda(), s.cache, s.d_table, s.ints(s.lens), s.ints(starts_of(new)),
                                      max_query_len=max(new), return_lse=True, **kw)


@pytest.mark.parametrize("lens,new,heads,kv_heads,dim,page,fmt,dtype,window,causal", ATTENTION)
def test_error_is_relative_to_what_a_row_sees(backend, lens, new, heads, kv_heads, dim, page, fmt, dtype, window, causal):
    s = Setup(backend, lens, kv_heads=kv_heads, dim=dim, page=page, fmt=fmt, seed=heads * dim + sum(lens) + 1)
    q = queries(s, sum(new), heads, dim, dtype)
    got, lse = attend(backend, s, q, new, window=window or None, causal=causal)
    check_rows(s, q, new, got, lse, scale=dim ** -0.5, dtype=dtype, causal=causal, window=window)


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("spread", [1.0, 4.0])
@pytest.mark.parametrize("gain", [1.0, 20.0])
def test_pages_of_all_sizes(backend, new, spread, gain):
    """Value scales over up to 46 powers of two, key scales as they are in a model."""
    lens = [400, 90]
    s = Setup(backend, lens, kv_heads=2, dim=64, page=16, seed=int(gain) + int(spread), spread=spread)
    for scale in s.scale[0]:
        scale[:] = 1 / float(O.LARGEST["int8"])
    s.to_device()
    q = torch.from_numpy((s.rng.standard_normal((2 * new, 4, 64)) * gain).astype(np.float32)).bfloat16()
    got, lse = attend(backend, s, q, [new, new])
    check_rows(s, q, [new, new], got, lse, scale=0.125, dtype=torch.bfloat16, telling=0.5)


def with_outlier(backend, fmt, dim, page, where, seed, lens=(400, 90)):
    """Keys so that page `where` of sequence 0 has scores near -70 and the others a spread of 2, for queries
    near the vector that is returned."""
    s = Setup(backend, list(lens), kv_heads=2, dim=dim, page=page, fmt=fmt, seed=seed)
    top = float(O.LARGEST[fmt])
    toward = np.where(s.rng.random(dim) < 0.5, -1.0, 1.0).astype(np.float32)
    s.scale[0][:] = 2 / (top / 3)
    page_id = s.table[0, where]
    s.data[0][page_id] = O.to_bytes(np.broadcast_to(-top * toward, s.data[0][page_id].shape).copy(), fmt)
    s.scale[0][page_id] = 70 / (top * dim ** 0.5)
    return s, page_id, toward


def near(s, toward, tokens, heads, dtype):
    noise = s.rng.standard_normal((tokens, heads, len(toward))).astype(np.float32)
    return torch.from_numpy(toward + 0.2 * noise).to(dtype)


@pytest.mark.parametrize("new", [1, 5, 70])
@pytest.mark.parametrize("power", [10, 14, 20, 30, 60])
@pytest.mark.parametrize("fmt,dim,where", [("int8", 64, 0), ("int8", 128, 3), ("e4m3", 80, 24), ("e4m3", 256, 1)])
def test_page_of_large_values_that_no_row_heeds(backend, fmt, dim, where, power, new):
    """A page whose values are 2^power larger and whose softmax weight is e^-70: the other pages keep their
    precision."""
    s, page_id, toward = with_outlier(backend, fmt, dim, 16, where, seed=power + dim)
    s.scale[1][page_id] *= np.float32(2.0 ** power)
    s.to_device()
    q = near(s, toward, 2 * new, 4, torch.float16)
    got, lse = attend(backend, s, q, [new, new])
    check_rows(s, q, [new, new], got, lse, scale=dim ** -0.5, dtype=torch.float16, telling=0.5)


@pytest.mark.parametrize("power", [14, 30])
def test_page_of_large_values_among_many_long_sequences(backend, power):
    """The same where a warp of the rows kernel meets many pages of one row."""
    lens = [2100] * 16
    s = Setup(backend, lens, kv_heads=8, dim=64, page=64, seed=power)
    top = 127.0
    toward = np.where(s.rng.random(64) < 0.5, -1.0, 1.0).astype(np.float32)
    s.scale[0][:] = 2 / (top / 3)
    large = s.table[:, 1]                                        # in every sequence
    s.data[0][large] = (-top * toward).astype(np.int8)
    s.scale[0][large] = 70 / (top * 8)
    s.scale[1][large] *= np.float32(2.0 ** power)
    s.to_device()
    q = near(s, toward, 16, 8, torch.float16)
    got, lse = attend(backend, s, q, [1] * 16)
    check_rows(s, q, [1] * 16, got, lse, scale=0.125, dtype=torch.float16, telling=0.5)


@pytest.mark.parametrize("new", [4, 90])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_later_page_of_large_values(backend, dim, new):
    """What a row gives does not depend on the value scale of a page that it does not see."""
    lens = [146]
    s = Setup(backend, lens, kv_heads=1, dim=dim, page=16, seed=dim)
    q = queries(s, new, 4, dim)
    clean, _ = attend(backend, s, q, [new])
    s.scale[1][s.table[0, 9]] *= np.float32(2.0 ** 40)           # positions 144, 145
    s.to_device()
    got, lse = attend(backend, s, q, [new])
    assert torch.equal(got[:new - 2], clean[:new - 2])


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("power", [-60, -20, 0, 60, 110])
def test_scales_near_the_ends_of_their_type(backend, power, new):
    lens = [400, 90]
    s = Setup(backend, lens, kv_heads=2, dim=64, page=16, seed=power + 100)
    s.scale[1] *= np.float32(2.0 ** power)
    s.to_device()
    q = queries(s, 2 * new, 4, 64, torch.bfloat16)
    got, lse = attend(backend, s, q, [new, new])
    check_rows(s, q, [new, new], got, lse, scale=0.125, dtype=torch.bfloat16, telling=0.3)


@pytest.mark.parametrize("new", [1, 70])
def test_pages_of_zeros(backend, new):
    """Value scales of zero on every page of one sequence and on some of the other's."""
    lens = [400, 90]
    s = Setup(backend, lens, kv_heads=2, dim=64, page=16, seed=41)
    s.scale[1][s.table[1, :6]] = 0
    s.scale[1][s.table[0, 1:20]] = 0
    s.to_device()
    q = queries(s, 2 * new, 4, 64)
    got, lse = attend(backend, s, q, [new, new])
    check_rows(s, q, [new, new], got, lse, scale=0.125, dtype=torch.float16)
    assert (got[new:] == 0).all()


@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("dim,fmt,heads", [(64, "int8", 4), (128, "int8", 8), (80, "e4m3", 4), (256, "e4m3", 2)])
def test_few_rows_are_as_exact_as_their_type(backend, dim, fmt, heads, new):
    """Weights meet the values in two fp16 parts, so an fp16 output is off by its own rounding and little else: the
    error's norm is within a tenth of that of the exact result rounded (weights rounded once make it 1.4 times)."""
    lens = [600] * 8
    s = Setup(backend, lens, kv_heads=2, dim=dim, page=64, fmt=fmt, seed=dim, spread=0.1)
    for scale in s.scale[0]:
        scale[:] = 2 / (float(O.LARGEST[fmt]) / 3)               # scores with a spread of 2
    s.to_device()
    q = queries(s, 8 * new, heads, dim)
    got, _ = attend(backend, s, q, [new] * 8)
    wrong = rounded = 0.0
    for b in range(8):
        rows = slice(b * new, (b + 1) * new)
        want = O.attention(q[rows].float().numpy(), s.values(b, 0), s.values(b, 1), 600, scale=dim ** -0.5)[0]
        wrong += float(((got[rows].double().cpu().numpy() - want) ** 2).sum())
        rounded += float(((want.astype(np.float16).astype(np.float64) - want) ** 2).sum())
    assert wrong <= 1.1 ** 2 * rounded, (wrong / rounded) ** 0.5


# ---------------------------------------------------------------------------------------
# values that are not finite
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_bytes_of_a_block_with_a_value_that_is_not_finite(backend, fmt, bad, dtype):
    """Scale NaN and bytes of zero, its earlier tokens' and later ones' too; every other block, scale and
    byte as the NumPy statement has it."""
    s = Setup(backend, [40, 20], fmt=fmt, seed=9)
    x = s.rng.standard_normal((12, 2, 64)).astype(np.float32)
    x = torch.from_numpy(x).to(dtype)
    lens, starts = [40, 20], [0, 8, 12]                          # positions 32 .. 39 and 16 .. 19
    x[3, 1, 7] = bad
    with np.errstate(invalid="ignore"):
        for which in range(2):
            O.write(s.data[which], s.scale[which], x.float().numpy(), s.table, lens, starts, fmt)
            s.data[which][s.table[0, 2], 1, :8] = 0
    backend.kv_cache_write(s.cache, x.cuda(), x.cuda(), s.d_table, s.ints(lens), s.ints(starts))
    s.check_bytes()
    y = torch.ones(1, 2, 64, dtype=dtype)                        # one more token for that page
    with np.errstate(invalid="ignore"):
        for which in range(2):
            O.write(s.data[which], s.scale[which], y.float().numpy(), s.table, [41], [0, 1], fmt)
            s.data[which][s.table[0, 2], 1, :9] = 0
    backend.kv_cache_write(s.cache, y.cuda(), y.cuda(), s.d_table[:1], s.ints([41]), s.ints([0, 1]))
    s.check_bytes()
    # a page that held tokens before
    z = torch.full((1, 2, 64), bad, dtype=dtype)
    with np.errstate(invalid="ignore"):
        for which in range(2):
            O.write(s.data[which], s.scale[which], z.float().numpy(), s.table[1:], [21 - 16], [0, 1], fmt)
            s.data[which][s.table[1, 0], :, :5] = 0
    backend.kv_cache_write(s.cache, z.cuda(), z.cuda(), s.d_table[1:], s.ints([5]), s.ints([0, 1]))
    s.check_bytes()
    backend.check_status()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length,new,at", [(40, 40, 35), (18, 4, 16), (300, 150, 290)])
def test_written_infinity_reaches_the_rows_that_see_it(backend, fmt, dim, length, new, at):
    """A value that is not finite is written among a prompt's: rows that see its page of 16 tokens are NaN, the
    others what they are without it."""
    gen = torch.Generator().manual_seed(dim)
    x = torch.randn(length, 1, dim, generator=gen).half()
    q = torch.randn(new, 2, dim, generator=gen).half().cuda()
    outs = []
    for bad in (None, float("inf"), float("nan")):
        v = x.clone()
        if bad is not None:
            v[at, 0, 5] = bad
        cache = backend.create_kv_cache(pages=-(-length // 16), kv_heads=1, head_dim=dim, page_tokens=16, format=fmt)
        table = torch.arange(cache.pages, dtype=torch.int32, device="cuda").view(1, -1)
        ints = lambda *n: torch.tensor(n, dtype=torch.int32, device="cuda")
        backend.kv_cache_write(cache, x.cuda(), v.cuda(), table, ints(length), ints(0, length))
        outs.append(backend.kv_cache_attention(q, cache, table, ints(length), ints(0, new)))
    clean, *rest = outs
    first = max(0, at // 16 * 16 - (length - new))               # row of the page's first token
    for out in rest:
        assert torch.equal(out[:first], clean[:first])
        assert torch.isnan(out[first:]).all()
    backend.check_status()


# ---------------------------------------------------------------------------------------
# bounds of zero
# ---------------------------------------------------------------------------------------
def test_a_bound_of_zero_is_reported(backend):
    """Tokens or rows that a bound of zero leaves out are flagged, as with any bound that is too small."""
    s = Setup(backend, [40, 20], seed=2)
    x = torch.ones(2, 2, 64, dtype=torch.float16, device="cuda")
    lens, starts = s.ints([40, 20]), s.ints([0, 1, 2])
    backend.kv_cache_write(s.cache, x, x, s.d_table, lens, starts, max_query_len=0)
    with pytest.raises(RuntimeError, match="out of range"):
        backend.check_status()
    s.check_bytes()
    out = tuple(torch.full((5, 2, 64), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    backend.kv_cache_read(s.cache, s.d_table, s.ints([0, 0]), s.ints([0, 2, 5]), rows=5, max_rows=0, out=out)
    with pytest.raises(RuntimeError, match="out of range"):
        backend.check_status()
    assert (out[0] == 7.0).all() and (out[1] == 7.0).all()
    # sequences without tokens stay within it
    backend.kv_cache_write(s.cache, x, x, s.d_table, lens, s.ints([0, 0, 0]), max_query_len=0)
    backend.kv_cache_read(s.cache, s.d_table, s.ints([0, 0]), s.ints([0, 0, 0]), rows=5, max_rows=0, out=out)
    backend.check_status()
    s.check_bytes()


# ---------------------------------------------------------------------------------------
# positions near 2^31
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("new,window", [(1, 200), (5, 3000), (300, 200)])
def test_positions_near_the_end_of_32_bits(backend, new, window):
    """The longest sequence that a page table may describe (its pages but the last few shared), beside one whose
    many new tokens make the grid of a write reach beyond 2^31 from there."""
    page, width = 128, 2 ** 24 - 33
    length, other = width * page, 9000
    own = 40                                                     # last pages of the long sequence
    cache, small = (backend.create_kv_cache(pages=1 + own + 71, kv_heads=1, head_dim=16, page_tokens=page) for _ in range(2))
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    tail = torch.arange(1, 1 + own, dtype=torch.int32, device="cuda")
    beside = torch.arange(1 + own, 1 + own + 71, dtype=torch.int32, device="cuda")
    table = torch.zeros((2, width), dtype=torch.int32, device="cuda")
    table[0, -own:], table[1, :71] = tail, beside
    small_table = torch.zeros((2, 71), dtype=torch.int32, device="cuda")
    small_table[0, :own], small_table[1] = tail, beside
    gen = torch.Generator(device="cuda").manual_seed(new)
    k, v = (torch.randn(new + other, 1, 16, generator=gen, device="cuda").half() for _ in range(2))
    before = [torch.randn(own * page - new, 1, 16, generator=gen, device="cuda").half() for _ in range(2)]
    q = torch.randn(new, 2, 16, generator=gen, device="cuda").half()
    results = []
    for c, t, n in ((cache, table, length), (small, small_table, own * page)):
        backend.kv_cache_write(c, *before, small_table[:1], ints(own * page - new), ints(0, own * page - new))
        backend.kv_cache_write(c, k, v, t, ints(n, other), ints(0, new, new + other))
        read = backend.kv_cache_read(c, t, ints(n - 700, 5), ints(0, 700, other + 695), rows=other + 695)
        out = backend.kv_cache_attention(q, c, t[:1], ints(n), ints(0, new), window=window, return_lse=True)
        results.append((c.k, c.v, c.k_scale, c.v_scale, *read, *out))
    backend.check_status()
    for a, b in zip(*results):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------
# outputs that overlap
# ---------------------------------------------------------------------------------------
def test_outputs_that_overlap_are_refused(backend):
    s = Setup(backend, [40, 20])
    lens, starts = s.ints([40, 20]), s.ints([0, 1, 2])
    wide = torch.ones(3, 8, 64, dtype=torch.float16, device="cuda")
    q = wide[:2, :4]
    for out in (wide[1:, :4], wide[:2, 2:6], wide[:2, :4], wide.view(-1)[64:64 + 512].view(2, 4, 64)):
        with pytest.raises(ValueError, match="overlap"):
            backend.kv_cache_attention(q, s.cache, s.d_table, lens, starts, out=out)
    want = backend.kv_cache_attention(q, s.cache, s.d_table, lens, starts)
    got = backend.kv_cache_attention(q, s.cache, s.d_table, lens, starts, out=wide[:2, 4:])     # beside it
    assert torch.equal(got, want) and (wide[:, :4] == 1).all() and (wide[2] == 1).all()
    rows = torch.zeros(5, 2, 64, dtype=torch.float16, device="cuda")
    for out in ((rows[:3], rows[:3]), (rows[:3], rows[2:]), (rows[:3],), (rows[:3],) * 3):
        with pytest.raises(ValueError):
            backend.kv_cache_read(s.cache, s.d_table, s.ints([0, 0]), s.ints([0, 2, 3]), rows=3, out=out)
    backend.check_status()
