"""Paged 8-bit key/value cache on the GPU against the plain NumPy statement in kv_oracle.py.

Writing and reading are compared bit for bit (both sides are correctly rounded fp32).  Attention is
compared with float64 element by element; the bound counts, per output,
* half a step of the output type,
* the rounding of each softmax weight to fp16 before it meets the values, 2^-11 of sum p|v|.  A weight
  below fp16's normal range, 2^-14, is off by up to half of its step 2^-24, in units of a value scale that
  is at most the largest of the pages: times the byte it meets that is 2^-25 of the largest value, for
  each of the `keys` weights; the sum they are divided by is at least 1 (the maximum's own weight);
* scores in fp32: head_dim + 8 roundings of 2^-22 (tensor cores truncate) of sum |q k|, which move a
  weight by that relative amount, twice (numerator and denominator), and so the output by that of
  sum p|v|;
* the same for the exponential and the sums over keys: 2^-20.
"""
import numpy as np
import pytest
import torch

import kv_oracle as O

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def backend():
    from rns_llm_b200.backends import CudaRNSBackend
    return CudaRNSBackend()


class Setup:
    """A cache with random contents on both sides and the page table of some sequences."""

    def __init__(self, backend, lens, *, kv_heads=2, dim=64, page=16, fmt="int8", seed=0, spare=2, spread=0.5):
        rng = np.random.default_rng(seed)
        self.backend, self.fmt, self.page, self.lens = backend, fmt, page, list(lens)
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + spare
        order = rng.permutation(pages)
        width = max(counts + [1])
        self.table = np.full((len(lens), width), -1, np.int32)     # entries behind a length are never read
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (pages, kv_heads, page, dim)
        self.data, self.scale = [], []
        for _ in range(2):
            scale = np.exp(rng.uniform(-spread, spread, shape[:2]) * 4).astype(np.float32) / O.LARGEST[fmt]
            x = rng.standard_normal(shape).astype(np.float32) * O.LARGEST[fmt] / 3
            self.data.append(O.to_bytes(np.clip(x, -O.LARGEST[fmt], O.LARGEST[fmt]), fmt))
            self.scale.append(scale)
        self.rng = rng
        self.to_device()

    def to_device(self):
        from rns_llm_b200.backends import QuantizedKVCache
        kind = torch.int8 if self.fmt == "int8" else torch.float8_e4m3fn
        k, v = (torch.from_numpy(d.copy()).cuda().view(kind) for d in self.data)
        ks, vs = (torch.from_numpy(s.copy()).cuda() for s in self.scale)
        self.cache = QuantizedKVCache(k=k, v=v, k_scale=ks, v_scale=vs)
        self.d_table = torch.from_numpy(self.table).cuda()

    def ints(self, values):
        return torch.tensor(list(values), dtype=torch.int32, device="cuda")

    def values(self, b, which):
        return O.tokens_of(self.data[which], self.scale[which], self.table, b, 0, self.lens[b], self.fmt)

    def check_bytes(self):
        for got, scale, want, want_scale in zip((self.cache.k, self.cache.v), (self.cache.k_scale, self.cache.v_scale),
                                                self.data, self.scale):
            assert np.array_equal(scale.cpu().numpy(), want_scale, equal_nan=True)
            assert np.array_equal(got.view(torch.int8).cpu().numpy(), want)


def starts_of(counts):
    return [0] + list(np.cumsum(counts))


# ---------------------------------------------------------------------------------------
# write
# ---------------------------------------------------------------------------------------
WRITES = [
    # lens after the write, new tokens, kv_heads, dim, page, format, type, layout
    ([1], [1], 1, 64, 16, "int8", torch.float16, "plain"),
    ([17, 16, 1, 0, 33], [1, 1, 1, 1, 1], 2, 64, 16, "int8", torch.float16, "plain"),
    ([5, 40, 129, 64], [5, 33, 1, 64], 3, 128, 64, "int8", torch.bfloat16, "fused"),
    ([200, 31, 77], [150, 31, 3], 2, 80, 32, "e4m3", torch.float16, "fused"),
    ([300, 128], [172, 128], 2, 256, 128, "int8", torch.float32, "plain"),
    ([300, 1], [45, 1], 1, 256, 128, "e4m3", torch.bfloat16, "odd"),
    ([70], [70], 12, 16, 16, "int8", torch.float32, "odd"),
    ([3, 20], [5, 20], 2, 96, 16, "e4m3", torch.float32, "head_major"),      # more new tokens than positions
]


def laid_out(x, layout):
    """The same [tokens, heads, dim] values in another memory layout."""
    t, h, d = x.shape
    if layout == "fused":                       # a column block of a wider projection
        wide = torch.zeros((t, 3 * h, d), dtype=x.dtype, device=x.device)
        wide[:, h:2 * h] = x
        return wide[:, h:2 * h]
    if layout == "odd":                         # rows that start on no 16-byte boundary
        wide = torch.zeros((t, h, d + 3), dtype=x.dtype, device=x.device)
        wide[:, :, 1:d + 1] = x
        return wide[:, :, 1:d + 1]
    if layout == "head_major":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    return x


@pytest.mark.parametrize("lens,new,heads,dim,page,fmt,dtype,layout", WRITES)
def test_write_is_bit_exact(backend, lens, new, heads, dim, page, fmt, dtype, layout):
    s = Setup(backend, lens, kv_heads=heads, dim=dim, page=page, fmt=fmt, seed=len(lens) * 100 + dim)
    starts = starts_of(new)
    x = []
    for which in range(2):
        values = s.rng.standard_normal((starts[-1], heads, dim)).astype(np.float32)
        values *= np.exp(s.rng.uniform(-4, 2, (starts[-1], heads, 1)))       # some blocks' scales grow, some do not
        x.append(torch.from_numpy(values).to(dtype))
        O.write(s.data[which], s.scale[which], x[which].float().numpy(), s.table, lens, starts, fmt)
    backend.kv_cache_write(s.cache, *(laid_out(t.cuda(), layout) for t in x), s.d_table, s.ints(lens), s.ints(starts),
                           max_query_len=max(new))
    backend.check_status()
    s.check_bytes()


def test_appending_token_by_token(backend):
    """80 single-token steps through two pages; the page that a sequence starts is taken over
    whatever scale it held before."""
    lens, heads, dim = [0, 0], 2, 64
    s = Setup(backend, [80, 70], kv_heads=heads, dim=dim, page=64, seed=5)
    for scale in s.scale:
        scale[:] = 1e6                           # stale contents of a reused page
    s.to_device()
    for step in range(80):
        live = [b for b in range(2) if step < s.lens[b]]
        lens = [min(step + 1, n) for n in s.lens]
        new = [1 if b in live else 0 for b in range(2)]
        starts = starts_of(new)
        x = [torch.from_numpy((s.rng.standard_normal((starts[-1], heads, dim)) * (1 + step / 10)).astype(np.float16))
             for _ in range(2)]
        for which in range(2):
            # the oracle walks pages of sequences with new tokens only
            for b in live:
                O.write(s.data[which], s.scale[which], x[which].float().numpy()[starts[b]:starts[b + 1]],
                        s.table[b:b + 1], [lens[b]], [0, 1], "int8")
        backend.kv_cache_write(s.cache, x[0].cuda(), x[1].cuda(), s.d_table, s.ints(lens), s.ints(starts), max_query_len=1)
    backend.check_status()
    s.check_bytes()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_block_with_a_value_that_is_not_finite(backend, fmt, bad):
    """Its scale is NaN, also after later writes to the page; other blocks are untouched."""
    s = Setup(backend, [40], fmt=fmt, seed=9)
    x = torch.randn(8, 2, 64, generator=torch.Generator().manual_seed(1)).half()
    x[3, 1, 7] = bad
    backend.kv_cache_write(s.cache, x.cuda(), x.cuda(), s.d_table, s.ints([40]), s.ints([0, 8]))
    scale = s.cache.k_scale.cpu().numpy()
    page = s.table[0, 2]
    assert np.isnan(scale[page, 1]) and np.isnan(s.cache.v_scale.cpu().numpy()[page, 1])
    scale[page] = s.scale[0][page]
    assert np.array_equal(scale, s.scale[0]) or np.isfinite(scale).all()
    y = torch.ones(1, 2, 64).half()
    backend.kv_cache_write(s.cache, y.cuda(), y.cuda(), s.d_table, s.ints([41]), s.ints([0, 1]))
    assert np.isnan(s.cache.k_scale.cpu().numpy()[page, 1]) and np.isfinite(s.cache.k_scale.cpu().numpy()[page, 0])
    backend.check_status()


def test_values_of_zero_and_of_the_type_s_ends(backend):
    s = Setup(backend, [16, 16, 16], seed=3)
    x = torch.zeros(48, 2, 64, dtype=torch.float32)
    x[16:32] = 1e-38
    x[32:48] = 3.0e38
    x[32:48, :, ::2] *= -1
    for which in range(2):
        O.write(s.data[which], s.scale[which], x.numpy(), s.table, [16] * 3, [0, 16, 32, 48], "int8")
    backend.kv_cache_write(s.cache, x.cuda(), x.cuda(), s.d_table, s.ints([16] * 3), s.ints([0, 16, 32, 48]))
    s.check_bytes()


# ---------------------------------------------------------------------------------------
# read
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens,first,heads,dim,page,fmt,dtype", [
    ([1], [0], 1, 64, 16, "int8", torch.float16),
    ([40, 0, 17, 200], [3, 0, 16, 0], 3, 80, 16, "int8", torch.bfloat16),
    ([300, 129], [128, 0], 2, 256, 128, "e4m3", torch.float32),
    ([1000], [1], 12, 64, 32, "e4m3", torch.float16),
    ([515, 64], [2, 64], 2, 16, 64, "int8", torch.float32),
])
def test_read_is_bit_exact(backend, lens, first, heads, dim, page, fmt, dtype):
    s = Setup(backend, lens, kv_heads=heads, dim=dim, page=page, fmt=fmt, seed=dim)
    starts = starts_of([n - f for n, f in zip(lens, first)])
    rows = starts[-1] + 2                        # two rows behind the last sequence
    out = tuple(torch.full((rows, heads, dim), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    got = backend.kv_cache_read(s.cache, s.d_table, s.ints(first), s.ints(starts), rows=rows, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    again = backend.kv_cache_read(s.cache, s.d_table, s.ints(first), s.ints(starts), rows=starts[-1],
                                  max_rows=max(n - f for n, f in zip(lens, first)), dtype=dtype)
    backend.check_status()
    for which in range(2):
        want = np.concatenate([O.tokens_of(s.data[which], s.scale[which], s.table, b, f, n, fmt)
                               for b, (f, n) in enumerate(zip(first, lens))])
        want = torch.from_numpy(want).to(dtype)
        assert torch.equal(out[which][:-2].cpu(), want) and torch.equal(again[which].cpu(), want)
        assert (out[which][-2:] == 7.0).all()


# ---------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------
def attention_bound(want, spread, loud, dim, dtype, keys, largest):
    score = (dim + 8) * 2.0 ** -22 * loud[:, :, None]
    return (HALF_STEP[dtype] * np.abs(want) + (2.0 ** -11 + 2.0 ** -20 + 2 * score) * spread * 1.01 +
            keys * 2.0 ** -25 * largest + 2.0 ** -24)


def check_attention(s, q, new, got, lse, *, scale, causal=True, window=0, dtype):
    starts, dim = starts_of(new), q.shape[2]
    got = got.float().cpu().numpy().astype(np.float64)
    for b, n in enumerate(new):
        keys, values = s.values(b, 0), s.values(b, 1)
        rows = slice(starts[b], starts[b + 1])
        want, want_lse, spread, loud = O.attention(q[rows].float().numpy(), keys, values, s.lens[b], scale=scale,
                                                   causal=causal, window=window)
        largest = float(np.abs(values).max()) if len(values) else 0.0
        bound = attention_bound(want, spread, loud, dim, dtype, len(keys), largest)
        error = np.abs(got[rows] - want)
        assert np.isfinite(got[rows]).all()
        assert (error <= bound).all(), (b, float((error - bound).max()), float((error / bound).max()))
        empty = np.isneginf(want_lse)
        assert (got[rows][empty] == 0).all()
        if lse is not None:
            l = lse.cpu().numpy().astype(np.float64)[rows]
            assert np.array_equal(np.isneginf(l), empty)
            with np.errstate(invalid="ignore"):
                slack = (dim + 8) * 2.0 ** -22 * loud + 2.0 ** -20 * (1 + np.abs(want_lse))
                assert (np.abs(l - want_lse) <= slack)[~empty].all()


ATTENTION = [
    # lens, new tokens, heads, kv_heads, dim, page, format, type, window, causal
    ([1], [1], 1, 1, 64, 16, "int8", torch.float16, 0, True),
    ([5, 64, 0, 1, 130], [1, 1, 1, 1, 1], 4, 2, 64, 16, "int8", torch.float16, 0, True),
    ([515, 3], [1, 1], 8, 1, 128, 64, "int8", torch.bfloat16, 0, True),        # one shared head
    ([700, 1300], [1, 1], 12, 12, 64, 64, "int8", torch.float16, 0, True),
    ([333, 90], [5, 2], 14, 2, 80, 32, "e4m3", torch.float16, 64, True),      # seven heads share one
    ([260, 100, 17], [3, 100, 17], 6, 2, 128, 16, "int8", torch.float16, 0, True),   # decode beside prompts
    ([200], [200], 4, 4, 64, 32, "e4m3", torch.bfloat16, 0, True),
    ([257, 129], [129, 65], 8, 2, 128, 128, "int8", torch.bfloat16, 0, True),
    ([150], [90], 3, 1, 256, 64, "int8", torch.float16, 0, True),
    ([333], [140], 4, 2, 96, 64, "e4m3", torch.float16, 50, True),
    ([40, 7], [12, 10], 4, 2, 64, 16, "int8", torch.float16, 0, True),        # more queries than tokens
    ([100, 30], [7, 30], 2, 2, 64, 16, "int8", torch.float16, 0, False),      # every query sees everything
    ([300], [130], 2, 1, 64, 64, "int8", torch.float16, 0, False),
    ([64, 65, 63], [1, 2, 64], 40, 1, 64, 64, "int8", torch.float16, 1, True),   # forty heads share one, itself only
    ([128, 31], [3, 31], 4, 2, 16, 16, "int8", torch.float16, 0, True),
    ([70, 3], [3, 1], 130, 1, 64, 64, "int8", torch.float16, 0, True),        # more heads share one than a tile has rows
    ([129, 257], [128, 129], 2, 2, 128, 32, "e4m3", torch.bfloat16, 2 ** 40, True),   # a window wider than anything
    ([700, 300, 0, 129], [300, 299, 0, 1], 6, 2, 256, 64, "e4m3", torch.float16, 0, True),   # wide heads: prompts, one token
    ([333], [333], 2, 2, 144, 16, "int8", torch.bfloat16, 100, True),
    ([260, 40], [200, 45], 40, 1, 208, 128, "int8", torch.float16, 0, True),
    ([515, 20], [129, 33], 3, 3, 160, 32, "e4m3", torch.bfloat16, 0, False),
    ([2000], [130], 2, 2, 256, 128, "int8", torch.bfloat16, 0, True),         # wide heads, keys split among many CTAs
]


@pytest.mark.parametrize("lens,new,heads,kv_heads,dim,page,fmt,dtype,window,causal", ATTENTION)
def test_attention(backend, lens, new, heads, kv_heads, dim, page, fmt, dtype, window, causal):
    s = Setup(backend, lens, kv_heads=kv_heads, dim=dim, page=page, fmt=fmt, seed=heads * dim + sum(lens))
    starts = starts_of(new)
    q = torch.from_numpy(s.rng.standard_normal((starts[-1] + 1, heads, dim)).astype(np.float32)).to(dtype)
    scale = dim ** -0.5
    out = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
    got, lse = backend.kv_cache_attention(q.cuda(), s.cache, s.d_table, s.ints(lens), s.ints(starts),
                                          max_query_len=max(new), causal=causal, window=window or None, out=out,
                                          return_lse=True)
    assert got is out and (out[-1] == 5.0).all()              # the row behind the last sequence
    check_attention(s, q, new, got, lse, scale=scale, causal=causal, window=window, dtype=dtype)
    # without the bound on the new tokens, q as a column block, out and q with other strides
    wide = torch.zeros((q.shape[0], heads + 3, dim), dtype=dtype, device="cuda")
    wide[:, 1:heads + 1] = q.cuda()
    out2 = torch.zeros((heads, q.shape[0], dim), dtype=dtype, device="cuda").transpose(0, 1)
    got2 = backend.kv_cache_attention(wide[:, 1:heads + 1], s.cache, s.d_table, s.ints(lens), s.ints(starts),
                                      causal=causal, window=window or None, softmax_scale=scale, out=out2)
    check_attention(s, q, new, got2, None, scale=scale, causal=causal, window=window, dtype=dtype)
    odd = torch.zeros((q.shape[0], heads, dim + 1), dtype=dtype, device="cuda")
    odd[:, :, 1:] = q.cuda()
    got3 = backend.kv_cache_attention(odd[:, :, 1:], s.cache, s.d_table, s.ints(lens), s.ints(starts),
                                      max_query_len=max(new), causal=causal, window=window or None)
    assert torch.equal(got3[:starts[-1]], got[:starts[-1]])
    backend.check_status()


@pytest.mark.parametrize("new", [2, 75])
@pytest.mark.parametrize("scale", [-0.25, 0.0, 1e-30, 3.0])
def test_attention_with_any_scale(backend, new, scale):
    lens = [140, 75]
    s = Setup(backend, lens, kv_heads=2, dim=64, page=32, seed=12)
    q = torch.from_numpy(s.rng.standard_normal((2 * new, 6, 64)).astype(np.float32)).bfloat16()
    got, lse = backend.kv_cache_attention(q.cuda(), s.cache, s.d_table, s.ints(lens), s.ints(starts_of([new, new])),
                                          softmax_scale=scale, return_lse=True)
    check_attention(s, q, [new, new], got, lse, scale=scale, dtype=torch.bfloat16)


def test_a_bound_that_is_too_small_costs_time_only(backend):
    """Attention uses max_query_len to choose its tiles; results do not depend on it."""
    lens, new = [300, 40], [90, 1]
    s = Setup(backend, lens, kv_heads=2, dim=64, page=32, seed=13)
    q = torch.from_numpy(s.rng.standard_normal((91, 4, 64)).astype(np.float32)).half()
    for bound in (0, 1, 5, 90, 1000):
        got = backend.kv_cache_attention(q.cuda(), s.cache, s.d_table, s.ints(lens), s.ints(starts_of(new)), max_query_len=bound)
        check_attention(s, q, new, got, None, scale=0.125, dtype=torch.float16)
    backend.check_status()


@pytest.mark.parametrize("new,bound", [(1, 2 ** 30), (2, 2 ** 31 - 1), (70, 2 ** 30)])
def test_workspace_covers_any_bound(backend, new, bound):
    """The C entry with a bound beyond the tokens stays inside the bytes that it asked for."""
    import ctypes as C
    from rns_llm_b200 import _native as N

    s = Setup(backend, [5000], kv_heads=2, dim=64, page=64, seed=16)
    q = torch.from_numpy(s.rng.standard_normal((new, 8, 64)).astype(np.float32)).half().cuda()
    lens, starts, out = s.ints([5000]), s.ints([0, new]), torch.empty_like(q)
    cache = backend._kv_args(s.cache, s.d_table, lens, starts)
    args = N.KVAttentionArgs(q.data_ptr(), N.F16, 8, new, q.stride(0), q.stride(1), lens.data_ptr(), starts.data_ptr(), bound,
                             1, 0, 0.125, out.data_ptr(), out.stride(0), out.stride(1), None, None, 0)
    lib = N.load()
    need = lib.rns_kv_attention_workspace(C.byref(cache), C.byref(args))
    work = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
    args.d_workspace, args.workspace_bytes = work.data_ptr(), need
    stream = torch.cuda.current_stream().cuda_stream
    N.check(lib.rns_kv_attention(C.byref(cache), C.byref(args), stream))
    assert (work[need:] == 0x5a).all()
    check_attention(s, q.cpu(), [new], out, None, scale=0.125, dtype=torch.float16)
    for bad in (dict(workspace_bytes=need - 1), dict(d_workspace=work.data_ptr() + 8), dict(d_workspace=None)):
        for name, value in bad.items():
            kept = getattr(args, name)
            setattr(args, name, value)
            assert lib.rns_kv_attention(C.byref(cache), C.byref(args), stream) == N.ERR_INVALID_ARGUMENT
            setattr(args, name, kept)


def test_many_sequences(backend):
    """More sequences than threads of a block, most of them empty or without queries."""
    rng = np.random.default_rng(3)
    lens = [int(n) if keep else 0 for n, keep in zip(rng.integers(1, 40, 1300), rng.random(1300) < 0.3)]
    new = [int(rng.integers(0, 3)) for _ in lens]
    s = Setup(backend, lens, kv_heads=1, dim=16, page=16, seed=14)
    q = torch.from_numpy(s.rng.standard_normal((sum(new), 2, 16)).astype(np.float32)).half()
    for bound in (2, 40):                                        # the rows kernel; the prompt kernel (by its bound)
        got, lse = backend.kv_cache_attention(q.cuda(), s.cache, s.d_table, s.ints(lens), s.ints(starts_of(new)),
                                              max_query_len=bound, return_lse=True)
        check_attention(s, q, new, got, lse, scale=0.25, dtype=torch.float16)


def test_other_device_and_stream_are_left_alone(backend):
    """The call runs on the current stream of the cache's device and leaves both as they were."""
    s = Setup(backend, [100], kv_heads=2, dim=64, page=32, seed=15)
    q = torch.from_numpy(s.rng.standard_normal((1, 4, 64)).astype(np.float32)).half().cuda()
    lens, starts = s.ints([100]), s.ints([0, 1])
    want = backend.kv_cache_attention(q, s.cache, s.d_table, lens, starts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = backend.kv_cache_attention(q, s.cache, s.d_table, lens, starts)
        assert torch.cuda.current_stream() == side
    side.synchronize()
    assert torch.equal(got, want) and torch.cuda.current_device() == 0


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("gain,spread", [(300.0, 0.5), (1e-6, 0.5), (1.0, 4.0), (20.0, 3.0)])
def test_attention_over_wide_ranges(backend, new, gain, spread):
    """Scores from nothing to one-hot, pages whose scales differ by many orders of magnitude."""
    lens = [400, 90]
    s = Setup(backend, lens, kv_heads=2, dim=64, page=16, seed=int(gain * 10) + int(spread), spread=spread)
    starts = starts_of([new, new])
    q = torch.from_numpy((s.rng.standard_normal((starts[-1], 4, 64)) * gain).astype(np.float32)).half()
    scale = 0.125 if spread < 1 else 1e-3
    got, lse = backend.kv_cache_attention(q.cuda(), s.cache, s.d_table, s.ints(lens), s.ints(starts),
                                          softmax_scale=scale, return_lse=True)
    check_attention(s, q, [new, new], got, lse, scale=scale, dtype=torch.float16)


@pytest.mark.parametrize("new", [1, 80])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_masked_places_have_no_part(backend, fmt, new):
    """Bytes behind a sequence's length (NaN patterns among them), pages with scale NaN or infinity
    that the queries do not see, and queries of other rows that are not finite."""
    lens = [150, 150]
    s = Setup(backend, lens, dim=64, page=16, fmt=fmt, seed=4)
    q = torch.from_numpy(s.rng.standard_normal((2 * new, 4, 64)).astype(np.float32)).half()
    starts, window = s.ints([0, new, 2 * new]), 32
    args = (s.d_table, s.ints(lens), starts)
    clean = backend.kv_cache_attention(q.cuda(), s.cache, *args, window=window)
    check_attention(s, q, [new, new], clean, None, scale=0.125, window=window, dtype=torch.float16)
    for b in range(2):                               # rows 150 .. 159 of the last page
        for data in s.data:
            data[s.table[b, 9], :, 6:] = 0x7f
    hidden = (150 - new - window) // 16              # pages wholly before every window
    for scale in s.scale:
        scale[s.table[0, :hidden]] = np.nan
        scale[s.table[1, :hidden]] = np.inf
    s.to_device()
    got = backend.kv_cache_attention(q.cuda(), s.cache, *args, window=window)
    assert torch.equal(got, clean)
    # a page whose scale is NaN reaches the rows that see it and no others
    for scale in s.scale:
        scale[s.table[0, 9]] = np.nan                # positions 144 .. 149
    s.to_device()
    got = backend.kv_cache_attention(q.cuda(), s.cache, *args, window=window)
    first = max(0, new - 6)
    assert torch.isnan(got[first:new]).all()
    assert torch.equal(got[:first], clean[:first]) and torch.equal(got[new:], clean[new:])
    # likewise a query
    q[0, 1, 3] = float("inf")
    q[new, 2, 0] = float("nan")
    s2 = Setup(backend, lens, dim=64, page=16, fmt=fmt, seed=4)
    got = backend.kv_cache_attention(q.cuda(), s2.cache, *args, window=window)
    assert torch.isnan(got[0, 1]).any() and torch.isnan(got[new, 2]).any()
    keep = torch.ones(2 * new, 4, dtype=torch.bool)
    keep[0, 1] = keep[new, 2] = False
    assert torch.equal(got[keep.cuda()], clean[keep.cuda()])
    backend.check_status()


@pytest.mark.parametrize("new", [1, 100])
def test_long_cache_and_shared_pages(backend, new):
    """Thousands of keys, so that the key axis is split; two sequences share their prefix pages."""
    lens = [5000, 4990, 120]
    s = Setup(backend, lens, kv_heads=2, dim=64, page=64, seed=8)
    s.table[1, :78] = s.table[0, :78]
    s.to_device()
    q = torch.from_numpy(s.rng.standard_normal((3 * new, 4, 64)).astype(np.float32)).half()
    got, lse = backend.kv_cache_attention(q.cuda(), s.cache, s.d_table, s.ints(lens), s.ints(starts_of([new] * 3)),
                                          max_query_len=new, return_lse=True)
    check_attention(s, q, [new] * 3, got, lse, scale=0.125, dtype=torch.float16)


def test_pages_beyond_32_bit_offsets(backend):
    """A cache of more than 2^32 bytes a side, its last pages in use."""
    page, heads, dim = 128, 8, 256
    pages = (1 << 32) // (page * heads * dim) + 5
    cache = backend.create_kv_cache(pages=pages, kv_heads=heads, head_dim=dim, page_tokens=page)
    gen = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(200, heads, dim, generator=gen, device="cuda").half() for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 2], [0, 1]], dtype=torch.int32, device="cuda")
    small = backend.create_kv_cache(pages=4, kv_heads=heads, head_dim=dim, page_tokens=page)
    small_table = torch.tensor([[3, 2], [0, 1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([200, 0], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 200, 200], dtype=torch.int32, device="cuda")
    q = torch.randn(200, 16, dim, generator=gen, device="cuda").half()
    results = []
    for c, t in ((cache, table), (small, small_table)):
        backend.kv_cache_write(c, k, v, t, lens, starts)
        read = backend.kv_cache_read(c, t, torch.zeros_like(lens), starts, rows=200)
        many = backend.kv_cache_attention(q, c, t, lens, starts)
        one = backend.kv_cache_attention(q[-1:], c, t, lens, torch.tensor([0, 1, 1], dtype=torch.int32, device="cuda"))
        results.append((*read, many, one))
    backend.check_status()
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert (cache.k_scale[:2] == 0).all()


def decode_steps(backend, s, x, q, table, lens, starts):
    outs = []
    for step in range(len(q)):
        lens += 1
        backend.kv_cache_write(s.cache, x[step], x[step], table, lens, starts, max_query_len=1)
        outs.append(backend.kv_cache_attention(q[step], s.cache, table, lens, starts, max_query_len=1))
    return outs


def test_captured_steps_replay(backend):
    """Write and attention of one token in a graph, replayed while lengths advance on the device;
    two graphs captured on one stream keep separate scratch and may run side by side."""
    lens0, heads = [700, 33], 4
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(6, 2, 2, 64, generator=gen, device="cuda").half()
    q = torch.randn(6, 2, heads, 64, generator=gen, device="cuda").half()
    whole = [720, 60]
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    eager = Setup(backend, whole, page=32, seed=6)
    want = decode_steps(backend, eager, x, q, eager.d_table, eager.ints(lens0), starts)
    runs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            s = Setup(backend, whole, page=32, seed=6)
            lens, xs, qs = s.ints(lens0), x[0].clone(), q[0].clone()
            # the shapes run once before the capture, on a copy of the cache
            warm = Setup(backend, whole, page=32, seed=6)
            decode_steps(backend, warm, x[:1], q[:1], warm.d_table, lens.clone(), starts)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                lens += 1
                backend.kv_cache_write(s.cache, xs, xs, s.d_table, lens, starts, max_query_len=1)
                out = backend.kv_cache_attention(qs, s.cache, s.d_table, lens, starts, max_query_len=1)
            runs.append((graph, s, lens, xs, qs, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(6):
        for stream, (graph, s, lens, xs, qs, out) in zip(streams, runs):
            with torch.cuda.stream(stream):
                xs.copy_(x[step])
                qs.copy_(q[step])
                graph.replay()
        torch.cuda.synchronize()
        for run in runs:
            assert torch.equal(run[5], want[step])
    for run in runs:
        assert torch.equal(run[1].cache.k, eager.cache.k) and torch.equal(run[1].cache.k_scale, eager.cache.k_scale)
    backend.check_status()
    del runs


def test_two_streams_at_once(backend):
    s = [Setup(backend, [3000, 2000], kv_heads=2, dim=128, page=64, seed=i) for i in range(2)]
    q = [torch.from_numpy(x.rng.standard_normal((2, 8, 128)).astype(np.float32)).half().cuda() for x in s]
    starts = s[0].ints([0, 1, 2])
    lens = s[0].ints([3000, 2000])
    alone = [backend.kv_cache_attention(q[i], s[i].cache, s[i].d_table, lens, starts) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(backend.kv_cache_attention(q[i], s[i].cache, s[i].d_table, lens, starts))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])      # and runs agree bit for bit


def test_out_of_range_indices_are_reported(backend):
    s = Setup(backend, [40, 20], seed=2)
    good = s.d_table.clone()
    q = torch.ones(2, 4, 64, dtype=torch.float16, device="cuda")
    x = torch.ones(2, 2, 64, dtype=torch.float16, device="cuda")
    starts, lens = s.ints([0, 1, 2]), s.ints([40, 20])
    before = (s.cache.k.clone(), s.cache.k_scale.clone())
    bad_table = good.clone()
    bad_table[0] = 10 ** 6
    fine = backend.kv_cache_attention(q, s.cache, good, lens, starts)
    for table, n, st in ((bad_table, lens, starts), (good, s.ints([10 ** 6, 20]), starts), (good, lens, s.ints([5, 1, 2]))):
        s.to_device()                                          # the writes below change sequence 1
        out = backend.kv_cache_attention(q, s.cache, table, n, st)
        with pytest.raises(RuntimeError, match="out of range"):
            backend.check_status()
        assert torch.equal(out[1], fine[1])                    # the other sequence is served
        backend.kv_cache_write(s.cache, x, x, table, n, st)
        with pytest.raises(RuntimeError, match="out of range"):
            backend.check_status()
        page = s.table[1, 1]
        changed = (s.cache.k_scale != before[1]).any(dim=1).cpu().numpy()
        assert changed.sum() <= 1 and not np.delete(changed, page).any()
    k, v = backend.kv_cache_read(s.cache, bad_table, s.ints([0, 0]), s.ints([0, 40, 60]), rows=60)
    assert (k[:40] == 0).all() and (k[40:] != 0).any()
    with pytest.raises(RuntimeError, match="out of range"):
        backend.check_status()
    backend.kv_cache_read(s.cache, good, s.ints([10 ** 6, -3]), s.ints([0, 40, 60]), rows=60)
    with pytest.raises(RuntimeError, match="out of range"):
        backend.check_status()
    # a bound on the new tokens that is too small is reported, and nothing is written
    scale = s.cache.k_scale.clone()
    many = torch.full((4, 2, 64), 1e4, dtype=torch.float16, device="cuda")
    backend.kv_cache_write(s.cache, many, many, good, lens, s.ints([0, 3, 4]), max_query_len=1)
    with pytest.raises(RuntimeError, match="out of range"):
        backend.check_status()
    assert torch.equal(s.cache.k_scale[s.table[0, :3]], scale[s.table[0, :3]])
    backend.check_status()


def test_refused_calls(backend):
    s = Setup(backend, [40, 20])
    q = torch.ones(2, 4, 64, dtype=torch.float16, device="cuda")
    x = torch.ones(2, 2, 64, dtype=torch.float16, device="cuda")
    lens, starts = s.ints([40, 20]), s.ints([0, 1, 2])

    def attend(q=q, table=s.d_table, lens=lens, starts=starts, **kw):
        return backend.kv_cache_attention(q, s.cache, table, lens, starts, **kw)

    for bad in (lambda: attend(q.float()), lambda: attend(q[:, :3]), lambda: attend(q[:, :, :32]), lambda: attend(q.cpu()),
                lambda: attend(q.transpose(1, 2).contiguous().transpose(1, 2)), lambda: attend(q[:, :0]),
                lambda: attend(table=s.d_table.long()), lambda: attend(table=s.d_table[:1]), lambda: attend(lens=lens.long()),
                lambda: attend(lens=lens.cpu()), lambda: attend(starts=starts[:2]), lambda: attend(starts=starts.float()),
                lambda: attend(window=0), lambda: attend(window=-1), lambda: attend(window=4, causal=False),
                lambda: attend(out=q), lambda: attend(out=torch.empty_like(q).float()),
                lambda: attend(out=torch.empty(1, 4, 64, dtype=q.dtype, device="cuda").expand(2, 4, 64)),
                lambda: attend(softmax_scale=float("nan")), lambda: attend(max_query_len=-1),
                lambda: backend.kv_cache_write(s.cache, x, x.float(), s.d_table, lens, starts),
                lambda: backend.kv_cache_write(s.cache, x.to(torch.int8), x.to(torch.int8), s.d_table, lens, starts),
                lambda: backend.kv_cache_write(s.cache, x[:, :1], x[:, :1], s.d_table, lens, starts),
                lambda: backend.kv_cache_write(s.cache, x.cpu(), x, s.d_table, lens, starts),
                lambda: backend.kv_cache_write(s.cache, x, x, s.d_table, lens, starts, max_query_len=-1),
                lambda: backend.kv_cache_read(s.cache, s.d_table, lens, starts, rows=-1),
                lambda: backend.kv_cache_read(s.cache, s.d_table, lens, starts, rows=2, dtype=torch.int8),
                lambda: backend.kv_cache_read(s.cache, s.d_table, lens, starts, rows=2, out=(x, x[:1])),
                lambda: backend.create_kv_cache(pages=2, kv_heads=2, head_dim=64, format="int4"),
                lambda: backend.create_kv_cache(pages=2, kv_heads=2, head_dim=72),
                lambda: backend.create_kv_cache(pages=0, kv_heads=2, head_dim=64),
                lambda: backend.create_kv_cache(pages=2, kv_heads=2, head_dim=64, page_tokens=24)):
        with pytest.raises(ValueError):
            bad()
    # calls without work
    none = torch.empty(0, 4, 64, dtype=torch.float16, device="cuda")
    assert backend.kv_cache_attention(none, s.cache, s.d_table, lens, s.ints([0, 0, 0])).shape == (0, 4, 64)
    assert attend(q[:0], s.d_table[:0], lens[:0], starts[:1]).shape == (0, 4, 64)
    backend.kv_cache_write(s.cache, x[:0], x[:0], s.d_table, lens, s.ints([0, 0, 0]))
    backend.check_status()
