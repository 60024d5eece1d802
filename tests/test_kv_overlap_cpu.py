"""Outputs of the quantised cache's calls that share memory with another tensor of the call are told apart from
those that do not (host side, on CPU tensors)."""
import random

import pytest
import torch

from rns_llm_b200.backends import QuantizedKVCache
from rns_llm_b200.backends.kv_cache import _rows_meet, _spans_meet


def elements(t):
    at = torch.arange(t.untyped_storage().nbytes() // t.element_size())
    return set(torch.as_strided(at, t.shape, t.stride(), t.storage_offset()).flatten().tolist())


def test_rows_that_meet_against_their_elements():
    rng = random.Random(1)
    buffer, seen = torch.zeros(4000, dtype=torch.float16), [0, 0]
    for _ in range(4000):
        rows, heads, dim = rng.randint(1, 5), rng.randint(1, 4), rng.choice((1, 2, 16))
        head = dim + rng.choice((0, 0, 1, dim))
        row = (heads - 1) * head + dim + rng.choice((0, 0, 3, 2 * heads * head))
        strides = (row, head, 1) if rng.random() < 0.7 else (dim + rng.choice((0, dim)), rows * 2 * dim, 1)
        a, b = (torch.as_strided(buffer, (rows, heads, dim), strides, rng.randint(0, 150)) for _ in range(2))
        meet = bool(elements(a) & elements(b))
        assert _rows_meet(a, b) == meet
        seen[meet] += 1
        other = torch.as_strided(buffer, (rows, heads, dim), (heads * dim, dim, 1), rng.randint(0, 150))
        if elements(a) & elements(other):
            assert _rows_meet(a, other) and _spans_meet(a, other)
    assert min(seen) > 500
    wide = torch.zeros(7, 9, 16)
    assert not _rows_meet(wide[:, :3], wide[:, 3:6]) and not _rows_meet(wide[:, ::3], wide[:, 1::3])
    assert _rows_meet(wide[1:, :3], wide[:-1, :3]) and _rows_meet(wide[:, :3], wide[:, 2:5])
    assert not _rows_meet(wide[:0], wide[:0])


def test_a_cache_whose_tensors_overlap_is_refused():
    both, scales = torch.zeros(3, 2, 16, 64, dtype=torch.int8), torch.zeros(3, 2)
    for change in (dict(v=both[:2]), dict(v=both[1:]), dict(v_scale=scales[:2]), dict(v_scale=scales[1:])):
        tensors = dict(k=both[:2], v=torch.zeros_like(both[:2]), k_scale=scales[:2], v_scale=torch.zeros(2, 2), **{})
        tensors.update(change)
        with pytest.raises(ValueError, match="overlap"):
            QuantizedKVCache(**tensors)
    with pytest.raises(ValueError, match="CUDA"):                  # halves of one allocation are apart
        QuantizedKVCache(k=both[:1], v=both[1:2], k_scale=scales[:1], v_scale=scales[1:2])
