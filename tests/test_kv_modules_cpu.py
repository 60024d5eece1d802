"""OPT blocks over the quantised cache without a GPU: which masks, models and calls they take.

The backend is a stand-in that keeps the cached keys and values as they are, in float32, so what a block
computes can be compared with the model's own attention.
"""
import types

import pytest
import torch

from rns_llm_b200.integration import use_quantized_cache
from rns_llm_b200.layers import QuantizedCacheAttention, QuantizedDecoderCache

transformers = pytest.importorskip("transformers")


class PlainBackend:
    """The two calls of the cache on rows [pages * page_tokens] of one page table, causal."""

    def create_kv_cache(self, *, pages, kv_heads, head_dim, page_tokens, format, device):
        if format not in ("int8", "e4m3"):
            raise ValueError("format")
        shape = (pages * page_tokens, kv_heads, head_dim)
        return types.SimpleNamespace(device=torch.device("cpu"), page=page_tokens, kv_heads=kv_heads, head_dim=head_dim,
                                     k=torch.zeros(shape), v=torch.zeros(shape), k_scale=torch.zeros(pages, kv_heads),
                                     v_scale=torch.zeros(pages, kv_heads))

    def rows(self, cache, table, b, n):
        at = torch.arange(n)
        return table[b].long()[at // cache.page] * cache.page + at % cache.page

    def kv_cache_write(self, cache, k, v, table, lens, starts, *, max_query_len):
        for b, n in enumerate(lens.tolist()):
            new = slice(int(starts[b]), int(starts[b + 1]))
            rows = self.rows(cache, table, b, n)[n - (new.stop - new.start):]
            cache.k[rows], cache.v[rows] = k[new].float(), v[new].float()

    def kv_cache_attention(self, q, cache, table, lens, starts, *, max_query_len, softmax_scale):
        out = torch.zeros_like(q)
        for b, n in enumerate(lens.tolist()):
            new = slice(int(starts[b]), int(starts[b + 1]))
            rows = self.rows(cache, table, b, n)
            scores = torch.einsum("qhd,khd->hqk", q[new].float(), cache.k[rows]) * softmax_scale
            first = n - (new.stop - new.start)
            hidden = torch.arange(n) > torch.arange(first, n)[:, None]
            weights = scores.masked_fill(hidden, float("-inf")).softmax(-1)
            out[new] = torch.einsum("hqk,khd->qhd", weights, cache.v[rows]).to(q.dtype)
        return out


def small_opt(implementation="sdpa", dtype=torch.bfloat16):
    config = transformers.OPTConfig(vocab_size=64, hidden_size=64, num_hidden_layers=2, num_attention_heads=2, ffn_dim=64,
                                    max_position_embeddings=64, word_embed_proj_dim=64)
    torch.manual_seed(7)
    return transformers.OPTForCausalLM._from_config(config, attn_implementation=implementation).to(dtype).eval()


def cache_for(model, batch=2, max_tokens=40, **kw):
    return QuantizedDecoderCache.for_model(model, PlainBackend(), batch=batch, max_tokens=max_tokens, page_tokens=16, **kw)


IDS = torch.arange(2 * 30).view(2, 30) % 61


@pytest.mark.parametrize("implementation", ["sdpa", "eager"])
def test_model_on_the_cache_is_the_model(implementation):
    """Prompt, a chunk behind it and single tokens, with and without a mask of ones."""
    model, wrapped = small_opt(implementation), small_opt(implementation)
    use_quantized_cache(wrapped)
    cache, own, at = cache_for(wrapped), None, 0
    with torch.no_grad():
        for n, ones in ((7, False), (5, True), (1, False), (1, True), (3, False)):
            mask = torch.ones(2, at + n, dtype=torch.long) if ones else None
            ids = IDS[:, at:at + n]
            want = model(input_ids=ids, past_key_values=own, attention_mask=mask, use_cache=True)
            own = want.past_key_values
            got = wrapped(input_ids=ids, past_key_values=cache, attention_mask=mask, use_cache=True).logits
            at += n
            # bfloat16 activations of about 1 through two layers
            assert (got - want.logits).abs().max() < 0.05
            assert cache.get_seq_length() == at


def causal(new, total, kind):
    seen = torch.arange(total) <= torch.arange(total - new, total)[:, None]
    if kind == "bool":
        return seen.expand(2, 1, new, total).clone()
    low = float("-inf") if kind == "inf" else torch.finfo(torch.bfloat16).min
    return torch.zeros(2, 1, new, total, dtype=torch.bfloat16).masked_fill(~seen, low)


@pytest.mark.parametrize("layer", [0, 1])
@pytest.mark.parametrize("kind", ["bool", "min", "inf"])
@pytest.mark.parametrize("past,new", [(0, 6), (4, 3), (5, 1)])
def test_masks_that_are_not_causal_are_refused(kind, past, new, layer):
    model = small_opt()
    use_quantized_cache(model)
    block = model.model.decoder.layers[layer].self_attn
    x = torch.randn(2, past + new, 64, generator=torch.Generator().manual_seed(1)).bfloat16()
    total = past + new

    def run(mask):
        cache = cache_for(model)
        with torch.no_grad():
            if past:
                block(x[:, :past], past_key_values=cache)
            return block(x[:, past:], past_key_values=cache, attention_mask=mask)[0]

    want = run(None)
    good = causal(new, total, kind)
    assert torch.equal(run(good), want)
    assert torch.equal(run(good[:1]), want) and torch.equal(run(good[:, :, :, :]), want)
    bad = []
    for query, key in ((new - 1, 0), (0, past), (new - 1, total - 1)):      # a key hidden that the query sees
        mask = good.clone()
        mask[1, 0, query, key] = False if kind == "bool" else good.min() if new > 1 else float("-inf")
        if not torch.equal(mask, good):
            bad.append(mask)
    if new > 1:
        mask = good.clone()
        mask[0, 0, 0, total - 1] = True if kind == "bool" else 0.0           # a later key seen
        bad.append(mask)
    if kind != "bool":
        mask = good.clone()
        mask[0, 0, new - 1, 0] = -0.5                                        # a bias on a score
        bad.append(mask)
    bad += [good[..., :-1], torch.cat((good, good[..., :1]), -1), good[:, :, :1] if new > 1 else good[..., :0],
            good[:, 0], good.expand(2, 2, new, total)[:, :, :, 1:]]
    for mask in bad:
        with pytest.raises(ValueError, match="mask"):
            run(mask)


def test_masks_of_other_forms():
    """[batch, tokens]: ones only; integers of four dimensions and objects that are no tensors are refused."""
    model = small_opt()
    use_quantized_cache(model)
    block = model.model.decoder.layers[0].self_attn
    x = torch.randn(2, 4, 64).bfloat16()
    run = lambda mask: block(x, past_key_values=cache_for(model), attention_mask=mask)
    with torch.no_grad():
        for dtype in (torch.long, torch.bool, torch.bfloat16):
            run(torch.ones(2, 4, dtype=dtype))
            for place in ((0, 0), (1, 3), (0, 2)):
                mask = torch.ones(2, 4, dtype=dtype)
                mask[place] = 0
                with pytest.raises(ValueError, match="padded"):
                    run(mask)
        for mask in (torch.ones(2, 3), torch.ones(2, 1, 4, 4, dtype=torch.long), torch.ones(4), object()):
            with pytest.raises(ValueError, match="mask"):
                run(mask)


def test_model_refuses_padding_and_custom_masks():
    """The same through the whole model, single tokens included; the cache is left as it was."""
    for implementation in ("sdpa", "eager"):
        model = small_opt(implementation)
        use_quantized_cache(model)
        cache = cache_for(model)
        left, right = torch.ones(2, 6, dtype=torch.long), torch.ones(2, 6, dtype=torch.long)
        left[0, :2] = 0
        right[1, 4:] = 0
        hidden = causal(6, 6, "bool")
        hidden[:, :, 3, 0] = False
        with torch.no_grad():
            for mask in (left, right, hidden):
                with pytest.raises(ValueError):
                    model(input_ids=IDS[:, :6], attention_mask=mask, position_ids=torch.arange(6).expand(2, 6),
                          past_key_values=cache, use_cache=True)
                assert cache.get_seq_length() == 0 and cache.seq_lens.tolist() == [0, 0]
            model(input_ids=IDS[:, :6], past_key_values=cache, use_cache=True)
            later = torch.ones(2, 7, dtype=torch.long)
            later[1, 2] = 0
            with pytest.raises(ValueError):
                model(input_ids=IDS[:, 6:7], attention_mask=later, past_key_values=cache, use_cache=True)
            assert cache.get_seq_length() == 6
            model(input_ids=IDS[:, 6:7], past_key_values=cache, use_cache=True)
            assert cache.get_seq_length() == 7


def test_wrapping_twice_changes_nothing():
    model = small_opt()
    names = use_quantized_cache(model)
    blocks = [layer.self_attn for layer in model.model.decoder.layers]
    assert names == [f"model.decoder.layers.{i}.self_attn" for i in range(2)]
    assert use_quantized_cache(model) == names
    for layer, block in zip(model.model.decoder.layers, blocks):
        assert layer.self_attn is block and not isinstance(block.attention, QuantizedCacheAttention)
    with torch.no_grad():
        out = model(input_ids=IDS[:, :6], past_key_values=cache_for(model), use_cache=True)
    assert torch.isfinite(out.logits).all()
    # a block that was wrapped by hand beside one that was not
    model = small_opt()
    layers = model.model.decoder.layers
    layers[0].self_attn = QuantizedCacheAttention(layers[0].self_attn)
    first = layers[0].self_attn
    assert use_quantized_cache(model) == names and layers[0].self_attn is first
    assert isinstance(layers[1].self_attn, QuantizedCacheAttention)


@pytest.mark.parametrize("training", [False, True])
def test_wrapping_keeps_the_mode_of_a_model(training):
    model = small_opt().train(training)
    model.model.decoder.layers[1].self_attn.q_proj.eval()
    modes = [m.training for m in model.modules()]
    use_quantized_cache(model)
    for layer in model.model.decoder.layers:
        assert layer.self_attn.training == training
    assert [m.training for m in model.modules() if not isinstance(m, QuantizedCacheAttention)] == modes


def test_keys_of_another_sequence_are_refused():
    """A block that is given other hidden states for its keys (cross attention) does not run on the cache."""
    model = small_opt()
    use_quantized_cache(model)
    block, x = model.model.decoder.layers[0].self_attn, torch.randn(2, 4, 64).bfloat16()
    cache = cache_for(model)
    with torch.no_grad():
        with pytest.raises(ValueError, match="cross"):
            block(x, past_key_values=cache, key_value_states=x)
        assert cache.get_seq_length() == 0
        block(x, past_key_values=cache, key_value_states=None)


def test_a_copy_goes_its_own_way():
    import copy

    model = small_opt()
    use_quantized_cache(model)
    cache = cache_for(model)
    step = lambda c, at, n: model(input_ids=IDS[:, at:at + n], past_key_values=c, use_cache=True).logits
    with torch.no_grad():
        step(cache, 0, 6)
        other = copy.deepcopy(cache)
        assert other.backend is cache.backend and other.caches[0].k.data_ptr() != cache.caches[0].k.data_ptr()
        step(other, 9, 3)
        assert (cache.get_seq_length(), other.get_seq_length()) == (6, 9)
        assert cache.seq_lens.tolist() == [6, 6] and other.seq_lens.tolist() == [9, 9]
        fresh = cache_for(model)
        step(fresh, 0, 6)
        assert torch.equal(step(cache, 6, 2), step(fresh, 6, 2))


def test_sequences_are_reordered():
    model = small_opt()
    use_quantized_cache(model)
    cache, swapped = cache_for(model), cache_for(model)
    with torch.no_grad():
        model(input_ids=IDS[:, :6], past_key_values=cache, use_cache=True)
        model(input_ids=IDS[[1, 1], :6], past_key_values=swapped, use_cache=True)
        cache.reorder_cache(torch.tensor([1, 1]))
        a, b = (model(input_ids=IDS[:, 6:8], past_key_values=c, use_cache=True).logits for c in (cache, swapped))
    assert torch.equal(a, b)
    with pytest.raises(ValueError, match="beam_idx"):
        cache.reorder_cache(torch.tensor([0]))


@pytest.mark.parametrize("beams", [1, 3])
def test_generate(beams):
    """The model library's search over the cache: greedy tokens are those of single steps by hand, beams follow
    the sequences that the search keeps."""
    model = small_opt()
    use_quantized_cache(model)
    cache, calls = cache_for(model, batch=2 * beams), []
    reorder, cache.reorder_cache = cache.reorder_cache, lambda index: calls.append(index) or reorder(index)
    got = model.generate(IDS[:, :6], attention_mask=torch.ones(2, 6, dtype=torch.long), past_key_values=cache,
                         max_new_tokens=8, num_beams=beams, do_sample=False, pad_token_id=1, eos_token_id=None)
    assert got.shape == (2, 14) and torch.equal(got[:, :6], IDS[:, :6])
    assert cache.get_seq_length() == 13
    if beams > 1:
        assert calls and all(tuple(index.shape) == (2 * beams,) for index in calls)
        return
    own, tokens, want = cache_for(model), IDS[:, :6], [IDS[:, :6]]
    with torch.no_grad():
        for _ in range(8):
            tokens = model(input_ids=tokens, past_key_values=own, use_cache=True).logits[:, -1:].float().argmax(-1)
            want.append(tokens)
    assert torch.equal(got, torch.cat(want, 1))


@pytest.mark.parametrize("where", ["kv_cache_write", "kv_cache_attention"])
def test_a_call_that_raises_appends_nothing(where, monkeypatch):
    """The lengths are those before it, and the conversation goes on as if it had not been."""
    model = small_opt()
    use_quantized_cache(model)
    cache, twin = cache_for(model), cache_for(model)
    step = lambda c, at, n: model(input_ids=IDS[:, at:at + n], past_key_values=c, use_cache=True).logits

    def broken(*args, **kw):
        raise RuntimeError("out of memory")

    with torch.no_grad():
        for c in (cache, twin):
            step(c, 0, 6)
        with monkeypatch.context() as patch:
            patch.setattr(cache.backend, where, broken)
            with pytest.raises(RuntimeError, match="out of memory"):
                step(cache, 6, 3)
        assert cache.get_seq_length() == 6 and cache.seq_lens.tolist() == [6, 6]
        assert torch.equal(step(cache, 6, 2), step(twin, 6, 2))
