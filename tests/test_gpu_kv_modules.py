"""OPT blocks over the quantised cache: a model runs on it, its blocks do exactly what the backend's
calls do on their projections, and other calls of the blocks are unchanged."""
import pytest
import torch

pytestmark = pytest.mark.gpu

transformers = pytest.importorskip("transformers")

C0 = (127, 126, 125, 121)


@pytest.fixture(scope="module")
def backend():
    from rns_llm_b200.backends import CudaRNSBackend
    return CudaRNSBackend()


def small_opt(dtype=torch.float16):
    config = transformers.OPTConfig(vocab_size=512, hidden_size=256, num_hidden_layers=2, num_attention_heads=4, ffn_dim=512,
                                    max_position_embeddings=512, word_embed_proj_dim=256, do_layer_norm_before=True)
    torch.manual_seed(7)
    return transformers.OPTForCausalLM(config).to(dtype).cuda().eval()


@pytest.mark.parametrize("rns", [False, True])
@pytest.mark.parametrize("format", ["int8", "e4m3"])
def test_blocks_compose_the_backend_calls(backend, rns, format):
    from rns_llm_b200.integration import replace_opt_attention_blocks, use_quantized_cache
    from rns_llm_b200.layers import QuantizedDecoderCache

    model = small_opt()
    if rns:
        replace_opt_attention_blocks(model, backend=backend, moduli=C0)
    plain_ids = torch.randint(0, 512, (3, 70), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    with torch.no_grad():
        before = model(input_ids=plain_ids, use_cache=True).logits
    assert len(use_quantized_cache(model)) == 2
    with torch.no_grad():
        assert torch.equal(model(input_ids=plain_ids, use_cache=True).logits, before)     # the library's own cache

    cache = QuantizedDecoderCache.for_model(model, backend, batch=3, max_tokens=100, page_tokens=32, format=format)
    twin = QuantizedDecoderCache.for_model(model, backend, batch=3, max_tokens=100, page_tokens=32, format=format)
    seen = []

    def record(module, args, kwargs, output):
        seen.append((module, args[0] if args else kwargs["hidden_states"], output[0]))

    hooks = [layer.self_attn.register_forward_hook(record, with_kwargs=True) for layer in model.model.decoder.layers]
    with torch.no_grad():
        tokens, steps = plain_ids, 0
        for _ in range(5):
            out = model(input_ids=tokens, past_key_values=cache, use_cache=True)
            assert out.past_key_values is cache and torch.isfinite(out.logits).all()
            tokens = out.logits[:, -1:].argmax(-1)
            steps += 1
        for hook in hooks:
            hook.remove()
        assert cache.get_seq_length() == 74 and cache.seq_lens.tolist() == [74] * 3
        # the same blocks by hand
        length = 0
        for i, (module, x, y) in enumerate(seen):
            block, new = module.attention, x.shape[1]
            if module.layer_idx == 0:
                length += new
            lens = torch.full((3,), length, dtype=torch.int32, device="cuda")
            starts = torch.arange(0, 4 * new, new, dtype=torch.int32, device="cuda")
            q, k, v = (p(x).reshape(3 * new, 4, 64) for p in (block.q_proj, block.k_proj, block.v_proj))
            own = twin.caches[module.layer_idx]
            backend.kv_cache_write(own, k, v, twin.page_table, lens, starts)
            a = backend.kv_cache_attention(q, own, twin.page_table, lens, starts, softmax_scale=64 ** -0.5)
            assert torch.equal(block.out_proj(a.view(3, new, 256)), y), i
    for a, b in zip(cache.caches, twin.caches):
        assert torch.equal(a.k.view(torch.int8), b.k.view(torch.int8)) and torch.equal(a.k_scale, b.k_scale)
        assert torch.equal(a.v.view(torch.int8), b.v.view(torch.int8)) and torch.equal(a.v_scale, b.v_scale)
    backend.check_status()
    # another conversation in the same pages
    cache.reset()
    with torch.no_grad():
        again = model(input_ids=plain_ids, past_key_values=cache, use_cache=True).logits
        fresh = QuantizedDecoderCache.for_model(model, backend, batch=3, max_tokens=100, page_tokens=32, format=format)
        assert torch.equal(again, model(input_ids=plain_ids, past_key_values=fresh, use_cache=True).logits)


def test_refusals(backend):
    from rns_llm_b200.integration import use_quantized_cache
    from rns_llm_b200.layers import QuantizedCacheAttention, QuantizedDecoderCache

    model = small_opt()
    with pytest.raises(ValueError, match="no attention modules"):
        use_quantized_cache(torch.nn.Linear(4, 4))
    with pytest.raises(TypeError):
        QuantizedCacheAttention(torch.nn.Linear(4, 4))
    use_quantized_cache(model)
    make = lambda **kw: QuantizedDecoderCache.for_model(model, backend, **{**dict(batch=2, max_tokens=40), **kw})
    ids = torch.ones(2, 20, dtype=torch.long, device="cuda")
    for kw in (dict(batch=0), dict(max_tokens=0), dict(format="int4"), dict(page_tokens=48)):
        with pytest.raises(ValueError):
            make(**kw)
    with torch.no_grad():
        with pytest.raises(ValueError, match="sequences"):
            model(input_ids=ids[:1, :3], past_key_values=make(), use_cache=True)
        cache = make()
        model(input_ids=ids, past_key_values=cache, use_cache=True)
        with pytest.raises(ValueError, match="do not fit"):
            model(input_ids=ids[:, :1].expand(2, 21), past_key_values=cache, use_cache=True)
        mask = torch.ones_like(ids)
        mask[0, :4] = 0                                   # left padding
        with pytest.raises(ValueError, match="padded"):
            model(input_ids=ids, attention_mask=mask, past_key_values=make(), use_cache=True)
        model.train()
        with pytest.raises(ValueError, match="inference"):
            model(input_ids=ids, past_key_values=make(), use_cache=True)
    with pytest.raises(ValueError):
        small = small_opt(torch.float32)                   # queries are float16 or bfloat16
        use_quantized_cache(small)
        with torch.no_grad():
            small(input_ids=ids, past_key_values=QuantizedDecoderCache.for_model(small, backend, batch=2, max_tokens=40))


def test_copies_and_pickles(backend):
    """A copied or unpickled cache has tensors and addresses of its own; a copied conversation goes its own way."""
    import copy
    import pickle

    from rns_llm_b200.integration import use_quantized_cache
    from rns_llm_b200.layers import QuantizedDecoderCache

    for format in ("int8", "e4m3"):
        cache = backend.create_kv_cache(pages=3, kv_heads=2, head_dim=64, page_tokens=16, format=format)
        x = torch.randn(20, 2, 64, device="cuda").half()
        table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
        ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
        backend.kv_cache_write(cache, x, x, table, ints(20), ints(0, 20))
        want = backend.kv_cache_read(cache, table, ints(0), ints(0, 20), rows=20)
        for other in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
            assert other.k.data_ptr() != cache.k.data_ptr() and other.k.dtype == cache.k.dtype
            for a, b in zip(backend.kv_cache_read(other, table, ints(0), ints(0, 20), rows=20), want):
                assert torch.equal(a, b)
            backend.kv_cache_write(other, x * 9, x * 9, table, ints(20), ints(0, 20))
            for a, b in zip(backend.kv_cache_read(cache, table, ints(0), ints(0, 20), rows=20), want):
                assert torch.equal(a, b)
    model = small_opt()
    use_quantized_cache(model)
    ids = torch.randint(0, 512, (2, 30), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    with torch.no_grad():
        first = QuantizedDecoderCache.for_model(model, backend, batch=2, max_tokens=40, page_tokens=16)
        model(input_ids=ids[:, :20], past_key_values=first, use_cache=True)
        second = copy.deepcopy(first)
        model(input_ids=ids[:, 25:], past_key_values=second, use_cache=True)
        a = model(input_ids=ids[:, 20:25], past_key_values=first, use_cache=True).logits
        third = QuantizedDecoderCache.for_model(model, backend, batch=2, max_tokens=40, page_tokens=16)
        model(input_ids=ids[:, :20], past_key_values=third, use_cache=True)
        assert torch.equal(a, model(input_ids=ids[:, 20:25], past_key_values=third, use_cache=True).logits)
        # beams: both sequences go on from the second
        first.reorder_cache(torch.tensor([1, 1], device="cuda"))
        third.reset()
        model(input_ids=ids[[1, 1], :20], past_key_values=third, use_cache=True)
        model(input_ids=ids[[1, 1], 20:25], past_key_values=third, use_cache=True)
        b, c = (model(input_ids=ids[:, 25:26], past_key_values=x, use_cache=True).logits for x in (first, third))
        assert torch.equal(b, c)
    backend.check_status()
