"""OPT attention over a quantised key/value cache.

The reference fuses the projections of an OPT attention block and leaves its cache and softmax to
the model (scripts/evaluate_ppl.py:53-94).  Here a block's attention can keep its keys and values in
8 bits as well: ``QuantizedDecoderCache`` takes the place of the model library's cache object
(``past_key_values``), and ``QuantizedCacheAttention`` runs a block on it.  Every other call of the
block goes to the module it wraps.
"""
from __future__ import annotations

import copy

import torch
from torch import nn

from ..backends.kv_cache import QuantizedKVCache


class QuantizedDecoderCache:
    """8-bit cache of a decoder: one paged cache a layer, a batch of sequences of one length.

    Passed to the model as ``past_key_values``; the model asks it for the cached length, the
    attention blocks write to it and read it.  ``max_tokens`` bounds the sequences; a call beyond
    it raises.  Batches are not padded: every sequence gets the same number of tokens a call, and
    each token sees those up to itself; a block refuses any other attention mask.  The
    lengths are counted on the host too, so its calls are not captured into CUDA graphs (the backend's
    own calls can be).
    """

    is_compileable = False
    is_initialized = True

    def __init__(self, backend, *, layers: int, batch: int, max_tokens: int, kv_heads: int, head_dim: int,
                 page_tokens: int = 64, format: str = "int8", device: torch.device | str = "cuda") -> None:
        if layers < 1 or batch < 1 or max_tokens < 1:
            raise ValueError("layers, batch and max_tokens must be at least 1")
        per_sequence = -(-int(max_tokens) // int(page_tokens))
        self.backend = backend
        self.batch = int(batch)
        self.max_tokens = int(max_tokens)
        self.caches: list[QuantizedKVCache] = [
            backend.create_kv_cache(pages=batch * per_sequence, kv_heads=kv_heads, head_dim=head_dim,
                                    page_tokens=page_tokens, format=format, device=device) for _ in range(layers)]
        device = self.caches[0].device
        self.page_table = torch.arange(batch * per_sequence, dtype=torch.int32, device=device).view(batch, per_sequence)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self._lengths = [0] * layers
        self._starts: dict[int, torch.Tensor] = {}

    @classmethod
    def for_model(cls, model: nn.Module, backend, *, batch: int, max_tokens: int, page_tokens: int = 64,
                  format: str = "int8") -> "QuantizedDecoderCache":
        """Sizes taken from an OPT model's configuration and device."""
        config = model.config
        return cls(backend, layers=config.num_hidden_layers, batch=batch, max_tokens=max_tokens,
                   kv_heads=config.num_attention_heads, head_dim=config.hidden_size // config.num_attention_heads,
                   page_tokens=page_tokens, format=format, device=next(model.parameters()).device)

    # what the model asks of its cache
    def get_seq_length(self, layer_idx: int = 0) -> int:
        return self._lengths[layer_idx or 0]

    def get_mask_sizes(self, query_length: int, layer_idx: int = 0) -> tuple[int, int]:
        return self._lengths[layer_idx or 0] + int(query_length), 0

    def __len__(self) -> int:
        return len(self.caches)

    def reset(self) -> None:
        """Forgets the sequences; their pages are taken over by the next ones."""
        self.seq_lens.zero_()
        self._lengths = [0] * len(self.caches)

    def reorder_cache(self, beam_idx: torch.Tensor) -> None:
        """Sequence i becomes a copy of sequence ``beam_idx[i]`` (beam search)."""
        if tuple(beam_idx.shape) != (self.batch,):
            raise ValueError(f"beam_idx must name a sequence for each of the cache's {self.batch}")
        for cache in self.caches:
            for tensor in (cache.k, cache.v, cache.k_scale, cache.v_scale):
                rows = tensor.view(torch.int8).view(self.batch, -1)      # a sequence's pages lie together
                rows.copy_(rows.index_select(0, beam_idx.to(rows.device)))

    def __deepcopy__(self, memo: dict) -> "QuantizedDecoderCache":
        """A cache of its own with the same sequences, on the same backend."""
        own = copy.copy(self)
        memo[id(self)] = own
        own.caches = copy.deepcopy(self.caches, memo)
        own.page_table, own.seq_lens = self.page_table.clone(), self.seq_lens.clone()
        own._lengths, own._starts = list(self._lengths), dict(self._starts)
        return own

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
               softmax_scale: float) -> torch.Tensor:
        """Appends the new tokens' keys and values to layer ``layer`` and attends causally: q, k, v
        [batch * new, heads, head_dim], sequence after sequence."""
        new, rest = divmod(q.shape[0], self.batch)
        if rest or new == 0:
            raise ValueError(f"the cache holds {self.batch} sequences: every call brings each as many new tokens")
        if q.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("attention over the quantised cache runs in float16 or bfloat16")
        length = self._lengths[layer] + new
        if length > self.max_tokens:
            raise ValueError(f"{length} tokens do not fit the cache's {self.max_tokens}")
        ahead = max(self._lengths)
        if ahead > self._lengths[layer] and ahead != length:
            raise ValueError("the layers of the cache are at different lengths")
        starts = self._starts.get(new)
        if starts is None:
            starts = torch.arange(0, (self.batch + 1) * new, new, dtype=torch.int32, device=self.seq_lens.device)
            self._starts[new] = starts
        cache = self.caches[layer]
        if ahead < length:                               # the first layer of this call
            self.seq_lens += new
        try:
            self.backend.kv_cache_write(cache, k, v, self.page_table, self.seq_lens, starts, max_query_len=new)
            out = self.backend.kv_cache_attention(q, cache, self.page_table, self.seq_lens, starts, max_query_len=new,
                                                  softmax_scale=softmax_scale)
        except Exception:
            if ahead < length:
                self.seq_lens -= new
            raise
        self._lengths[layer] = length
        return out


class QuantizedCacheAttention(nn.Module):
    """An OPT attention block that attends over a ``QuantizedDecoderCache`` when it is given one,
    and is the block it wraps otherwise.  Inference only, in float16 or bfloat16."""

    def __init__(self, attention: nn.Module, layer_idx: int | None = None) -> None:
        super().__init__()
        for name in ("q_proj", "k_proj", "v_proj", "out_proj"):
            if not isinstance(getattr(attention, name, None), nn.Module):
                raise TypeError(f"attention.{name} must be a module")
        layer_idx = getattr(attention, "layer_idx", None) if layer_idx is None else layer_idx
        if layer_idx is None:
            raise ValueError("the attention block has no layer_idx")
        self.attention = attention
        self.layer_idx = int(layer_idx)
        self.training = attention.training

    def forward(self, hidden_states: torch.Tensor, past_key_values=None, attention_mask: torch.Tensor | None = None,
                output_attentions: bool = False, **kwargs):
        block = self.attention
        if not isinstance(past_key_values, QuantizedDecoderCache):
            return block(hidden_states, past_key_values=past_key_values, attention_mask=attention_mask,
                         output_attentions=output_attentions, **kwargs)
        if output_attentions:
            raise ValueError("attention weights are not formed over a quantised cache")
        if self.training:
            raise ValueError("attention over a quantised cache is for inference")
        if kwargs.get("key_value_states") is not None:
            raise ValueError("cross attention does not run on a quantised cache")
        batch, new, width = hidden_states.shape
        if attention_mask is not None:
            _check_mask(attention_mask, batch, block.num_heads, past_key_values.get_seq_length(self.layer_idx), new)
        q, k, v = (proj(hidden_states) for proj in (block.q_proj, block.k_proj, block.v_proj))
        heads = (batch * new, block.num_heads, block.head_dim)
        out = past_key_values.attend(self.layer_idx, q.view(heads), k.view(heads), v.view(heads),
                                     softmax_scale=block.scaling)
        return block.out_proj(out.view(batch, new, width)), None


def _check_mask(mask, batch: int, heads: int, cached: int, new: int) -> None:
    """Refuses every mask but one that says what the cache's attention does anyway: causal, nothing padded.
    Reads the mask on the host (the model passes none for unpadded prompts and single tokens, unless its
    attention is the eager one)."""
    total = cached + new
    shape = tuple(mask.shape) if isinstance(mask, torch.Tensor) else ()
    if len(shape) == 2 and shape[0] in (1, batch) and shape[1] == total:
        good = mask != 0
    elif (len(shape) == 4 and shape[0] in (1, batch) and shape[1] in (1, heads) and shape[2:] == (new, total) and
          (mask.dtype == torch.bool or mask.is_floating_point())):
        at = torch.arange(total, device=mask.device)
        seen = at <= at[cached:, None]
        # scores get 0 added where a key is seen; a type's lowest value or -inf hides it
        good = mask == seen if mask.dtype == torch.bool else torch.where(seen, mask == 0, mask <= -1e4)
    else:
        raise ValueError(f"the quantised cache takes attention masks of [batch, {total}], or boolean or floating ones of "
                         f"[batch, 1, {new}, {total}]")
    if not bool(good.all()):
        raise ValueError("the attention mask is not the causal one: padded batches and masks of other forms are not "
                         "supported by the quantised cache")
