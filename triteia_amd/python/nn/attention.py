"""The attention block of a layer that serves many fine-tuned variants at once."""
import torch
import torch.nn as nn

from .linear import multi_delta_linear


class multi_delta_attention(nn.Module):
    """qkv projection, rotary positions (with norms of queries and keys, if `qk_norm`), the write into the layer's paged cache, attention
    over it and the output projection, for a batch of sequences whose tokens each pick a variant of both projections (index -1: none).

    Attention is causal over the whole context; heads have 64 or 128 elements.  `qkv_proj` and `o_proj` are `multi_delta_linear` layers; queries,
    keys and values stay views of the former's output.  Every method runs on the current stream without a synchronisation and can be recorded into a graph."""

    def __init__(self, hidden, n_heads, n_kv_heads, head_dim, n_deltas, with_base=True, qk_norm=False, interleaved=False, eps=1e-6):
        super().__init__()
        assert n_heads % n_kv_heads == 0, f"{n_heads} heads over {n_kv_heads} heads of the cache"
        assert head_dim in (64, 128), f"attention takes heads of 64 or 128 elements, got {head_dim}"
        self.n_heads, self.n_kv_heads, self.head_dim, self.interleaved, self.eps = n_heads, n_kv_heads, head_dim, interleaved, eps
        self.qkv_proj = multi_delta_linear(hidden, (n_heads + 2 * n_kv_heads) * head_dim, n_deltas, with_base)
        self.o_proj = multi_delta_linear(n_heads * head_dim, hidden, n_deltas, with_base)
        for name in ("q_norm", "k_norm"):
            self.register_buffer(name, torch.ones(head_dim, dtype=torch.float16) if qk_norm else None)

    def plan(self, cache, q_starts, kv_lens, n_tokens, max_q=None):
        """The attention's work list for a batch: one serves every layer of a forward pass."""
        from triteia_amd.python.ops import attention_plan
        return attention_plan(cache, q_starts, kv_lens, self.n_heads, n_tokens, max_q)

    def forward(self, x, indices, positions, table, cache, slots, pages, q_starts, kv_lens, plan=None, route=None, max_q=None):
        """x [tokens, hidden] fp16, the new tokens of all sequences one after the other -> [tokens, hidden].

        indices: each token's variant (`route`: a routing plan of them, shared by all layers); positions, slots: each token's position and place in
        `cache` (a PagedCache, this layer's); table: from ops.rotary_table; pages, q_starts, kv_lens, plan, max_q: as for ops.paged_attention."""
        from triteia_amd.python.ops import paged_attention, rotary_cache_write
        tokens = x.shape[0]
        qkv = self.qkv_proj(x, indices, route).view(tokens, self.n_heads + 2 * self.n_kv_heads, self.head_dim)
        q, k, v = qkv.split([self.n_heads, self.n_kv_heads, self.n_kv_heads], 1)
        q = rotary_cache_write(q, k, v, positions, table, cache, slots, self.interleaved, self.q_norm, self.k_norm, self.eps)
        out = paged_attention(q, cache, pages, q_starts, kv_lens, plan=plan, max_q=max_q)
        return self.o_proj(out.view(tokens, self.n_heads * self.head_dim), indices, route)
