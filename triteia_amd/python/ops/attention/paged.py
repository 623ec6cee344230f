"""Attention of new tokens over a paged cache, and the plan that a forward pass makes of its batch once."""
from triteia_amd.python import capi

__all__ = ["attention_plan", "paged_attention"]


def attention_plan(cache, q_starts, kv_lens, n_heads, n_tokens, max_q=None, causal=True, window=0):
    """The work list of a batch, made on the device without a synchronisation: for every layer's `paged_attention` with `n_heads` heads over caches of as many
    heads as `cache`.

    q_starts int32 [sequences + 1]: where each sequence's new tokens begin, from 0 on; kv_lens int32 [sequences]: tokens of its context, the
    new ones among them; n_tokens: rows of the queries (behind q_starts[-1]: padding, whose outputs are zeros); max_q: no sequence brings more new tokens than this.  It
    chooses kernels, grids and scratch: a batch of single tokens should say 1 (None: n_tokens, which runs it as prompts).  Any number is right; which one may change the
    order of sums."""
    return capi.attention_plan(q_starts, kv_lens, n_tokens, n_heads, cache.kv_heads, max_q, causal, window)


def paged_attention(q, cache, pages, q_starts, kv_lens, plan=None, max_q=None, causal=True, window=0, scale=None):
    """softmax(scale * q k^T) v [tokens, heads, dim] of new tokens q [tokens, heads, dim] over their sequences' contexts, head h on head
    h // (heads / kv_heads) of the cache.  Heads of 64 or 128 elements.

    pages int32 [sequences, pages of one]: a sequence's pages in order (entries behind its last are not read; tokens behind the last column are not seen).  causal: the last of a sequence's new tokens sees all of its context,
    each one before it one token less; with `window` it sees the last `window` of those only.  causal=False: every token sees the whole context (cross attention
    to states of another length).  A token that sees nothing gets zeros.  `plan`: from `attention_plan` with the same
    lengths, causal and window (None: made here); scale: dim^-0.5 if None.  Serving only: no gradient is recorded."""
    if plan is None:
        plan = attention_plan(cache, q_starts, kv_lens, q.shape[1], q.shape[0], max_q, causal, window)
    elif plan.causal != bool(causal) or plan.window != window:
        raise RuntimeError(f"the plan is for causal={plan.causal}, window={plan.window}")
    return capi.paged_attention(q, cache, pages, plan, cache.dim ** -0.5 if scale is None else scale)
