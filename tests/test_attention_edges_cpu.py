"""The attention side's refusals and sizes that need no GPU."""
import pytest

from triteia_amd.python import ops
from triteia_amd.python.nn import multi_delta_attention


@pytest.mark.parametrize("head_dim", [32, 96, 256])
def test_a_layer_refuses_heads_that_attention_does_not_take(head_dim):
    with pytest.raises(AssertionError, match="heads of 64 or 128"):
        multi_delta_attention(512, 8, 2, head_dim, 1)
    multi_delta_attention(512, 8, 2, 64, 1)


@pytest.mark.parametrize("scaling,match", [
    ({"factor": 8.0}, "unknown scaling"), ({}, "unknown scaling"), ({"type": None, "factor": 2.0}, "unknown scaling"), ({"type": "other", "factor": 2.0}, "unknown scaling"),
    ({"type": "linear"}, "needs factor"), ({"type": "ntk"}, "needs factor"), ({"type": "yarn", "original": 64}, "needs factor"), ({"type": "yarn", "factor": 2.0}, "needs original"),
    ({"type": "bands", "factor": 2.0, "low": 1.0}, "needs high, original"), ({"type": "bands", "factor": 2.0, "low": 4.0, "high": 4.0, "original": 64}, "bands from"),
    ({"type": "linear", "factor": 0.5}, "factor of 0.5"), ({"type": "linear", "factor": float("nan")}, "factor of nan"), ({"type": "linear", "factor": 2.0, "beta": 1}, "unknown settings")])
def test_a_scaling_of_positions_that_is_not_whole_is_refused(scaling, match):
    """(A missing type or factor gave the table without any scaling.)"""
    with pytest.raises(RuntimeError, match=match):
        ops.rotary_table(10, 64, scaling=scaling, device="cpu")


def test_scratch_does_not_shrink_with_the_batch():
    """More tokens of as many sequences, or more sequences of as many tokens, never need less."""
    from triteia_amd.python.capi import _ffi
    bytes_of = _ffi.lib().triteia_hip_attention_scratch_bytes
    for heads, kv_heads in ((32, 32), (64, 8), (20, 1), (3, 3)):
        for max_q in (1, 2, 16, 1000):
            sizes = [bytes_of(8, tokens, heads, kv_heads, max_q, 128) for tokens in range(1, 600)]
            assert all(0 < a <= b for a, b in zip(sizes, sizes[1:]))
            sizes = [bytes_of(seqs, 4000, heads, kv_heads, max_q, 128) for seqs in range(1, 600, 7)]
            assert all(0 < a <= b for a, b in zip(sizes, sizes[1:]))
