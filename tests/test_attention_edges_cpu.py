"""The attention side's refusals and sizes that need no GPU."""
import pytest

from triteia_amd.python.nn import multi_delta_attention


@pytest.mark.parametrize("head_dim", [32, 96, 256])
def test_a_layer_refuses_heads_that_attention_does_not_take(head_dim):
    with pytest.raises(AssertionError, match="heads of 64 or 128"):
        multi_delta_attention(512, 8, 2, head_dim, 1)
    multi_delta_attention(512, 8, 2, 64, 1)
