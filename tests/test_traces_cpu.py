"""A trace follows torch's operations.  A kernel launched beside them leaves it an output that nothing fills, so every op refuses to be recorded into one."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from triteia_amd.python import capi, ops

E4M3 = torch.float8_e4m3fn
half = lambda *shape: torch.zeros(shape, dtype=torch.float16)  # noqa: E731
whole = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731


class Cache:
    k, v, k_scale, v_scale = half(2, 2, 16, 64), half(2, 2, 16, 64), None, None
    _tensors = (k, v, None, None)
    kv_heads, dim, device, dtype, kind = 2, 64, torch.device("cpu"), torch.float16, 0


def plan():
    return capi.AttentionPlan(torch.zeros(64, dtype=torch.uint8), 1, 2, 4, 2, 2, True, 0)


x = half(2, 256)
CALLS = {
    "quantize_fp8": lambda x: ops.quantize_fp8(x),
    "dequantize_fp8": lambda x: ops.dequantize_fp8(x.to(E4M3), torch.zeros(2, 2)),
    "matmul_fp8": lambda x: ops.matmul_fp8(x, torch.zeros(128, 256).to(E4M3), torch.zeros(1, 2)),
    "rotary": lambda x: ops.rotary(x.view(2, 4, 64), x.view(2, 4, 64), whole(2), torch.zeros(4, 32, 2)),
    "cache_read": lambda x: ops.cache_read(Cache, whole(2)),
    "attention_plan": lambda x: ops.attention_plan(Cache, whole(2), whole(1), 4, 2),
    "shared_plan": lambda x: ops.attention_plan(Cache, whole(2), whole(1), 4, 2, group_starts=whole(2), prefix_lens=whole(1)),
    "paged_attention": lambda x: ops.paged_attention(x.view(2, 4, 64), Cache, whole(1, 1), whole(2), whole(1), plan=plan()),
    "matmul": lambda x: ops.matmul_4bit_2_4(whole(8, 512), x, torch.zeros(256, 16, dtype=torch.int16), half(1, 256)),
    "bmm": lambda x: ops.bmm_4bit_2_4(whole(1, 8, 512), x[None], torch.zeros(1, 256, 16, dtype=torch.int16), half(1, 1, 256)),
    "sbmm": lambda x: ops.sbmm_4bit_2_4_native(whole(1, 8, 512), x, torch.zeros(1, 256, 16, dtype=torch.int16), half(1, 1, 256), whole(2)),
    "ldmm": lambda x: ops.ldmm(whole(2), x, half(1, 256, 16), half(1, 16, 256), whole(1, 8, 512), torch.zeros(1, 256, 16, dtype=torch.int16), half(1, 1, 256)),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_no_op_is_recorded_into_a_trace(name):
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(CALLS[name], (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="trace"):
        make_fx(CALLS[name])(x)
    with pytest.raises(RuntimeError, match="GPU tensor"):              # the same call outside of one
        CALLS[name](x)
