"""Projections of many variants, rotary positions, cache and attention as a layer runs them, and the ops' Python path."""
import numpy as np
import pytest
import torch

from oracle import triteia_oracle as orc
from tests.helpers import activations, make_deltas, to_gpu

pytestmark = pytest.mark.gpu


def test_layer_of_many_variants():
    from triteia_amd.python import ops
    from triteia_amd.python.nn import multi_delta_attention
    hidden, heads, kv_heads, dim, n, page = 512, 4, 2, 64, 3, 16
    lengths = [(1, 40), (9, 9), (30, 70), (1, 1)]
    tokens = sum(new for new, _ in lengths)
    layer = multi_delta_attention(hidden, heads, kv_heads, dim, n, qk_norm=True).cuda()
    rng = np.random.default_rng(1)
    packed = {}
    for seed, name in ((2, "qkv_proj"), (3, "o_proj")):
        proj = getattr(layer, name)
        packed[name] = make_deltas(n, proj.infeatures, proj.outfeatures, seed)
        for buffer, value in zip((proj.qweight, proj.meta, proj.scale), to_gpu(*packed[name])):
            buffer.copy_(value.view(buffer.shape))
        proj.base.copy_(torch.from_numpy(rng.standard_normal((proj.outfeatures, proj.infeatures)).astype(np.float16) * np.float16(0.04)))
    for norm in (layer.q_norm, layer.k_norm):
        norm.copy_(torch.from_numpy(1 + 0.1 * rng.standard_normal(dim)))
    x, idx = activations(tokens, hidden, 4), rng.integers(-1, n, size=tokens).astype(np.int32)
    cache, table = ops.paged_cache(24, kv_heads, dim, page), ops.rotary_table(100, dim)
    pages = torch.randperm(24, generator=torch.Generator().manual_seed(5))[:20].to(torch.int32).view(4, 5)
    starts = np.concatenate([[0], np.cumsum([new for new, _ in lengths])])
    # the contexts' earlier tokens
    history = []
    for b, (new, kv) in enumerate(lengths):
        k, v = (torch.from_numpy(activations((kv - new) * kv_heads, dim, 10 + 2 * b + i)).view(kv - new, kv_heads, dim) for i in range(2))
        at = torch.arange(kv - new)
        ops.cache_write(cache, k.cuda(), v.cuda(), (pages[b, at // page].long() * page + at % page).cuda())
        history.append((k.double().numpy(), v.double().numpy()))
    positions = torch.cat([torch.arange(kv - new, kv) for new, kv in lengths])
    owner = torch.repeat_interleave(torch.arange(4), torch.tensor([new for new, _ in lengths]))
    slots = pages[owner, positions // page].long() * page + positions % page
    args = (*to_gpu(x, idx), positions.cuda(), table, cache, slots.cuda(), pages.cuda(), torch.from_numpy(starts.astype(np.int32)).cuda(),
            torch.tensor([kv for _, kv in lengths], dtype=torch.int32).cuda())
    plan = layer.plan(cache, args[7], args[8], tokens, max_q=30)
    got = layer(*args, plan=plan)
    assert torch.equal(got, layer(*args, max_q=30))               # (its own plan; the same tokens written again)

    def project(x, name):
        y = orc.sbmm_4bit_2_4(packed[name][0], x.astype(np.float16), packed[name][1], packed[name][2], idx).astype(np.float64)
        return y + x @ getattr(layer, name).base.cpu().numpy().astype(np.float64).T

    qkv = project(x.astype(np.float64), "qkv_proj").reshape(tokens, -1, dim)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    rotate = table.double().cpu().numpy()[positions.numpy()]       # [tokens, pairs, 2]
    turned = []
    for y, weight in ((q, layer.q_norm), (k, layer.k_norm)):
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + layer.eps) * weight.double().cpu().numpy()
        a, b, c, s = y[..., :dim // 2], y[..., dim // 2:], rotate[:, None, :, 0], rotate[:, None, :, 1]
        turned.append(np.concatenate([a * c - b * s, b * c + a * s], -1))
    q, k = turned
    out = np.zeros((tokens, heads, dim))
    for b, (new, kv) in enumerate(lengths):
        rows = slice(starts[b], starts[b + 1])
        keys, values = (np.concatenate([old, x[rows]]).repeat(heads // kv_heads, 1) for old, x in zip(history[b], (k, v)))
        score = np.einsum("thd,shd->hts", q[rows], keys) * dim ** -0.5
        score = np.where(np.arange(kv) <= np.arange(kv - new, kv)[:, None], score, -np.inf)
        p = np.exp(score - score.max(-1, keepdims=True))
        out[rows] = np.einsum("hts,shd->thd", p / p.sum(-1, keepdims=True), values)
    want = project(out.reshape(tokens, -1), "o_proj")
    # three products and an attention, each within the framework's 2e-3 of its own reference
    error = orc.rel_frobenius(got.float().cpu().numpy(), want)
    assert error <= 8e-3, error


@pytest.mark.parametrize("dtype,kind", [(torch.float16, "same"), (torch.bfloat16, "int8"), (torch.float16, "fp8")])
def test_the_python_path_gives_the_same_bits(monkeypatch, dtype, kind):
    """What the native calls leave to Python (a tensor subclass, say) comes out the same."""
    from tests.test_gpu_attention import Batch, randn
    from triteia_amd.python import ops
    from triteia_amd.python.capi import attention as capi

    batch = Batch([(1, 100), (40, 90)], 4, 2, 64, 16, kind, dtype)
    table, x = ops.rotary_table(50, 64), randn(7, 6, 64, seed=3, dtype=dtype).cuda()
    positions, norm = torch.arange(7).cuda(), torch.ones(64, dtype=dtype, device="cuda")
    asked = []

    class Declines:
        def __getattr__(self, name):
            return lambda *args: asked.append(name)

    def everything():
        q, k, v = x.split([2, 2, 2], 1)
        out = list(ops.rotary(q, k, positions, table, True, norm, None))
        out.append(ops.rotary_cache_write(q, k, v, positions, table, batch.cache, positions + 3, k_norm=norm))
        out += ops.cache_read(batch.cache, positions, dtype)
        out.append(ops.paged_attention(*batch.inputs(), window=33, max_q=40))
        return out

    first = everything()
    monkeypatch.setattr(capi, "native", Declines)
    second = everything()
    assert set(asked) == {"rotary_cache", "cache_read", "attention_plan", "paged_attention"}
    assert all(torch.equal(a, b) for a, b in zip(first, second)) and len(first) == len(second) == 6
