"""What the variants of a base model share, together as a serving step uses it: base weights in 8 bits under the deltas, and the requests' common prefixes."""
import numpy as np
import pytest
import torch

from oracle import triteia_oracle as orc
from tests.helpers import activations, make_deltas, to_gpu

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def ops():
    from triteia_amd.python import ops
    return ops


def values(codes, scales, rows):
    """In 64 bits, on the CPU."""
    n, k = codes.shape
    return (codes.double() * scales.double().repeat_interleave(rows, 0)[:n].repeat_interleave(128, 1)[:, :k]).cpu().numpy()


def dense(m, k, seed):
    return torch.from_numpy((np.random.default_rng(seed).standard_normal((m, k)) * 0.04).astype(np.float16)).cuda()


@pytest.mark.parametrize("tokens", [1, 4, 5, 37, 300])
@pytest.mark.parametrize("k,m", [(512, 256), (1024, 768)])
def test_base_in_8_bits_under_deltas(tokens, k, m):
    """The layer and the ops give the bits of the base product and the routed deltas added to it; the base product that of the codes, the deltas the oracle's."""
    from triteia_amd.python.capi import route_plan, sbmm_2_4_routed
    from triteia_amd.python.nn import multi_delta_linear
    n = 5
    layer = multi_delta_linear(k, m, n, with_base="fp8").cuda()
    packed = make_deltas(n, k, m, 3)
    for buffer, value in zip((layer.qweight, layer.meta, layer.scale), to_gpu(*packed)):
        buffer.copy_(value.view(buffer.shape))
    layer.load_base(dense(m, k, 4))
    x, idx = activations(tokens, k, 5), np.random.default_rng(6).integers(-1, n, size=tokens).astype(np.int32)
    gx, gi = to_gpu(x, idx)
    want = ops().matmul_fp8(gx, layer.base, layer.base_scale)
    sbmm_2_4_routed(gx, layer.qweight, layer.meta, want, layer.scale, gi, accumulate=True)
    got = layer(gx, gi)
    assert torch.equal(got, want)
    assert torch.equal(ops().sbmm_4bit_2_4_native(layer.qweight, gx, layer.meta, layer.scale, gi, layer.base, layer.base_scale), want)
    planned = layer(gx, gi, route_plan(gi, n)) if tokens > 1 else got
    x8, xs = ops().quantize_fp8(gx)
    exact = orc.sbmm_4bit_2_4(packed[0], x, packed[1], packed[2], idx).astype(np.float64) + values(x8, xs, 1) @ values(layer.base, layer.base_scale, 128).T
    for y in (got, planned):
        assert orc.rel_frobenius(y.float().cpu().numpy(), exact) <= 2e-3
    state = {name: t.clone() for name, t in layer.state_dict().items()}
    other = multi_delta_linear(k, m, n, with_base="fp8").cuda()
    other.load_state_dict(state)
    assert torch.equal(other(gx, gi), got) and "base_scale" not in multi_delta_linear(k, m, n, with_base=True).state_dict()


@pytest.mark.parametrize("tokens", [3, 64, 2100])
def test_base_in_8_bits_under_adapters_and_deltas(tokens):
    """ldmm, on one stream and (large batches) on two: the LoRA product and the deltas are added to the base product of the codes."""
    k, m, n, adapters, rank = 1024, 512, 4, 3, 16
    if tokens > 2000:
        k, m = 4096, 4096                                                      # (where the pair runs beside the base product)
    packed = make_deltas(n, k, m, 7)
    rng = np.random.default_rng(8)
    A, B = (rng.standard_normal((adapters, k, rank)) * 0.05).astype(np.float16), (rng.standard_normal((adapters, rank, m)) * 0.05).astype(np.float16)
    x, idx = activations(tokens, k, 9), rng.integers(-1, adapters + n, size=tokens).astype(np.int32)
    gq, gm, gs, gA, gB, gx, gi = to_gpu(packed[0], packed[1], packed[2], A, B, x, idx)
    w, ws = ops().quantize_fp8(dense(m, k, 10), rows=128)
    got = ops().ldmm(gi, gx, gA, gB, gq, gm, gs, w, base_scale=ws)
    assert torch.equal(got, ops().ldmm(gi, gx, gA, gB, gq, gm, gs, w, base_scale=ws))
    rest = ops().ldmm(gi, gx, gA, gB, gq, gm, gs).double()
    base = ops().matmul_fp8(gx, w, ws, dtype=torch.float32).double()
    # Each product rounded to fp16 and their sum once more: three roundings of values that are not above the sum of magnitudes.
    # x A is rounded to fp16 between the pair's products, and with a base its sums over K come in another order: a value that
    # lies beside a rounding's middle goes the other way, a whole step (2^-10 of it) that B carries into all of its token's row.
    chosen = gi.clamp(0, adapters - 1).long()
    inner = torch.stack([gx.double() @ a for a in gA.double()])[chosen, torch.arange(tokens)]
    step = torch.stack([inner.abs() @ b for b in gB.double().abs()])[chosen, torch.arange(tokens)] * ((gi >= 0) & (gi < adapters))[:, None]
    bound = 3 * 2.0 ** -11 * (rest.abs() + base.abs()) + 2.0 ** -10 * step + 2.0 ** -23
    assert bool(((got.double() - rest - base).abs() <= bound).all())


def test_one_row_of_any_stride_over_a_base_in_8_bits():
    """A single row is adjacent elements whatever the strides of its view say: the newest token of a long sequence, a column."""
    from triteia_amd.python.nn import multi_delta_linear
    k, m, n, adapters, rank = 4096, 256, 3, 2, 16
    layer = multi_delta_linear(k, m, n, with_base="fp8").cuda()
    for buffer, value in zip((layer.qweight, layer.meta, layer.scale), to_gpu(*make_deltas(n, k, m, 3))):
        buffer.copy_(value.view(buffer.shape))
    layer.load_base(dense(m, k, 4))
    rng = np.random.default_rng(8)
    gA, gB = to_gpu((rng.standard_normal((adapters, k, rank)) * 0.05).astype(np.float16), (rng.standard_normal((adapters, rank, m)) * 0.05).astype(np.float16))
    row = torch.from_numpy(activations(1, k, 5)).cuda()
    hidden = torch.zeros(1, 4100, k, dtype=torch.float16, device="cuda")
    hidden[:, -1] = row
    views = hidden[:, -1], row.reshape(k, 1).t(), row.as_strided((1, k), (8, 1))
    assert views[0].stride(0) > 1 << 24 and views[1].stride(0) == 1 and all(v.is_contiguous() and torch.equal(v, row) for v in views)
    packed = layer.qweight, layer.meta, layer.scale
    for index in (-1, 0, 2, 3):
        idx = torch.tensor([index], dtype=torch.int32, device="cuda")
        delta = idx.clamp(max=n - 1)
        want = layer(row, delta), ops().ldmm(idx, row, gA, gB, *packed, layer.base, base_scale=layer.base_scale), ops().matmul_fp8(row, layer.base, layer.base_scale)
        for x in views:
            got = (ops().sbmm_4bit_2_4_native(packed[0], x, *packed[1:], delta, layer.base, layer.base_scale),
                   ops().ldmm(idx, x, gA, gB, *packed, layer.base, base_scale=layer.base_scale), ops().matmul_fp8(x, layer.base, layer.base_scale))
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(layer(x, delta), want[0])
    assert torch.equal(layer(hidden[:, -1:], delta)[0], want[0])


def test_refusals_of_the_base():
    from triteia_amd.python.nn import multi_delta_linear
    with pytest.raises(AssertionError, match="with_base"):
        multi_delta_linear(256, 256, 1, with_base="int8")
    layer = multi_delta_linear(256, 256, 1, with_base="fp8").cuda()
    with pytest.raises(AssertionError, match="a base of"):
        layer.load_base(torch.zeros(128, 256))
    x, idx = torch.zeros(2, 256, dtype=torch.float16, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    args = layer.qweight, x, layer.meta, layer.scale, idx
    with pytest.raises(RuntimeError, match="weight_scale"):
        ops().sbmm_4bit_2_4_native(*args, layer.base, layer.base_scale[:1])
    with pytest.raises(RuntimeError, match="weight must be"):
        ops().sbmm_4bit_2_4_native(*args, torch.zeros(256, 256, dtype=torch.float16, device="cuda"), layer.base_scale)
    for call in (lambda: ops().sbmm_4bit_2_4_native(*args, None, layer.base_scale),
                 lambda: ops().ldmm(idx, x, x.new_zeros(1, 256, 16), x.new_zeros(1, 16, 256), *args[:1], *args[2:4], base_scale=layer.base_scale)):
        with pytest.raises(ValueError, match="without a base_weight"):
            call()
    with pytest.raises(RuntimeError, match="gradient"):
        layer(x.clone().requires_grad_(), idx)


class Step:
    """A layer whose base is in 8 bits, and requests of three variants, most of them behind their variant's prefix; one new token each, a prompt among them."""

    def __init__(self, cache_dtype):
        from triteia_amd.python.nn import multi_delta_attention
        self.heads, self.kv_heads, self.dim, self.page, n, hidden = 8, 2, 64, 16, 3, 512
        self.layer = layer = multi_delta_attention(hidden, self.heads, self.kv_heads, self.dim, n, with_base="fp8", qk_norm=True).cuda()
        for seed, proj in ((2, layer.qkv_proj), (3, layer.o_proj)):
            for buffer, value in zip((proj.qweight, proj.meta, proj.scale), to_gpu(*make_deltas(n, proj.infeatures, proj.outfeatures, seed))):
                buffer.copy_(value.view(buffer.shape))
            proj.load_base(dense(proj.outfeatures, proj.infeatures, 10 + seed))
        # (variant, prefix, [(new tokens, tokens of its own)])
        groups = [(0, 832, [(1, 5), (1, 40), (1, 1)]), (1, 1104, [(1, 77), (20, 50), (1, 9), (1, 16)]), (-1, 0, [(1, 60)])]
        self.prefix_lens = [p for _, p, _ in groups]
        self.group_starts = np.concatenate([[0], np.cumsum([len(seqs) for _, _, seqs in groups])])
        lengths = [(new, p + own) for _, p, seqs in groups for new, own in seqs]
        self.new, self.kv = [a for a, _ in lengths], [b for _, b in lengths]
        variant = [v for v, _, seqs in groups for _ in seqs]
        page, g = self.page, torch.Generator().manual_seed(5)
        n_pages = sum(p // page for p in self.prefix_lens) + sum(-(-own // page) for _, _, seqs in groups for _, own in seqs) + 1
        order = torch.randperm(n_pages, generator=g).to(torch.int32)
        self.pages = torch.zeros((len(lengths), max(-(-kv // page) for kv in self.kv)), dtype=torch.int32)
        self.cache = ops().paged_cache(n_pages, self.kv_heads, self.dim, page, cache_dtype)
        at = b = 0
        for _, p, seqs in groups:
            shared = order[at:at + p // page]
            at += p // page
            for _, own in seqs:
                have = -(-own // page)
                self.pages[b, :len(shared)], self.pages[b, len(shared):len(shared) + have] = shared, order[at:at + have]
                at, b = at + have, b + 1
        history = [torch.randn((n_pages * page, self.kv_heads, self.dim), generator=g).half().cuda() for _ in range(2)]
        ops().cache_write(self.cache, *history, torch.arange(n_pages * page).cuda())
        positions = torch.cat([torch.arange(kv - new, kv) for new, kv in lengths])
        owner = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(self.new))
        slots = self.pages[owner, positions // page].long() * page + positions % page
        self.tokens = len(positions)
        self.x = torch.from_numpy(activations(self.tokens, hidden, 4)).cuda()
        whole = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32).cuda()  # noqa: E731
        self.starts = whole(np.concatenate([[0], np.cumsum(self.new)]))
        self.args = (whole(np.repeat(variant, self.new)), positions.cuda(), ops().rotary_table(1400, self.dim), self.cache, slots.cuda(), self.pages.cuda(), self.starts, whole(self.kv))
        self.groups = dict(group_starts=whole(self.group_starts), prefix_lens=whole(self.prefix_lens))

    def plan(self, **groups):
        return self.layer.plan(self.cache, self.starts, self.args[7], self.tokens, max_q=20, **groups)


@pytest.mark.parametrize("dtype", [torch.float16, torch.int8, E4M3])
def test_step_of_variants_with_shared_prefixes(dtype):
    s = Step(dtype)
    plan = s.plan(**s.groups)
    assert int(plan.buffer.view(torch.int32)[[1, 3, 5]].sum()) >= 7             # (the groups' sequences are joined from shares)
    got = s.layer(s.x, *s.args, plan=plan)
    # the same by its operators, the attention against its formula on what the cache holds then
    idx, positions, table, cache, slots, pages, starts, lens = s.args
    qkv = s.layer.qkv_proj(s.x, idx).view(s.tokens, -1, s.dim)
    q, k, v = qkv.split([s.heads, s.kv_heads, s.kv_heads], 1)
    q = ops().rotary_cache_write(q, k, v, positions, table, cache, slots, False, s.layer.q_norm, s.layer.k_norm, s.layer.eps)
    out = ops().paged_attention(q, cache, pages, starts, lens, plan=plan)
    assert torch.equal(s.layer.o_proj(out.view(s.tokens, -1), idx), got)
    at = 0
    for b, (new, kv) in enumerate(zip(s.new, s.kv)):
        where = (s.pages[b, torch.arange(kv) // s.page].long() * s.page + torch.arange(kv) % s.page).cuda()
        k, v = (t.double().repeat_interleave(s.heads // s.kv_heads, 1) for t in ops().cache_read(cache, where, torch.float16))
        score = torch.matmul(q[at:at + new].double().transpose(0, 1), k.permute(1, 2, 0).contiguous()) * s.dim ** -0.5
        score = score.masked_fill(torch.arange(kv, device="cuda") > torch.arange(kv - new, kv, device="cuda")[:, None], -torch.inf)
        p = torch.softmax(score, -1)
        want, size = (torch.matmul(p, x.transpose(0, 1).contiguous()).transpose(0, 1) for x in (v, v.abs()))
        # P and the output are rounded once, scores by 2^-13, and what cache_read gives of 8 bits once more
        assert bool(((out[at:at + new].double() - want).abs() <= (4 * 2.0 ** -11 + 2.0 ** -13) * size + 2.0 ** -24 * kv * v.abs().max()).all())
        at += new
    alone = s.layer(s.x, *s.args, plan=s.plan())
    # Each by itself: the attention's outputs x differ by d, up to four roundings to fp16 or 2^-9 of their sizes.  The projection's
    # base quantises x to codes that are up to 2^-3 x apart: such a d takes one code in (2^-3 x / d) over to the next, by a whole
    # 2^-3 x, so the mean square of what reaches the products is 2^-3 x d, at most 2^-12 x^2, whose root is 2^-6.
    assert float((alone.double() - got.double()).norm() / got.double().norm()) < 2.0 ** -6


def test_step_in_a_graph():
    """Plan, projections, cache write, attention and output recorded once; replayed for other tokens, lengths and prefixes between eager steps."""
    s = Step(torch.float16)
    layer = s.layer

    def step():
        return layer(s.x, *s.args, plan=s.plan(**s.groups))

    want = step().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(3):
        s.x.copy_(torch.from_numpy(activations(s.tokens, s.x.shape[1], 50 + turn)).cuda())
        s.groups["prefix_lens"].copy_(torch.tensor([p // (turn + 1) for p in s.prefix_lens], dtype=torch.int32))
        fresh = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, fresh) and not torch.equal(fresh, want)
