"""The attention side where the range of a type, a table or a list ends, and the kernels' builds and the plan's branches that the ordinary batches do not reach.

Bounds are those of test_gpu_attention.py unless a test derives its own."""
import math

import pytest
import torch

from tests.test_gpu_attention import HALF, KINDS, U, Batch, empty_cache, ops, randn, rows_of

pytestmark = pytest.mark.gpu


def attend_into_nan(batch, starts, lens, pages, most, causal=True, window=0):
    """paged_attention by the C ABI with an output and a scratch full of NaN: what no kernel writes, or reads without having written it, shows."""
    from triteia_amd.python.capi import _ffi
    q, cache = batch.q.cuda(), batch.cache
    plan = ops().attention_plan(cache, starts, lens, batch.heads, q.shape[0], most, causal, window)
    out = torch.full_like(q, math.nan)
    nbytes = _ffi.lib().triteia_hip_attention_scratch_bytes(plan.n_seqs, plan.n_tokens, plan.heads, plan.kv_heads, plan.max_q, cache.dim)
    scratch = torch.full((nbytes,), 0xff, dtype=torch.uint8, device="cuda")
    code = _ffi.lib().triteia_hip_paged_attention(
        _ffi.ptr(q), q.stride(0), q.stride(1), _ffi.ptr(out), *cache._pointers(), cache._strides, cache.n_pages, cache.page, cache.kind, _ffi.ptr(pages),
        pages.stride(0), pages.shape[1], _ffi.ptr(plan.buffer), plan.buffer.numel(), plan.n_seqs, plan.n_tokens, plan.heads, plan.kv_heads, cache.dim, plan.max_q,
        int(causal), window, cache.dim ** -0.5, _ffi.ptr(scratch), nbytes, int(q.dtype == torch.bfloat16), _ffi.device_index(q), _ffi.stream_of(q))
    assert code == 0, _ffi.last_error()
    return out


# --- lengths, offsets and tables that do not fit each other -----------------------------------------------------------------------

def answer_within(batch, limit, lens, causal=True, window=0):
    """Batch.answer with contexts of `lens` of which the table holds the first `limit` tokens."""
    want = torch.zeros(batch.q.shape, dtype=torch.float64)
    size, most = torch.zeros_like(want), torch.zeros(want.shape[:2] + (1,), dtype=torch.float64)
    group = batch.heads // batch.kv_heads
    for b, (n, _) in enumerate(batch.lengths):
        rows = slice(batch.starts[b], batch.starts[b + 1])
        k, v = (x[b][:limit].repeat_interleave(group, 1) for x in (batch.k, batch.v))
        score = torch.einsum("thd,shd->hts", batch.q[rows].double(), k) * batch.dim ** -0.5
        position, token = torch.arange(n)[:, None] + (lens[b] - n), torch.arange(k.shape[0])
        seen = (token < lens[b]).expand(n, -1)
        if causal:
            seen = seen & (token <= position)
        if window:
            seen = seen & (token > position - window)
        p = torch.nan_to_num(torch.softmax(score.masked_fill(~seen, -math.inf), -1))
        want[rows], size[rows] = torch.einsum("hts,shd->thd", p, v), torch.einsum("hts,shd->thd", p, v.abs())
        most[rows] = k.shape[0] * v.abs().max()
    return want, size, most


def close(batch, got, want, size, most):
    bound = (2 * U[batch.dtype] + 2.0 ** -13) * size + 2.0 ** -24 * most + 1e-30
    got = got.double().cpu()
    assert bool(((got - want).abs() <= bound).all()), f"{float(((got - want).abs() / bound).nan_to_num(math.inf).max()):.3f} of the bound"


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("most", [1, None])
@pytest.mark.parametrize("columns", [3, 10, 40])
def test_tokens_that_the_table_does_not_hold_are_not_seen(kind, most, columns):
    """The plan cuts by lengths, the attention joins by what the table can hold: every row is written all the same."""
    batch = Batch([(1, 3000), (1, 40), (100, 2500), (6, 700), (1, 1030)], 4, 2, 64, 16, kind)
    lens, pages = [kv for _, kv in batch.lengths], batch.pages[:, :columns].contiguous().cuda()
    args = (torch.tensor(batch.starts, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), pages)
    for how in ({}, {"window": 50}, {"window": 2400}, {"causal": False}):
        close(batch, attend_into_nan(batch, *args, most, **how), *answer_within(batch, 16 * columns, lens, **how))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("most", [1, None])
def test_the_largest_lengths_cost_what_the_table_holds(kind, most):
    batch = Batch([(1, 300), (5, 300), (130, 300)], 4, 2, 64, 16, kind)
    starts, pages = torch.tensor(batch.starts, dtype=torch.int32).cuda(), batch.pages[:, :18].contiguous().cuda()
    for lens in ([2 ** 31 - 1] * 3, [2 ** 31 - 70, 300, 2 ** 30], [2 ** 31 - 1, 2 ** 31 - 129, 299]):
        for how in ({}, {"window": 60}, {"causal": False}):
            got = attend_into_nan(batch, starts, torch.tensor(lens, dtype=torch.int32).cuda(), pages, most, **how)
            close(batch, got, *answer_within(batch, 288, lens, **how))


@pytest.mark.parametrize("most", [1, None])
@pytest.mark.parametrize("starts", [[0, 500, -3, 140], [0, 140, 0, 140], [-7, 1, 2, 10 ** 9], [3, 20, 50, 140], [140, 0, 0, 0], [50, 60, 10, 30], [9, 9, 9, 9]])
def test_offsets_in_any_order_leave_no_row_out(most, starts):
    """An offset is taken as the largest of those up to it, the first as 0: every token has one sequence, or none."""
    batch = Batch([(1, 40), (9, 77), (130, 200)], 6, 3, 64, 16)
    got = attend_into_nan(batch, torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor([kv for _, kv in batch.lengths], dtype=torch.int32).cuda(),
                          batch.pages.cuda(), most)
    taken = [0]
    for s in starts[1:]:
        taken.append(max(taken[-1], min(max(s, 0), 140)))
    batch.starts, batch.lengths = taken, [(b - a, kv) for a, b, (_, kv) in zip(taken, taken[1:], batch.lengths)]
    batch.check(got)


# --- weights, scores and scales far apart -----------------------------------------------------------------------------------------

def put(batch, b, k, v):
    """Other keys and values [tokens, heads of the cache, dim] for sequence b."""
    place = batch.slots(b, torch.arange(batch.lengths[b][1]))
    ops().cache_write(batch.cache, k.to(batch.dtype).cuda(), v.to(batch.dtype).cuda(), place)
    for keep, raw, scale in ((batch.k, batch.cache.k, batch.cache.k_scale), (batch.v, batch.cache.v, batch.cache.v_scale)):
        x = rows_of(raw, batch.page)[place.cpu()].double()
        keep[b] = x if scale is None else x * rows_of(scale, batch.page)[place.cpu()].double()[..., None]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("seqs,n", [(64, 1), (32, 128)])
def test_many_small_weights_count(kind, seqs, n):
    """Ten thousand weights of 2^-26 of the largest, whose value is zero: below what fp16 holds beside 1, and all of the answer.  As many sequences as leave the
    context whole, on the same pages.

    A row's largest weight stands at 2^7 or more in fp16, so that a smaller one is off by 2^-32 of it at most."""
    kv, heads, dim = 10000, 32, 64
    batch = Batch([(1, kv)], heads, heads, dim, 64, kind)
    k, v = torch.zeros(kv, heads, dim), torch.ones(kv, heads, dim)
    k[0, :, 0], v[0] = 26 * math.log(2.0), 0.0
    put(batch, 0, k, v)
    batch.q[:] = 0
    batch.q[..., 0] = 1
    want, size, _ = batch.answer(scale=1.0)
    starts, lens = torch.arange(seqs + 1, dtype=torch.int32).cuda() * n, torch.full((seqs,), kv, dtype=torch.int32, device="cuda")
    got = ops().paged_attention(batch.q.repeat(seqs * n, 1, 1).cuda(), batch.cache, batch.pages.repeat(seqs, 1).cuda(), starts, lens, causal=False, scale=1.0,
                                max_q=n).double().cpu()
    assert want.min() > 1e-4
    bound = (2 * U[batch.dtype] + 2.0 ** -13) * size + kv * 2.0 ** -32
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n", [1, 5, 90])
def test_large_values_of_no_weight_do_not_hide_small_ones(kind, dtype, n):
    """Visible tokens whose values are 10^7 times the others' and whose weight is next to nothing: from the first on, later on, and with all of the weight until other
    tokens come.  Weights times scales are kept in fp16's range by the largest such product of the row, which stands at 1 or more there: an error of
    2^-25 of it for a token."""
    kv, dim, most_code = 700, 64, 127 if kind == "int8" else 448
    for case in ("first", "apart", "last", "until"):
        batch = Batch([(n, kv)], 4, 2, dim, 16, kind, dtype)
        big = {"first": [0], "apart": list(range(3, 600, 50)), "last": [kv - n - 1], "until": [0, 1, 17]}[case]
        k, v = randn(kv, 2, dim, seed=1) * 0.1, randn(kv, 2, dim, seed=2) * 2e-3
        v[big] = randn(len(big), 2, dim, seed=3) * 10000
        k[..., 0] = 0
        k[big, :, 0] = -40.0
        if case == "until":
            k[100:, :, 0] = 40.0
            k[big, :, 0] = 0.0
            k[2:17, :, 0], k[18:100, :, 0] = -40.0, -40.0
        put(batch, 0, k, v)
        batch.q[..., 0] = 1
        want, size, _ = batch.answer(scale=1.0)
        got = ops().paged_attention(*batch.inputs(), scale=1.0, max_q=n).double().cpu()
        # the largest weight times scale of every row
        top = torch.zeros(want.shape[:2] + (1,), dtype=torch.float64)
        v_scale = (batch.v[0].abs().amax(-1) / most_code).repeat_interleave(2, 1)                # [kv, heads]
        score = torch.einsum("thd,shd->hts", batch.q.double(), batch.k[0].repeat_interleave(2, 1))
        p = torch.softmax(score.masked_fill(torch.arange(kv) > torch.arange(kv - n, kv)[:, None], -math.inf), -1)
        top[..., 0] = (p * v_scale.t()[:, None]).amax(-1).t()
        bound = (2 * U[dtype] + 2.0 ** -13) * size + kv * 2.0 ** -25 * most_code * top + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert bool(((got - want).abs() <= bound).all()), (case, float(((got - want).abs() / bound).max()))


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n", [1, 90])
def test_scales_of_either_sign(kind, dtype, n):
    """A cache that a program has filled itself may hold negative scales, large ones among them."""
    batch = Batch([(n, 300)], 4, 2, 64, 16, kind, dtype)
    flip = torch.where(torch.arange(16) % 3 == 0, -3e4, 1.0).cuda()
    batch.cache.v_scale.mul_(flip)
    place = batch.slots(0, torch.arange(300)).cpu()
    batch.v[0] = rows_of(batch.cache.v, 16)[place].double() * rows_of(batch.cache.v_scale, 16)[place].double()[..., None]
    want, size, most = batch.answer()
    got = ops().paged_attention(*batch.inputs(), max_q=n).double().cpu()
    bound = (2 * U[dtype] + 2.0 ** -13) * size + 2.0 ** -24 * most
    finite = want.abs() < (60000 if dtype == torch.float16 else 1e30)
    assert bool(((got - want).abs() <= bound)[finite].all())


@pytest.mark.parametrize("kind", ["same", "int8"])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 3e4), (torch.bfloat16, 1e5), (torch.bfloat16, 1e16), (torch.bfloat16, 1e18)])
@pytest.mark.parametrize("n", [1, 5, 90])
def test_scores_near_the_end_of_32_bits(kind, dtype, size, n):
    """Scores of 10^10 to 3 * 10^38 of either sign, further apart than any exponential reaches: the largest takes all of the weight."""
    kv, dim = 200, 64
    for most, others in ((-0.5, -1.0), (1.0, 0.5), (1.0, -1.0)):
        batch = Batch([(n, kv)], 2, 1, dim, 16, kind, dtype)
        k, v = torch.full((kv, 1, dim), others * size), randn(kv, 1, dim, seed=2)
        k[37] = most * size
        put(batch, 0, k, v)
        batch.q[:] = size / 8
        got = ops().paged_attention(*batch.inputs(), max_q=n).double().cpu()
        want = batch.v[0][37, 0].expand_as(got)
        assert bool(((got - want).abs() <= 2 * U[dtype] * want.abs() + 2.0 ** -25).all())


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n", [1, 5, 90])
def test_equal_scores_of_any_size(kind, dtype, n):
    """Keys that are all the same: the mean of what a row sees, at scores of 0 to 10^10 of either sign, with values small enough to move fp16's range."""
    kv, dim = 700, 64
    for size, sign in ((0.0, 1), (30.0, 1), (3e3, -1), (3e4, 1), (3e4, -1)):
        batch = Batch([(n, kv)], 2, 1, dim, 16, kind, dtype)
        put(batch, 0, torch.full((kv, 1, dim), sign * size), randn(kv, 1, dim, seed=2) * 1e-2)
        batch.q[:] = size
        batch.check(ops().paged_attention(*batch.inputs(), max_q=n))


# --- the cache ----------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", HALF)
def test_codes_are_the_nearest_to_the_quotient(kind, dtype):
    """code = x / scale, as 32 bits round it, to the nearest code, on rows that hold quotients near the middle of two (a product with 1 / scale takes the other one of
    some of them)."""
    dim, tokens, held = 256, 4000, KINDS[kind]
    x = torch.rand(tokens, 1, dim, generator=torch.Generator().manual_seed(1))
    top = torch.rand(tokens, 1, 1, generator=torch.Generator().manual_seed(2)) * 4 + 0.1
    middle = torch.randint(0, 127, x.shape, generator=torch.Generator().manual_seed(3)).float() + 0.5
    x = torch.where(x < 0.9, middle / 127 * top, x * top).to(dtype)
    x[..., :1] = top.to(dtype)
    x = torch.minimum(x, x[..., :1])
    cache = ops().paged_cache(tokens // 16, 1, dim, 16, held)
    ops().cache_write(cache, x.cuda(), -x.cuda(), torch.arange(tokens).cuda())
    for y, raw, scale in ((x, cache.k, cache.k_scale), (-x, cache.v, cache.v_scale)):
        quotient = y.float() / rows_of(scale, 16)[..., None]
        want = quotient.round() if kind == "int8" else quotient.clamp(-448, 448).to(held).float()
        assert torch.equal(rows_of(raw, 16), want)


# --- the layer ------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("seqs", [0, 2])
@pytest.mark.parametrize("planned", [False, True])
def test_a_layer_of_no_tokens(seqs, planned):
    from triteia_amd.python.capi import route_plan
    from triteia_amd.python.nn import multi_delta_attention
    layer = multi_delta_attention(512, 4, 2, 64, 3).cuda()
    cache, table = ops().paged_cache(4, 2, 64, 16), ops().rotary_table(100, 64)
    int32 = dict(dtype=torch.int32, device="cuda")
    indices, starts, lens = torch.zeros(0, **int32), torch.zeros(seqs + 1, **int32), torch.full((seqs,), 9, **int32)
    extra = dict(plan=layer.plan(cache, starts, lens, 0), route=route_plan(indices, 3)) if planned else {}
    out = layer(torch.zeros(0, 512, dtype=torch.float16, device="cuda"), indices, indices, table, cache, indices, torch.zeros(seqs, 1, **int32), starts, lens, **extra)
    assert out.shape == (0, 512) and out.dtype == torch.float16


# --- the plan's branches and the builds that other batches do not reach -------------------------------------------------------------

def many(n, new, kv, seed=0):
    """n lengths of up to `new` new tokens (none among them) on contexts of up to `kv`."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for i in range(n):
        tokens = int(torch.randint(0 if i % 5 == 0 else 1, new + 1, (), generator=g))
        out.append((tokens, max(tokens, int(torch.randint(1, kv + 1, (), generator=g)))))
    return out


@pytest.mark.parametrize("n", [63, 64, 65, 130, 300])
@pytest.mark.parametrize("kind", ["same", "fp8"])
@pytest.mark.parametrize("new,most", [(1, 1), (1, None), (5, 5), (40, None)])
def test_many_sequences(n, kind, new, most):
    """The plan's sums over the sequences in rounds of 64, its order of tiles up to 256 of them and beyond."""
    batch = Batch(many(n, new, 90, n), 4, 2, 64, 16, kind, padding=5)
    batch.check(ops().paged_attention(*batch.inputs(), max_q=most))
    batch.check(ops().paged_attention(*batch.inputs(), max_q=most, window=20), window=20)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("most", [1, None])
def test_lists_of_many_tiles_are_cut(kind, most):
    """300 single tokens over one head of the cache, two on long contexts: their tiles are cut in a list that is not sorted."""
    lengths = many(300, 1, 60, 3)
    lengths[7], lengths[290] = (1, 9000), (1, 5001)
    batch = Batch(lengths, 2, 1, 64, 16, kind, torch.bfloat16)
    got = ops().paged_attention(*batch.inputs(), max_q=most)
    batch.check(got)
    long = torch.tensor([batch.starts[7], batch.starts[290]])
    near(got[long.cuda()], batch.answer()[0][long], batch.dtype)


@pytest.mark.parametrize("kind", ["same", "int8"])
def test_lists_of_many_long_tiles_are_cut(kind):
    lengths = [(17 + i % 9, 30 + i % 70) for i in range(262)]
    lengths[100], lengths[3] = (300, 6000), (1, 4000)
    batch = Batch(lengths, 1, 1, 64, 16, kind)
    got = ops().paged_attention(*batch.inputs())
    batch.check(got)
    rows = slice(batch.starts[100], batch.starts[101])
    near(got[rows], batch.answer()[0][rows], batch.dtype)


def near(got, want, dtype):
    """Beside the bound on each element, the norm of the error.  Weights are off by u (their rounding) and 2^-13 (scores), the output by u.  Random values of either sign
    add up like their squares, weights' errors with them: 2 u + 2^-13 of the norm.  (A block of 64 tokens that is lost or counted twice among 9000 is 8 %.)"""
    error = (got.double().cpu() - want).norm() / want.norm()
    assert error <= 2 * U[dtype] + 2.0 ** -13, float(error)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("lengths", [[(1, 9000)], [(4, 9001), (1, 5000)], [(150, 9001), (1, 12345), (20, 4100)]])
def test_cut_contexts_by_their_norm(kind, dtype, lengths):
    batch = Batch(lengths, 4, 1, 128, 64, kind, dtype)
    most = max(n for n, _ in lengths)
    for how in ({}, {"window": 4000}, {"causal": False}):
        got = ops().paged_attention(*batch.inputs(), max_q=most, **how)
        batch.check(got, **how)
        want = batch.answer(**how)[0]
        for b in range(len(lengths)):
            rows = slice(batch.starts[b], batch.starts[b + 1])
            near(got[rows], want[rows], dtype)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seqs,most", [(60, 1), (3, 1), (40, 4), (5, 4)], ids=["16 rows, 4 wavefronts", "16 rows, 8", "32 rows, 4", "32 rows, 8"])
def test_each_build_for_few_rows(kind, dtype, dim, seqs, most):
    """Tiles of 16 or 32 rows (8 heads of a group, 1 or 4 tokens) on four wavefronts (more than 128 workgroups by the plan's bounds) or eight."""
    group, kv_heads = 8, 4
    batch = Batch(many(seqs, most, 200, seqs + most), group * kv_heads, kv_heads, dim, 32, kind, dtype)
    tokens = batch.starts[-1]
    bound = min(seqs + 1, tokens) + tokens * group // (32 if most * group > 16 else 16)
    assert most * group <= 32 and (bound * kv_heads > 128) == (seqs >= 40)
    for how in ({}, {"window": 33}, {"causal": False}):
        got = ops().paged_attention(*batch.inputs(), max_q=most, **how)
        batch.check(got, **how)
        near(got, batch.answer(**how)[0], dtype)


@pytest.mark.parametrize("kind", ["same", "fp8"])
def test_a_mixed_step_in_a_graph(kind):
    """The launch of long and short tiles, a plan whose cuts and joins change, recorded once and replayed on other offsets, lengths, pages and tokens with work between."""
    heads, kv_heads, dim, page, tokens = 8, 2, 64, 16, 230
    batch = Batch([(1, 9000), (130, 9000), (99, 9000)], heads, kv_heads, dim, page, kind)
    q, cache, pages, starts, lens = batch.inputs()

    def step():
        return ops().paged_attention(q, cache, pages, starts, lens)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    batches = [([0, 1, 131, 230], [9000, 9000, 9000]), ([0, 1, 131, 230], [40, 130, 99]), ([0, 200, 200, 201], [8000, 0, 5000]), ([0, 3, 20, 228], [9000, 20, 208]),
               ([0, 1, 131, 230], [9000, 9000, 9000]), ([0, 0, 0, 0], [1, 2, 3])]
    for i, (s, n) in enumerate(batches):
        new = randn(tokens, heads, dim, seed=i).to(q.dtype)
        q.copy_(new)
        starts.copy_(torch.tensor(s, dtype=torch.int32))
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, step())
        torch.cuda.synchronize()
        # (the cache stays; sequences see the first tokens of their contexts)
        now = Batch.__new__(Batch)
        now.__dict__.update(batch.__dict__)
        now.q, now.starts, now.lengths = new, s, [(b - a, kv) for a, b, kv in zip(s, s[1:], n)]
        now.k, now.v = ([x[b][:n[b]] for b in range(3)] for x in (batch.k, batch.v))
        now.check(got)


# --- refusals -----------------------------------------------------------------------------------------------------------------------

def test_tangents_are_refused():
    """Forward mode: a tangent that the kernels would drop."""
    import torch.autograd.forward_ad as fwd
    x, table, positions = randn(3, 2, 64, dtype=torch.float16).cuda(), ops().rotary_table(10, 64), torch.zeros(3, dtype=torch.int32, device="cuda")
    cache = ops().paged_cache(4, 2, 64, page=16)
    pages, starts, lens = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([[0]], [0, 3], [3]))
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops().rotary(dual, x, positions, table), lambda: ops().rotary(x, dual, positions, table),
                     lambda: ops().cache_write(cache, x, dual, positions), lambda: ops().paged_attention(dual, cache, pages, starts, lens),
                     lambda: ops().rotary(x, x, positions, table, q_norm=fwd.make_dual(x[0, 0].clone(), x[0, 0].clone()))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        assert ops().rotary(x, x, positions, table)[0].shape == x.shape


def test_arguments_that_belong_together():
    x, table, positions = randn(3, 2, 64, dtype=torch.float16).cuda(), ops().rotary_table(10, 64), torch.arange(3).cuda()
    cache = ops().paged_cache(4, 2, 64, page=16)
    for call in (lambda: ops().rotary(x, x, positions, None), lambda: ops().rotary(x, x, None, table),
                 lambda: ops().rotary_cache_write(x, x, x, positions, None, cache, positions)):
        with pytest.raises(RuntimeError, match="positions and table"):
            call()
    for call in (lambda: ops().rotary(x, None, positions, table), lambda: ops().rotary_cache_write(x, x, None, positions, table, cache, positions),
                 lambda: ops().cache_write(cache, x, x, None), lambda: ops().cache_write(cache, None, x, positions), lambda: ops().cache_read(cache, None)):
        with pytest.raises(TypeError, match="must be a torch.Tensor"):
            call()
    # (norms alone, without a rotation, are a pass of their own)
    w = torch.full((64,), 2.0, dtype=torch.float16, device="cuda")
    y = ops().rotary(x, x, None, None, q_norm=w)
    assert torch.equal(y[1], x) and torch.allclose(y[0].float().pow(2).mean(-1), torch.tensor(4.0, device="cuda"), rtol=2e-3)


def test_no_heads_of_queries():
    x, table, positions = randn(3, 2, 64, dtype=torch.float16).cuda(), ops().rotary_table(10, 64), torch.arange(3).cuda()
    q, k = ops().rotary(x[:, :0], x, positions, table)
    assert q.shape == (3, 0, 64) and torch.equal(k, ops().rotary(x, x, positions, table)[1])
    q, k = ops().rotary(x, x[:, :0], positions, table)
    assert k.shape == (3, 0, 64) and torch.equal(q, ops().rotary(x, x, positions, table)[0])
    cache = ops().paged_cache(4, 2, 64, page=16)
    assert ops().rotary_cache_write(x[:, :0], x, x, positions, table, cache, positions).shape == (3, 0, 64)


def test_lazily_negated_tensors():
    """(torch gives such a view for the imaginary part of a conjugate: its memory holds the other sign.)"""
    x, table, positions = randn(3, 2, 64, dtype=torch.float16).cuda(), ops().rotary_table(10, 64), torch.arange(3).cuda()
    w = randn(64, seed=1, dtype=torch.float16).cuda()
    cache = ops().paged_cache(4, 2, 64, page=16)
    lazy = torch._neg_view
    for args in ((lazy(x), x, positions, table, False, w), (x, lazy(x), positions, table, False, w), (x, x, positions, lazy(table), False, w),
                 (x, x, positions, table, False, lazy(w), lazy(w))):
        plain = [a.resolve_neg().clone() if isinstance(a, torch.Tensor) else a for a in args]
        assert all(torch.equal(a, b) for a, b in zip(ops().rotary(*args), ops().rotary(*plain)))
    ops().cache_write(cache, lazy(x), x, positions)
    assert torch.equal(ops().cache_read(cache, positions)[0], -x)
    pages, starts, lens = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([[0]], [0, 3], [3]))
    assert torch.equal(ops().paged_attention(lazy(x), cache, pages, starts, lens), ops().paged_attention(-x, cache, pages, starts, lens))
    with pytest.raises(RuntimeError, match="negated"):
        ops().PagedCache(lazy(cache.k), cache.v)
