"""Attention of sequences in groups that share a prefix: the answer of every sequence by itself.

Bounds are those of test_gpu_attention.py: which tokens go into which partial sum changes no rounding but those of sums in 32 bits."""
import math

import pytest
import torch

from tests.test_gpu_attention import HALF, KINDS, Batch, empty_cache, ops, rows_of

pytestmark = pytest.mark.gpu


class Shared(Batch):
    """Groups (tokens of the prefix, [(new tokens, tokens of its own), ..]); a group with prefix None: sequences that belong to none.  Whole pages of a prefix are the same
    ones for all of its sequences, a page that it ends in is copied."""

    def __init__(self, groups, heads=4, kv_heads=2, dim=128, page=16, kind="same", dtype=torch.float16, padding=0, seed=0, big=1.0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page, self.kind, self.dtype = heads, kv_heads, dim, page, kind, dtype
        self.lengths = [(n, (prefix or 0) + own) for prefix, seqs in groups for n, own in seqs]
        need = sum((prefix or 0) // page for prefix, _ in groups) + sum(-(-kv // page) for _, kv in self.lengths)
        n_pages = need + 2
        self.cache = empty_cache(kind, dtype, n_pages, kv_heads, page, dim)
        order = torch.randperm(n_pages, generator=g).to(torch.int32)
        self.width = max((-(-kv // page) for _, kv in self.lengths), default=0) + 1
        self.pages = torch.full((len(self.lengths), self.width), 2 ** 31 - 1, dtype=torch.int32)
        self.group_starts, self.prefix_lens, self.k, self.v = [], [], [], []
        at = b = 0
        for prefix, seqs in groups:
            if prefix is not None:
                assert not self.group_starts or self.group_starts[-1] == b
                self.group_starts += [b, b + len(seqs)] if not self.group_starts else [b + len(seqs)]
                self.prefix_lens.append(prefix)
            whole = (prefix or 0) // page
            shared = order[at:at + whole]
            at += whole
            first = [torch.randn(((prefix or 0), kv_heads, dim), generator=g) * big for _ in range(2)]
            for n, own in seqs:
                kv = (prefix or 0) + own
                mine = -(-kv // page) - whole
                self.pages[b, :whole], self.pages[b, whole:whole + mine] = shared, order[at:at + mine]
                at += mine
                k, v = (torch.cat([x, torch.randn((own, kv_heads, dim), generator=g) * big]) for x in first)
                ops().cache_write(self.cache, k.to(dtype).cuda(), v.to(dtype).cuda(), self.slots(b, torch.arange(kv)))
                b += 1
        # what the cache holds, from its own codes
        for keep, raw, scale in ((self.k, self.cache.k, self.cache.k_scale), (self.v, self.cache.v, self.cache.v_scale)):
            held, scales = rows_of(raw, page), None if scale is None else rows_of(scale, page)
            for b, (_, kv) in enumerate(self.lengths):
                place = self.slots(b, torch.arange(kv)).cpu()
                x = held[place].double()
                keep.append(x if scale is None else x * scales[place].double()[..., None])
        self.starts = [0]
        for n, _ in self.lengths:
            self.starts.append(self.starts[-1] + n)
        self.q = (torch.randn((self.starts[-1] + padding, heads, dim), generator=g) * 2).to(dtype)

    def groups(self):
        return dict(group_starts=torch.tensor(self.group_starts or [0], dtype=torch.int32).cuda(), prefix_lens=torch.tensor(self.prefix_lens, dtype=torch.int32).cuda())

    def plan(self, max_q=None, causal=True, window=0, **groups):
        q, cache, _, starts, lens = self.inputs()
        return ops().attention_plan(cache, starts, lens, self.heads, q.shape[0], max_q, causal, window, **(groups or self.groups()))

    def attend(self, max_q=None, causal=True, window=0, scale=None, **groups):
        q, cache, pages, starts, lens = self.inputs()
        return ops().paged_attention(q, cache, pages, starts, lens, plan=self.plan(max_q, causal, window, **groups), causal=causal, window=window, scale=scale)


DECODES = [(300, [(1, 1), (1, 15), (1, 70)]), (0, [(1, 40), (1, 3)]), (64, [(1, 1), (1, 64)]), (1100, [(1, 5), (1, 130), (1, 1), (1, 200), (1, 64), (1, 63), (1, 65)]),
           (500, [(1, 20)]), (None, [(1, 90), (1, 1), (1, 900)])]
CHUNKS = [(None, [(3, 100)]), (190, [(5, 5), (1, 40), (70, 70), (2, 9)]), (400, [(64, 128), (33, 33), (1, 1), (1, 900)]), (1000, [(200, 263), (129, 129), (1, 1), (40, 41), (2, 30)])]
MANY = [(1900, [(1, 1 + 7 * i % 90) for i in range(24)]), (130, [(1, 3)] * 30), (None, [(1, 100)] * 5)]
PROMPTS = [(700, [(64, 128), (33, 33), (90, 100)]), (1000, [(200, 263), (129, 129)])]


def shared(batch, plan):
    """Whether the plan has every sequence of a group with a prefix joined from shares: the prefix's and its own."""
    joins = int(plan.buffer.view(torch.int32)[[1, 3, 5]].sum())
    at = [b for g, p in enumerate(batch.prefix_lens) if p >= 64 for b in range(batch.group_starts[g], batch.group_starts[g + 1])]
    return joins >= sum(batch.lengths[b][0] > 0 for b in at) > 0


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,page", [(4, 4, 16), (8, 2, 32), (20, 1, 64), (3, 1, 128)])
@pytest.mark.parametrize("groups", [DECODES, CHUNKS, MANY, PROMPTS], ids=["decodes", "chunks", "many", "prompts"])
def test_shared_prefix(kind, dtype, dim, heads, kv_heads, page, groups):
    batch = Shared(groups, heads, kv_heads, dim, page, kind, dtype)
    most = max(n for n, _ in batch.lengths)
    assert groups is PROMPTS or shared(batch, batch.plan(most))
    batch.check(batch.attend(most))
    batch.check(batch.attend(most, causal=False, scale=0.2), causal=False, scale=0.2)
    batch.check(batch.attend(most, window=50), window=50)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("most", [None, 1, 2, 7, 100000])
@pytest.mark.parametrize("groups", [DECODES, CHUNKS], ids=["decodes", "chunks"])
def test_the_largest_number_of_new_tokens_is_a_hint(kind, most, groups):
    batch = Shared(groups, 8, 2, 128, 16, kind)
    batch.check(batch.attend(most))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("most", [1, None])
def test_groups_of_nothing(kind, most):
    """Sequences without new tokens, groups without sequences, new tokens that reach back into the prefix or ahead of the context, no tokens of their own, padding."""
    batch = Shared([(1000, [(0, 0), (1, 30), (0, 10), (1, 7)]), (300, []), (128, [(6, 2), (40, 3)]), (100, [(150, 30), (1, 1)]), (256, [(0, 9), (0, 1)]), (64, []),
                    (None, [(2, 50)])], 6, 2, 64, 16, kind, padding=21)
    batch.check(batch.attend(most))
    batch.check(batch.attend(most, causal=False), causal=False)
    cross = Shared([(960, [(3, 0), (1, 0), (20, 0)]), (70, [(1, 0), (2, 0)])], 6, 2, 64, 16, kind)
    cross.check(cross.attend(most, causal=False), causal=False)                 # states that all rows see all of, and nothing else
    none = Shared([(None, [])], padding=3)
    assert not none.attend(most).any()
    assert Shared([(100, [(0, 5), (0, 1)])]).attend(most).shape == (0, 4, 128)
    no_groups = Shared([(None, [(1, 100), (3, 70)])], 4, 2, 128, 16, kind)
    no_groups.check(no_groups.attend(most))


@pytest.mark.parametrize("kind", list(KINDS))
def test_prefixes_that_are_cut_into_shares(kind):
    for groups in ([(9000, [(1, 30), (1, 700), (2, 5)])], [(20000, [(3, 40), (40, 5000)]), (5000, [(1, 1), (1, 1)])], [(12000, [(150, 151), (1, 12), (90, 3000)])]):
        batch = Shared(groups, 4, 1, 128, 64, kind, torch.bfloat16)
        most = max(n for n, _ in batch.lengths)
        for how in ({}, {"causal": False}):
            batch.check(batch.attend(most, **how), **how)


@pytest.mark.parametrize("kind", list(KINDS))
def test_prompts_that_are_cut_into_two_rounds(kind):
    """Prompts share nothing; 42 tiles over 8 heads are cut into more shares than the 64 of one round, and joined."""
    batch = Shared([(1300, [(203, 203), (200, 251), (196, 199)]), (1280, [(203, 210), (193, 230), (200, 200)])], 32, 8, 64, 64, kind, torch.bfloat16, padding=3)
    counts = batch.plan(203).buffer.view(torch.int32)[:6].tolist()
    assert counts[3] == 42 and 64 < counts[2] <= 128 and counts[4:] == [0, 0], counts
    batch.check(batch.attend(203))
    batch.check(batch.attend(203, causal=False), causal=False)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 32, 64), (30, 30, 128), (64, 32, 128)])
def test_a_wavefront_for_each_sequence(kind, dtype, heads, kv_heads, dim):
    """Enough sequences times heads of the cache that each one's own part is a wavefront's; a prompt, sequences that share little and long parts among them."""
    batch = Shared([(1300, [(1, 1 + 37 * i % 300) for i in range(13)] + [(1, 700)]), (64, [(1, 9), (0, 5), (3, 70)]), (900, [(30, 40), (1, 1), (1, 64)]), (None, [(1, 900), (1, 20)])],
                   heads, kv_heads, dim, 16, kind, dtype, padding=2)
    assert shared(batch, batch.plan(1)) and len(batch.lengths) * kv_heads > 512
    batch.check(batch.attend(1))
    batch.check(batch.attend(30, causal=False, scale=0.2), causal=False, scale=0.2)


MIXED = [(2048, [(1, 1 + 9 * i % 100) for i in range(40)])]


@pytest.mark.parametrize("at", [0, 13, 40])
def test_a_prompt_beside_requests_of_few_tokens(at):
    """A prompt of a group walks its own context and leaves the others to share: as many tiles are joined as without it, wherever it stands."""
    few = MIXED[0][1]
    alone = Shared(MIXED, 8, 8, 64, 64)
    mixed = Shared([(2048, few[:at] + [(1500, 1500)] + few[at:])], 8, 8, 64, 64)
    joins = [batch.plan(most).buffer.view(torch.int32)[[1, 3, 5]].tolist() for batch, most in ((alone, 1), (mixed, 1500))]
    assert joins[0][0] + joins[0][2] == len(few) == joins[1][0] + joins[1][2], joins
    for most in (1, 1500):
        mixed.check(mixed.attend(most))


BETWEEN = [(1000, [(1, 30), (100, 120), (2, 5), (1, 1), (300, 310), (70, 70), (0, 9), (3, 200), (65, 90), (1, 2)]),
           (800, [(80, 300), (1, 7), (257, 257), (66, 66), (129, 140), (4, 4), (1, 600), (70, 70)]), (640, [(70, 70), (1, 3), (2, 3), (80, 80)]), (600, [(100, 100), (1, 9), (67, 67)]), (900, [(1, 1), (1, 70)]),
           (None, [(1, 50), (90, 90)])]
PACKED = [(1024, [(15, 20), (270, 270), (16, 16), (14, 90), (90, 91), (64, 70), (64, 64), (1, 1), (99, 99), (260, 300), (60, 60)]), (700, [(64, 64), (666, 670), (64, 64), (1, 1)])]


@pytest.mark.parametrize("many", [29, 30])
def test_sequences_of_some_rows_share_while_they_are_few(many):
    """Sequences of 65 to 256 rows are in the prefix as long as they have 6144 rows together."""
    some = [(210, 220 + i) for i in range(many)]
    batch = Shared([(768, [*some[:9], (1, 9), (1, 200), (0, 3), (3, 3), (2, 2), *some[9:]])], 2, 2, 64, 64)
    counts = batch.plan(210).buffer.view(torch.int32)[:6].tolist()
    assert counts[1] == 4 and (counts[4] > 0) == (many == 30), counts           # (a prefix of 7 rows is in the list of long walks, one of thousands among the tiles)
    for most in (1, 210):
        batch.check(batch.attend(most))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 128), (8, 2, 64), (20, 1, 128), (48, 48, 64)])
@pytest.mark.parametrize("groups", [BETWEEN, PACKED], ids=["between", "packed"])
def test_prompts_between_requests_of_few_tokens(kind, dtype, heads, kv_heads, dim, groups):
    """The rows that share are not adjacent: in prefixes of few rows, of several tiles, in more than one group, with groups beside them whose rows are."""
    batch = Shared(groups, heads, kv_heads, dim, 16, kind, dtype, padding=3)
    for most in (1, 666):
        batch.check(batch.attend(most))
    batch.check(batch.attend(666, causal=False, scale=0.2), causal=False, scale=0.2)
    few = [n for _, seqs in groups for n, _ in seqs if 0 < n * heads // kv_heads <= 64]
    joins = batch.plan(666).buffer.view(torch.int32)[[1, 3, 5]].tolist()
    assert len(few) < 2 or sum(joins) >= 2, joins


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("groups", [BETWEEN, PACKED], ids=["between", "packed"])
def test_plan_and_scratch_of_nan_with_prompts(kind, groups):
    """What a plan or a kernel reads without its having been written shows: both begin as NaN, and as the plan's largest numbers; twice, with the same bits."""
    from triteia_amd.python.capi import _ffi
    batch = Shared(groups, 8, 2, 128, 16, kind, padding=9)
    q, cache, pages, starts, lens = batch.inputs()
    at = batch.groups()
    sizes = (len(batch.lengths), len(batch.prefix_lens), q.shape[0], 8, 2)
    lib, most, where = _ffi.lib(), 666, (_ffi.device_index(q), _ffi.stream_of(q))
    plan_bytes, nbytes = lib.triteia_hip_shared_plan_bytes(*sizes, most), lib.triteia_hip_shared_scratch_bytes(*sizes, most, cache.dim)
    outs = []
    for fill in (0xff, 0x7f):
        out, scratch, plan = (torch.full_like(q, math.nan), *(torch.full((n,), fill, dtype=torch.uint8, device="cuda") for n in (nbytes, plan_bytes)))
        codes = [lib.triteia_hip_shared_plan(_ffi.ptr(starts), _ffi.ptr(lens), _ffi.ptr(at["group_starts"]), _ffi.ptr(at["prefix_lens"]), *sizes, most, 1, 0, _ffi.ptr(plan), plan_bytes, *where),
                 lib.triteia_hip_shared_attention(
                     _ffi.ptr(q), q.stride(0), q.stride(1), _ffi.ptr(out), *cache._pointers(), cache._strides, cache.n_pages, cache.page, cache.kind, _ffi.ptr(pages), pages.stride(0),
                     pages.shape[1], _ffi.ptr(plan), plan_bytes, *sizes, cache.dim, most, 1, 0, cache.dim ** -0.5, _ffi.ptr(scratch), nbytes, 0, *where)]
        assert codes == [0, 0], _ffi.last_error()
        outs.append(out)
    batch.check(outs[0])
    assert torch.equal(*outs)


def test_prompts_in_hundreds_of_groups():
    groups = [(1024, [(1, 1 + i % 30), (65 + i % 7, 65 + i % 40), (1 + i % 3, 9)]) for i in range(400)]
    batch = Shared(groups, 1, 1, 64, 64)
    joins = batch.plan(1).buffer.view(torch.int32)[[1, 3, 5]].tolist()
    assert joins[0] >= 800, joins
    batch.check(batch.attend(1))


def test_prompts_that_come_and_go_between_replays():
    """Which sequences are prompts is the device's to say: one graph, whose offsets change between replays."""
    batch = Shared([(700, [(1, 100), (170, 200), (2, 100), (1, 100), (166, 200), (3, 100)]), (900, [(1, 100), (1, 100), (180, 200), (1, 100)])], 4, 2, 64, 16)
    q, cache, pages, starts, lens = batch.inputs()
    groups = batch.groups()

    def call():
        plan = ops().attention_plan(cache, starts, lens, batch.heads, q.shape[0], 180, **groups)
        return ops().paged_attention(q, cache, pages, starts, lens, plan=plan)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    total = batch.starts[-1]
    for new in ([n for n, _ in batch.lengths], [170, 1, 1, 66, 2, 3, 180, 1, 1, 1], [1] * 10, [20, 30, 1, 2, 60, 2, 1, 1, 50, 1], [1, 1, 129, 1, 128, 1, 2, 150, 1, 64], [n for n, _ in batch.lengths]):
        batch.lengths = [(n, kv) for n, (_, kv) in zip(new, batch.lengths)]
        batch.starts = [sum(new[:i]) for i in range(len(new) + 1)]
        assert batch.starts[-1] <= total
        starts.copy_(torch.tensor(batch.starts, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        alone = call()
        torch.cuda.synchronize()
        assert torch.equal(alone, out)
        batch.check(alone)


@pytest.mark.parametrize("most", [1, None])
def test_more_groups_and_tiles_than_a_wavefront_has_lanes(most):
    groups = [(64 * (15 + i % 3) + 5, [(1, 1 + i % 5)] * (4 + i % 3)) for i in range(75)]
    batch = Shared(groups, 2, 1, 64, 16)
    assert shared(batch, batch.plan(most))
    batch.check(batch.attend(most))
    batch = Shared([(130, [(20, 20)] * 6)] * 70, 8, 1, 64, 16)                  # more than 256 tiles
    batch.check(batch.attend(most))


def test_sharing_that_does_not_pay():
    """Short prefixes of a few requests are read again; the answer is the same."""
    for groups, heads, kv_heads, pays in (([(512, [(1, 20)] * 16)], 64, 8, False), ([(4096, [(1, 20)] * 16)], 16, 8, True), ([(1024, [(1, 9), (1, 40)])], 8, 8, True),
                                          ([(640, [(1, 10)] * 20)], 32, 32, True), ([(256, [(1, 10)] * 20)], 32, 8, False)):
        batch = Shared(groups, heads, kv_heads, 64, 64)
        assert shared(batch, batch.plan(None)) == pays, groups
        batch.check(batch.attend(None))


def test_a_prefix_is_what_the_pages_say():
    """Prefix lengths shorter than what is shared are as right as the whole; longer ones end where some row's own context begins."""
    batch = Shared([(1024, [(1, 30), (1, 90), (4, 200)])], 8, 2, 128, 16)
    starts = torch.tensor([0, 3], dtype=torch.int32).cuda()
    for prefix in (-5, 0, 1, 63, 64, 500, 1024):
        batch.check(batch.attend(4, group_starts=starts, prefix_lens=torch.tensor([prefix], dtype=torch.int32).cuda()))
    twins = Shared([(1024, [(3, 0), (3, 0)])], 8, 2, 128, 16)                   # the same context twice
    for prefix in (1024, 2000, 2 ** 31 - 1):
        twins.check(twins.attend(3, group_starts=torch.tensor([0, 2], dtype=torch.int32).cuda(), prefix_lens=torch.tensor([prefix], dtype=torch.int32).cuda()))


@pytest.mark.parametrize("starts", [[0, 3, 2, 7], [5, 0, 3, 9], [-4, 2, 100, 50], [7, 7, 7, 7], [2 ** 31 - 1, 0, 0, -2 ** 31]])
def test_group_offsets_in_no_order(starts):
    """Each is taken as the largest ahead of it, inside the batch: any sequence is in one group at most, and every row is written.  (All share all of the prefix here, so that
    any grouping is right.)"""
    batch = Shared([(1000, [(1, 5), (2, 40), (1, 1), (3, 9), (1, 30), (1, 2), (1, 70)])], 4, 2, 64, 16)
    for prefixes in ([1000, 1000, 1000], [64, 0, 800]):
        batch.check(batch.attend(3, group_starts=torch.tensor(starts, dtype=torch.int32).cuda(), prefix_lens=torch.tensor(prefixes, dtype=torch.int32).cuda()))


def test_a_table_shorter_than_the_prefix():
    """Tokens behind the table's last column are not seen, of a prefix as of any context."""
    batch = Shared([(1280, [(1, 40), (2, 10)]), (320, [(1, 1), (1, 1)])], 4, 2, 64, 16)
    assert shared(batch, batch.plan(2, causal=False))
    q, cache, pages, starts, lens = batch.inputs()
    for columns in (1, 3, 20, 70):
        plan = ops().attention_plan(cache, starts, lens, 4, q.shape[0], 2, causal=False, **batch.groups())
        got = ops().paged_attention(q, cache, pages[:, :columns], starts, lens, plan=plan, causal=False)
        held = Batch.__new__(Batch)
        held.__dict__.update(batch.__dict__)
        held.lengths = [(n, min(kv, 16 * columns)) for n, kv in batch.lengths]
        held.k, held.v = ([x[:16 * columns] for x in held] for held in (batch.k, batch.v))
        held.check(got, causal=False)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_what_is_no_number_reaches_the_rows_that_see_it(bad):
    """In the shared part all of the group, in a sequence's own part its own rows, behind the last token of a page none."""
    for most in (1, None):
        batch = Shared([(1024, [(1, 20), (2, 30), (1, 90)]), (128, [(1, 3), (1, 4)])], 4, 2, 64, 16)
        assert shared(batch, batch.plan(most))
        clean = batch.attend(most)
        batch.check(clean)
        page, slot = divmod(int(batch.slots(1, torch.tensor([1024 + 29]))), 16)      # the second sequence's newest token
        batch.cache.v[page, :, slot, 5] = bad
        got = batch.attend(most)
        assert not got[2, :, 5].isfinite().any() and torch.equal(got[[0, 1, 3, 4, 5]], clean[[0, 1, 3, 4, 5]])
        page, slot = divmod(int(batch.slots(0, torch.tensor([70]))), 16)
        batch.cache.v[page, :, slot, 9] = bad
        got = batch.attend(most)
        assert not got[:4, :, 9].isfinite().any() and torch.equal(got[4:], clean[4:])


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("groups,most", [(DECODES, 1), (CHUNKS, None), (MANY, 1)])
def test_scratch_and_output_of_nan(kind, groups, most):
    """What no kernel writes, or reads without having written it, shows; twice, with the same bits."""
    from triteia_amd.python.capi import _ffi
    batch = Shared(groups, 8, 2, 128, 16, kind, padding=9)
    q, cache, pages, starts, lens = batch.inputs()
    plan = ops().attention_plan(cache, starts, lens, batch.heads, q.shape[0], most, **batch.groups())
    sizes = (plan.n_seqs, plan.n_groups, plan.n_tokens, plan.heads, plan.kv_heads)
    nbytes = _ffi.lib().triteia_hip_shared_scratch_bytes(*sizes, plan.max_q, cache.dim)
    outs = []
    for _ in range(2):
        out, scratch = torch.full_like(q, math.nan), torch.full((nbytes,), 0xff, dtype=torch.uint8, device="cuda")
        code = _ffi.lib().triteia_hip_shared_attention(
            _ffi.ptr(q), q.stride(0), q.stride(1), _ffi.ptr(out), *cache._pointers(), cache._strides, cache.n_pages, cache.page, cache.kind, _ffi.ptr(pages),
            pages.stride(0), pages.shape[1], _ffi.ptr(plan.buffer), plan.buffer.numel(), *sizes, cache.dim, plan.max_q, 1, 0, cache.dim ** -0.5, _ffi.ptr(scratch), nbytes,
            0, _ffi.device_index(q), _ffi.stream_of(q))
        assert code == 0, _ffi.last_error()
        outs.append(out)
    batch.check(outs[0])
    assert torch.equal(*outs)


def test_large_scores():
    """Sums of both parts meet under one maximum, however far apart their own are."""
    for big in (0.01, 30.0, 300.0):
        for kind in KINDS:
            batch = Shared([(1000, [(1, 60), (1, 3), (5, 90)])], 4, 2, 64, 16, kind, torch.bfloat16, big=big)
            batch.q = (batch.q.float() * 0.2).to(batch.dtype)
            got = batch.attend(None)
            want, size, _ = batch.answer()
            exact = torch.stack([torch.ones(())])                               # (a score of 32 bits is off by 2^-24 of its terms' sum, and a weight by as much)
            terms = (batch.q.double().abs().amax() * max(k.abs().max() for k in batch.k) * 64 * 64 ** -0.5 * 1.45) * 2.0 ** -23 * 64 * exact
            bound = (2 * 2.0 ** -8 + 2.0 ** -13 + 2 * terms) * size + 1e-30
            assert bool(((got.double().cpu() - want).abs() <= bound).all())


def test_replays_and_streams():
    """A plan and a call recorded into a graph, its lengths, groups and cache changed between replays; two graphs, and eager calls on another stream, side by side."""
    batch = Shared(DECODES, 8, 2, 128, 16)
    q, cache, pages, starts, lens = batch.inputs()
    groups = batch.groups()

    def call():
        plan = ops().attention_plan(cache, starts, lens, batch.heads, q.shape[0], 1, **groups)
        return ops().paged_attention(q, cache, pages, starts, lens, plan=plan)

    want = call()
    batch.check(want)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(call())
    side = torch.cuda.Stream()
    for turn, prefixes in enumerate((batch.prefix_lens, [0] * len(batch.prefix_lens), [64] * len(batch.prefix_lens), batch.prefix_lens)):
        groups["prefix_lens"].copy_(torch.tensor([min(p, most) for p, most in zip(prefixes, batch.prefix_lens)], dtype=torch.int32))
        q.copy_(batch.q * (turn + 1) / 4)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            beside = call()
        alone = call()
        torch.cuda.synchronize()
        assert all(torch.equal(alone, x) for x in (*outs, beside))
        held, batch.q = batch.q, q.cpu()
        batch.check(alone)
        batch.q = held


def test_refusals_and_the_python_path(monkeypatch):
    from triteia_amd.python.capi import attention
    batch = Shared(DECODES, 8, 2, 128, 16)
    q, cache, pages, starts, lens = batch.inputs()
    groups = batch.groups()
    plan = lambda **how: ops().attention_plan(cache, starts, lens, 8, q.shape[0], 1, **{**groups, **how})  # noqa: E731
    for how, text in ((dict(group_starts=None), "together"), (dict(prefix_lens=None), "together"), (dict(prefix_lens=groups["prefix_lens"][:-1].contiguous()), "group_starts must have"),
                      (dict(prefix_lens=groups["prefix_lens"].long()), "int32"), (dict(group_starts=groups["group_starts"].float()), "int32"),
                      (dict(prefix_lens=groups["prefix_lens"].cpu()), "GPU tensor"), (dict(prefix_lens=groups["prefix_lens"].repeat(2)[::2]), "contiguous"),
                      (dict(group_starts=torch.zeros(1026, dtype=torch.int32).cuda(), prefix_lens=torch.zeros(1025, dtype=torch.int32).cuda()), "groups")):
        with pytest.raises(RuntimeError, match=text):
            plan(**how)
    with pytest.raises(RuntimeError, match="causal"):
        ops().paged_attention(q, cache, pages, starts, lens, plan=plan(), causal=False)
    want = batch.attend(1)

    class Nothing:
        def __getattr__(self, name):
            return lambda *args: None

    assert attention.native().shared_plan(starts, lens, groups["group_starts"], groups["prefix_lens"], q.shape[0], 8, 2, 1, True, 0) is not None
    monkeypatch.setattr(attention, "native", lambda: Nothing())
    assert torch.equal(batch.attend(1), want)
