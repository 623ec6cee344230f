"""Rotary positions, the paged cache and the attention over it, against their formulas in 64 bits.

Bounds.  u is the unit roundoff of the output's type (2^-11 in fp16, 2^-8 in bf16).  A rotated element is one rounding of a 32-bit value: u |y| and
2^-20 of the row's largest magnitude for the 32-bit steps.  Attention rounds P once and the output once: 2 u sum(p |v|), 2^-13 sum(p |v|) for the scores
(sums of 64 or 128 products in 32 bits and a hardware exponential), and 2^-24 max|v| per token for weights below fp16's normal range.  Codes of 8 bits may lie
one step from the nearest where x / scale is within 2^-20 of the middle between two."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
HALF = [torch.float16, torch.bfloat16]
KINDS = {"same": None, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


def ops():
    from triteia_amd.python import ops
    return ops


def randn(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype)


# --- rotary ---------------------------------------------------------------------------------------------------------------------

def turned(x, positions, table, interleaved, weight, eps):
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    y, half = x.clone(), table.shape[1]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = table[positions, i, 0].double()[:, None], table[positions, i, 1].double()[:, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def close_rows(got, want, dtype):
    got = got.double().cpu()
    bound = U[dtype] * want.abs() + 2.0 ** -20 * want.abs().amax(-1, keepdim=True) + 2.0 ** -25
    assert got.shape == want.shape and bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 64), (64, 16), (80, 80), (80, 32), (256, 256), (96, 48), (16, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", HALF)
def test_rotary(dim, rot, interleaved, dtype):
    for tokens, heads, kv_heads, norm in ((1, 3, 1, False), (5, 8, 8, True), (700, 6, 2, True), (301, 33, 5, False)):
        table = ops().rotary_table(1000, rot)
        qkv = randn(tokens, heads + 2 * kv_heads, dim, seed=tokens, dtype=dtype)
        positions = torch.randint(0, 1000, (tokens,), generator=torch.Generator().manual_seed(1))
        weights = [1 + 0.2 * randn(dim, seed=s) for s in (2, 3)] if norm else [None, None]
        weights = [w if w is None else w.to(dtype) for w in weights]
        q, k, _ = qkv.cuda().split([heads, kv_heads, kv_heads], 1)          # views with the projection's strides
        for wide in (torch.int32, torch.int64):
            got = ops().rotary(q, k, positions.to(wide).cuda(), table, interleaved, *(w if w is None else w.cuda() for w in weights), eps=1e-5)
            for y, x, w in zip(got, qkv.split([heads, kv_heads, kv_heads], 1), weights):
                close_rows(y, turned(x, positions, table.cpu(), interleaved, w, 1e-5), dtype)


def test_rotary_with_one_norm_and_other_layouts():
    x, table, dtype = randn(9, 4, 64, seed=1), ops().rotary_table(50, 64), torch.float16
    x = x.to(dtype)
    positions, w = torch.arange(9), randn(64, seed=2).to(dtype)
    flat = torch.zeros(9 * 4 * 64 + 3, dtype=dtype, device="cuda")
    flat[3:] = x.cuda().flatten()
    layouts = [flat[3:].view(9, 4, 64), x.cuda().transpose(0, 1).contiguous().transpose(0, 1), x.cuda().transpose(1, 2).contiguous().transpose(1, 2)]
    for q in layouts:                                                          # not on 16 bytes, heads first, elements apart
        for weights in ((w, None), (None, w)):
            got = ops().rotary(q, q, positions.cuda(), table, q_norm=None if weights[0] is None else w.cuda(), k_norm=None if weights[1] is None else w.cuda())
            for y, weight in zip(got, weights):
                close_rows(y, turned(x, positions, table.cpu(), False, weight, 1e-6), dtype)


def test_positions_outside_the_table_are_loud():
    x, table = randn(4, 2, 64, dtype=torch.float16).cuda(), ops().rotary_table(10, 32)
    q, k = ops().rotary(x, x, torch.tensor([0, 10, -1, 9]).cuda(), table)
    bad = torch.tensor([False, True, True, False])
    assert q[bad, :, :32].isnan().all() and k[bad, :, :32].isnan().all() and not q[~bad].isnan().any()
    assert torch.equal(q[bad][..., 32:], x[bad][..., 32:])


def test_infinities_stay_in_their_pair():
    x, table = randn(1, 1, 64, dtype=torch.float16), ops().rotary_table(10, 32)
    x[0, 0, 3], x[0, 0, 40] = math.inf, math.nan
    q, _ = ops().rotary(x.cuda(), x.cuda(), torch.tensor([1]).cuda(), table)
    assert set((~q[0, 0].isfinite()).nonzero().flatten().tolist()) == {3, 19, 40}


def test_no_tokens_or_heads():
    table = ops().rotary_table(10, 64)
    none = torch.zeros(0, 4, 64, dtype=torch.float16, device="cuda")
    q, k = ops().rotary(none, none, torch.zeros(0, dtype=torch.int32, device="cuda"), table)
    assert q.shape == k.shape == (0, 4, 64)


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
                                     {"type": "bands", "factor": 8.0, "low": 1.0, "high": 4.0, "original": 512}, {"type": "yarn", "factor": 4.0, "original": 512}])
def test_table(scaling):
    rot, base = 64, 10000.0
    table = ops().rotary_table(100, rot, base, scaling).double().cpu()
    for i in (0, 1, 9, 17, 31):
        rate, size = base ** (-2 * i / rot), 1.0
        if scaling:
            f = scaling["factor"]
            if scaling["type"] == "linear":
                rate /= f
            elif scaling["type"] == "ntk":
                rate = (base * f ** (rot / (rot - 2))) ** (-2 * i / rot)
            elif scaling["type"] == "bands":
                turns = 512 * rate / (2 * math.pi)
                if turns < 1:
                    rate /= f
                elif turns <= 4:
                    s = (turns - 1) / 3
                    rate = (1 - s) * rate / f + s * rate
            else:
                lo, hi = (rot * math.log(512 / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32.0, 1.0))
                lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
                s = min(max((i - lo) / (hi - lo), 0), 1)
                rate, size = rate / f * s + rate * (1 - s), 0.1 * math.log(f) + 1
        for p in (0, 1, 37, 99):
            assert abs(table[p, i, 0] - size * math.cos(p * rate)) < 2e-7 and abs(table[p, i, 1] - size * math.sin(p * rate)) < 2e-7


# --- the cache --------------------------------------------------------------------------------------------------------------------

def empty_cache(kind, dtype, n_pages, kv_heads, page, dim, tokens_first=False):
    """A cache full of what must not be read: NaN (in int8: the scales)."""
    held = KINDS[kind] or dtype
    parts = []
    for _ in range(2):
        shape = (n_pages, page, kv_heads, dim) if tokens_first else (n_pages, kv_heads, page, dim)
        x = torch.full(shape, 127, dtype=torch.int8, device="cuda") if held == torch.int8 else torch.full(shape, math.nan, device="cuda").to(held)
        parts.append(x.transpose(1, 2) if tokens_first else x)
    if kind != "same":
        parts += [torch.full((n_pages, kv_heads, page), math.nan, device="cuda") for _ in range(2)]
    return ops().PagedCache(*parts)


def rows_of(t, page):
    """[slots, heads, ..] of a cache tensor, on the CPU."""
    return t.float().cpu().transpose(1, 2).reshape(-1, t.shape[1], *t.shape[3:])


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dim,page,tokens_first", [(128, 16, False), (64, 64, True), (128, 32, True), (80, 16, False), (256, 16, False), (8, 32, False)])
def test_write_and_read(kind, dtype, dim, page, tokens_first):
    kv_heads, n_pages = 3, 9
    for tokens in (1, 50, 140):
        cache = empty_cache(kind, dtype, n_pages, kv_heads, page, dim, tokens_first)
        k, v = (randn(tokens, kv_heads, dim, seed=s).mul(10.0 ** randn(tokens, kv_heads, 1, seed=s + 2)).to(dtype) for s in (1, 2))
        k[0, 1], v[tokens // 2, 2] = 0, 0
        slots = torch.randperm(n_pages * page, generator=torch.Generator().manual_seed(3))[:tokens]
        hidden = slots.clone()
        hidden[tokens // 3::7] = -1
        if tokens > 1:
            hidden[1] = n_pages * page
        ops().cache_write(cache, k.cuda(), v.cuda(), hidden.to(torch.int32 if tokens == 50 else torch.int64).cuda())
        kept = (hidden >= 0) & (hidden < n_pages * page)
        got = ops().cache_read(cache, hidden.cuda(), dtype)
        for x, y, raw, scale in zip((k, v), got, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
            y = y.float().cpu()
            assert not y[~kept].any()
            untouched = torch.ones(n_pages * page, dtype=torch.bool)
            untouched[hidden[kept]] = False
            if kind == "same":
                assert torch.equal(y[kept], x[kept].float()) and rows_of(raw, page)[untouched].isnan().all()
                continue
            # the scale is a division of 32-bit values; the code the nearest, or beside it where the quotient is in the middle
            most = 127 if kind == "int8" else 448
            want = x.double().abs().amax(-1) / most
            s = rows_of(scale, page)
            assert s[untouched].isnan().all()
            assert bool(((s[hidden[kept]].double() - want[kept]).abs() <= 2.0 ** -23 * want[kept]).all())
            code = rows_of(raw, page)[hidden[kept]].double()
            quotient = x[kept].double() / s[hidden[kept]].double().clamp_min(1e-38)[..., None]
            step = torch.ones_like(code) if kind == "int8" else 2.0 ** (code.abs().clamp_min(2.0 ** -6).log2().floor() - 3)
            assert bool(((code - quotient).abs() <= step * (0.5 + 2.0 ** -16) + 1e-9).all())
            value = code * s[hidden[kept]].double()[..., None]
            assert bool(((y[kept].double() - value).abs() <= U[dtype] * value.abs() * 1.001 + 2.0 ** -25).all())


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_rows_that_hold_no_number_read_back_as_none(kind):
    cache = ops().paged_cache(1, 2, 64, page=16, dtype=KINDS[kind])
    k = randn(4, 2, 64, dtype=torch.float16)
    k[1, 0, 5], k[2, 1, 60] = math.inf, math.nan
    ops().cache_write(cache, k.cuda(), k.cuda(), torch.arange(4).cuda())
    for x in ops().cache_read(cache, torch.arange(4).cuda()):
        bad = x.isnan().all(-1).cpu()
        assert bad.tolist() == [[False, False], [True, False], [False, True], [False, False]] and torch.equal(bad, x.isnan().any(-1).cpu())


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotated_keys_are_rounded_once(kind, interleaved):
    dtype, dim, tokens = torch.bfloat16, 128, 70
    qkv, table = randn(tokens, 8 + 2 * 2, dim, seed=5, dtype=dtype), ops().rotary_table(200, 64)
    positions, norm = torch.arange(tokens) + 100, (1 + 0.1 * randn(dim, seed=6)).to(dtype)
    cache = empty_cache(kind, dtype, 6, 2, 16, dim)
    q, k, v = qkv.cuda().split([8, 2, 2], 1)
    slots = torch.randperm(96, generator=torch.Generator().manual_seed(1))[:tokens]
    got = ops().rotary_cache_write(q, k, v, positions.cuda(), table, cache, slots.cuda(), interleaved, norm.cuda(), norm.cuda())
    xq, xk, xv = qkv.split([8, 2, 2], 1)
    close_rows(got, turned(xq, positions, table.cpu(), interleaved, norm, 1e-6), dtype)
    want = turned(xk, positions, table.cpu(), interleaved, norm, 1e-6)
    back, back_v = ops().cache_read(cache, slots.cuda(), dtype)
    if kind == "same":
        close_rows(back, want, dtype)
        assert torch.equal(back_v.cpu(), xv)
    else:
        # half a step of the code, the value's own rounding
        for y, x in ((back, want), (back_v, xv.double())):
            top = x.abs().amax(-1, keepdim=True)
            half = top / 254 if kind == "int8" else (x.abs() * 2.0 ** -4).clamp_min(top / 448 * 2.0 ** -10)
            assert bool(((y.double().cpu() - x).abs() <= 1.01 * half + U[dtype] * x.abs()).all())


# --- attention --------------------------------------------------------------------------------------------------------------------

class Batch:
    """Sequences of (new tokens, tokens of the context), their cache in pages of any order with NaN wherever no token lies, and the answer."""

    def __init__(self, lengths, heads=4, kv_heads=2, dim=128, page=16, kind="same", dtype=torch.float16, padding=0, seed=0, tokens_first=False, big=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.heads, self.kv_heads, self.dim, self.page, self.kind, self.dtype = lengths, heads, kv_heads, dim, page, kind, dtype
        need = [-(-kv // page) for _, kv in lengths]
        n_pages = sum(need) + 2
        self.cache = empty_cache(kind, dtype, n_pages, kv_heads, page, dim, tokens_first)
        order = torch.randperm(n_pages, generator=g)
        self.width = max(need, default=0) + 1
        self.pages = torch.full((len(lengths), self.width), 2 ** 31 - 1, dtype=torch.int32)      # (entries behind the last page are not read)
        at, self.k, self.v = 0, [], []
        for b, (_, kv) in enumerate(lengths):
            self.pages[b, :need[b]] = order[at:at + need[b]].to(torch.int32)
            at += need[b]
            k, v = (torch.randn((kv, kv_heads, dim), generator=g) * big for _ in range(2))
            place = self.slots(b, torch.arange(kv))
            ops().cache_write(self.cache, k.to(dtype).cuda(), v.to(dtype).cuda(), place)
            # what the cache holds, from its own codes
            for keep, raw, scale in ((self.k, self.cache.k, self.cache.k_scale), (self.v, self.cache.v, self.cache.v_scale)):
                x = rows_of(raw, page)[place.cpu()].double()
                keep.append(x if scale is None else x * rows_of(scale, page)[place.cpu()].double()[..., None])
        self.starts = [0]
        for n, _ in lengths:
            self.starts.append(self.starts[-1] + n)
        self.q = (torch.randn((self.starts[-1] + padding, heads, dim), generator=g) * 2).to(dtype)

    def slots(self, b, tokens):
        return (self.pages[b, tokens // self.page].long() * self.page + tokens % self.page).cuda()

    def inputs(self):
        return (self.q.cuda(), self.cache, self.pages.cuda(), torch.tensor(self.starts, dtype=torch.int32).cuda(),
                torch.tensor([kv for _, kv in self.lengths], dtype=torch.int32).cuda())

    def answer(self, causal=True, window=0, scale=None):
        """(outputs, sum(p |v|), max |v|) in 64 bits."""
        scale = self.dim ** -0.5 if scale is None else scale
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        size, most = torch.zeros_like(out), torch.zeros(out.shape[:2] + (1,), dtype=torch.float64)
        group = self.heads // self.kv_heads
        for b, (n, kv) in enumerate(self.lengths):
            if not n or not kv:
                continue
            q = self.q[self.starts[b]:self.starts[b + 1]].double()
            k, v = (x[b].repeat_interleave(group, 1) for x in (self.k, self.v))
            score = torch.einsum("thd,shd->hts", q, k) * scale
            position, token = torch.arange(kv - n, kv)[:, None], torch.arange(kv)
            seen = torch.ones(n, kv, dtype=torch.bool)
            if causal:
                seen = token <= position
            if window:
                seen = seen & (token > position - window)
            score = score.masked_fill(~seen, -math.inf)
            p = torch.nan_to_num(torch.softmax(score, -1)) if not score.isnan().any() else torch.softmax(score, -1)
            p = torch.where(seen.any(-1)[:, None], p, 0.0)
            rows = slice(self.starts[b], self.starts[b + 1])
            out[rows] = torch.einsum("hts,shd->thd", p, v)
            size[rows] = torch.einsum("hts,shd->thd", p, v.abs())
            most[rows] = kv * v.abs().max()
        return out, size, most

    def check(self, got, **how):
        want, size, most = self.answer(**how)
        bound = (2 * U[self.dtype] + 2.0 ** -13) * size + 2.0 ** -24 * most + 1e-30
        got = got.double().cpu()
        assert got.shape == want.shape
        worst = ((got - want).abs() / bound).max() if want.numel() else 0
        assert bool(((got - want).abs() <= bound).all()), f"{float(worst):.3f} of the bound"


DECODES = [(1, 1), (1, 15), (1, 16), (1, 17), (1, 300), (1, 64), (1, 2050)]
CHUNKS = [(5, 5), (1, 40), (70, 70), (64, 128), (33, 500), (200, 263), (129, 129)]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,page", [(4, 4, 16), (8, 2, 32), (20, 1, 64), (3, 1, 128)])
@pytest.mark.parametrize("lengths", [DECODES, CHUNKS], ids=["decodes", "chunks"])
def test_attention(kind, dtype, dim, heads, kv_heads, page, lengths):
    batch = Batch(lengths, heads, kv_heads, dim, page, kind, dtype)
    most = max(n for n, _ in lengths)
    batch.check(ops().paged_attention(*batch.inputs(), max_q=most))
    batch.check(ops().paged_attention(*batch.inputs(), max_q=most, causal=False, scale=0.2), causal=False, scale=0.2)
    for window in (1, 50, 128):
        batch.check(ops().paged_attention(*batch.inputs(), max_q=most, window=window), window=window)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("most", [None, 1, 2, 7, 100000])
def test_the_largest_number_of_new_tokens_is_a_hint(kind, most):
    batch = Batch(CHUNKS, 8, 2, 128, 16, kind)
    batch.check(ops().paged_attention(*batch.inputs(), max_q=most))


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("most", [1, None])
def test_the_scale_of_a_value_that_is_masked_changes_no_bit(kind, dtype, most):
    for n, kv, heads, kv_heads, at in ((6, 40, 4, 2, 37), (20, 300, 8, 1, 290), (100, 150, 2, 2, 120), (1, 70, 2, 1, 10)):
        window = 20 if n == 1 else 0
        batch = Batch([(n, kv)], heads, kv_heads, 64, 16, kind, dtype)
        clean = ops().paged_attention(*batch.inputs(), max_q=most, window=window)
        page, slot = divmod(int(batch.slots(0, torch.tensor([at]))), 16)
        batch.cache.v_scale[page, :, slot] *= 2.0 ** 14
        got = ops().paged_attention(*batch.inputs(), max_q=most, window=window)
        first = kv - n
        sees = torch.tensor([first + t >= at and (not window or at > first + t - window) for t in range(n)])
        assert torch.equal(got[~sees.cuda()], clean[~sees.cuda()])


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("most", [1, None])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30])
def test_windows_longer_than_any_context(kind, most, window):
    batch = Batch([(1, 300), (6, 2), (200, 30), (40, 0), (129, 263)], 6, 2, 64, 16, kind)
    batch.check(ops().paged_attention(*batch.inputs(), max_q=most, window=window), window=window)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("most", [1, None])
def test_sequences_of_nothing(kind, most):
    """No new tokens, no context, new tokens that reach back ahead of the first token of the context, padding behind the last sequence."""
    batch = Batch([(0, 0), (1, 0), (0, 50), (1, 7), (6, 2), (40, 0), (200, 30), (0, 0)], 6, 2, 64, 16, kind, padding=21)
    for how in ({}, {"window": 3}, {"causal": False}):
        batch.check(ops().paged_attention(*batch.inputs(), max_q=most, **how), **how)
    none = Batch([], padding=3)
    assert not ops().paged_attention(*none.inputs()).any()
    empty = Batch([(0, 5)])
    assert ops().paged_attention(*empty.inputs()).shape == (0, 4, 128)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("lengths", [[(1, 9000), (1, 3), (2, 7777)], [(3, 20000), (40, 5000)], [(150, 9001), (1, 12345), (1, 64)]])
def test_contexts_that_are_cut_into_shares(kind, lengths):
    batch = Batch(lengths, 4, 1, 128, 64, kind, torch.bfloat16)
    most = max(n for n, _ in lengths)
    for how in ({}, {"window": 4000}, {"causal": False}):
        batch.check(ops().paged_attention(*batch.inputs(), max_q=most, **how), **how)


@pytest.mark.parametrize("kind", ["same", "fp8"])
@pytest.mark.parametrize("most", [1, None])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_is_masked_is_not_seen_whatever_it_holds(kind, most, bad):
    """A key or value that is no number reaches the rows that see its token and no other."""
    for n, kv, heads, kv_heads, at in ((6, 40, 4, 2, 37), (100, 150, 2, 2, 120), (1, 70, 2, 1, 10)):
        window = 20 if n == 1 else 0
        batch = Batch([(n, kv)], heads, kv_heads, 64, 16, kind)
        clean = ops().paged_attention(*batch.inputs(), max_q=most, window=window)
        page, slot = divmod(int(batch.slots(0, torch.tensor([at]))), 16)
        if kind == "same":
            batch.cache.v[page, :, slot, 5] = bad
            batch.cache.k[page, :, slot, 7] = math.nan
        else:
            batch.cache.v.view(torch.uint8)[page, :, slot, 5] = 0x7F
            batch.cache.k_scale[page, :, slot] = math.nan
        got = ops().paged_attention(*batch.inputs(), max_q=most, window=window)
        first = kv - n
        sees = torch.tensor([first + t >= at and (not window or at > first + t - window) for t in range(n)])
        assert torch.equal(got[~sees.cuda()], clean[~sees.cuda()])
        assert got[sees.cuda()].isnan().all()
    # values alone: the rows that see them get what they add up to
    batch = Batch([(100, 150)], 2, 2, 64, 16, "same")
    clean = ops().paged_attention(*batch.inputs(), max_q=most)
    for token, what in ((60, math.inf), (120, bad), (120, math.inf)):
        page, slot = divmod(int(batch.slots(0, torch.tensor([token]))), 16)
        batch.cache.v[page, :, slot, 11 if token == 120 else 12] = what
        got = ops().paged_attention(*batch.inputs(), max_q=most)
        column = got[:, :, 11 if token == 120 else 12]
        sees = (torch.arange(50, 150) >= token).cuda()
        assert torch.equal(column[~sees], clean[:, :, 11 if token == 120 else 12][~sees])
        assert bool((column[sees].isnan() if math.isnan(what) else column[sees] == what).all())
        rest = torch.ones(64, dtype=torch.bool)
        rest[11], rest[12] = False, False
        assert torch.equal(got[..., rest.cuda()], clean[..., rest.cuda()])


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", HALF)
def test_scores_and_values_of_any_size(kind, dtype):
    """Scores hundreds apart, a maximum that comes last, values near the ends of the types."""
    batch = Batch([(1, 700), (3, 333), (90, 400)], 4, 2, 128, 16, kind, dtype, big=8.0)
    batch.check(ops().paged_attention(*batch.inputs(), scale=3.0), scale=3.0)
    for big in (1e-4, 2000.0):
        batch = Batch([(1, 700), (3, 333), (90, 400)], 4, 2, 64, 16, kind, dtype, big=big)
        want, size, most = batch.answer(scale=1e-3 / big)
        got = ops().paged_attention(*batch.inputs(), scale=1e-3 / big).double().cpu()
        bound = (2 * U[dtype] + 2.0 ** -13) * size + 2.0 ** -24 * most + (2.0 ** -25 if dtype == torch.float16 else 0)   # (an fp16 output below its normal range)
        assert bool(((got - want).abs() <= bound).all())


def test_other_layouts_and_streams():
    batch = Batch([(1, 100), (9, 77), (130, 200)], 6, 3, 128, 32, tokens_first=True, padding=2)
    q, cache, pages, starts, lens = batch.inputs()
    plain = ops().paged_attention(q, cache, pages, starts, lens)
    batch.check(plain)
    wide = torch.zeros(q.shape[0], 12, 128, dtype=q.dtype, device="cuda")
    wide[:, 3:9] = q
    odd = torch.zeros(q.numel() + 1, dtype=q.dtype, device="cuda")
    odd[1:] = q.flatten()
    table = torch.full((3, batch.width + 5), -1, dtype=torch.int32, device="cuda")
    table[:, 2:2 + batch.width] = pages
    for one in (wide[:, 3:9], odd[1:].view(q.shape), q.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(ops().paged_attention(one, cache, table[:, 2:2 + batch.width], starts, lens), plain)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        again = ops().paged_attention(q, cache, pages, starts, lens)
    side.synchronize()
    assert torch.equal(again, plain)


def test_a_plan_serves_every_layer_and_repeats_its_bits():
    batch = Batch([(1, 5000), (70, 300), (1, 90)], 4, 2, 128, 16, "int8")
    q, cache, pages, starts, lens = batch.inputs()
    plan = ops().attention_plan(cache, starts, lens, n_heads=4, n_tokens=q.shape[0], max_q=70)
    first = ops().paged_attention(q, cache, pages, starts, lens, plan=plan)
    batch.check(first)
    for _ in range(3):
        assert torch.equal(ops().paged_attention(q, cache, pages, starts, lens, plan=plan), first)
    with pytest.raises(RuntimeError, match="plan is for"):
        ops().paged_attention(q, cache, pages, starts, lens, plan=plan, causal=False)
    with pytest.raises(RuntimeError, match="plan is for"):
        ops().paged_attention(q[1:], cache, pages, starts, lens, plan=plan)


def test_a_step_in_a_graph():
    """Positions, write, plan and attention recorded once and replayed on other tokens, lengths and pages, with work between the replays."""
    heads, kv_heads, dim, page, seqs = 8, 2, 128, 16, 5
    cache = ops().paged_cache(60, kv_heads, dim, page, torch.int8)
    table = ops().rotary_table(500, dim)
    qkv = torch.zeros(seqs, heads + 2 * kv_heads, dim, dtype=torch.float16, device="cuda")
    positions, slots, lens = (torch.zeros(seqs, dtype=torch.int32, device="cuda") for _ in range(3))
    pages = torch.arange(60, dtype=torch.int32, device="cuda").view(seqs, 12)
    starts = torch.arange(seqs + 1, dtype=torch.int32, device="cuda")

    def step():
        q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
        q = ops().rotary_cache_write(q, k, v, positions, table, cache, slots)
        return ops().paged_attention(q, cache, pages, starts, lens, max_q=1)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(6):
        qkv.copy_(randn(*qkv.shape, seed=i))
        at = torch.tensor([i, 3 * i + 1, 20, 150 + i, 7]).cuda()
        positions.copy_(at)
        slots.copy_(pages.gather(1, (at // page).long()[:, None])[:, 0] * page + at % page)
        lens.copy_(at + 1)
        graph.replay()
        got = out.clone()
        codes = cache.k.clone()
        assert torch.equal(got, step()) and torch.equal(cache.k, codes)
        torch.cuda.synchronize()


def test_offsets_that_pass_32_bits():
    """Pages whose bytes lie beyond 2^32 from the cache's first, in 8 and 16 bits."""
    for dtype, held, n_pages in ((torch.float16, torch.float16, 40000), (torch.float16, torch.float8_e4m3fn, 70000)):
        kv_heads, dim, page = 8, 128, 64
        k, v = (torch.empty((n_pages, kv_heads, page, dim), dtype=held, device="cuda") for _ in range(2))
        assert k.numel() * k.element_size() > 2 ** 32
        scales = [] if held == dtype else [torch.empty((n_pages, kv_heads, page), device="cuda") for _ in range(2)]
        cache = ops().PagedCache(k, v, *scales)
        for lengths in ([(1, 300), (1, 190)], [(100, 300), (30, 190)]):
            batch = Batch(lengths, 16, kv_heads, dim, page, "same", dtype)
            far = batch.pages.clone()
            for b, (_, kv) in enumerate(lengths):
                for j in range(-(-kv // page)):
                    far[b, j] = n_pages - 1 - 7 * j - 50 * b
                    inside = torch.arange(j * page, min(kv, (j + 1) * page))
                    ops().cache_write(cache, batch.k[b][inside].to(dtype).cuda(), batch.v[b][inside].to(dtype).cuda(), int(far[b, j]) * page + (inside % page).cuda())
                place = far[b, torch.arange(kv) // page].long() * page + torch.arange(kv) % page
                for keep, back in zip((batch.k, batch.v), ops().cache_read(cache, place.cuda(), torch.float16)):
                    if held == dtype:
                        assert torch.equal(back.double().cpu(), keep[b])
                # (of codes: what the cache holds, in 32 bits)
                if held != dtype:
                    for keep, raw, scale in ((batch.k, k, cache.k_scale), (batch.v, v, cache.v_scale)):
                        at_page, at_slot = place.cuda() // page, place.cuda() % page
                        keep[b] = (raw.view(torch.uint8)[at_page, :, at_slot].view(held).double() * scale[at_page, :, at_slot].double()[..., None]).cpu()
            q, _, _, starts, lens = batch.inputs()
            batch.check(ops().paged_attention(q, cache, far.cuda(), starts, lens))
        del k, v, cache, scales


def test_lengths_and_tables_that_make_no_sense_stay_inside():
    """Offsets that do not ascend or pass the tokens, lengths beyond the table, pages that the cache does not have: some numbers, no access out of bounds."""
    batch = Batch([(1, 40), (9, 77), (130, 200)], 6, 3, 64, 16)
    q, cache, pages, starts, lens = batch.inputs()
    for s in ([0, 500, -3, 140], [0, 140, 0, 140], [-7, 1, 2, 10 ** 9]):
        out = ops().paged_attention(q, cache, pages, torch.tensor(s, dtype=torch.int32).cuda(), lens)
        torch.cuda.synchronize()
        assert out.shape == q.shape
    ops().paged_attention(q, cache, torch.full_like(pages, -5), starts, lens + 10000)
    ops().paged_attention(q, cache, pages, starts, lens - 10000)
    torch.cuda.synchronize()
    batch.check(ops().paged_attention(*batch.inputs()))


# --- refusals ---------------------------------------------------------------------------------------------------------------------

def test_refusals():
    half = dict(dtype=torch.float16, device="cuda")
    table, x = ops().rotary_table(10, 64), torch.zeros(3, 2, 64, **half)
    positions = torch.zeros(3, dtype=torch.int32, device="cuda")
    cache = ops().paged_cache(4, 2, 64, page=16)
    cases = [
        ("GPU tensor", lambda: ops().rotary(x.cpu(), x, positions, table)),
        ("fp16|float16", lambda: ops().rotary(x.float(), x, positions, table)),
        ("expected 3 tokens", lambda: ops().rotary(x[:2], x, positions, table)),
        ("int32 or torch.int64", lambda: ops().rotary(x, x, positions.float(), table)),
        ("each of 3 tokens", lambda: ops().rotary(x, x, positions[:2], table)),
        ("contiguous float32", lambda: ops().rotary(x, x, positions, table.half())),
        ("rotates 64 of 32", lambda: ops().rotary(x[..., :32], x[..., :32], positions, table)),
        ("multiple of 16", lambda: ops().rotary_table(10, 24)),
        ("unknown scaling", lambda: ops().rotary_table(10, 64, scaling={"type": "other"})),
        ("unknown settings", lambda: ops().rotary_table(10, 64, scaling={"type": "linear", "factor": 2.0, "beta": 1})),
        ("q_norm must be", lambda: ops().rotary(x, x, positions, table, q_norm=torch.ones(32, **half))),
        ("requires a gradient", lambda: ops().rotary(x.clone().requires_grad_(), x, positions, table)),
        ("elements: a multiple of 8", lambda: ops().rotary(torch.zeros(3, 2, 272, **half), torch.zeros(3, 2, 272, **half), positions, table)),
        ("does not go with", lambda: ops().cache_write(cache, x.bfloat16(), x.bfloat16(), positions)),
        ("expected \\[tokens, 2, 64\\]", lambda: ops().cache_write(cache, x[:, :1], x[:, :1], positions)),
        ("does not go with", lambda: ops().cache_read(cache, positions, torch.bfloat16)),
        ("does not go with", lambda: ops().cache_read(ops().paged_cache(4, 2, 64, dtype=torch.int8), positions, torch.float32)),
        ("pages of 16", lambda: ops().paged_cache(4, 2, 64, page=24)),
        ("belongs to caches of 8 bits", lambda: ops().PagedCache(cache.k.to(torch.int8), cache.v.to(torch.int8))),
        ("holds fp16", lambda: ops().PagedCache(cache.k.float(), cache.v.float())),
        ("adjacent elements", lambda: ops().PagedCache(cache.k.transpose(2, 3).contiguous().transpose(2, 3), cache.v)),
        ("n_pages, kv_heads", lambda: ops().PagedCache(cache.k, cache.v[:2])),
    ]
    q, pages = torch.zeros(3, 4, 64, **half), torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    starts, lens = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda"), torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    attend = ops().paged_attention
    odd = ops().paged_cache(4, 2, 96, page=16)
    cases += [
        ("multiple, up to 1024", lambda: attend(torch.zeros(3, 5, 64, **half), cache, pages, starts, lens)),
        ("64 or 128", lambda: attend(torch.zeros(3, 4, 96, **half), odd, pages, starts, lens)),
        ("expected \\[tokens, 4, 64\\]", lambda: attend(torch.zeros(3, 4, 128, **half), cache, pages, starts, lens)),
        ("does not go with", lambda: attend(q.bfloat16(), cache, pages, starts, lens)),
        ("int32 \\[2, pages", lambda: attend(q, cache, pages.long(), starts, lens)),
        ("int32 \\[2, pages", lambda: attend(q, cache, pages[:1], starts, lens)),
        ("contiguous vector", lambda: attend(q, cache, pages, starts.long(), lens)),
        ("must have 3 entries", lambda: attend(q, cache, pages, starts[:2], lens)),
        ("positive number", lambda: attend(q, cache, pages, starts, lens, scale=-1.0)),
        ("window needs causal", lambda: attend(q, cache, pages, starts, lens, causal=False, window=4)),
        ("window -1", lambda: attend(q, cache, pages, starts, lens, window=-1)),
        ("column at least", lambda: attend(q, cache, pages[:, :0], starts, lens)),
        ("up to 4096 sequences", lambda: attend(q, cache, torch.zeros(5000, 1, dtype=torch.int32, device="cuda"), torch.zeros(5001, dtype=torch.int32, device="cuda"),
                                                 torch.zeros(5000, dtype=torch.int32, device="cuda"))),
    ]
    for text, call in cases:
        with pytest.raises(RuntimeError, match=text):
            call()
    with pytest.raises(TypeError):
        ops().rotary([1.0], x, positions, table)
    torch.cuda.synchronize()
