"""The base weight in 8 bits: quantiser, read-back and product against their formulas.

Bounds.  Scales and codes are what 32-bit divisions and the nearest code give: no difference.  The matrix instruction adds the products of eight adjacent codes in
fixed point: measured on the instruction, a product keeps its bits down to 2^-13 of the largest of the eight and loses those below, so each of the seven others is off
by less than 2^-13 of that, together 7 2^-13 of the largest.  Those sums, 16 of a block, then the blocks are added in 32 bits, each addition off by 2^-23 of the sum of
magnitudes at most, the two roundings of a block's scales among them; the result is rounded once.  With u the unit roundoff of the output's type:
7 2^-13 sum(largest of eight |x w|) + (16 + blocks + 2) 2^-23 sum(|x w|) + u |y|, and half of fp16's least number."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
HALF = [torch.float16, torch.bfloat16]
E4M3 = torch.float8_e4m3fn


def ops():
    from triteia_amd.python import ops
    return ops


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def spread(scales, rows, n, k):
    return scales.repeat_interleave(rows, 0)[:n].repeat_interleave(128, 1)[:, :k]


def quantised(x, rows):
    """On the CPU, whose divisions are rounded to nearest."""
    n, k = x.shape
    padded = torch.nn.functional.pad(x.float(), (0, -k % 128, 0, -n % rows))
    top = padded.view(-1, rows, padded.shape[1] // 128, 128).abs().amax((1, 3))
    strange = ~top.isfinite()
    scale = torch.where(top < 1e-30, 0.0, top / 448.0)
    y = (x.float() / spread(torch.where(scale > 0, scale, 1.0), rows, n, k)).clamp(-448, 448).to(E4M3)
    y = torch.where(spread(strange, rows, n, k), 0.0, y.float()).to(E4M3)
    return y, torch.where(strange, math.nan, scale)


def same(a, b):
    a, b = (t.cpu().float() for t in (a, b))
    return a.shape == b.shape and torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def values(codes, scales, rows):
    return codes.double() * spread(scales.double(), rows, *codes.shape)


def largest(x, w):
    """For every token and feature, the largest product of each eight, added up.  x [tokens, k], w [m, k] in 64 bits."""
    x, w = (t.abs().float().cuda().view(t.shape[0], -1, 8) for t in (x, w))
    out = torch.zeros(x.shape[0], w.shape[0], device="cuda")
    step = max(1, (1 << 28) // (x.shape[0] * w.shape[0] * 8))
    for i in range(0, x.shape[1], step):
        out += (x[:, None, i:i + step] * w[None, :, i:i + step]).amax(-1).sum(-1)
    return out.double()


def close(got, x, w, dtype):
    """x, w: the values in 64 bits, on any device.  Of large products a part."""
    assert got.dtype == dtype and got.shape == (x.shape[0], w.shape[0])
    g = torch.Generator().manual_seed(1)
    rows = torch.randperm(x.shape[0], generator=g)[:128].sort().values
    columns = torch.randperm(w.shape[0], generator=g)[:max(512, (1 << 31) // (len(rows) * x.shape[1]))].sort().values
    got, x, w = got.cuda()[rows.cuda()][:, columns.cuda()].double(), x.cuda()[rows.cuda()], w.cuda()[columns.cuda()]
    want, most = x @ w.t(), x.abs() @ w.abs().t()
    bound = 7 * 2.0 ** -13 * largest(x, w) + (16 + -(-x.shape[1] // 128) + 2) * 2.0 ** -23 * most + U[dtype] * want.abs() + 2.0 ** -25
    off = (got - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


# --- quantiser -------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("n,k", [(1, 16), (1, 4096), (3, 128), (13, 4096), (17, 144), (128, 256), (129, 48), (300, 2000), (1000, 1040), (2500, 1168)])
@pytest.mark.parametrize("dtype", HALF)
def test_quantise_and_back(rows, n, k, dtype):
    x = (randn(n, k, seed=n + k) * torch.exp(2 * randn(k, seed=1))).to(dtype)
    codes, scales = ops().quantize_fp8(x.cuda(), rows=rows)
    want, want_scales = quantised(x, rows)
    assert codes.dtype == E4M3 and same(scales, want_scales) and same(codes, want)
    for out in (torch.float16, torch.bfloat16, torch.float32):
        back = ops().dequantize_fp8(codes, scales, dtype=out)
        assert back.dtype == out and same(back, (want.float() * spread(want_scales, rows, n, k)).to(out))


@pytest.mark.parametrize("rows", [1, 128])
def test_quantise_blocks_without_numbers(rows):
    x = randn(260, 400, seed=3, dtype=torch.bfloat16)
    x[:2, :128] = 0
    x[128:256, 128:256] = 0                                  # a whole tile of zeros
    x[3, 130], x[130, 5], x[257, 399], x[4, 0] = math.inf, math.nan, -math.inf, 1e-36
    x[5, :128] = 1e-35
    codes, scales = ops().quantize_fp8(x.cuda(), rows=rows)
    want, want_scales = quantised(x, rows)
    assert same(scales, want_scales) and same(codes, want)
    assert same(ops().dequantize_fp8(codes, scales, dtype=torch.float32), want.float() * spread(want_scales, rows, 260, 400))


def test_quantise_the_ends_of_the_types():
    for dtype in HALF:
        info = torch.finfo(dtype)
        x = torch.tensor([[info.max, -info.max, info.tiny, 1.0] * 4, [info.tiny] * 16, [info.smallest_normal / 4] * 16, [448.0, 447.0, 17.0, 0.1171875] * 4]).to(dtype)
        for rows in (1, 128):
            assert all(same(a, b) for a, b in zip(ops().quantize_fp8(x.cuda(), rows=rows), quantised(x, rows)))


def test_quantise_layouts():
    x = randn(40, 512, seed=4, dtype=torch.float16).cuda()
    want = [t.float() for t in ops().quantize_fp8(x[:, 128:384].contiguous())]
    flat = torch.zeros(40 * 256 + 3, dtype=torch.float16, device="cuda")
    flat[3:] = x[:, 128:384].flatten()
    for view in (x[:, 128:384], flat[3:].view(40, 256), x[:, 128:384].t().contiguous().t(), torch._neg_view(-x[:, 128:384])):
        assert all(torch.equal(a.float(), b) for a, b in zip(ops().quantize_fp8(view), want))
    one = x[:1, :256].expand(40, 256)                        # rows that are one row
    codes, scales = ops().quantize_fp8(one)
    assert torch.equal(codes.float(), ops().quantize_fp8(one.contiguous())[0].float()) and scales.shape == (40, 2)
    back = ops().dequantize_fp8(codes, scales.contiguous())
    assert torch.equal(back, ops().dequantize_fp8(codes, scales)) and torch.equal(back, ops().dequantize_fp8(codes.t().contiguous().t(), scales))


def test_quantise_nothing():
    for rows in (1, 128):
        codes, scales = ops().quantize_fp8(torch.zeros(0, 256, dtype=torch.float16, device="cuda"), rows=rows)
        assert codes.shape == (0, 256) and scales.shape == (0, 2)
        assert ops().dequantize_fp8(codes, scales).shape == (0, 256)


# --- product ---------------------------------------------------------------------------------------------------------------------

def weight(m, k, seed=0):
    """Blocks of sizes of their own, so that a scale in the wrong place shows."""
    w = randn(m, k, seed=seed) * torch.exp(randn(-(-m // 128), -(-k // 128), seed=seed + 1)).repeat_interleave(128, 0)[:m].repeat_interleave(128, 1)[:, :k]
    codes, scales = quantised(w.half(), 128)
    return codes, scales


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 33, 63, 64, 65, 100, 130, 300])
@pytest.mark.parametrize("k,m", [(16, 16), (48, 1), (128, 128), (144, 3), (256, 129), (2000, 1001), (4096, 640), (1040, 2050)])
def test_product(tokens, k, m):
    x = (randn(tokens, k, seed=tokens) * torch.exp(randn(k, seed=5)) * torch.exp(randn(tokens, 1, seed=6))).half()
    w, ws = weight(m, k, seed=k + m)
    x8, xs = quantised(x, 1)
    xv, wv = values(x8, xs, 1), values(w, ws, 128)
    wg, wsg = w.cuda(), ws.cuda()
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        close(ops().matmul_fp8(x.cuda(), wg, wsg, dtype=dtype).cpu(), xv, wv, dtype)
        close(ops().matmul_fp8(x8.cuda(), wg, wsg, x_scale=xs.cuda(), dtype=dtype).cpu(), xv, wv, dtype)
    xb = x.bfloat16()
    x8, xs = quantised(xb, 1)
    close(ops().matmul_fp8(xb.cuda(), wg, wsg).cpu(), values(x8, xs, 1), wv, torch.bfloat16)


@pytest.mark.parametrize("tokens,k,m", [(1, 8192, 8192), (5, 28672, 512), (16, 4096, 11008), (64, 11008, 4096), (200, 8192, 1024), (513, 2048, 5000), (1000, 4096, 1408),
                                        (2049, 1024, 4097), (4000, 2064, 2560)])
def test_product_of_real_sizes(tokens, k, m):
    x = randn(tokens, k, seed=1).bfloat16().cuda()
    w, ws = ops().quantize_fp8(0.02 * torch.randn(m, k, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).half(), rows=128)
    x8, xs = ops().quantize_fp8(x)
    xv, wv = values(x8, xs, 1), values(w, ws, 128)
    for dtype in (torch.bfloat16, torch.float32):
        close(ops().matmul_fp8(x, w, ws, dtype=dtype), xv, wv, dtype)
    assert torch.equal(ops().matmul_fp8(x8, w, ws, x_scale=xs, dtype=torch.bfloat16), ops().matmul_fp8(x, w, ws))      # the same codes, the same sums


def sizes_of_every_tile():
    """For each tile, whole and in shares of K, the smallest of a grid of ragged sizes that are multiplied on it."""
    from triteia_amd.python.capi import _ffi
    found = {}
    for tokens in (1, 15, 17, 31, 33, 47, 61, 67, 97, 131, 193, 259, 389, 515, 771, 1027, 2051):
        for k in (272, 1040, 2000, 4112, 8208, 11024):
            for m in (131, 515, 1001, 2050, 4097, 8199, 11012, 20004):
                tile = _ffi.lib().triteia_hip_fp8_tile(tokens, m, k)
                key = (tile % 10 ** 6, tile >= 2 * 10 ** 6)
                if key not in found or tokens * k * m < found[key][0]:
                    found[key] = (tokens * k * m, (tokens, k, m))
    return {key: size for key, (_, size) in sorted(found.items())}


@pytest.mark.parametrize("tile", [16016, 32016, 32032, 128016, 128032, 64064, 128064, 128096, 128128, 128160, 256096, 256128, 256192, 256224, 256256])
def test_every_tile(tile):
    sizes = [size for key, size in sizes_of_every_tile().items() if key[0] == tile]
    assert sizes
    for tokens, k, m in sizes:
        x = (randn(tokens, k, seed=1) * torch.exp(randn(tokens, 1, seed=2))).half().cuda()
        w, ws = (t.cuda() for t in weight(m, k, seed=3))
        x8, xs = ops().quantize_fp8(x)
        xv, wv = values(x8, xs, 1), values(w, ws, 128)
        for dtype in (torch.float16, torch.bfloat16, torch.float32):
            close(ops().matmul_fp8(x, w, ws, dtype=dtype), xv, wv, dtype)
        twice = [ops().matmul_fp8(x8, w, ws, x_scale=by, dtype=torch.float32) for by in (xs, xs.contiguous())]
        assert torch.equal(*twice)


@pytest.mark.parametrize("tile", [16016, 32016, 32032, 128016, 128032, 64064, 128064, 128096, 128128, 128160, 256096, 256128, 256192, 256224, 256256])
def test_every_tile_adds_every_product(tile):
    """Whole numbers of -8 to 8 under scales of powers of two that change from block to block: products of up to 64, whole, lie within the 13 bits that the instruction keeps, and sums of up to 11024 of them
    times 4, in quarters, within 24.  So every sum is exact, and one product left out, taken twice or under another block's scale shows in its element.

    And random codes in norm: of eight products seven are off by less than 2^-13 of the largest, each with a sign of its own: sqrt(7 / 3) 2^-13 of it in the mean, whose square is at most the sum
    of all eight's, so the result is off by that part of its norm, below 2^-12.  One product in 4096 left out everywhere is 2^-6."""
    for tokens, k, m in [size for key, size in sizes_of_every_tile().items() if key[0] == tile]:
        g = torch.Generator("cuda").manual_seed(tokens + k + m)
        pick = lambda lo, hi, *shape: torch.randint(lo, hi + 1, shape, generator=g, device="cuda").float()  # noqa: E731
        blocks = -(-k // 128)
        x, w = pick(-8, 8, tokens, k).to(E4M3), pick(-8, 8, m, k).to(E4M3)
        xs, ws = torch.exp2(pick(-1, 1, tokens, blocks)), torch.exp2(pick(-1, 1, -(-m // 128), blocks))
        want = values(x, xs, 1) @ values(w, ws, 128).t()
        assert torch.equal(want, want.float().double()) and torch.equal(ops().matmul_fp8(x, w, ws, x_scale=xs, dtype=torch.float32).double(), want)
        for dtype in HALF:
            assert torch.equal(ops().matmul_fp8(x, w, ws, x_scale=xs, dtype=dtype), want.float().to(dtype))
        x, xs = ops().quantize_fp8(torch.randn(tokens, k, generator=g, device="cuda").half())
        w, ws = ops().quantize_fp8(torch.randn(m, k, generator=g, device="cuda").half(), rows=128)
        want = values(x, xs, 1) @ values(w, ws, 128).t()
        off = (ops().matmul_fp8(x, w, ws, x_scale=xs, dtype=torch.float32).double() - want).norm() / want.norm()
        assert float(off) <= 2.0 ** -12, (tokens, k, m, float(off))


@pytest.mark.parametrize("tokens", [1, 40])
def test_what_cancels_in_eight_products(tokens):
    """Small products beside large ones that cancel: kept to 2^-13 of the largest in its eight, and whole in another."""
    one, w, x = torch.ones(1, 1, device="cuda"), torch.zeros(16, 128, device="cuda"), torch.zeros(tokens, 128, device="cuda")
    x[:, 8:10], w[:, 8], w[:, 9] = 448.0, 448.0, -448.0
    for a, b in ((2.0, 2.0), (3.0, 4.0), (15.0, 15.0), (0.25, 0.5), (-7.0, 8.0)):
        for place, bound in ((10, 2.0 ** -13 * 448 * 448), (15, 2.0 ** -13 * 448 * 448), (7, 0.0), (16, 0.0), (127, 0.0)):
            near_x, near_w = x.clone(), w.clone()
            near_x[:, place], near_w[:, place] = a, b
            got = ops().matmul_fp8(near_x.to(E4M3), near_w.to(E4M3), one, x_scale=one.expand(tokens, 1), dtype=torch.float32)
            assert bool(((got - a * b).abs() <= bound).all()), (a, b, place, got[0, 0])


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("tokens", [1, 3, 4, 5, 8])
def test_few_tokens_quantised_on_the_way(tokens, dtype):
    """The bits of the quantiser and the product apart, for any K, values that are no numbers and views among the inputs."""
    from triteia_amd.python.capi import _ffi
    for k, m in ((16, 16), (48, 40), (128, 1000), (144, 129), (1040, 3001), (2000, 515), (4096, 4096), (11024, 1027)):
        x = (randn(tokens, k, seed=k) * torch.exp(2 * randn(k, seed=1))).to(dtype).cuda()
        w, ws = (t.cuda() for t in weight(m, k, seed=4))
        if tokens <= 4 and _ffi.lib().triteia_hip_fp8_tile(tokens, m, k) == 1016016:
            assert _ffi.lib().triteia_hip_fp8_scratch_bytes(tokens, m, k, 0) == 0
        for bad in (None, math.inf, math.nan):
            if bad is not None:
                x[tokens // 2, k - 1] = bad
                x[0, :min(k, 128)] = 0
            x8, xs = ops().quantize_fp8(x)
            want = ops().matmul_fp8(x8, w, ws, x_scale=xs, dtype=torch.float32)
            wide = torch.full((tokens + 1, k + 200), math.nan, dtype=dtype, device="cuda")
            wide[:tokens, 72:72 + k] = x
            for view in (x, wide[:tokens, 72:72 + k], x.clone()):
                got = ops().matmul_fp8(view, w, ws, dtype=torch.float32)
                assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_shares_of_k_are_tested():
    assert sum(split for _, split in sizes_of_every_tile()) >= 3


def test_product_layouts():
    tokens, k, m = 37, 400, 260
    w, ws = (t.cuda() for t in weight(m, k, seed=8))
    x = randn(tokens, k, seed=9, dtype=torch.float16).cuda()
    x8, xs = ops().quantize_fp8(x)
    want = ops().matmul_fp8(x, w, ws)
    wide = torch.zeros(m, 3 * k + 80, dtype=torch.uint8, device="cuda").view(E4M3)
    wide[:, 80:80 + k] = w
    wide_x = torch.zeros(tokens, 2 * k, dtype=torch.float16, device="cuda")
    wide_x[:, 8:8 + k] = x
    flat = torch.zeros(tokens * k + 1, dtype=torch.float16, device="cuda")
    flat[1:] = x.flatten()
    for weights in (w, wide[:, 80:80 + k]):
        for scales in (ws, ws.t().contiguous().t(), ws.double().float().repeat(1, 2)[:, :ws.shape[1]]):
            for view in (x, wide_x[:, 8:8 + k], flat[1:].view(tokens, k), x.t().contiguous().t(), torch._neg_view(-x)):
                assert torch.equal(ops().matmul_fp8(view, weights, scales), want)
            for view, by in ((x8, xs), (x8, xs.contiguous()), (torch.cat([x8.view(torch.uint8)] * 2, 1).view(E4M3)[:, :k], xs)):
                assert torch.equal(ops().matmul_fp8(view, weights, scales, x_scale=by), want)
    assert torch.equal(ops().matmul_fp8(x[0], w, ws), ops().matmul_fp8(x[:1], w, ws)[0])
    more = ops().matmul_fp8(x[:36].view(3, 4, 3, k), w, ws)
    assert more.shape == (3, 4, 3, m) and torch.equal(more.view(36, m), ops().matmul_fp8(x[:36], w, ws))
    more = ops().matmul_fp8(x8[:36].reshape(4, 9, k), w, ws, x_scale=xs[:36].reshape(4, 9, -1))
    assert more.shape == (4, 9, m) and torch.equal(more.view(36, m), ops().matmul_fp8(x[:36], w, ws))
    one = x[:1].expand(tokens, k)
    assert torch.equal(ops().matmul_fp8(one, w, ws), ops().matmul_fp8(one.contiguous(), w, ws))


def test_single_rows_of_any_stride():
    """A row of adjacent elements, whatever its view's stride says: of x, of codes and of a weight with one feature."""
    k = 4096
    w, ws = (t.cuda() for t in weight(256, k, seed=2))
    x = randn(1, k, seed=3, dtype=torch.float16).cuda()
    x8, xs = ops().quantize_fp8(x)

    def views(t):
        far = torch.zeros(1, (1 << 25) // k + 4, k, dtype=torch.uint8, device="cuda").view(torch.uint8)
        raw = t.view(torch.uint8) if t.dtype == E4M3 else None
        if raw is None:
            far = torch.zeros(1, (1 << 25) // k + 4, k, dtype=t.dtype, device="cuda")
            far[:, -1] = t
            return t, far[:, -1], t.reshape(k, 1).t(), t.as_strided((1, k), (24, 1))
        far[:, -1] = raw
        return t, far.view(E4M3)[:, -1], raw.reshape(k, 1).t().view(E4M3), raw.as_strided((1, k), (24, 1)).view(E4M3)

    want, one = ops().matmul_fp8(x, w, ws), ops().matmul_fp8(x, w[:1], ws[:1])
    assert torch.equal(one, want[:, :1])
    for view in views(x):
        assert view.stride(1) == 1 and torch.equal(ops().matmul_fp8(view, w, ws), want)
        codes, scales = ops().quantize_fp8(view)
        assert torch.equal(codes.view(torch.uint8), x8.view(torch.uint8)) and torch.equal(scales, xs)
    for view in views(x8):
        assert torch.equal(ops().matmul_fp8(view, w, ws, x_scale=xs, dtype=torch.float16), want) and torch.equal(ops().dequantize_fp8(view, xs), ops().dequantize_fp8(x8, xs))
    for view in views(w[:1].clone()):
        assert torch.equal(ops().matmul_fp8(x, view, ws[:1]), one)


def test_product_without_tokens_or_features():
    w, ws = (t.cuda() for t in weight(130, 256))
    assert ops().matmul_fp8(torch.zeros(0, 256, dtype=torch.float16, device="cuda"), w, ws).shape == (0, 130)
    assert ops().matmul_fp8(torch.zeros(3, 256, dtype=torch.float16, device="cuda"), w[:0], ws[:0]).shape == (3, 0)


@pytest.mark.parametrize("tokens", [3, 40, 300, 1100])
def test_what_is_no_number_stays_in_its_row(tokens):
    k, m = 528, 300
    w, ws = (t.cuda() for t in weight(m, k, seed=3))
    x = randn(tokens, k, seed=4, dtype=torch.float16).cuda()
    want = ops().matmul_fp8(x, w, ws)
    bad = x.clone()
    bad[1, 5], bad[2, 527] = math.inf, math.nan
    got = ops().matmul_fp8(bad, w, ws)
    assert got[1:3].isnan().all() and torch.equal(got[3:], want[3:]) and torch.equal(got[0], want[0])
    codes = w.view(torch.uint8).clone()
    codes[7, 520] = 0x7f                                     # a weight that is no number: its feature
    got = ops().matmul_fp8(x, codes.view(E4M3), ws)
    live = torch.arange(m, device="cuda") != 7
    assert got[:, 7].isnan().all() and torch.equal(got[:, live], want[:, live])
    scales = ws.clone()
    scales[1, 2] = math.nan                                  # a block's scale: the block's features
    got = ops().matmul_fp8(x, w, scales)
    assert got[:, 128:256].isnan().all() and torch.equal(got[:, :128], want[:, :128]) and torch.equal(got[:, 256:], want[:, 256:])


@pytest.mark.parametrize("tokens", [1, 16, 50, 300, 1100])
def test_nothing_is_read_behind_the_rows(tokens):
    """What lies behind the last element of a row, or behind the last row, changes no bit: codes of NaN around all of it."""
    k, m = 272, 140
    w, ws = (t.cuda() for t in weight(m, k, seed=5))
    x8, xs = (t.cuda() for t in quantised(randn(tokens, k, seed=6, dtype=torch.float16), 1))
    want = ops().matmul_fp8(x8, w, ws, x_scale=xs)
    around = []
    for t in (x8, w):
        big = torch.full((t.shape[0] + 300, k + 256), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)
        big[:t.shape[0], :k] = t
        around.append(big[:t.shape[0], :k])
    nan = torch.full((400, 9), math.nan, device="cuda")
    nan[:ws.shape[0], :ws.shape[1]] = ws
    nan_x = torch.full((tokens + 300, 9), math.nan, device="cuda")
    nan_x[:tokens, :xs.shape[1]] = xs
    assert torch.equal(ops().matmul_fp8(around[0], around[1], nan[:ws.shape[0], :ws.shape[1]], x_scale=nan_x[:tokens, :xs.shape[1]]), want)


def test_weights_of_more_than_4_gib():
    m, k, tokens = 70016, 65536, 3
    w = torch.empty(m, k, dtype=torch.uint8, device="cuda")
    for i in range(0, m, 8752):
        w[i:i + 8752] = torch.randint(0, 120, (8752, k), generator=torch.Generator("cuda").manual_seed(i), device="cuda", dtype=torch.uint8)
    w = w.view(E4M3)
    ws = torch.rand(m // 128, k // 128, generator=torch.Generator("cuda").manual_seed(1), device="cuda") + 0.5
    x8, xs = ops().quantize_fp8(randn(tokens, k, seed=2).bfloat16().cuda())
    got = ops().matmul_fp8(x8, w, ws, x_scale=xs, dtype=torch.float32)
    xv = values(x8, xs, 1)
    for lo in (0, 32768, 65536, m - 128):
        rows = slice(lo, lo + 128)
        close(got[:, rows], xv, values(w[rows], ws[lo // 128:lo // 128 + 1], 128), torch.float32)


def test_repeats_and_replays():
    """Calls side by side on two streams, and a graph replayed between eager work: the same bits as a call alone."""
    sizes = [(1, 4096, 1024), (13, 8192, 640), (64, 2048, 4096), (300, 1040, 1001), (2000, 1024, 2048)]
    inputs = []
    for tokens, k, m in sizes:
        w, ws = ops().quantize_fp8(0.02 * randn(m, k, seed=k).half().cuda(), rows=128)
        inputs.append((randn(tokens, k, seed=m).half().cuda(), w, ws))
    want = [ops().matmul_fp8(*i).clone() for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([ops().matmul_fp8(*i) for i in inputs])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [ops().matmul_fp8(*i) for i in inputs]
        codes = [ops().quantize_fp8(i[0]) for i in inputs]
    for turn in range(3):
        for i in inputs:
            i[0].copy_(randn(*i[0].shape, seed=turn + 40).half())
        fresh = [ops().matmul_fp8(*i) for i in inputs]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, fresh))
        for i, (c, s) in zip(inputs, codes):
            a, b = ops().quantize_fp8(i[0])
            assert torch.equal(c.view(torch.uint8), a.view(torch.uint8)) and torch.equal(s, b)


# --- refusals --------------------------------------------------------------------------------------------------------------------

def test_refusals():
    w, ws = (t.cuda() for t in weight(256, 256))
    x = torch.zeros(4, 256, dtype=torch.float16, device="cuda")
    x8, xs = ops().quantize_fp8(x)
    bad = [((x.float(), w, ws), {}, "x must be"), ((x, w.float(), ws), {}, "weight must be"), ((x, w, ws.double()), {}, "weight_scale"), ((x, w, ws[:1]), {}, "weight_scale"),
           ((x[:, :128], w, ws), {}, "expected rows"), ((x, w, ws), dict(x_scale=xs), "x_scale belongs"), ((x8, w, ws), {}, "x_scale belongs"),
           ((x8, w, ws), dict(x_scale=xs[:2]), "x_scale"), ((x, w, ws), dict(dtype=torch.float64), "product in"), ((x.cpu(), w, ws), {}, "GPU tensor"),
           ((x, w.cpu(), ws), {}, "GPU tensor"), ((x, w.t(), ws), {}, "adjacent"), ((x[:, :200], w[:, :200], ws), {}, "multiple of 16"),
           ((x.clone().requires_grad_(), w, ws), {}, "gradient")]
    for args, more, text in bad:
        with pytest.raises(RuntimeError, match=text):
            ops().matmul_fp8(*args, **more)
    with torch.no_grad():
        assert torch.equal(ops().matmul_fp8(x.clone().requires_grad_(), w, ws), ops().matmul_fp8(x, w, ws))
    for args, text in (((x.float(),), "float16"), ((x, 64), "rows of a scale"), ((x[:, :8],), "multiple of 16"), ((x[0],), "rows, elements"), ((x.cpu(),), "GPU")):
        with pytest.raises(RuntimeError, match=text):
            ops().quantize_fp8(*args)
    for args, text in (((x, ws), "float8"), ((x8, ws), "scales"), ((x8, xs, torch.int32), "values in"), ((x8, xs.half()), "scales"), ((x8.cpu(), xs), "GPU")):
        with pytest.raises(RuntimeError, match=text):
            ops().dequantize_fp8(*args)


@pytest.mark.parametrize("call", ["native", "python"])
def test_both_ways_in_are_the_same(call, monkeypatch):
    from triteia_amd.python.capi import fp8
    w, ws = (t.cuda() for t in weight(200, 272))
    x = randn(5, 272, seed=2, dtype=torch.float16).cuda()
    want = ops().matmul_fp8(x, w, ws), *ops().quantize_fp8(x), ops().dequantize_fp8(*ops().quantize_fp8(x))
    if call == "python":
        class Nothing:
            def __getattr__(self, name):
                return lambda *args: None
        monkeypatch.setattr(fp8, "native", lambda: Nothing())
    else:
        assert fp8.native().matmul_fp8(x, w, ws, None, None) is not None and fp8.native().quantize_fp8(x, 1) is not None
    got = ops().matmul_fp8(x, w, ws), *ops().quantize_fp8(x), ops().dequantize_fp8(*ops().quantize_fp8(x))
    assert all(torch.equal(a.float(), b.float()) and a.stride() == b.stride() for a, b in zip(got, want))
