"""What a serving step of many variants shares: the base weight, in 8 bits with a scale for each block of 128, and the prefix that the requests of
one variant have in common.

Three operators, each in a plain form of elementary torch operations and through the framework's own entry points: the quantiser (activations
with a scale for every token and 128 channels, weights with one for every 128 x 128) with its read-back; the product of activations with such
a weight; attention of a batch in groups, each of which shares a prefix.

A case is a dict of plain values.  `op` names the call.
"quant": `rows` x `k` values in `dtype`, `block` rows a scale, quantised and read back.
"product": `tokens` x `k` activations times a weight of `m` x `k`; `codes`: the activations are in 8 bits already, else they are quantised in the call.
"prefix": `groups` of `seqs` requests in all share a prefix of up to `prefix` tokens each; every request has up to `ctx` tokens of its own, `new` of them new ones;
`heads` / `kv_heads` / `dim`, `cache` ("same", "int8", "fp8") and `page` as the paged cache has them; not `causal`: every row sees all of its context.
"""
import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _quant(rows, k, dtype="fp16", block=1):
    return {"op": "quant", "rows": rows, "k": k, "dtype": dtype, "block": block}


def _product(tokens, k, m, dtype="fp16", codes=False):
    return {"op": "product", "tokens": tokens, "k": k, "m": m, "dtype": dtype, "codes": codes}


def _prefix(seqs, prefix, ctx, dtype="fp16", groups=1, new=1, heads=32, kv_heads=32, dim=128, cache="same", page=16, causal=True):
    return {"op": "prefix", "seqs": seqs, "groups": groups, "prefix": prefix, "ctx": ctx, "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "cache": cache, "page": page, "causal": causal, "dtype": dtype}


def listed():
    cases = {
        # a few requests' activations ahead of a projection
        "quant_decode": _quant(13, 4096),
        # a batch of prompts' activations
        "quant_prefill": _quant(8000, 8192, "bf16"),
        # a base weight on its way into 8 bits when a model is loaded, checked against what it stood for
        "quant_weight": _quant(11008, 4096, block=128),
        # one request's token through a projection
        "product_one": _product(1, 4096, 4096),
        # the framework's decode batch through the widest layer that its benchmark has
        "product_decode": _product(64, 8192, 28672, "bf16"),
        # a mixed step on a layer of odd sizes: neither the channels nor the features end on a block
        "product_ragged": _product(203, 2000, 1001),
        # activations that another layer has quantised already
        "product_codes": _product(1000, 4096, 11008, codes=True),
        # prompts through the widest layer
        "product_prefill": _product(8000, 8192, 28672, "bf16"),
        # a handful of chats behind one system prompt
        "prefix_chats": _prefix(5, 1000, 100),
        # a decode batch whose requests ask about the same long document
        "prefix_decode": _prefix(64, 8200, 500, "bf16", heads=64, kv_heads=8, page=64),
        # six variants, each with a prompt of its own, in one batch over a cache in 8 bits
        "prefix_variants": _prefix(96, 3000, 400, groups=6, cache="fp8", page=32),
        # prompts that begin alike: the rest of each is attended to for the first time
        "prefix_prompts": _prefix(8, 6000, 231, "bf16", new=203, heads=32, kv_heads=8, page=64),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [work(c) for c in listed()]
    most_flops, most_bytes = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    op = rng.choice(["quant", "product", "product", "product", "prefix", "prefix", "prefix"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "quant":
        c = _quant(_log_int(rng, 1, 20000), 16 * _log_int(rng, 4, 1800), dtype, rng.choice([1, 1, 128]))
        grow = "rows"
    elif op == "product":
        c = _product(_log_int(rng, 1, 8000), 16 * _log_int(rng, 8, 1800), _log_int(rng, 16, 30000), dtype, rng.random() < 0.3)
        grow = "tokens"
    else:
        heads, kv_heads = rng.choice([(32, 32), (40, 40), (64, 8), (32, 8), (16, 16), (12, 4), (20, 1)])
        seqs = _log_int(rng, 2, 128)
        c = _prefix(seqs, _log_int(rng, 64, 30000), _log_int(rng, 16, 2000), dtype, min(seqs, rng.choice([1, 1, 2, 5])),
                    rng.choice([1, 1, 1, _log_int(rng, 2, 300)]), heads, kv_heads, rng.choice([64, 128, 128]), rng.choice(["same", "same", "int8", "fp8"]),
                    rng.choice([16, 32, 64, 128]), rng.random() < 0.85)
        c["new"] = min(c["new"], c["ctx"])
        while c["new"] > 1 and _scores(c) > 1 << 29:           # (what the plain form has to hold)
            c["new"] //= 2
        grow = "prefix"
        while c["prefix"] > 64 and (_scores(c) > 1 << 29 or _held_values(c) > 1 << 31):
            c["prefix"] //= 2
    while c[grow] > 1 and (work(c)["flops"] > most_flops or work(c)["bytes"] > most_bytes):
        c[grow] //= 2
    return c


def _scores(case):
    return case["seqs"] * case["heads"] * case["new"] * (case["prefix"] + case["ctx"])


def _held_values(case):
    return case["seqs"] * case["kv_heads"] * case["dim"] * (case["prefix"] + case["ctx"])


def _batch(case):
    """Per group its prefix (whole pages), per request (its group, new tokens, tokens of its own with the new ones).  One group has the whole prefix and
    one request the whole length; the others are spread over the range.  Shapes only: the same for every seed."""
    rng = random.Random("%(seqs)d %(groups)d %(prefix)d %(ctx)d %(new)d" % case)
    page = case["page"]
    prefixes = [(case["prefix"] if g == 0 else rng.randint(case["prefix"] // 2, case["prefix"])) // page * page for g in range(case["groups"])]
    ends = sorted(rng.sample(range(1, case["seqs"]), case["groups"] - 1)) + [case["seqs"]]
    out = []
    for b in range(case["seqs"]):
        new = case["new"] if b == 0 or case["new"] == 1 else rng.randint((case["new"] + 1) // 2, case["new"])
        out.append((sum(b >= e for e in ends), new, case["ctx"] if b == 0 else rng.randint(max(new, case["ctx"] // 10), case["ctx"])))
    return prefixes, out


# --- inputs -----------------------------------------------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(g, rows, k, dtype):
    """Channels of different sizes, a few of them far larger, as behind a norm's weight."""
    channel = torch.exp(0.5 * _randn(g, k)) * torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    return (_randn(g, rows, k) * channel).to(dtype)


def _blocked(x, rows):
    """x [n, k] as [n / rows, rows, k / 128, 128], zeros behind its ends."""
    n, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % 128, 0, -n % rows))
    return x.view(-1, rows, x.shape[1] // 128, 128)


def _spread(scales, rows, n, k):
    """Scales [n / rows, k / 128] as one for every element."""
    return scales.repeat_interleave(rows, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _quantised(x, rows):
    """(codes, scales) of x [n, k] in 32 bits: blocks of rows x 128, the largest magnitude at the end of the codes' range."""
    n, k = x.shape
    top = _blocked(x.abs(), rows).amax((1, 3))
    scale = torch.where(top < 1e-30, 0.0, top / torch.full((), 448.0, device=x.device))     # (a divisor on the GPU: a number would be multiplied by)
    y = x / _spread(torch.where(scale > 0, scale, 1.0), rows, n, k)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _rows_quantised(x, kind):
    """The cache's codes of 8 bits: x [..., dim] with one scale for every row."""
    most = 127.0 if kind == "int8" else 448.0
    scale = x.abs().amax(-1) / most
    y = x / torch.where(scale > 0, scale, 1.0)[..., None]
    return (y.round().to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)), scale


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    s = {"op": case["op"], "dtype": dtype}
    if case["op"] == "quant":
        s["block"] = case["block"]
        s["x"] = _activations(g, case["rows"], case["k"], dtype) if case["block"] == 1 else (0.02 * _randn(g, case["rows"], case["k"])).to(dtype)
        return s
    if case["op"] == "product":
        s["w"], s["w_scale"] = _quantised(0.02 * _randn(g, case["m"], case["k"]), 128)
        s["x"], s["x_scale"] = _activations(g, case["tokens"], case["k"], dtype), None
        if case["codes"]:
            s["x"], scale = _quantised(s["x"].float(), 1)
            s["x_scale"] = scale.t().contiguous().t()            # (a block's scales of all tokens adjacent, as the quantiser leaves them)
        return s
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    prefixes, requests = _batch(case)
    lengths = [prefixes[group] + length for group, _, length in requests]
    n_pages = sum(p // page for p in prefixes) + sum(-(-length // page) for _, _, length in requests)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    s["pages"] = torch.zeros((len(requests), max(-(-n // page) for n in lengths)), dtype=torch.int32, device="cuda")
    at, shared = 0, []
    for p in prefixes:
        shared.append(order[at:at + p // page])
        at += p // page
    for b, (group, _, length) in enumerate(requests):
        first, have = len(shared[group]), -(-length // page)
        s["pages"][b, :first] = shared[group]
        s["pages"][b, first:first + have] = order[at:at + have]
        at += have
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    s["q_starts"] = whole([sum(new for _, new, _ in requests[:b]) for b in range(len(requests) + 1)])
    s["kv_lens"] = whole(lengths)
    s["group_starts"] = whole([sum(group < i for group, _, _ in requests) for i in range(len(prefixes) + 1)])
    s["prefix_lens"] = whole(prefixes)
    s.update(heads=heads, kv_heads=kv_heads, dim=dim, page=page, kind=case["cache"], causal=case["causal"], scale=dim ** -0.5,
             max_q=max(new for _, new, _ in requests))
    # a cache with history in it: keys whose channels differ in size, as they do behind a projection
    spread = torch.exp(0.3 * _randn(g, kv_heads, 1, dim))
    for name in ("k", "v"):
        x = _randn(g, n_pages, kv_heads, page, dim)
        if name == "k":
            x *= spread
        s[name], s[name + "_scale"] = (x.to(dtype), None) if case["cache"] == "same" else _rows_quantised(x, case["cache"])
    s["q"] = (1.5 * _randn(g, sum(new for _, new, _ in requests), heads, dim)).to(dtype)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["op"] == "prefix":
        from triteia_amd.python import ops
        s["handle"] = ops.PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        # made once for a forward pass and used by every layer of it
        s["plan"] = ops.attention_plan(s["handle"], s["q_starts"], s["kv_lens"], n_heads=s["heads"], n_tokens=s["q"].shape[0], max_q=s["max_q"],
                                       causal=s["causal"], group_starts=s["group_starts"], prefix_lens=s["prefix_lens"])
    return s


# --- the operators --------------------------------------------------------------------------------------------------------------

def _run_own(s):
    from triteia_amd.python import ops
    if s["op"] == "quant":
        codes, scales = ops.quantize_fp8(s["x"], rows=s["block"])
        return ops.dequantize_fp8(codes, scales, dtype=s["dtype"]), scales
    if s["op"] == "product":
        return ops.matmul_fp8(s["x"], s["w"], s["w_scale"], x_scale=s["x_scale"], dtype=s["dtype"])
    return ops.paged_attention(s["q"], s["handle"], s["pages"], s["q_starts"], s["kv_lens"], plan=s["plan"], causal=s["causal"], scale=s["scale"])


def _values(s, name):
    """Each request's keys or values in 32 bits, [seqs, kv_heads, columns, dim]."""
    pages = s["pages"].long()
    if s["kind"] == "same":
        x = s[name][pages].float()
    else:
        x = s[name].view(torch.uint8)[pages].view(s[name].dtype).float() * s[name + "_scale"][pages][..., None]
    return x.permute(0, 2, 1, 3, 4).reshape(pages.shape[0], s["kv_heads"], -1, s["dim"])


def _attend(s):
    q, n_seqs, kv_heads, dim, most = s["q"], s["pages"].shape[0], s["kv_heads"], s["dim"], s["max_q"]
    group = s["heads"] // kv_heads
    starts, new = s["q_starts"][:-1].long(), s["q_starts"].diff().long()
    row = torch.arange(most, device=q.device)
    live = row < new[:, None]                                                      # [seqs, most]
    at = torch.where(live, starts[:, None] + row, 0)
    rows = q.float()[at].view(n_seqs, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n_seqs, kv_heads, group * most, dim)
    column = torch.arange(s["pages"].shape[1] * s["page"], device=q.device)
    inside = column < s["kv_lens"][:, None]
    seen = inside[:, None, :].expand(-1, most, -1)
    if s["causal"]:
        seen = seen & (column <= ((s["kv_lens"].long() - new)[:, None] + row)[..., None])
    score = torch.matmul(rows, _values(s, "k").transpose(2, 3)).view(n_seqs, kv_heads, group, most, -1) * s["scale"]
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top > -math.inf, top, 0)).exp_()
    total = weight.sum(-1, keepdim=True)
    v = torch.where(inside[:, None, :, None], _values(s, "v"), 0)
    out = torch.matmul(weight.view(n_seqs, kv_heads, group * most, -1), v).view(n_seqs, kv_heads, group, most, dim)
    out = (out / torch.where(total > 0, total, 1)).permute(0, 3, 1, 2, 4).reshape(n_seqs, most, -1, dim)
    return out[live].to(q.dtype)


def _run_plain(s):
    if s["op"] == "quant":
        n, k = s["x"].shape
        codes, scales = _quantised(s["x"].float(), s["block"])
        return (codes.float() * _spread(scales, s["block"], n, k)).to(s["dtype"]), scales
    if s["op"] == "product":
        x, scale = (s["x"], s["x_scale"]) if s["x_scale"] is not None else _quantised(s["x"].float(), 1)
        x = x.float() * _spread(scale, 1, *x.shape)
        w = s["w"].float() * _spread(s["w_scale"], 128, *s["w"].shape)
        return torch.matmul(x, w.t()).to(s["dtype"])
    return _attend(s)


def run(s):
    return _run_own(s) if own else _run_plain(s)


# --- what the operators are defined as, in 64 bits ------------------------------------------------------------------------------

def _codes64(x, rows):
    """(codes, scales) in 64 bits of x [n, k]: scales and quotients are rounded to 32 bits, then quotients to the nearest code."""
    n, k = x.shape
    blocks = x.double().new_zeros((-(-n // rows) * rows, -(-k // 128) * 128))
    blocks[:n, :k] = x.double()
    blocks = blocks.unflatten(1, (-1, 128)).unflatten(0, (-1, rows))
    top = blocks.abs().max(3).values.max(1).values
    scale = torch.where(top < 1e-30, torch.zeros_like(top), (top / 448).float().double())
    quotient = (blocks / torch.where(scale == 0, 1.0, scale)[:, None, :, None]).float().clamp(-448, 448)
    codes = quotient.to(torch.float8_e4m3fn).double()
    return codes, scale[:, None, :, None]


def _whole(blocks, n, k):
    return blocks.flatten(2, 3).flatten(0, 1)[:n, :k]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "quant":
        codes, scale = _codes64(s["x"], case["block"])
        return _whole(codes * scale, case["rows"], case["k"]), scale[:, 0, :, 0]
    if case["op"] == "product":
        tokens, k, m = case["tokens"], case["k"], case["m"]
        if s["x_scale"] is None:
            codes, scale = _codes64(s["x"], 1)
            x = _whole(codes * scale, tokens, k)
        else:
            x = s["x"].double()
            for b in range(s["x_scale"].shape[1]):
                x[:, 128 * b:128 * b + 128] *= s["x_scale"][:, b:b + 1].double()
        out = torch.empty((tokens, m), dtype=torch.float64, device=x.device)
        for j in range(0, m, 128):
            w = s["w"][j:j + 128].double()
            for b in range(s["w_scale"].shape[1]):
                w[:, 128 * b:128 * b + 128] *= s["w_scale"][j // 128, b].double()
            out[:, j:j + 128] = x @ w.t()
        return out
    held = {n: s[n].double() if s[n + "_scale"] is None else s[n].double() * s[n + "_scale"].double().unsqueeze(-1) for n in ("k", "v")}
    q, group = s["q"].double(), case["heads"] // case["kv_heads"]
    out = torch.zeros_like(q)
    starts, lens = s["q_starts"].tolist(), s["kv_lens"].tolist()
    for b, kv in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        own_pages = s["pages"][b, :-(-kv // case["page"])].long()
        k, v = (held[n][own_pages].transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :kv] for n in ("k", "v"))
        for h in range(case["kv_heads"]):
            rows = q[lo:hi, h * group:(h + 1) * group]
            score = torch.matmul(rows, k[h].t()) * s["scale"]                   # [rows, group, kv]
            if case["causal"]:
                position = kv - (hi - lo) + torch.arange(hi - lo, device=q.device)[:, None, None]
                score[(torch.arange(kv, device=q.device) > position).expand_as(score)] = -math.inf
            out[lo:hi, h * group:(h + 1) * group] = torch.softmax(score, -1) @ v[h]
    return out


# --- what a pass cannot do without -----------------------------------------------------------------------------------------------

def work(case):
    """Bytes: inputs and outputs once, scales and indices among them, of contexts a group's prefix once; operations: two for each product."""
    if case["op"] == "quant":
        n, k = case["rows"], case["k"]
        codes = n * k + 4.0 * -(-n // case["block"]) * -(-k // 128)
        return {"bytes": 2 * (2.0 * n * k + codes), "flops": 0.0}
    if case["op"] == "product":
        t, k, m = case["tokens"], case["k"], case["m"]
        blocks = -(-k // 128)
        x = t * k + 4.0 * t * blocks if case["codes"] else 2.0 * t * k
        return {"bytes": x + m * k + 4.0 * -(-m // 128) * blocks + 2.0 * t * m, "flops": 2.0 * t * k * m}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    row = 2.0 * kv_heads * (dim * 2 if case["cache"] == "same" else dim + 4)           # one token's keys and values
    prefixes, requests = _batch(case)
    bytes_, pairs = sum(prefixes) * (row + 4.0 / case["page"]), 0.0
    for group, new, length in requests:
        bytes_ += length * (row + 4.0 / case["page"]) + 4.0 * new * heads * dim + 8
        seen = prefixes[group] + length
        pairs += new * seen - (new * (new - 1) / 2 if case["causal"] else 0)
    return {"bytes": bytes_, "flops": 4.0 * pairs * heads * dim}
