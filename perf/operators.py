"""The attention side of a serving step as cases that can be timed: rotary positions (with the norms of queries and keys), the
write into a paged cache, the read-back and the attention of new tokens over it.

Every case exists twice: in a plain form of elementary torch operations in 32 bits, and through the framework's own operators.

A case is a dict of plain values.  `op` names the call.  `heads` / `kv_heads` / `dim`: heads of the queries, heads of the cache
and elements of a head; `dtype`: type of activations; `cache`: what the cache holds ("same": the activations' type; "int8",
"fp8": codes with one 32-bit scale for every token and head); `page`: tokens of a page.  `tokens`: new tokens (rotary, write) or
tokens read back (read).  For attention `seqs` requests have a context of up to `ctx` tokens; `chunks` of them bring `new` tokens, the
others one.  `rot` elements of a head are rotated; `limit`: positions in the table.
"""
import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"same": 2, "int8": 1, "fp8": 1}


def _case(op, dtype="fp16", heads=32, kv_heads=32, dim=128, cache="same", page=16, tokens=0, seqs=0, chunks=0, new=1, ctx=0,
          causal=True, window=0, rot=128, interleaved=False, norm=False, limit=4096):
    return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "cache": cache, "page": page, "tokens": tokens,
            "seqs": seqs, "chunks": chunks, "new": new, "ctx": ctx, "causal": causal, "window": window, "rot": rot,
            "interleaved": interleaved, "norm": norm, "limit": limit}


def listed():
    cases = {
        # a few requests being decoded: queries and keys of one layer are rotated
        "rotary_decode": _case("rotary", tokens=13),
        # prompts of a model with norms on queries and keys, which rotates half of a head in the interleaved layout, positions far out
        "rotary_prefill": _case("rotary", "bf16", 40, 40, tokens=8000, rot=64, interleaved=True, norm=True, limit=131072),
        # a decode batch: one new token of each request goes into the cache
        "write_decode": _case("write", tokens=64, page=16),
        # a chunk of prompts quantised into the cache, read back as what later steps will see of it
        "write_prefill": _case("write", "bf16", 64, 8, cache="int8", page=64, tokens=2000, norm=True, limit=32768),
        # one request's context handed on to another program
        "read_one": _case("read", "bf16", 8, 8, dim=64, page=32, tokens=777),
        # the contexts of many requests out of an 8-bit cache
        "read_many": _case("read", cache="fp8", page=64, tokens=20000),
        # one user, one token, a short chat
        "attend_one": _case("attend", page=16, seqs=1, ctx=500),
        # the framework's usual decode batch, contexts of any length
        "attend_decode": _case("attend", page=16, seqs=64, ctx=4096),
        # a few long documents, few cache heads, in 8 bits
        "attend_long": _case("attend", "bf16", 64, 8, cache="int8", page=64, seqs=3, ctx=100000),
        # the prompt of one model from its first token on
        "attend_prefill": _case("attend", page=64, seqs=1, chunks=1, new=4000, ctx=4000),
        # prompts taken in chunks behind long contexts
        "attend_chunk": _case("attend", "bf16", 64, 8, page=64, seqs=4, chunks=4, new=500, ctx=8200),
        # one layer of a serving step: decodes and two prompts in one batch, written to an 8-bit cache, planned and attended over
        "step_mixed": _case("step", "fp16", 32, 8, cache="fp8", page=32, seqs=26, chunks=2, new=203, ctx=2000),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [work(c) for c in listed()]
    most_flops, most_bytes = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    op = rng.choice(["rotary", "write", "read", "attend", "attend", "attend", "step"])
    heads, kv_heads = rng.choice([(32, 32), (40, 40), (64, 8), (32, 8), (16, 16), (12, 4), (20, 1)])
    dim = rng.choice([64, 128, 128])
    c = _case(op, rng.choice(["fp16", "bf16"]), heads, kv_heads, dim, rng.choice(["same", "same", "int8", "fp8"]), rng.choice([16, 32, 64, 128]),
              rot=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.4, limit=rng.choice([4096, 32768, 131072]))
    if op in ("rotary", "write"):
        c["tokens"] = _log_int(rng, 1, 8000)
        grow = "tokens"
    elif op == "read":
        c["tokens"] = _log_int(rng, 1, 40000)
        grow = "tokens"
    else:
        c["seqs"] = _log_int(rng, 1, 64)
        c["ctx"] = _log_int(rng, 16, 100000 if c["seqs"] <= 4 else 8000)
        c["chunks"] = rng.choice([0, 0, min(c["seqs"], 3), c["seqs"]])
        c["new"] = _log_int(rng, 2, 4000) if c["chunks"] else 1
        if op == "attend":
            kind = rng.choice(["causal", "causal", "cross", "window"])
            c["causal"], c["window"] = kind != "cross", _log_int(rng, 16, 4000) if kind == "window" else 0
        c["limit"] = max(c["limit"], 131072 if c["ctx"] > 32768 else 32768 if c["ctx"] > 4096 else 4096)
        while c["chunks"] and c["new"] > 1 and _scores(c) > 1 << 30:     # (what the plain form has to hold)
            c["new"] //= 2
        while c["seqs"] > 1 and _scores(c) > 1 << 30:
            c["seqs"] //= 2
            c["chunks"] = min(c["chunks"], c["seqs"])
        c["new"] = max(1, min(c["new"], c["ctx"]))
        grow = "ctx"
    while c[grow] > 16 and (work(c)["flops"] > most_flops or work(c)["bytes"] > most_bytes):
        c[grow] //= 2
        c["new"] = max(1, min(c["new"], c["ctx"])) if grow == "ctx" else c["new"]
    return c


def _scores(case):
    return case["seqs"] * case["heads"] * (case["new"] if case["chunks"] else 1) * case["ctx"]


def _lengths(case):
    """Per request: (new tokens, tokens of its context with the new ones).  One request has all of `ctx`; the others' lengths are spread
    over the range, odd ones among them.  Shapes only: the same for every seed."""
    rng = random.Random("%(seqs)d %(chunks)d %(new)d %(ctx)d" % case)
    out = []
    for i in range(case["seqs"]):
        new = case["new"] if i < case["chunks"] else 1
        if case["chunks"] > 1 and 0 < i < case["chunks"]:
            new = rng.randint((new + 1) // 2, new)
        kv = case["ctx"] if i == 0 else rng.randint(max(1, case["ctx"] // 20), case["ctx"])
        out.append((new, max(kv, new) if case["causal"] else kv))
    order = list(range(len(out)))
    rng.shuffle(order)
    return [out[i] for i in order]


# --- inputs -----------------------------------------------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _quantised(x, kind):
    """(codes, scales): x [..., dim] as codes with one scale for every row, the row's largest magnitude at the end of the range."""
    most = 127.0 if kind == "int8" else 448.0
    scale = x.abs().amax(-1) / most
    y = x / torch.where(scale > 0, scale, 1.0)[..., None]
    return (y.round().to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)), scale


def _held(case, g, n_pages):
    """A cache with history in it: keys whose channels differ in size, as they do behind a projection."""
    shape = (n_pages, case["kv_heads"], case["page"], case["dim"])
    spread = torch.exp(0.3 * _randn(g, case["kv_heads"], 1, case["dim"]))
    out = {}
    for name in ("k", "v"):
        x = _randn(g, *shape)
        if name == "k":
            x *= spread
        if case["cache"] == "same":
            out[name], out[name + "_scale"] = x.to(_DTYPES[case["dtype"]]), None
        else:
            out[name], out[name + "_scale"] = _quantised(x, case["cache"])
    return out


def _table(case):
    """cos and sin of every position and pair, worked out in 64 bits."""
    rate = 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
    angle = torch.arange(case["limit"], device="cuda", dtype=torch.float64)[:, None] * rate
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, dim, page = _DTYPES[case["dtype"]], case["dim"], case["page"]
    s = {"op": case["op"], "dtype": dtype, "heads": case["heads"], "kv_heads": case["kv_heads"], "dim": dim, "page": page,
         "kind": case["cache"], "causal": case["causal"], "window": case["window"], "interleaved": case["interleaved"], "eps": 1e-6,
         "scale": dim ** -0.5, "q_norm": None, "k_norm": None}
    attends = case["op"] in ("attend", "step")
    if attends:
        lengths = _lengths(case)
        tokens = sum(n for n, _ in lengths)
        width = max(1, -(-max(kv for _, kv in lengths) // page))
        n_pages = max(1, sum(-(-kv // page) for _, kv in lengths))
        order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        s["pages"] = torch.zeros((len(lengths), width), dtype=torch.int32, device="cuda")
        at, positions, slots = 0, [], []
        for b, (new, kv) in enumerate(lengths):
            have = -(-kv // page)
            s["pages"][b, :have] = order[at:at + have]
            at += have
            if case["op"] == "step":
                p = torch.arange(kv - new, kv, device="cuda", dtype=torch.int32)
                positions.append(p)
                slots.append(s["pages"][b, (p // page).long()] * page + p % page)
        s["q_starts"] = torch.tensor([0] + [sum(n for n, _ in lengths[:b + 1]) for b in range(len(lengths))], dtype=torch.int32, device="cuda")
        s["kv_lens"] = torch.tensor([kv for _, kv in lengths], dtype=torch.int32, device="cuda")
        s["max_q"], s["max_kv"] = max(n for n, _ in lengths), max(kv for _, kv in lengths)
        s.update(_held(case, g, n_pages))
        if case["op"] == "step":
            s["positions"], s["slots"] = torch.cat(positions), torch.cat(slots)
    else:
        tokens = case["tokens"]
        n_pages = -(-tokens // page) + 3
        if case["op"] == "read":
            # whole pages in any order, the last one not full
            order = torch.randperm(n_pages, generator=g, device="cuda")[:-(-tokens // page)]
            s["slots"] = (order[:, None] * page + torch.arange(page, device="cuda")).flatten()[:tokens].to(torch.int32)
            s.update(_held(case, g, n_pages))
        else:
            s["positions"] = torch.randint(0, case["limit"], (tokens,), generator=g, device="cuda", dtype=torch.int32)
        if case["op"] == "write":
            s["slots"] = torch.randperm(n_pages * page, generator=g, device="cuda")[:tokens].to(torch.int32)
            s.update(_held(case, g, n_pages))
    if case["op"] != "read":
        # queries, keys and values as views of the fused projection's output, a row a token
        n = case["heads"] + (0 if case["op"] == "attend" else 2 * case["kv_heads"])
        x = _randn(g, tokens, n, dim)
        x[:, :case["heads"]] *= 1.5
        qkv = x.to(dtype)
        s["q"], s["k_new"], s["v_new"] = qkv.split([case["heads"], (n - case["heads"]) // 2, (n - case["heads"]) // 2], 1)
    if "positions" in s:
        s["table"] = _table(case)
        if case["norm"]:
            s["q_norm"], s["k_norm"] = ((1 + 0.1 * _randn(g, dim)).to(dtype) for _ in range(2))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from triteia_amd.python import ops
        if "k" in s:
            s["handle"] = ops.PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if case["op"] == "attend":
            # made once for a forward pass and used by every layer of it (the step makes its own, within the call)
            s["plan"] = ops.attention_plan(s["handle"], s["q_starts"], s["kv_lens"], n_heads=s["heads"], n_tokens=s["q"].shape[0],
                                           max_q=s["max_q"], causal=s["causal"], window=s["window"])
    return s


# --- the operators --------------------------------------------------------------------------------------------------------------

def _run_own(s):
    from triteia_amd.python import ops
    op = s["op"]
    how = dict(interleaved=s["interleaved"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=s["eps"])
    if op == "rotary":
        return ops.rotary(s["q"], s["k_new"], s["positions"], s["table"], **how)
    if op == "read":
        return ops.cache_read(s["handle"], s["slots"], dtype=s["dtype"])
    if op == "attend":
        return ops.paged_attention(s["q"], s["handle"], s["pages"], s["q_starts"], s["kv_lens"], plan=s["plan"], causal=s["causal"],
                                   window=s["window"], scale=s["scale"])
    q = ops.rotary_cache_write(s["q"], s["k_new"], s["v_new"], s["positions"], s["table"], s["handle"], s["slots"], **how)
    if op == "write":
        if s["kind"] == "same":
            return q, s["k"], s["v"]
        return q, ops.cache_read(s["handle"], s["slots"], dtype=s["dtype"])
    plan = ops.attention_plan(s["handle"], s["q_starts"], s["kv_lens"], n_heads=s["heads"], n_tokens=q.shape[0], max_q=s["max_q"],
                              causal=s["causal"], window=s["window"])
    return ops.paged_attention(q, s["handle"], s["pages"], s["q_starts"], s["kv_lens"], plan=plan, causal=s["causal"], window=s["window"],
                               scale=s["scale"])


def _turned(x, positions, table, interleaved, weight, eps):
    """x [tokens, heads, dim] in 32 bits: each head normalised if it has a weight, its first elements rotated."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.float()
    half = table.shape[1]
    cos, sin = table[positions.long()][:, None].unbind(-1)
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _put(s, k, v):
    """k, v [tokens, kv_heads, dim] in 32 bits into the cache."""
    page, slot = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
    for name, x in (("k", k), ("v", v)):
        if s["kind"] == "same":
            s[name][page, :, slot] = x.to(s["dtype"])
        else:
            codes, scale = _quantised(x, s["kind"])
            s[name].view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
            s[name + "_scale"][page, :, slot] = scale


def _values(s, name, page, slot=None):
    """Pages (or single tokens) of the cache in 32 bits."""
    at = (page,) if slot is None else (page, slice(None), slot)
    if s["kind"] == "same":
        return s[name][at].float()
    return s[name].view(torch.uint8)[at].view(s[name].dtype).float() * s[name + "_scale"][at][..., None]


def _attend(s, q):
    n_seqs, kv_heads, dim = s["pages"].shape[0], s["kv_heads"], s["dim"]
    group, most = q.shape[1] // kv_heads, s["max_q"]
    starts, new = s["q_starts"][:-1].long(), s["q_starts"].diff().long()
    row = torch.arange(most, device=q.device)
    live = row < new[:, None]                                                      # [seqs, most]
    at = torch.where(live, starts[:, None] + row, 0)
    rows = q.float()[at].view(n_seqs, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n_seqs, kv_heads, group * most, dim)
    column = torch.arange(s["pages"].shape[1] * s["page"], device=q.device)
    inside = column < s["kv_lens"][:, None]                                        # [seqs, columns]
    k, v = (_values(s, name, s["pages"].long()).permute(0, 2, 1, 3, 4).reshape(n_seqs, kv_heads, -1, dim) for name in ("k", "v"))
    v = torch.where(inside[:, None, :, None], v, 0)
    seen = inside[:, None, :].expand(-1, most, -1)
    if s["causal"]:
        position = (s["kv_lens"].long() - new)[:, None] + row
        seen = seen & (column <= position[..., None])
        if s["window"]:
            seen = seen & (column > position[..., None] - s["window"])
    score = torch.matmul(rows, k.transpose(2, 3)).view(n_seqs, kv_heads, group, most, -1) * s["scale"]
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top > -math.inf, top, 0)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(n_seqs, kv_heads, group * most, -1), v).view(n_seqs, kv_heads, group, most, dim)
    out = (out / torch.where(total > 0, total, 1)).permute(0, 3, 1, 2, 4).reshape(n_seqs, most, -1, dim)
    return out[live].to(q.dtype)


def _run_plain(s):
    op, dtype = s["op"], s["dtype"]
    if op == "read":
        page, slot = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
        return tuple(_values(s, name, page, slot).to(dtype) for name in ("k", "v"))
    if op == "attend":
        return _attend(s, s["q"])
    q = _turned(s["q"], s["positions"], s["table"], s["interleaved"], s["q_norm"], s["eps"]).to(dtype)
    k = _turned(s["k_new"], s["positions"], s["table"], s["interleaved"], s["k_norm"], s["eps"])
    if op == "rotary":
        return q, k.to(dtype)
    _put(s, k, s["v_new"].float())
    if op == "write":
        if s["kind"] == "same":
            return q, s["k"], s["v"]
        page, slot = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
        return q, tuple(_values(s, name, page, slot).to(dtype) for name in ("k", "v"))
    return _attend(s, q)


def run(s):
    return _run_own(s) if own else _run_plain(s)


# --- what the operators are defined as, in 64 bits ------------------------------------------------------------------------------

def _turned64(x, positions, table, interleaved, weight, eps):
    x = x.double()
    if weight is not None:
        x = x / ((x * x).sum(-1, keepdim=True) / x.shape[-1] + eps).sqrt() * weight.double()
    out = x.clone()
    for i in range(table.shape[1]):
        one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + table.shape[1])
        c, d = (table[positions.long(), i, j].double()[:, None] for j in (0, 1))
        out[..., one] = x[..., one] * c - x[..., two] * d
        out[..., two] = x[..., one] * d + x[..., two] * c
    return out


def _rounded(x, kind, dtype):
    """What the cache holds of x, in 64 bits."""
    if kind == "same":
        return x.to(dtype).double()
    top = x.abs().max(-1, keepdim=True).values
    scale = (top / (127 if kind == "int8" else 448)).float().double()
    y = x / torch.where(scale > 0, scale, 1.0)
    return (y.round() if kind == "int8" else y.float().to(torch.float8_e4m3fn).double()) * scale


def exact(case, seed):
    s = _inputs(case, seed)
    held = {}
    if "k" in s:
        for name in ("k", "v"):
            held[name] = s[name].double() if s[name + "_scale"] is None else s[name].double() * s[name + "_scale"].double().unsqueeze(-1)
    if case["op"] == "read":
        index = s["slots"].long()
        return tuple(held[name].transpose(1, 2).reshape(-1, s["kv_heads"], s["dim"])[index] for name in ("k", "v"))
    if case["op"] != "attend":
        q, k = (_turned64(x, s["positions"], s["table"], s["interleaved"], w, s["eps"]) for x, w in ((s["q"], s["q_norm"]), (s["k_new"], s["k_norm"])))
        if case["op"] == "rotary":
            return q, k
        page, slot = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
        for name, x in (("k", k), ("v", s["v_new"].double())):
            if case["op"] == "write" and s["kind"] == "same":
                held[name][page, :, slot] = x
            else:
                held[name][page, :, slot] = _rounded(x, s["kind"], s["dtype"])
        if case["op"] == "write":
            return (q, held["k"], held["v"]) if s["kind"] == "same" else (q, tuple(held[n][page, :, slot] for n in ("k", "v")))
        q = q.to(s["dtype"]).double()
    else:
        q = s["q"].double()
    out = torch.zeros_like(q)
    starts, lens = s["q_starts"].tolist(), s["kv_lens"].tolist()
    for b, kv in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        own_pages = s["pages"][b, :-(-kv // s["page"])].long()
        k, v = (held[name][own_pages].transpose(0, 1).reshape(s["kv_heads"], -1, s["dim"])[:, :kv] for name in ("k", "v"))
        group = q.shape[1] // s["kv_heads"]
        block = max(1, (1 << 27) // (max(1, kv) * group))
        for h in range(s["kv_heads"]):
            for r in range(lo, hi, block):
                rows = q[r:min(hi, r + block), h * group:(h + 1) * group]
                score = torch.matmul(rows, k[h].t()) * s["scale"]                   # [rows, group, kv]
                if s["causal"]:
                    position = kv - (hi - lo) + torch.arange(r - lo, r - lo + rows.shape[0], device=q.device)[:, None, None]
                    far = torch.arange(kv, device=q.device) - position
                    score[((far > 0) | (far <= -s["window"]) if s["window"] else far > 0).expand_as(score)] = -math.inf
                out[r:r + rows.shape[0], h * group:(h + 1) * group] = torch.nan_to_num(torch.softmax(score, -1)) @ v[h]
    return out


# --- what a pass cannot do without -----------------------------------------------------------------------------------------------

def work(case):
    """Bytes: inputs and outputs once (of a context what some new token sees), table rows, scales and indices among them;
    operations: two for each product of the attention."""
    heads, kv_heads, dim, tokens = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    a_row = kv_heads * (dim * _SIZE[case["cache"]] + (0 if case["cache"] == "same" else 4))     # one token's keys (or values) in the cache
    rotated = lambda n: n * (2 * 2.0 * heads * dim + 4 * case["rot"] + 4)   # queries in and out, table, positions  # noqa: E731
    if case["op"] == "rotary":
        return {"bytes": rotated(tokens) + tokens * 4.0 * kv_heads * dim, "flops": 3.0 * tokens * (heads + kv_heads) * case["rot"]}
    if case["op"] == "read":
        return {"bytes": tokens * 2.0 * (a_row + 2 * kv_heads * dim) + 4 * tokens, "flops": 0.0}
    write = lambda n: rotated(n) + n * 2.0 * (2 * kv_heads * dim + a_row) + 4 * n  # noqa: E731
    if case["op"] == "write":
        back = 0.0 if case["cache"] == "same" else tokens * 2.0 * (a_row + 2 * kv_heads * dim) + 4 * tokens
        return {"bytes": write(tokens) + back, "flops": 3.0 * tokens * (heads + kv_heads) * case["rot"]}
    bytes_, flops = 0.0, 0.0
    for new, kv in _lengths(case):
        seen = kv if not case["causal"] else min(kv, case["window"] + new - 1) if case["window"] else kv
        pairs = float(new) * kv
        if case["causal"]:
            first = kv - new
            w = case["window"] or kv
            pairs = float(sum(min(first + i + 1, w) for i in range(new)))
        bytes_ += 2.0 * seen * a_row + 2 * 2.0 * new * heads * dim + 4 * (seen / case["page"]) + 8
        flops += 4.0 * pairs * heads * dim
        if case["op"] == "step":
            bytes_ += write(new)
    return {"bytes": bytes_, "flops": flops}
