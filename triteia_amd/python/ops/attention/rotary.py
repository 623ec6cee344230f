"""Rotary positions of queries and keys, with the norms of both and the write into the paged cache in the same launch."""
import math

import torch

from triteia_amd.python import capi

__all__ = ["rotary_table", "rotary", "rotary_cache_write"]
_NEEDED = {"linear": ("factor",), "ntk": ("factor",), "bands": ("factor", "low", "high", "original"), "yarn": ("factor", "original")}


def rotary_table(limit, rotary_dim, base=10000.0, scaling=None, device="cuda"):
    """cos and sin of positions 0 .. limit - 1: float32 [limit, rotary_dim / 2, 2], worked out in 64 bits.  Pair i turns by position * base^(-2 i / rotary_dim).

    `scaling` for contexts longer than those of training, a dict with `type` and `factor` and what else is named here:
      "linear": positions divided by `factor`;
      "ntk":    the base multiplied by factor^(d / (d - 2)), so that the slowest pair is stretched by `factor` and the fastest is not;
      "bands":  pairs that turn fewer than `low` times over `original` positions slowed by `factor`, more than `high` times not, between the two linear
                in the number of turns;
      "yarn":   a ramp over the pairs' indices between those that turn `fast` and `slow` times (32 and 1) over `original` positions, and cos and sin
                multiplied by `magnitude` (0.1 ln(factor) + 1)."""
    if rotary_dim < 16 or rotary_dim % 16:
        raise RuntimeError(f"{rotary_dim} elements to rotate: a multiple of 16")
    if limit < 1:
        raise RuntimeError(f"a table of {limit} positions")
    pair = torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64)
    kind, how, factor, magnitude = None, {}, 1.0, 1.0
    if scaling is not None:
        how = dict(scaling)
        kind = how.pop("type", None)
        if kind not in ("linear", "ntk", "bands", "yarn"):
            raise RuntimeError(f"unknown scaling of positions: {scaling}")
        missing = [name for name in _NEEDED[kind] if name not in how]
        if missing:
            raise RuntimeError(f"{kind} scaling needs {', '.join(missing)}: {scaling}")
        factor = float(how.pop("factor"))
        if not 1.0 <= factor < math.inf:
            raise RuntimeError(f"a factor of {factor}: 1 at least")
    if kind == "ntk":
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    rate = float(base) ** (-pair / rotary_dim)
    if kind == "linear":
        rate = rate / factor
    elif kind == "bands":
        low, high, original = float(how.pop("low")), float(how.pop("high")), float(how.pop("original"))
        if not low < high:
            raise RuntimeError(f"bands from {low} to {high} turns")
        keep = ((original * rate / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        rate = rate * keep + rate / factor * (1 - keep)
    elif kind == "yarn":
        fast, slow, original = float(how.pop("fast", 32.0)), float(how.pop("slow", 1.0)), float(how.pop("original"))
        index = lambda turns: rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rotary_dim - 1)
        slowed = ((pair / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        rate = rate * (1 - slowed) + rate / factor * slowed
        magnitude = float(how.pop("magnitude", 0.1 * math.log(factor) + 1.0))
    if how:
        raise RuntimeError(f"unknown settings {sorted(how)} of {kind} scaling")
    angle = torch.arange(limit, device=device, dtype=torch.float64)[:, None] * rate
    return (torch.stack([angle.cos(), angle.sin()], -1) * magnitude).float()


def rotary(q, k, positions, table, interleaved=False, q_norm=None, k_norm=None, eps=1e-6):
    """(q, k) [tokens, heads, dim] with each head normalised (x * rsqrt(mean(x^2) + eps) * norm, where there is one) and its first
    2 * table.shape[1] elements rotated: pairs (i, i + half), or (2 i, 2 i + 1) if `interleaved`.  Inputs may be views, e.g. of the fused projection's output.

    positions int32 / int64 [tokens]; one outside the table gives NaN in the rotated elements.  Serving only: no gradient is recorded."""
    return capi.rotary_cache(q, k, None, positions, table, None, None, interleaved, q_norm, k_norm, eps)


def rotary_cache_write(q, k, v, positions, table, cache, slots, interleaved=False, q_norm=None, k_norm=None, eps=1e-6):
    """`rotary` of q and k, with k and v going into the cache at `slots` (int32 / int64 [tokens], distinct; outside the cache: not written) in the
    cache's type: -> q.  Keys are rounded once, from the rotated 32-bit values."""
    return capi.rotary_cache(q, k, v, positions, table, cache, slots, interleaved, q_norm, k_norm, eps)[0]
