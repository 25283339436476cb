"""The operators of a cache held in 4 bits from their definitions, in 64 bits, one request and head at a time."""
import math

import torch

GROUP = 32


def held(x):
    """What 4 bits hold of x [..., dim]: groups of 32, step float16(largest * 1/7 in float), codes to the nearest whole number within -7 .. 7."""
    groups = x.double().unflatten(-1, (-1, GROUP))
    top = groups.abs().amax(-1, keepdim=True)
    step = (top.float() * (1 / 7)).clamp(max=65504.0).half().double()
    code = torch.where(step > 0, (groups / step).round().clamp(-7, 7), torch.zeros_like(groups))
    bad = ~torch.isfinite(top)
    return torch.where(bad, torch.full_like(groups, math.nan), code * step).flatten(-2)


def seen(n, ctx, window=None, keep_first=0):
    """[n, ctx] whether the n newest tokens of a sequence of ctx see its keys."""
    at = torch.arange(ctx - n, ctx)[:, None]
    j = torch.arange(ctx)[None, :]
    ok = j <= at
    return ok if window is None else ok & ((at - j < window) | (j < keep_first))


def weights(q, k, scale, ok, sink=None):
    """Softmax weights [heads, n, ctx] of q [n, heads, dim] over k [kv_heads, ctx, dim], masked by ok [n, ctx]."""
    group = q.shape[1] // k.shape[0]
    s = torch.einsum("nhd,hjd->hnj", q.double(), k.double().repeat_interleave(group, 0)) * scale
    s = s.masked_fill(~ok.to(s.device), -math.inf)
    top = s.amax(-1, keepdim=True)
    if sink is not None:
        sink = torch.as_tensor(sink, dtype=torch.float64, device=s.device).reshape(-1, 1, 1).expand(s.shape[0], 1, 1)
        top = torch.maximum(top, sink)
    e = (s - top).exp()
    den = e.sum(-1, keepdim=True) + (0 if sink is None else (sink - top).exp())
    return e / den


def attention(q, k, v, scale, ok, sink=None):
    """out [n, heads, dim], the same with |v| for v (what rounding errors are relative to), and the weights."""
    p = weights(q, k, scale, ok, sink)
    v = v.double().repeat_interleave(q.shape[1] // k.shape[0], 0)
    # a key out of sight takes no part, whatever is held there
    clean = torch.nan_to_num(v, 0.0, 0.0, 0.0)
    return torch.einsum("hnj,hjd->nhd", p, clean), torch.einsum("hnj,hjd->nhd", p, clean.abs()), p


def stepped(p, v):
    """sum over keys of weight times step, [n, heads, dim]: p [heads, n, rows] as `attention` gives it, v [rows, kv_heads, dim] as it was stored."""
    step = v.double().unflatten(-1, (-1, GROUP)).abs().amax(-1) / 7
    step = torch.nan_to_num(step, 0.0, 0.0, 0.0).repeat_interleave(GROUP, -1).transpose(0, 1).repeat_interleave(p.shape[0] // v.shape[1], 0)
    return torch.einsum("hnj,hjd->nhd", p, step)


def evicted(mass, keep, recent, first):
    """Places that stay of one head's sums, in order."""
    n = mass.numel()
    if n <= keep:
        return list(range(n))
    between = list(range(first, n - recent))
    value = lambda i: math.inf if math.isnan(float(mass[i])) else float(mass[i])
    nan = lambda i: math.isnan(float(mass[i]))
    best = sorted(between, key=lambda i: (not nan(i), -value(i), i))[:keep - first - recent]
    return sorted(list(range(first)) + best + list(range(n - recent, n)))
