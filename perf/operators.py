"""The operators of a cache held in 4 bits, as they are measured: storing keys and values, attention over them, the weight that
attention has given each key, and the eviction of the keys that had least of it.

Kinds of cases (`run` is one pass of each):

  store      new keys and values of a step go into the paged cache and are handed back as the cache holds them
  decode     attention of a few new tokens per request over its cache: one token (a decode step) or several (a drafted
             continuation that is checked in one step)
  weigh      the same for a decode step that also adds every key's attention weights to its sum
  prompt     attention of portions of prompts behind a history in the cache
  evict      of every request's rows the first, the latest and the weightiest go to new pages with their sums; the rows are
             handed back as values

A value is held as c s: s the largest magnitude of its 32 neighbours along the head times 1/7 (in float), rounded to float16 (at most 65504),
c = x / s rounded to the nearest whole number, at most 7 in size.  A page of one key head holds blocks of 8 rows: 8 rows of
4-bit codes c + 8, then the scales.  `places` says where in a block a code and a scale are.

Inputs are seeded: keys with channels of uneven spread, values normal, weight sums of uneven size.
"""
from __future__ import annotations

import math

import torch

own = False

# query heads, key heads, head size: the shapes of the presets, and layouts between and beside them
LAYOUTS = {"smollm2-135m": (9, 3, 64), "smollm2-1.7b": (32, 32, 64), "llama-3.1-8b": (32, 8, 128), "one key head": (16, 1, 128),
           "head size 32": (8, 4, 32), "head size 96": (12, 2, 96)}
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
GROUP, BLOCK = 32, 8


def listed():
    return [
        # a decode step of three users on the smallest shape: latency
        {"name": "store 3 tokens 135m", "kind": "store", "layout": "smollm2-135m", "requests": 3, "tokens": 1, "before": 200, "page": 16, "dtype": "bfloat16"},
        # the float mode of the engine, a portion of no round length behind an earlier one
        {"name": "store 700 135m float", "kind": "store", "layout": "smollm2-135m", "requests": 2, "tokens": 351, "before": 77, "page": 16, "dtype": "float32"},
        # whole prompts on the largest shape
        {"name": "store 4 x 2048 8b", "kind": "store", "layout": "llama-3.1-8b", "requests": 4, "tokens": 2048, "before": 0, "page": 16, "dtype": "bfloat16"},
        # one user of the smallest shape: latency
        {"name": "decode 1 x 700 135m", "kind": "decode", "layout": "smollm2-135m", "requests": 1, "tokens": 1, "context": 700, "page": 16, "dtype": "bfloat16"},
        # the float mode, as many key heads as query heads
        {"name": "decode 5 x 1500 1.7b float", "kind": "decode", "layout": "smollm2-1.7b", "requests": 5, "tokens": 1, "context": 1500, "page": 16, "dtype": "float32"},
        # a server's decode step: many users, long contexts of mixed length
        {"name": "decode 64 x 8000 8b", "kind": "decode", "layout": "llama-3.1-8b", "requests": 64, "tokens": 1, "context": 8000, "page": 16, "dtype": "bfloat16"},
        # drafted tokens checked in one step
        {"name": "decode 8 x 5 behind 3000 8b", "kind": "decode", "layout": "llama-3.1-8b", "requests": 8, "tokens": 5, "context": 3005, "page": 16, "dtype": "bfloat16"},
        # a decode step that keeps account of what is looked at
        {"name": "weigh 32 x 4000 8b", "kind": "weigh", "layout": "llama-3.1-8b", "requests": 32, "tokens": 1, "context": 4000, "page": 16, "dtype": "bfloat16"},
        {"name": "weigh 3 x 600 135m float", "kind": "weigh", "layout": "smollm2-135m", "requests": 3, "tokens": 1, "context": 600, "page": 16, "dtype": "float32"},
        # portions of prompts behind a history
        {"name": "prompt 2 x 1000 behind 2500 8b", "kind": "prompt", "layout": "llama-3.1-8b", "requests": 2, "tokens": 1000, "context": 3500, "page": 16, "dtype": "bfloat16"},
        # one user's cache cut down
        {"name": "evict 1 x 900 to 512 135m", "kind": "evict", "layout": "smollm2-135m", "requests": 1, "context": 900, "keep": 512, "page": 16, "dtype": "bfloat16"},
        # a server's caches cut down to half
        {"name": "evict 24 x 4096 to 2048 8b", "kind": "evict", "layout": "llama-3.1-8b", "requests": 24, "context": 4096, "keep": 2048, "page": 16, "dtype": "bfloat16"},
    ]


def spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["store", "decode", "decode", "decode", "weigh", "prompt", "evict"])
    layout = rng.choice(["smollm2-135m", "smollm2-1.7b", "llama-3.1-8b", "llama-3.1-8b", "one key head", "head size 32", "head size 96"])
    heads = LAYOUTS[layout][1] * LAYOUTS[layout][2]
    case = {"kind": kind, "layout": layout, "page": rng.choice([8, 16, 16, 16, 24, 64]), "dtype": "float32" if rng.random() < 0.2 else "bfloat16"}
    if kind == "store":
        case.update(requests=spread(rng, 1, 32), before=rng.choice([0, spread(rng, 1, 2000)]))
        case["tokens"] = spread(rng, 1, max(1, min(4096, 8 * 1024 * 1024 // (heads * case["requests"]))))
        return case
    case["requests"] = spread(rng, 1, 64)
    most = max(64, min(16000, 300 * 1024 * 1024 // (heads * case["requests"])))     # rows a request may have
    if kind == "prompt":
        case["requests"] = rng.randint(1, 4)
        case["tokens"] = spread(rng, 17, 1500 if case["dtype"] == "bfloat16" else 400)
        case["context"] = case["tokens"] + rng.choice([0, spread(rng, 1, 2500)])
    elif kind == "evict":
        case["context"] = spread(rng, 40, max(64, min(6000, 44 * 1024 * 1024 // (heads * case["requests"]))))
        case["keep"] = max(16, int(case["context"] * rng.uniform(0.2, 0.95)))
    else:
        case["tokens"] = 1 if kind == "weigh" or rng.random() < 0.7 else rng.randint(2, 8)
        case["context"] = max(case["tokens"], spread(rng, 1, most // 2 if kind == "weigh" else most))
        if case["dtype"] == "float32":
            case["requests"] = min(16, case["requests"])
    if kind != "evict" and rng.random() < 0.2:
        case["window"] = spread(rng, 1, 2000)
    return case


# ---------------------------------------------------------------- sizes
def contexts(case):
    """Rows in each request's cache, this step's included: half to all of the longest, mixed, and never fewer than the step brings."""
    n, longest = case["requests"], case["context"]
    return [max(case.get("tokens", 1), longest - (longest // 2) * ((7 * i) % n) // n) for i in range(n)]


def portions(case):
    if case["kind"] == "store":          # uneven shares, the first whole
        return [max(1, case["tokens"] - (case["tokens"] // 3) * ((5 * i) % case["requests"]) // case["requests"]) for i in range(case["requests"])]
    return [case.get("tokens", 0)] * case["requests"]


def ends(case):
    if case["kind"] == "store":
        return [n + (case["before"] * (2 + i) // (1 + case["requests"])) for i, n in enumerate(portions(case))]
    return contexts(case)


def first_and_recent(case):
    """Rows that stay whatever their weight: the sequence's first, and the latest."""
    return min(4, case["keep"] // 4), case["keep"] // 4


def page_bytes(case):
    return case["page"] * 9 * LAYOUTS[case["layout"]][2] // 16


# ---------------------------------------------------------------- the packed form
def places(dim, values, device):
    """Where a block of 8 rows keeps a code (in half bytes) and a scale (in float16 numbers behind the codes): [8, dim] and [8, dim / 32].
    Keys: the 8 codes of a 32-bit word are 8 neighbours, and a quarter of a row has one word of every group of 32.
    Values: the even rows come first; the 4 codes of a 16-bit half are 4 neighbours, an eighth of a row has one half of every group,
    and at head size 128 the eighths of every other pair of rows are exchanged four by four; scales of two rows lie side by side."""
    row = torch.arange(BLOCK, device=device)[:, None]
    d = torch.arange(dim, device=device)[None, :]
    groups = dim // GROUP
    group, within = d // GROUP, d % GROUP
    g = torch.arange(groups, device=device)[None, :]
    if not values:
        return row * dim + ((within // 8) * groups + group) * 8 + within % 8, row * groups + g
    slot = row // 2 + 4 * (row % 2)
    eighth = within // 4
    if dim == 128:
        eighth = eighth ^ (4 * ((slot // 2) % 2))
    return slot * dim + (eighth * groups + group) * 4 + within % 4, ((row // 2) * groups + g) * 2 + row % 2


def pack(codes, scales, values):
    """codes [..., rows, dim] (-7 to 7) and scales [..., rows, dim / 32] as the bytes of whole blocks, rows a multiple of 8."""
    lead, rows, dim = codes.shape[:-2], codes.shape[-2], codes.shape[-1]
    at, scale_at = places(dim, values, codes.device)
    nibbles = torch.empty(*lead, rows // BLOCK, BLOCK * dim, dtype=torch.uint8, device=codes.device)
    nibbles[..., at.reshape(-1)] = (codes + 8).to(torch.uint8).reshape(*lead, rows // BLOCK, BLOCK * dim)
    held = torch.empty(*lead, rows // BLOCK, BLOCK * (dim // GROUP), dtype=torch.float16, device=codes.device)
    held[..., scale_at.reshape(-1)] = scales.reshape(*lead, rows // BLOCK, -1)
    return torch.cat((nibbles[..., 0::2] | (nibbles[..., 1::2] << 4), held.view(torch.uint8)), dim=-1)


def unpack(blocks, dim, values):
    """The values [..., rows, dim] in float that blocks [..., n, 9 dim / 2] of bytes stand for."""
    at, scale_at = places(dim, values, blocks.device)
    code, scale = blocks[..., :4 * dim], blocks[..., 4 * dim:].contiguous().view(torch.float16)
    nibbles = torch.stack((code & 15, code >> 4), dim=-1).flatten(-2)
    codes = nibbles[..., at.reshape(-1)].float() - 8
    lead, n = blocks.shape[:-2], blocks.shape[-2]
    scales = scale[..., scale_at.reshape(-1)].float().reshape(*lead, n * BLOCK, dim // GROUP, 1)
    return (codes.reshape(*lead, n * BLOCK, dim // GROUP, GROUP) * scales).flatten(-2)


def quantized(x):
    """x [..., dim] as codes and scales."""
    groups = x.unflatten(-1, (-1, GROUP))
    top = groups.abs().amax(-1).float()
    scales = (top * (1 / 7)).clamp(max=65504.0).to(torch.float16)
    held = scales.double()[..., None]
    codes = torch.where(held > 0, (groups.double() / held).round().clamp(-7, 7), torch.zeros_like(held))
    return codes.flatten(-2), scales


# ---------------------------------------------------------------- inputs, made from the seed alone
def normal(shape, seed, stream, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + stream)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def keys_like(shape, seed, stream, dtype):
    """Normal numbers whose channels have spreads of their own, a few of them much wider."""
    wide = 0.5 + normal((shape[-1],), 1, 77).abs()
    wide[::29] *= 4
    return (normal(shape, seed, stream) * wide).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def tiles(case):
    """Queries of the prompts as (request, first query) in tiles of `span`, a portion's last tile first."""
    hq, _, dim = LAYOUTS[case["layout"]]
    span = 64
    if case["dtype"] == "bfloat16" and dim in (64, 128):
        span = 256 if sum(-(-n // 128) for n in portions(case)) * hq > 148 else 128
    pairs = [(r, q0) for r, n in enumerate(portions(case)) for q0 in range((n - 1) // span * span, -1, -span)]
    return span, i32([r for r, _ in pairs]), i32([q for _, q in pairs])


def prepare(case, seed):
    hq, hkv, dim = LAYOUTS[case["layout"]]
    dtype, page, kind = DTYPES[case["dtype"]], case["page"], case["kind"]
    lens, new = ends(case), portions(case)
    n, longest = len(lens), max(lens)
    width = -(-longest // page)
    per = [-(-c // page) for c in lens]
    fresh = [-(-min(c, case["keep"]) // page) for c in lens] if kind == "evict" else []
    total = sum(per) + sum(fresh)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32)
    at = 0
    for r, k in enumerate(per):
        table[r, :k] = order[at:at + k]
        at += k
    q_start = [sum(new[:r]) for r in range(n)]
    state = dict(case, kind=kind, lens=lens, longest=longest, dim=dim, hq=hq, hkv=hkv, scale=dim ** -0.5, dtype=dtype,
                 req_slot=i32(list(range(n))), block_table=table.cuda(), ctx_len=i32(lens), q_start=i32(q_start), q_len=i32(new))
    state["k_cache"] = torch.empty((total, hkv, page_bytes(case)), dtype=torch.uint8, device="cuda")
    state["v_cache"] = torch.empty_like(state["k_cache"])
    step = max(1, (1 << 25) // (hkv * page * dim))
    for values, cache in ((False, state["k_cache"]), (True, state["v_cache"])):
        for a in range(0, total, step):
            m = min(step, total - a)
            rows = (m, hkv, page, dim)
            x = normal(rows, seed, 100 + 2 * a + 1, dtype) if values else keys_like(rows, seed, 100 + 2 * a, dtype)
            cache[a:a + m] = pack(*quantized(x), values).flatten(-2)
    tokens = sum(new)
    if kind == "store":
        # keys and values as one projection leaves them: rows of both side by side
        rows = torch.empty((tokens, 2, hkv, dim), dtype=dtype, device="cuda")
        rows[:, 0] = keys_like((tokens, hkv, dim), seed, 1, dtype)
        rows[:, 1] = normal((tokens, hkv, dim), seed, 2, dtype)
        state.update(k=rows[:, 0], v=rows[:, 1], token_req=i32([r for r, m in enumerate(new) for _ in range(m)]),
                     positions=i32([c - m + i for c, m in zip(lens, new) for i in range(m)]))
    elif kind != "evict":
        state["q"] = (normal((tokens, hq, dim), seed, 3) * 1.5).to(dtype)
        state["queries"] = max(new)
    if kind in ("weigh", "evict"):
        state["mass"] = (normal((total, hkv, page), seed, 4) * 1.5).exp()
    if kind == "evict":
        to = torch.full((n, max(fresh)), -1, dtype=torch.int32)
        for r, k in enumerate(fresh):
            to[r, :k] = order[at:at + k]
            at += k
        state["to_table"] = to.cuda()
        state["new_len"] = i32([min(c, case["keep"]) for c in lens])
    if kind == "prompt":
        state["span"], state["tile_req"], state["tile_q0"] = tiles(case)
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        return run_own(state)
    return {"store": plain_store, "decode": plain_attention, "weigh": plain_attention, "prompt": plain_attention, "evict": plain_evict}[state["kind"]](state)


def run_own(s):
    from cisr_b200.ops import kernels

    kind, page = s["kind"], s["page"]
    cache = (s["k_cache"], s["v_cache"])
    if kind == "store":
        kernels.int4_store(s["k"], s["v"], *cache, s["token_req"], s["positions"], s["req_slot"], s["block_table"], page)
        k_out, v_out = torch.empty(s["k"].shape, dtype=s["dtype"], device="cuda"), torch.empty(s["v"].shape, dtype=s["dtype"], device="cuda")
        kernels.int4_read(*cache, k_out, v_out, s["token_req"], s["positions"], s["req_slot"], s["block_table"], page)
        return k_out, v_out
    if kind == "evict":
        first, recent = first_and_recent(s)
        kept = torch.empty((s["requests"], s["hkv"], s["keep"]), dtype=torch.int32, device="cuda")
        kernels.int4_evict(*cache, s["mass"], s["req_slot"], s["block_table"], s["ctx_len"], s["to_table"], kept, page, s["longest"], recent, first)
        shape = (s["requests"], s["hkv"], s["keep"], s["dim"])
        k_out, v_out = torch.empty(shape, dtype=s["dtype"], device="cuda"), torch.empty(shape, dtype=s["dtype"], device="cuda")
        kernels.int4_expand(*cache, k_out, v_out, s["req_slot"], s["to_table"], s["new_len"], page)
        return kept, s["mass"], k_out, v_out
    out = torch.empty_like(s["q"])
    if kind == "prompt":
        kernels.attn_prefill_int4(s["q"], out, *cache, s["req_slot"], s["block_table"], s["tile_req"], s["tile_q0"], s["q_start"], s["q_len"],
                                  s["ctx_len"], s["longest"], page, s["scale"], s.get("window"), span=s["span"])
        return out
    kernels.attn_decode_int4(s["q"], out, *cache, s["req_slot"], s["block_table"], s["q_start"], s["q_len"], s["ctx_len"], s["queries"], s["longest"],
                             page, s["scale"], s.get("window"), mass=s.get("mass"))
    return (out, s["mass"]) if kind == "weigh" else out


def rows_of(s, cache, values, table, rows):
    """The first `rows` rows of every request in `table`, [requests, key heads, rows, dim] in float; nothing where there is no page."""
    pages = cache[table.clamp(min=0).long()]                                        # [requests, width, key heads, bytes]
    blocks = pages.unflatten(-1, (s["page"] // BLOCK, -1)).transpose(1, 2).flatten(2, 3)
    return unpack(blocks, s["dim"], values)[:, :, :rows]


def plain_store(s):
    req = s["token_req"].long()
    page = s["block_table"][req, s["positions"].long() // s["page"]].long()
    row = s["positions"].long() % s["page"]
    out = []
    for values, x, cache in ((False, s["k"], s["k_cache"]), (True, s["v"], s["v_cache"])):
        codes, scales = quantized(x)
        at, scale_at = places(s["dim"], values, x.device)
        # a row's codes are whole bytes of its block, and its scales whole float16 numbers
        mine, mine_scale = at[row % BLOCK], scale_at[row % BLOCK]                    # [tokens, dim], [tokens, groups]
        order = mine.argsort(-1)
        nibbles = (codes + 8).to(torch.uint8).gather(-1, order[:, None].expand_as(codes))
        bytes_ = nibbles[..., 0::2] | (nibbles[..., 1::2] << 4)
        byte_at = mine.gather(-1, order)[:, 0::2] // 2
        block = (row // BLOCK * (9 * s["dim"] // 2))[:, None]
        head = torch.arange(s["hkv"], device=x.device)[None, :, None]
        cache[page[:, None, None], head, (block + byte_at)[:, None]] = bytes_
        two = (4 * s["dim"] + 2 * mine_scale)[..., None] + torch.arange(2, device=x.device)
        cache[page[:, None, None], head, (block + two.flatten(-2))[:, None]] = scales.contiguous().view(torch.uint8)
        held = cache[page[:, None, None], head, (block + byte_at)[:, None]]
        back = torch.stack((held & 15, held >> 4), -1).flatten(-2).float() - 8
        back = back.gather(-1, order.argsort(-1)[:, None].expand_as(back))
        held = cache[page[:, None, None], head, (block + two.flatten(-2))[:, None]].contiguous().view(torch.float16).float()
        out.append((back.unflatten(-1, (-1, GROUP)) * held[..., None]).flatten(-2).to(s["dtype"]))
    return tuple(out)


def plain_attention(s):
    n, most, longest = s["requests"], max(1, s["queries"]), s["longest"]
    k = rows_of(s, s["k_cache"], False, s["block_table"], longest)
    v = rows_of(s, s["v_cache"], True, s["block_table"], longest)
    group = s["hq"] // s["hkv"]
    i = torch.arange(most, device=k.device)
    token = s["q_start"].long()[:, None] + i[None, :].minimum(s["q_len"].long()[:, None] - 1)
    q = s["q"].float()[token].view(n, most, s["hkv"], group, s["dim"]).permute(0, 2, 1, 3, 4).flatten(2, 3)
    scores = torch.matmul(q, k.transpose(-1, -2)).unflatten(2, (most, group)) * s["scale"]       # [n, hkv, queries, group, keys]
    at = (s["ctx_len"] - s["q_len"]).long()[:, None] + i[None, :]
    j = torch.arange(longest, device=k.device)
    seen = j <= at[..., None]
    if s.get("window"):
        seen &= at[..., None] - j < s["window"]
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), v).unflatten(2, (most, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    out = out[i[None, :] < s["q_len"].long()[:, None]].to(s["dtype"])
    if s["kind"] != "weigh":
        return out
    weight = torch.nn.functional.pad(p.sum((2, 3)), (0, s["block_table"].shape[1] * s["page"] - longest)).unflatten(2, (-1, s["page"])).transpose(1, 2)
    held = s["block_table"] >= 0
    pages = s["block_table"][held].long()
    s["mass"][pages] = s["mass"][pages] + weight[held]
    return out, s["mass"]


def plain_evict(s):
    first, recent = first_and_recent(s)
    longest, keep = s["longest"], s["keep"]
    mass = s["mass"][s["block_table"].clamp(min=0).long()].transpose(1, 2).flatten(2, 3)[..., :longest]       # [n, hkv, rows]
    j = torch.arange(longest, device=mass.device)
    lens = s["ctx_len"].long()[:, None, None]
    rank = torch.where((j < first) | (j >= lens - recent), math.inf, mass).masked_fill(j >= lens, -1.0)
    best = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    alive = rank.gather(-1, best) >= 0
    place = torch.where(alive, best, longest).sort(-1).values
    place = torch.nn.functional.pad(place, (0, keep - place.shape[-1]), value=longest)
    kept = torch.where(place < longest, place, -1).to(torch.int32)
    at = kept.clamp(min=0).long()
    out = []
    for values, cache in ((False, s["k_cache"]), (True, s["v_cache"])):
        rows = rows_of(s, cache, values, s["block_table"], longest)
        rows = rows.gather(2, at[..., None].expand(-1, -1, -1, s["dim"]))
        out.append(torch.where(kept[..., None] >= 0, rows, 0).to(s["dtype"]))
    width = s["to_table"].shape[1] * s["page"]
    new = torch.nn.functional.pad(torch.where(kept >= 0, mass.gather(-1, at), 0), (0, width - keep))
    valid = torch.nn.functional.pad(kept, (0, width - keep), value=-1) >= 0
    new, valid = (t.unflatten(2, (-1, s["page"])).transpose(1, 2) for t in (new, valid))                      # [n, pages, hkv, page]
    held = s["to_table"] >= 0
    pages = s["to_table"][held].long()
    s["mass"][pages] = torch.where(valid[held], new[held], s["mass"][pages])
    return kept, s["mass"], out[0], out[1]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    hq, hkv, dim = LAYOUTS[case["layout"]]
    size = 4 if case["dtype"] == "float32" else 2
    row = 2 * hkv * dim                                             # values of one cache row, keys and values
    held = row * 9 / 16
    lens, new = ends(case), portions(case)
    tokens = sum(new)
    if case["kind"] == "store":
        return {"bytes": tokens * (2 * row * size + 2 * held), "flops": 4 * tokens * row}
    if case["kind"] == "evict":
        kept = sum(min(c, case["keep"]) for c in lens)
        return {"bytes": sum(lens) * hkv * 4 + kept * (3 * held + row * size + 8 * hkv), "flops": kept * row}
    window = case.get("window")
    reach = sum(c if not window else min(c, window + n - 1) for c, n in zip(lens, new))
    pairs = sum(sum(min(c - n + i + 1, window or c) for i in range(n)) for c, n in zip(lens, new))
    weights = 8 * hkv * reach if case["kind"] == "weigh" else 0
    return {"bytes": reach * held + 2 * tokens * hq * dim * size + weights, "flops": 4 * hq * dim * pairs}


# ---------------------------------------------------------------- the same from the definitions, in 64 bits
def nearest(x):
    """What 4 bits hold of x [..., dim], in 64 bits: the definition of the format, group by group."""
    x = x.double().unflatten(-1, (-1, GROUP))
    step = (x.abs().max(-1, keepdim=True).values.float() * (1.0 / 7.0)).to(torch.float16).double()
    step = torch.where(step.isinf(), torch.full_like(step, 65504.0), step)
    whole = torch.round(x / step).nan_to_num(0.0, 0.0, 0.0).clamp(-7.0, 7.0)
    return (whole * step).flatten(-2)


def exact_rows(state, request, cache, values, rows, table="block_table"):
    """A request's rows as values [key heads, rows, dim], read block by block with the places of codes and scales."""
    dim, page = state["dim"], state["page"]
    pages = [p for p in state[table][request].tolist() if p >= 0]
    raw = cache[pages].view(len(pages), state["hkv"], page // 8, 9 * dim // 2).permute(1, 0, 2, 3).reshape(state["hkv"], -1, 9 * dim // 2)
    at, scale_at = places(dim, values, raw.device)
    byte = raw[..., (at // 2).flatten()].view(*raw.shape[:2], 8, dim)
    code = torch.where(at % 2 == 1, byte >> 4, byte & 15).double() - 8.0
    scale = raw[..., 4 * dim:].contiguous().view(torch.float16)[..., scale_at.flatten()].view(*raw.shape[:2], 8, dim // 32).double()
    return (code * scale.repeat_interleave(32, dim=-1)).reshape(state["hkv"], -1, dim)[:, :rows]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        return nearest(s["k"]), nearest(s["v"])
    if case["kind"] == "evict":
        return exact_evict(case, s)
    outs, group = [], s["hq"] // s["hkv"]
    mass = s["mass"].double() if case["kind"] == "weigh" else None
    start = 0
    for r, (length, n) in enumerate(zip(s["lens"], portions(case))):
        k = exact_rows(s, r, s["k_cache"], False, length).repeat_interleave(group, 0)
        v = exact_rows(s, r, s["v_cache"], True, length).repeat_interleave(group, 0)
        got = torch.empty((n, s["hq"], s["dim"]), dtype=torch.float64, device=k.device)
        weight = torch.zeros((s["hkv"], length), dtype=torch.float64, device=k.device)
        for a in range(0, n, 128):
            b = min(n, a + 128)
            score = torch.einsum("qhd,hkd->hqk", s["q"][start + a:start + b].double(), k) * s["scale"]
            at = torch.arange(length - n + a, length - n + b, device=k.device)[:, None]
            key = torch.arange(length, device=k.device)[None, :]
            hidden = (key > at) | ((at - key >= case["window"]) if case.get("window") else torch.zeros_like(key > at))
            p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            got[a:b] = torch.einsum("hqk,hkd->qhd", p, v)
            weight += p.sum(1).view(s["hkv"], group, length).sum(1)
        outs.append(got)
        start += n
        if mass is not None:
            for i, p in enumerate(s["block_table"][r].tolist()):
                part = weight[:, i * s["page"]:(i + 1) * s["page"]]
                if part.shape[1]:
                    mass[p, :, :part.shape[1]] += part
    out = torch.cat(outs)
    return out if mass is None else (out, mass)


def exact_evict(case, s):
    first, recent = first_and_recent(case)
    keep, hkv, dim, page = case["keep"], s["hkv"], s["dim"], s["page"]
    mass = s["mass"].double()
    rows = [torch.zeros((len(s["lens"]), hkv, keep, dim), dtype=torch.float64, device=mass.device) for _ in range(2)]
    for r, length in enumerate(s["lens"]):
        own_mass = torch.cat([s["mass"][p].double() for p in s["block_table"][r].tolist() if p >= 0], dim=1)[:, :length]
        weight = own_mass.clone()
        weight[:, :first] = math.inf
        weight[:, max(0, length - recent):] = math.inf
        keys, values = exact_rows(s, r, s["k_cache"], False, length), exact_rows(s, r, s["v_cache"], True, length)
        for h in range(hkv):
            place = torch.sort(torch.sort(-weight[h], stable=True).indices[:keep]).values
            m = place.numel()
            rows[0][r, h, :m], rows[1][r, h, :m] = keys[h, place], values[h, place]
            for i in range(0, m, page):
                mass[int(s["to_table"][r, i // page]), h, :min(page, m - i)] = own_mass[h, place[i:i + page]]
    return None, mass, rows[0], rows[1]
