"""Attention over a cache held in 4 bits where numbers, scales or lengths are unusual."""
import math

import pytest
import torch

import plain_int4 as plain
from cisr_b200.ops import kernels
from cisr_b200.ops.kernels import KernelError
from test_int4_cache_gpu import Cache, bound, i32, prompt_bound, queries

pytestmark = pytest.mark.gpu


def portions(cache, q, q_len, span, scale, **kw):
    """Every request's portion, in tiles of `span`."""
    starts = [sum(q_len[:r]) for r in range(len(q_len))]
    pairs = [(r, a) for r, n in enumerate(q_len) for a in range(0, n, span)]
    out = torch.full_like(q, 7.0)
    kernels.attn_prefill_int4(q, out, cache.k_cache, cache.v_cache, cache.slots, cache.table, i32([r for r, _ in pairs]), i32([a for _, a in pairs]), i32(starts), i32(q_len),
                              cache.ctx, max(cache.lens), cache.page, scale, span=span, **kw)
    kernels.raise_if_kernel_gave_up()
    return out


def check_portions(cache, q, got, q_len, span, scale, sink=None):
    at = 0
    for r, n in enumerate(q_len):
        want, size, p = plain.attention(q[at:at + n], *cache.held(r), scale, plain.seen(n, cache.lens[r]), sink)
        off = (got[at:at + n].double() - want).abs()
        most = bound(q.dtype, want, size, plain.stepped(p, cache.v[r]) if span == 64 else 0) + prompt_bound(q.dtype, span) * size
        assert (off <= most).all(), (r, float(torch.nan_to_num(off / most, 1e9).max()))
        at += n


@pytest.mark.parametrize("dim,span", [(64, 128), (64, 256), (128, 128), (128, 256), (96, 64), (32, 64)])
@pytest.mark.parametrize("size,scale", [(1.0, 0.125), (1e-4, 0.125), (1e-5, 1e-3), (1.0, 1e-19), (1e-4, 1e-30), (1.0, 0.0)])
def test_queries_of_zeros(dim, span, size, scale):
    """The mean of what such a row sees, whatever the sizes of keys and scale, with keys out of sight among a tile's."""
    hq, hkv = 4, 2
    lens, q_len = [300, 130], [200, 130]
    g = torch.Generator(device="cuda").manual_seed(3)
    k = [torch.randn((n, hkv, dim), generator=g, device="cuda") * size for n in lens]
    cache = Cache(lens, hkv, dim, 16, k=k, v=[torch.randn((n, hkv, dim), generator=g, device="cuda") for n in lens])
    q = queries(sum(q_len), hq, dim, torch.bfloat16)
    q[::3] = 0
    q[1::3, 1] = 0
    check_portions(cache, q, portions(cache, q, q_len, span, scale), q_len, span, scale)


@pytest.mark.parametrize("dtype,dim,span", [(torch.bfloat16, 64, 128), (torch.bfloat16, 128, 256), (torch.bfloat16, 32, 64), (torch.float32, 64, 64)])
@pytest.mark.parametrize("scale", [-0.125, -2.0, -1e-19, 3.0, 0.0])
@pytest.mark.parametrize("sink", [None, 0.5])
def test_scales_of_either_sign(dtype, dim, span, scale, sink):
    hq, hkv = 4, 2
    lens, q_len = [300, 130], [200, 130]
    cache = Cache(lens, hkv, dim, 16)
    q = queries(sum(q_len), hq, dim, dtype, std=1.0 if abs(scale) < 1 else 0.1)
    check_portions(cache, q, portions(cache, q, q_len, span, scale, sink=sink), q_len, span, scale, sink)


@pytest.mark.parametrize("scale", [math.inf, -math.inf, math.nan, 1e39])
def test_scales_that_are_no_numbers_are_refused(scale):
    for dtype, span in ((torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)):
        cache = Cache([20], 2, 64, 16)
        q = queries(3, 4, 64, dtype)
        with pytest.raises(KernelError):
            portions(cache, q, [3], span, scale)
        with pytest.raises(KernelError):
            cache.attend(q, [3], scale=scale)
    kernels.raise_if_kernel_gave_up()


def test_tile_lists_have_the_same_length_and_place():
    cache = Cache([300, 40], 2, 64, 16)
    q = queries(100, 4, 64, torch.bfloat16)
    one, two = i32([0]), i32([0, 0])
    for req, q0 in ((two, one), (one, two), (two.cpu(), two), (two, two.cpu()), (two[None], two[None]), (two.long(), two), (two, i32([0, 0, 0, 0])[::2])):
        with pytest.raises(KernelError):
            kernels.attn_prefill_int4(q, torch.empty_like(q), cache.k_cache, cache.v_cache, cache.slots, cache.table, req, q0, i32([0, 60]), i32([60, 40]), cache.ctx, 300, 16, 0.125,
                                      span=128)
    kernels.raise_if_kernel_gave_up()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 64), (8, 2, 128), (4, 2, 96)])
@pytest.mark.parametrize("n", [1, 3, 5])
@pytest.mark.parametrize("large,small", [(2000.0, 1e-3), (4e5, 1.0), (60.0, 1e-2)])
def test_a_large_group_among_small_ones(dtype, hq, hkv, dim, n, large, small):
    """One key of a tile has a large group of 32 values; every other group is held and weighed as exactly as beside small ones."""
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = torch.randn((2, 700, hkv, dim), generator=g, device="cuda")
    v = v * small
    v[100, :, 32:64] = large * torch.randn((hkv, 32), generator=g, device="cuda")
    v[650, 0, :32] = large
    q = queries(n, hq, dim, dtype)
    for again in (False, True):
        if again:
            k[100] = -3 * q[0, ::hq // hkv].float()              # the key itself has next to no weight with some rows, and all of it with others
        cache = Cache([700], hkv, dim, 16, k=[k], v=[v])
        out, size, p = plain.attention(q, *cache.held(0), dim ** -0.5, plain.seen(n, 700))
        # Float: the second float16 term of a product below 2^-14 is off by half of the smallest float16, 2^-25, which is 2^-34 of a weight times a
        # step since weights are held times 2^9, and codes are 7 at most: where one key takes nearly all the weight and has
        # code 0, that is what is left of the others.
        small = 0 if dtype == torch.bfloat16 else 7 * 700 * 2.0 ** -34
        off, most = (cache.attend(q, [n]).double() - out).abs(), bound(dtype, out, size, plain.stepped(p, cache.v[0])) + small
        assert (off <= most).all(), (again, float((off / most).max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2), (16, 2)])
@pytest.mark.parametrize("sink", [None, 0.3])
def test_tokens_that_see_nothing_give_no_weight(dtype, hq, hkv, sink):
    """More tokens than rows: the first ones lie before the first row, see nothing, give zeros and add nothing."""
    lens, q_len, dim, page = [3, 200, 1], [5, 6, 4], 64, 16
    cache = Cache(lens, hkv, dim, page)
    q = queries(sum(q_len), hq, dim, dtype)
    mass = torch.full((cache.pages, hkv, page), 0.25, device="cuda")
    got = cache.attend(q, q_len, mass=mass, sink=sink)
    at = 0
    for r, n in enumerate(q_len):
        blind = max(0, n - lens[r])
        assert not got[at:at + blind].any()
        ok = plain.seen(n, lens[r])[blind:]
        out, size, p = plain.attention(q[at + blind:at + n], *cache.held(r), dim ** -0.5, ok, sink)
        off = (got[at + blind:at + n].double() - out).abs()
        assert (off <= bound(dtype, out, size, plain.stepped(p, cache.v[r]))).all()
        sums = torch.cat([mass[i] for i in cache.table[r].tolist() if i >= 0], 1)[:, :lens[r]].double() - 0.25
        want = p.view(hkv, -1, lens[r]).sum(1)
        # weights as far off as `bound` says of scores, and float sums beside 0.25
        assert ((sums - want).abs() <= 2 * 70 * 8 * 2.0 ** -23 * want + 2.0 ** -22).all(), (r, sums, want)
        at += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lists_made_just_before_the_attention(monkeypatch, dtype):
    """With dependent launch: the call that gathers the listed requests' lists itself says so to the kernel (which must not read them before it
    waits), a call with lists from before does not, and replays follow the lists that the step makes."""
    hq, hkv, dim, page = 8, 2, 96, 16
    cache = Cache([300, 180, 90], hkv, dim, page)
    q = queries(60, hq, dim, dtype)
    q_len, q_start, which = i32([20, 30, 10]), i32([0, 20, 50]), i32([2, 0])
    tiles, places, out = i32([0]), i32([1, -9, 0]), torch.zeros_like(q)
    said = []
    pack = kernels._ATTN_INT4_CALL
    monkeypatch.setattr(kernels, "_ATTN_INT4_CALL", lambda *args: (said.append(args[-1]), pack(*args))[1])
    first = i32([0, 20, 50])

    def turn():
        q_start.copy_(first + 0)
        kernels.attn_prefill_int4(q, out, cache.k_cache, cache.v_cache, cache.slots, cache.table, tiles, tiles, q_start, q_len, cache.ctx, 300, page, dim ** -0.5, span=64,
                                  portions=(which, places))

    turn()
    kernels.attn_decode_int4(q, out, cache.k_cache, cache.v_cache, cache.slots, cache.table, q_start, q_len, cache.ctx, 30, 300, page, dim ** -0.5)
    assert said == [True, False]
    graph = torch.cuda.CUDAGraph()
    kernels.set_pdl(True)
    try:
        with torch.cuda.graph(graph):
            turn()
    finally:
        kernels.set_pdl(False)
    for listed in ([2, 0], [1, 2], [0, 0]):
        which.copy_(i32(listed))
        out.fill_(7.0)
        graph.replay()
        want = torch.full_like(q, 7.0)
        for r in set(listed):
            only = i32([n if i == r else 0 for i, n in enumerate((20, 30, 10))])
            kernels.attn_decode_int4(q, want, cache.k_cache, cache.v_cache, cache.slots, cache.table, first, only, cache.ctx, 60, 300, page, dim ** -0.5)
        assert torch.equal(out == 7, want == 7) and torch.allclose(out.float(), want.float(), rtol=2 ** -6, atol=2 ** -8)


def squared_errors(q, k, v, p, scale):
    """What the portions' float16 operands are off by in the mean square, [n, heads, dim], errors of one place independent of another's: a rounding is 2^-11 of
    a number at most and 2^-11 / sqrt 3 in the mean square (a bound for all mantissas).  Probabilities and values: as much of p v each.
    Keys: of every product q k of a score, and a score's error e turns p into p (1 + e - the mean of e): p (v - out) e."""
    u = 2.0 ** -22 / 3
    group = q.shape[1] // k.shape[0]
    k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    e = torch.einsum("nhd,hjd->hnj", q.double().square(), k.square()) * scale ** 2 * u
    out = torch.einsum("hnj,hjd->nhd", p, v)
    spread = torch.einsum("hnj,hjd->nhd", p.square() * e, v.square()) - 2 * out * torch.einsum("hnj,hjd->nhd", p.square() * e, v)
    spread += out.square() * (p.square() * e).sum(-1).transpose(0, 1)[..., None]
    return 2 * u * torch.einsum("hnj,hjd->nhd", p.square(), v.square()) + spread


@pytest.mark.parametrize("hq,hkv,dim,span", [(8, 2, 64, 128), (8, 2, 128, 128), (32, 8, 128, 256), (9, 3, 64, 256)])
@pytest.mark.parametrize("std", [0.3, 1.5, 3.0])
def test_portions_are_as_exact_as_their_operands(hq, hkv, dim, span, std):
    """In the mean square over each request: the output's own rounding, which is known to the digit, and what float16 operands add.  In a
    model on the CPU float16 operands are at 0.96 to 0.98 of the two; bfloat16 ones, eight times as coarse, at 1.27 and more (probabilities, queries of 0.3),
    1.3 (values) and 1.7 (keys, queries of 1.5 and more)."""
    lens, q_len = [1000, 300, 140], [290, 300, 40]
    cache = Cache(lens, hkv, dim, 16)
    q = queries(sum(q_len), hq, dim, torch.bfloat16, std=std)
    got = portions(cache, q, q_len, span, dim ** -0.5)
    at = 0
    for r, n in enumerate(q_len):
        held = cache.held(r)
        want, size, p = plain.attention(q[at:at + n], *held, dim ** -0.5, plain.seen(n, lens[r]))
        own = (want.to(torch.bfloat16).double() - want).square().mean()
        rest = squared_errors(q[at:at + n], *held, p, dim ** -0.5).mean()
        off = (got[at:at + n].double() - want).square().mean()
        assert off <= 1.1 ** 2 * (own + rest), (r, float((off / (own + rest)).sqrt()), float((own / want.square().mean()).sqrt()), float((rest / want.square().mean()).sqrt()))
        at += n


@pytest.mark.parametrize("dim,span", [(64, 128), (128, 256), (96, 64)])
@pytest.mark.parametrize("large,small", [(2000.0, 1e-3), (4e5, 1.0), (60.0, 1e-2)])
def test_portions_with_a_large_group_among_small_ones(dim, span, large, small):
    """Values down to 2^-28 of a key head's largest keep all their digits in float16 (its normal numbers reach from 2^-14 to 2^16)."""
    hq, hkv, scale = 8, 2, dim ** -0.5
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = torch.randn((2, 700, hkv, dim), generator=g, device="cuda")
    v = v * small
    v[100, :, 32:64] = large * torch.randn((hkv, 32), generator=g, device="cuda")
    v[650, 0, :32] = large
    cache = Cache([700], hkv, dim, 16, k=[k], v=[v])
    q = queries(200, hq, dim, torch.bfloat16)
    check_portions(cache, q, portions(cache, q, [200], span, scale), [200], span, scale)


@pytest.mark.parametrize("dim,span", [(64, 128), (128, 256)])
def test_tiles_of_requests_that_are_not_listed_are_reported(dim, span):
    """They are left alone, and the listed ones come out as they do alone."""
    hq, hkv = 4, 2
    cache = Cache([300, 200, 90], hkv, dim, 16)
    q = queries(120, hq, dim, torch.bfloat16)
    lists = (i32([0, 50, 90]), i32([50, 40, 30]), cache.ctx, 300, 16, dim ** -0.5)
    outs = []
    for tiles, places in (([0, 1, 2], [-1, 0, 5]), ([1], [-1, 0, -1])):
        out = torch.full_like(q, 7.0)
        kernels.attn_prefill_int4(q, out, cache.k_cache, cache.v_cache, cache.slots, cache.table, i32(tiles), i32([0] * len(tiles)), *lists, span=span,
                                  portions=(i32([1]), i32(places)))
        if len(tiles) == 3:
            with pytest.raises(KernelError, match="not among the portions"):
                kernels.raise_if_kernel_gave_up()
        kernels.raise_if_kernel_gave_up()
        assert (out[:50] == 7).all() and (out[90:] == 7).all()
        outs.append(out)
    assert torch.equal(*outs)
