"""A cache held in 4 bits against its definitions in 64 bits: rows in and out, attention and the weights it gives, eviction."""
import math

import pytest
import torch

import plain_int4 as plain
from cisr_b200.ops import kernels
from cisr_b200.ops.kernels import KernelError

pytestmark = pytest.mark.gpu

LAYOUTS = [(9, 3, 64), (8, 8, 32), (12, 2, 96), (32, 8, 128), (20, 1, 128)]


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Cache:
    """Pages in a shuffled order for requests of the given lengths; pages and steps of other owners hold NaN."""

    def __init__(self, lens, hkv, dim, page, seed=0, spare=3, k=None, v=None, dtype=torch.float32):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hkv, self.dim, self.page = lens, hkv, dim, page
        per = [-(-n // page) for n in lens]
        self.pages = sum(per) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        self.table = torch.full((len(lens), max(1, max(per))), -1, dtype=torch.int32)
        for r, n in enumerate(per):
            self.table[r, :n] = torch.tensor(order[:n])
            order = order[n:]
        self.free = order
        self.table = self.table.cuda()
        shape = (self.pages, hkv, kernels.int4_page_bytes(page, dim))
        self.k_cache = torch.full(shape, 0x7e, dtype=torch.uint8, device="cuda")       # steps 0x7e7e: NaN
        self.v_cache = self.k_cache.clone()
        self.slots = i32(list(range(len(lens))))
        self.ctx = i32(lens)
        cuda = torch.Generator(device="cuda").manual_seed(seed)
        self.k = [torch.randn((n, hkv, dim), generator=cuda, device="cuda").to(dtype) for n in lens] if k is None else k
        self.v = [torch.randn((n, hkv, dim), generator=cuda, device="cuda").to(dtype) for n in lens] if v is None else v
        for r, n in enumerate(lens):
            if n:
                self.store(r, 0, self.k[r], self.v[r])

    def store(self, r, start, k, v):
        n = k.shape[0]
        kernels.int4_store(k, v, self.k_cache, self.v_cache, i32([r] * n), i32(list(range(start, start + n))), self.slots, self.table, self.page)

    def held(self, r):
        """What is held of request r: keys and values [kv_heads, rows, dim] in 64 bits."""
        return plain.held(self.k[r]).transpose(0, 1), plain.held(self.v[r]).transpose(0, 1)

    def attend(self, q, q_len, longest=None, **kw):
        out = torch.full_like(q, 7.0)
        starts = [sum(q_len[:r]) for r in range(len(q_len))]
        kernels.attn_decode_int4(q, out, self.k_cache, self.v_cache, self.slots, self.table, i32(starts), i32(q_len), self.ctx, kw.pop("max_queries", max(q_len)),
                                 longest or max(self.lens), self.page, kw.pop("scale", self.dim ** -0.5), **kw)
        kernels.raise_if_kernel_gave_up()
        return out


def queries(tokens, hq, dim, dtype, seed=5, std=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((tokens, hq, dim), generator=g, device="cuda") * std).to(dtype)


def bound(dtype, out, size, steps=0):
    """bfloat16: the output's rounding, half of eps; the probability and its product with a step rounded to float16, half of its eps
    each; and scores, whose float sums of some 70 units of the softmax's exponent at most are 2^-23 of that off for each of 8 sums, so
    that a weight is 7e-5 off.  float: scores as before, probabilities of two float16 terms, 2^-22, and as much for the exponential.

    bfloat16 with single tokens, besides: the matrix instructions sum codes 0 .. 15 that are subnormal, n 2^-24, beside a
    product with 8, and align the products by exponent fields, 2^-14 for all of them, keeping 24 binary digits: every product is cut at
    2^-14 2^-24 = 2^-14 of a code's unit times its p s.  So both sums, 8 and n, are off by 2^-14 of sum p s at most, of sums of up to
    16 keys by one cut more for what was there: 2^-12 of `steps` = sum p s for the two is enough, and with code 0 against 8 - 8 of the
    weightiest key nothing of it shows in `size`."""
    score = 70 * 8 * 2.0 ** -23
    if dtype == torch.bfloat16:
        return torch.finfo(dtype).eps / 2 * out.abs() + (torch.finfo(torch.float16).eps + 2 * score) * size + 2.0 ** -12 * steps
    return (2 * score + 2.0 ** -21) * size + 1e-30


def check(cache, q, got, q_len, window=None, keep_first=0, sink=None, scale=None):
    at = 0
    for r, n in enumerate(q_len):
        if n:
            ok = plain.seen(n, cache.lens[r], window, keep_first)
            out, size, p = plain.attention(q[at:at + n], *cache.held(r), scale or cache.dim ** -0.5, ok, sink)
            off = (got[at:at + n].double() - out).abs()
            most = bound(q.dtype, out, size, plain.stepped(p, cache.v[r]))
            assert (off <= most).all(), (r, n, float((off / most).max()))
        at += n


# ------------------------------------------------------------------ rows
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hkv,dim", [(3, 64), (8, 128), (1, 32), (2, 96)])
@pytest.mark.parametrize("page", [8, 16, 40])
def test_rows_are_held_as_defined(hkv, dim, page, dtype):
    lens = [1, 45, 8, 0, 17]
    cache = Cache(lens, hkv, dim, page, dtype=dtype)
    for r, n in enumerate(lens):
        for into in (torch.float32, torch.bfloat16):
            k, v = torch.empty((2, n, hkv, dim), dtype=into, device="cuda")
            at = torch.randperm(n)
            kernels.int4_read(cache.k_cache, cache.v_cache, k, v, i32([r] * n), at.int().cuda(), cache.slots, cache.table, page)
            want_k, want_v = (plain.held(x[r])[at.cuda()].to(into) for x in (cache.k, cache.v))
            assert torch.equal(k, want_k) and torch.equal(v, want_v)


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_where_codes_and_steps_are(dim):
    """The bytes of a block, place by place."""
    page, groups = 16, dim // 32
    cache = Cache([page], 2, dim, page)
    raw = [c[cache.table[0, 0].item(), 1].cpu() for c in (cache.k_cache, cache.v_cache)]
    for values, bytes_, x in ((False, raw[0], cache.k[0]), (True, raw[1], cache.v[0])):
        want = plain.held(x[:, 1]).cpu()
        for row in (0, 3, 5, 8, 14):
            block, r = bytes_[row // 8 * (9 * dim // 2):][:9 * dim // 2], row % 8
            steps = block[4 * dim:].clone().view(torch.float16).double()
            for d in range(0, dim, 5):
                j, e = d // 32, d % 32
                if values:
                    slot = r // 2 + 4 * (r % 2)
                    eighth = (e // 4) ^ (4 if dim == 128 and slot // 2 % 2 else 0)
                    nibble, step = slot * dim + (eighth * groups + j) * 4 + e % 4, steps[(r // 2 * groups + j) * 2 + r % 2]
                else:
                    nibble, step = r * dim + (e // 8 * groups + j) * 8 + e % 8, steps[r * groups + j]
                code = (int(block[nibble // 2]) >> (4 * (nibble % 2)) & 15) - 8
                assert code * float(step) == float(want[row, d])


def test_numbers_of_every_kind():
    """Groups of zeros, of subnormals, of numbers that are cut, with infinities and NaN; quotients on a half and next to one."""
    dim, page = 128, 8
    x = torch.zeros((16, 1, dim))
    x[1] = torch.linspace(-1e-8, 1e-8, dim)                      # the step is a subnormal float16, then zero
    x[2] = 1e-42
    x[3] = torch.linspace(-1, 1, dim) * 3e38                     # magnitudes beyond 7 * 65504 are cut
    x[4] = torch.linspace(-5e5, 5e5, dim)
    x[5] = torch.randn(dim); x[5, 0, 40] = math.inf
    x[6] = torch.randn(dim); x[6, 0, 3] = -math.inf
    x[7] = torch.randn(dim); x[7, 0, 127] = math.nan
    x[8] = (torch.arange(dim) % 15 - 7) * 0.5                    # whole codes of step 0.5
    x[9] = ((torch.arange(dim) % 14) - 6.5) * 0.25; x[9, 0, ::32] = 1.75      # halves of step 0.25: ties
    x[10] = x[9] * (1 + 2.0 ** -23); x[10, 0, ::32] = 1.75
    x[11] = x[9] * (1 - 2.0 ** -24); x[11, 0, ::32] = 1.75
    x[12] = -x[10]
    x[13] = torch.randn(dim) * 1e-3
    x[14] = torch.randn(dim) * 1e4
    x[15] = torch.full((dim,), -0.0)
    x = x.cuda()
    cache = Cache([16], 1, dim, page, k=[x], v=[x])
    k, v = torch.empty((2, 16, 1, dim), device="cuda")
    kernels.int4_read(cache.k_cache, cache.v_cache, k, v, i32([0] * 16), i32(list(range(16))), cache.slots, cache.table, page)
    want = plain.held(x).float()
    assert torch.equal(torch.nan_to_num(k, 1234.5), torch.nan_to_num(want, 1234.5)) and torch.equal(torch.nan_to_num(v, 1234.5), torch.nan_to_num(want, 1234.5))
    assert torch.isnan(want[5:8]).any(-1).all() and torch.isfinite(want[:5]).all() and float(want[3].abs().max()) == 7 * 65504.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_million_quotients(dtype):
    """Every code of numbers of uneven size, next to halves among them, is the one that 64 bits give."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n, hkv, dim = 1024, 8, 128
    top = torch.rand((n, hkv, dim // 32, 1), generator=g, device="cuda") * 4 + 0.1
    step = (top / 7).half().float()
    whole = torch.randint(-7, 8, (n, hkv, dim // 32, 32), generator=g, device="cuda") + torch.randint(0, 2, (n, hkv, dim // 32, 32), generator=g, device="cuda") * 0.5
    x = step * whole * (1 + (torch.randint(-2, 3, whole.shape, generator=g, device="cuda") * 2.0 ** -23))
    x = torch.where(x.abs() > top, top, x)
    x[..., :1] = top
    x = x.flatten(-2).to(dtype)
    cache = Cache([n], hkv, dim, 16, k=[x], v=[-x])
    k, v = torch.empty((2, n, hkv, dim), device="cuda")
    kernels.int4_read(cache.k_cache, cache.v_cache, k, v, i32([0] * n), i32(list(range(n))), cache.slots, cache.table, 16)
    assert torch.equal(k, plain.held(x).float()) and torch.equal(v, plain.held(-x).float())


def test_strides_missing_pages_and_what_stays():
    """Rows out of a wider projection, at odd addresses too; a place without a page is left out, every other byte stays."""
    hkv, dim, page = 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn((5, 3 * hkv * dim + 3), generator=g, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        for shift in (0, 3):                                     # 3 numbers on: no wide loads
            rows = wide.to(dtype)[:, shift:]
            k, v = rows[:, :hkv * dim].unflatten(1, (hkv, dim)), rows[:, hkv * dim:2 * hkv * dim].unflatten(1, (hkv, dim))
            cache = Cache([20, 40], hkv, dim, page)
            cache.table[1, 2] = -1
            before = (cache.k_cache.clone(), cache.v_cache.clone())
            kernels.int4_store(k, v, cache.k_cache, cache.v_cache, i32([0, 1, 1, 0, 1]), i32([3, 33, 31, 17, 4000]), cache.slots, cache.table, page)
            got_k, got_v = torch.empty((2, 5, hkv, dim), device="cuda")
            kernels.int4_read(cache.k_cache, cache.v_cache, got_k, got_v, i32([0, 1, 1, 0, 1]), i32([3, 33, 31, 17, 4000]), cache.slots, cache.table, page)
            there = torch.tensor([True, False, True, True, False])
            assert torch.equal(got_k[there], plain.held(k)[there].float()) and torch.equal(got_v[there], plain.held(v)[there].float())
            assert not got_k[~there].any() and not got_v[~there].any()
            back_k, back_v = torch.empty((2, 3, hkv, dim), device="cuda")
            kernels.int4_read(*before, back_k, back_v, i32([0, 1, 0]), i32([3, 31, 17]), cache.slots, cache.table, page)
            # put the old rows back: the codes of held values are the codes they came from
            kernels.int4_store(cache.k[0][[3]], cache.v[0][[3]], cache.k_cache, cache.v_cache, i32([0]), i32([3]), cache.slots, cache.table, page)
            kernels.int4_store(cache.k[0][[17]], cache.v[0][[17]], cache.k_cache, cache.v_cache, i32([0]), i32([17]), cache.slots, cache.table, page)
            kernels.int4_store(cache.k[1][[31]], cache.v[1][[31]], cache.k_cache, cache.v_cache, i32([1]), i32([31]), cache.slots, cache.table, page)
            assert torch.equal(cache.k_cache, before[0]) and torch.equal(cache.v_cache, before[1])


def test_new_rows_have_no_weight_yet():
    cache = Cache([20, 30], 2, 64, 16)
    mass = torch.rand((cache.pages, 2, 16), device="cuda") + 1
    want = mass.clone()
    x = torch.randn((2, 2, 64), device="cuda")
    kernels.int4_store(x, x, cache.k_cache, cache.v_cache, i32([0, 1]), i32([19, 3]), cache.slots, cache.table, 16, mass=mass)
    want[cache.table[0, 1].item(), :, 3] = 0
    want[cache.table[1, 0].item(), :, 3] = 0
    assert torch.equal(mass, want)


@pytest.mark.parametrize("into", [torch.float32, torch.bfloat16])
def test_whole_requests(into):
    lens, hkv, dim, page = [0, 70, 24, 1], 2, 128, 24
    cache = Cache(lens, hkv, dim, page)
    k, v = torch.full((2, 4, hkv, 80, dim), 9.0, dtype=into, device="cuda")
    kernels.int4_expand(cache.k_cache, cache.v_cache, k, v, cache.slots, cache.table, cache.ctx, page)
    for r, n in enumerate(lens):
        want_k, want_v = cache.held(r)
        assert torch.equal(k[r, :, :n], want_k.to(into)) and torch.equal(v[r, :, :n], want_v.to(into)) and not k[r, :, n:].any() and not v[r, :, n:].any()
    some, _ = torch.full((2, 2, hkv, 80, dim), 9.0, dtype=into, device="cuda")
    kernels.int4_expand(cache.k_cache, cache.v_cache, some, some.clone(), cache.slots, cache.table, cache.ctx, page, requests=i32([2, 1]))
    assert torch.equal(some, k[[2, 1]])


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,dim", LAYOUTS)
@pytest.mark.parametrize("page", [8, 16, 24, 64])
def test_single_tokens(hq, hkv, dim, page, dtype):
    lens = [1, 7, 8, 9, 31, 32, 33, 127, 128, 129, 300, 2047, 2049]
    cache = Cache(lens, hkv, dim, page, seed=page)
    q = queries(len(lens), hq, dim, dtype)
    check(cache, q, cache.attend(q, [1] * len(lens)), [1] * len(lens))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,dim", [(9, 3, 64), (32, 8, 128)])
def test_several_tokens(hq, hkv, dim, dtype):
    lens, q_len = [5, 40, 1, 130, 257, 64, 900], [5, 3, 1, 16, 2, 0, 9]
    cache = Cache(lens, hkv, dim, 16)
    q = queries(sum(q_len), hq, dim, dtype)
    check(cache, q, cache.attend(q, q_len), q_len)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window,keep_first,sink", [(1, 0, None), (5, 0, 0.5), (64, 3, None), (100, 40, -2.0), (4000, 0, None), (None, 0, 1.5), (200, 150, None)])
def test_windows_and_sinks(window, keep_first, sink, dtype):
    hq, hkv, dim = 8, 2, 64
    lens, q_len = [1, 90, 300, 700, 2500], [1, 1, 4, 1, 2]
    cache = Cache(lens, hkv, dim, 16)
    q = queries(sum(q_len), hq, dim, dtype)
    check(cache, q, cache.attend(q, q_len, window=window, keep_first=keep_first, sink=sink), q_len, window, keep_first, sink)
    each = torch.linspace(-1, 2, hq, device="cuda")
    check(cache, q, cache.attend(q, q_len, window=window, keep_first=keep_first, sink=each), q_len, window, keep_first, each)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_no_query_sees_does_not_matter(dtype):
    """NaN in a window's passed keys (their pages gone or not), behind the end, and in keys that only later tokens see."""
    hq, hkv, dim = 8, 2, 128
    lens, q_len = [300, 200, 77], [1, 4, 3]
    cache = Cache(lens, hkv, dim, 16)
    q = queries(sum(q_len), hq, dim, dtype)
    good = cache.attend(q, q_len, window=40, keep_first=5)
    check(cache, q, good, q_len, 40, 5)
    bad = torch.full((1, hkv, dim), math.nan, device="cuda")
    for r, pos in ((0, 100), (0, 259), (0, 5), (1, 30), (1, 156), (2, 20)):
        cache.store(r, pos, bad, bad)
    cache.table[0, 3] = -1                                       # places 48 .. 63: passed
    assert torch.equal(cache.attend(q, q_len, window=40, keep_first=5), good)
    cache.store(1, 199, bad, bad)                                # the newest token of request 1 alone sees it
    got = cache.attend(q, q_len, window=40, keep_first=5)
    assert torch.isnan(got[4]).all() and torch.equal(got[:1], good[:1]) and torch.equal(got[5:], good[5:])
    # such a step counts as a large one, with which a tile's probabilities are held on another scale: roundings, not numbers, change
    rest = got.clone()
    rest[4] = good[4]
    check(cache, q, rest, q_len, 40, 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e-4, 1e-2, 30.0, 1e3, 4e5])
def test_values_of_any_size(size, dtype):
    """Steps below and above 2, alone and mixed in one request."""
    hq, hkv, dim = 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    k = [torch.randn((400, hkv, dim), generator=g, device="cuda") for _ in range(2)]
    v = [torch.randn((400, hkv, dim), generator=g, device="cuda") * size / 4 for _ in range(2)]
    v[1][:200] *= 1e-2
    cache = Cache([400, 400], hkv, dim, 16, k=k, v=v)
    q = queries(2, hq, dim, dtype)
    check(cache, q, cache.attend(q, [1, 1]), [1, 1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e-20, 1e-3, 1e4, 1e18])
def test_queries_of_any_size(size, dtype):
    hq, hkv, dim = 8, 2, 64
    cache = Cache([333], hkv, dim, 16)
    q = queries(1, hq, dim, dtype, std=size)
    check(cache, q, cache.attend(q, [1], scale=dim ** -0.5 / size), [1], scale=dim ** -0.5 / size)
    q[:, 0] = 0                                                  # a query of zeros: the mean
    check(cache, q, cache.attend(q, [1], scale=dim ** -0.5 / size), [1], scale=dim ** -0.5 / size)


def test_scores_that_are_far_apart_and_numbers_that_are_none():
    hq, hkv, dim = 4, 2, 64
    cache = Cache([500], hkv, dim, 16)
    q = queries(1, hq, dim, torch.float32, std=400.0)            # one key takes all the weight
    got = cache.attend(q, [1])
    out, size, p = plain.attention(q, *cache.held(0), dim ** -0.5, plain.seen(1, 500))
    clear = (p.amax(-1) > 1 - 1e-9)[:, 0]
    assert clear.any() and torch.allclose(got[0][clear].double(), out[0][clear], rtol=1e-4, atol=1e-5)
    q = queries(1, hq, dim, torch.bfloat16)
    q[0, 1, 5], q[0, 2, 9] = math.nan, math.inf
    got = cache.attend(q, [1])
    assert torch.isnan(got[0, 1]).all() and torch.isnan(got[0, 2]).all() and torch.isfinite(got[0, [0, 3]]).all()


def test_no_keys_no_tokens_and_requests_left_alone():
    hq, hkv, dim = 8, 2, 64
    cache = Cache([0, 50, 60], hkv, dim, 16)
    q = queries(6, hq, dim, torch.bfloat16)
    out = torch.full_like(q, 7.0)
    kernels.attn_decode_int4(q, out, cache.k_cache, cache.v_cache, cache.slots, cache.table, i32([0, 1, 5]), i32([1, 4, 1]), cache.ctx, 3, 60, 16, 0.125)
    assert not out[0].any() and (out[1:5] == 7).all() and (out[5] != 7).any()       # no keys: zeros; four tokens are more than three


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_few_and_many_requests(n, dtype):
    """Keys in one part, in a cluster of parts, in parts that a kernel of their own puts together: whatever the sizes choose."""
    hq, hkv, dim = 4, 1, 64
    for longest in (20, 600, 5000, 30000):
        lens = [max(1, longest - 37 * i * i) for i in range(n)]
        if sum(lens) > 400000:
            continue
        cache = Cache(lens, hkv, dim, 64)
        q = queries(n, hq, dim, dtype)
        mass = torch.zeros((cache.pages, hkv, 64), device="cuda")
        got = cache.attend(q, [1] * n, mass=mass)
        check(cache, q, got, [1] * n)
        assert torch.equal(cache.attend(q, [1] * n), got)
        for r in range(n):
            total = float(sum(mass[p].double().sum() for p in cache.table[r].tolist() if p >= 0))
            assert abs(total - hq) < hq * 1e-3                   # every query head's weights are one in all


def test_a_request_longer_than_the_bound_is_reported():
    cache = Cache([100], 2, 64, 16)
    q = queries(1, 4, 64, torch.bfloat16)
    with pytest.raises(KernelError, match="longer than the bound"):
        cache.attend(q, [1], longest=99)
    kernels.raise_if_kernel_gave_up()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,dim", [(9, 3, 64), (32, 8, 128), (20, 1, 128)])
@pytest.mark.parametrize("window,sink", [(None, None), (50, None), (None, 0.7)])
def test_weights_of_keys(hq, hkv, dim, window, sink, dtype):
    lens, q_len = [1, 60, 700, 2300, 40], [1, 1, 3, 1, 0]
    cache = Cache(lens, hkv, dim, 16)
    q = queries(sum(q_len), hq, dim, dtype)
    g = torch.Generator(device="cuda").manual_seed(9)
    mass = torch.rand((cache.pages, hkv, 16), generator=g, device="cuda")
    before = mass.clone()
    got = cache.attend(q, q_len, mass=mass, window=window, sink=sink)
    check(cache, q, got, q_len, window, 0, sink)
    want = before.double()
    at = 0
    for r, n in enumerate(q_len):
        if n:
            p = plain.weights(q[at:at + n], cache.held(r)[0], dim ** -0.5, plain.seen(n, lens[r], window), sink)
            p = p.view(hkv, hq // hkv * n, lens[r]).sum(1)
            for j in range(0, lens[r], 16):
                m = min(16, lens[r] - j)
                want[cache.table[r, j // 16].item(), :, :m] += p[:, j:j + m]
        at += n
    # a weight is off by its score's error (`bound`), the exponential's and the denominator's; a sum by one rounding for each of its terms
    off = (mass.double() - want).abs()
    assert (off <= 3 * 70 * 8 * 2.0 ** -23 * (want - before) + 64 * 2.0 ** -24 * want + 1e-12).all()
    assert torch.equal(mass == before, (want == before) | (mass == before))       # keys of no one stay as they were
    assert torch.equal(cache.attend(q, q_len, window=window, sink=sink), got)


def test_nothing_to_do():
    """No tokens, no requests, no rows: nothing is written, nothing fails."""
    cache = Cache([20], 2, 64, 16)
    none, empty = i32([]), torch.empty((0, 2, 64), device="cuda")
    before = cache.k_cache.clone()
    places = (cache.k_cache, cache.v_cache)
    kernels.int4_store(empty, empty, *places, none, none, cache.slots, cache.table, 16)
    kernels.int4_read(*places, empty, empty, none, none, cache.slots, cache.table, 16)
    kernels.int4_expand(*places, empty.view(0, 2, 0, 64), empty.view(0, 2, 0, 64), none, cache.table, none, 16)
    for dtype, span in ((torch.float32, 64), (torch.bfloat16, 128)):
        q = torch.empty((0, 4, 64), dtype=dtype, device="cuda")
        kernels.attn_decode_int4(q, q, *places, none, cache.table, none, none, none, 1, 20, 16, 0.125)
        kernels.attn_prefill_int4(q, q, *places, none, cache.table, none, none, none, none, none, 20, 16, 0.125, span=span)
        kernels.attn_prefill_int4(q, q, *places, cache.slots, cache.table, none, none, i32([0]), i32([0]), cache.ctx, 20, 16, 0.125, span=span)
    mass = torch.zeros((cache.pages, 2, 16), device="cuda")
    kernels.int4_evict(*places, mass, none, cache.table, none, torch.empty((0, 1), dtype=torch.int32, device="cuda"), torch.empty((0, 2, 8), dtype=torch.int32, device="cuda"), 16, 20, 2)
    kernels.int4_evict(*places, mass, cache.slots, cache.table, cache.ctx, i32([[0]]), torch.empty((1, 2, 0), dtype=torch.int32, device="cuda"), 16, 20, 0)
    kernels.raise_if_kernel_gave_up()
    assert torch.equal(cache.k_cache, before)


def test_a_prompt_longer_than_the_bound_is_reported():
    cache = Cache([300], 2, 64, 16)
    q = queries(40, 4, 64, torch.bfloat16)
    for longest in (128, 256):
        kernels.attn_prefill_int4(q, torch.empty_like(q), cache.k_cache, cache.v_cache, cache.slots, cache.table, i32([0]), i32([0]), i32([0]), i32([40]), cache.ctx, longest, 16,
                                  0.125, span=128)
        with pytest.raises(KernelError, match="longer than the bound"):
            kernels.raise_if_kernel_gave_up()
    kernels.raise_if_kernel_gave_up()


# ------------------------------------------------------------------ portions of prompts
def prompt_bound(dtype, span):
    """Beside `bound`, of the outputs' sizes: over the pages (tiles of 64) nothing.  float16 operands are three binary digits of a code times
    eleven of a step, rounded to eleven, 2^-12: of values once, of keys in scores with terms of 70 units at most, which a weight and the sum
    that it is divided by are off by; and probabilities are rounded so, as they are in `bound`."""
    return 0 if span == 64 else 2.0 ** -12 + 2 * 70 * 2.0 ** -12


@pytest.mark.parametrize("hq,hkv,dim,dtype,span", [(8, 2, 64, torch.bfloat16, 128), (8, 2, 128, torch.bfloat16, 256), (6, 2, 96, torch.bfloat16, 64), (8, 4, 32, torch.bfloat16, 64),
                                                   (9, 3, 64, torch.float32, 64), (4, 1, 128, torch.float32, 64)])
@pytest.mark.parametrize("window,keep_first", [(None, 0), (70, 6)])
def test_portions(hq, hkv, dim, dtype, span, window, keep_first):
    lens, q_len = [150, 1000, 33, 61], [150, 290, 2, 61]
    cache = Cache(lens, hkv, dim, 24)
    q = queries(sum(q_len), hq, dim, dtype)
    starts = [sum(q_len[:r]) for r in range(4)]

    def tiles(which):
        pairs = [(r, a) for r in which for a in range((q_len[r] - 1) // span * span, -1, -span)]
        return i32([r for r, _ in pairs]), i32([a for _, a in pairs])

    extra = prompt_bound(dtype, span)
    for which in (range(4), (3, 1)):
        out = torch.full_like(q, 7.0)
        places = i32([which.index(r) if r in which else -9 for r in range(4)])
        portions = None if len(which) == 4 else (i32(list(which)), places)
        kernels.attn_prefill_int4(q, out, cache.k_cache, cache.v_cache, cache.slots, cache.table, *tiles(which), i32(starts), i32(q_len), cache.ctx,
                                  max(lens), 24, dim ** -0.5, window, keep_first=keep_first, span=span, portions=portions)
        kernels.raise_if_kernel_gave_up()
        for r in range(4):
            got = out[starts[r]:starts[r] + q_len[r]]
            if r not in which:
                assert (got == 7).all()
                continue
            want, size, _ = plain.attention(q[starts[r]:starts[r] + q_len[r]], *cache.held(r), dim ** -0.5, plain.seen(q_len[r], lens[r], window, keep_first))
            off = (got.double() - want).abs()
            assert (off <= bound(dtype, want, size) + extra * size).all(), float((off / size).max())


@pytest.mark.parametrize("dim,span", [(64, 128), (128, 256), (32, 64)])
@pytest.mark.parametrize("size,query", [(1e-4, 1.5), (1e-2, 1e-20), (30.0, 1e18), (4e5, 1e4)])
def test_portions_of_any_size(dim, span, size, query):
    """Values and queries far from 1, some rows of them much smaller than the rest, and one request of zeros."""
    hq, hkv = 4, 2
    lens, q_len = [300, 130, 40], [200, 130, 40]
    g = torch.Generator(device="cuda").manual_seed(3)
    k = [torch.randn((n, hkv, dim), generator=g, device="cuda") for n in lens]
    v = [torch.randn((n, hkv, dim), generator=g, device="cuda") * size / 4 for n in lens]
    v[0][:100] *= 1e-2
    k[2].zero_(); v[2].zero_()
    cache = Cache(lens, hkv, dim, 16, k=k, v=v)
    q = queries(sum(q_len), hq, dim, torch.bfloat16, std=query)
    q[3::7] *= 2.0 ** -10
    starts = [0, 200, 330]
    pairs = [(r, a) for r in range(3) for a in range(0, q_len[r], span)]
    out = torch.empty_like(q)
    kernels.attn_prefill_int4(q, out, cache.k_cache, cache.v_cache, cache.slots, cache.table, i32([r for r, _ in pairs]), i32([a for _, a in pairs]), i32(starts), i32(q_len),
                              cache.ctx, 300, 16, dim ** -0.5 / query * 1.5, sink=0.3, span=span)
    for r, n in enumerate(q_len):
        rows = slice(starts[r], starts[r] + n)
        want, weight, _ = plain.attention(q[rows], *cache.held(r), dim ** -0.5 / query * 1.5, plain.seen(n, lens[r]), 0.3)
        off = (out[rows].double() - want).abs()
        # products of a probability (times 2^9) and a step are float16: below its normal numbers they are off by half of 2^-24, times codes up to 7
        small = 7 * lens[r] * 2.0 ** -34 if span == 64 else 1e-30
        assert (off <= bound(torch.bfloat16, want, weight) + prompt_bound(torch.bfloat16, span) * weight + small).all(), (r, float((off / weight).max()))


# ------------------------------------------------------------------ eviction
def evict(cache, mass, keep, recent, first, longest=None, fresh=None):
    n = len(cache.lens)
    width = -(-keep // cache.page)
    to = i32(cache.free[:n * width]).view(n, width) if fresh is None else fresh
    kept = torch.full((n, cache.hkv, keep), -5, dtype=torch.int32, device="cuda")
    kernels.int4_evict(cache.k_cache, cache.v_cache, mass, cache.slots, cache.table, cache.ctx, to, kept, cache.page, longest or max(cache.lens), recent, first)
    return to, kept


@pytest.mark.parametrize("hkv,dim,page", [(3, 64, 16), (2, 128, 8), (1, 32, 64), (2, 96, 24), (2, 128, 40)])
@pytest.mark.parametrize("keep,recent,first", [(64, 16, 4), (37, 0, 0), (50, 30, 20), (1, 0, 0), (90, 1, 7)])
def test_eviction(hkv, dim, page, keep, recent, first):
    lens = [200, 64, 65, 0, 12, 1030, 91]
    width = -(-keep // page)
    cache = Cache(lens, hkv, dim, page, spare=len(lens) * width + 2)
    g = torch.Generator(device="cuda").manual_seed(4)
    mass = torch.randint(0, 30, (cache.pages, hkv, page), generator=g, device="cuda").float() / 7      # many equal sums
    mass[cache.table[0, 1], 0, 3] = math.nan
    mass[cache.table[5, 2], :, 1] = math.inf
    mass[cache.table[5, 3], :, 1:4] = torch.tensor([-0.0, 0.0, -3.0], device="cuda")
    before, k0, v0 = mass.clone(), cache.k_cache.clone(), cache.v_cache.clone()
    to, kept = evict(cache, mass, keep, recent, first)
    touched = set()
    for r, n in enumerate(lens):
        m = min(n, keep)
        sums = torch.cat([before[p] for p in cache.table[r].tolist() if p >= 0] or [torch.zeros((hkv, 0), device="cuda")], 1)[:, :n].cpu()
        new = torch.cat([mass[p] for p in to[r].tolist()], 1)
        for h in range(hkv):
            want = plain.evicted(sums[h], keep, recent, first)
            assert kept[r, h].tolist() == want + [-1] * (keep - m), (r, h)
            assert torch.equal(torch.nan_to_num(new[h, :m].cpu(), 1e9), torch.nan_to_num(sums[h][want], 1e9))
            if m:
                k, v = torch.empty((2, m, hkv, dim), device="cuda")
                kernels.int4_read(cache.k_cache, cache.v_cache, k, v, i32([r] * m), i32(list(range(m))), cache.slots, to, page)
                held_k, held_v = cache.held(r)
                assert torch.equal(k[:, h], held_k[h][want].float()) and torch.equal(v[:, h], held_v[h][want].float())
        touched |= set(to[r].tolist())
        # rows behind the last one stay as they were
        assert torch.equal(torch.nan_to_num(new[:, m:]), torch.nan_to_num(torch.cat([before[p] for p in to[r].tolist()], 1)[:, m:]))
    rest = [p for p in range(cache.pages) if p not in touched]
    assert torch.equal(cache.k_cache[rest], k0[rest]) and torch.equal(cache.v_cache[rest], v0[rest])
    assert torch.equal(torch.nan_to_num(mass[rest]), torch.nan_to_num(before[rest]))


def test_eviction_of_long_requests():
    """More sums than shared memory takes, and a bound that is too low."""
    n, keep, page = 60000, 1000, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((n, 1, 32), generator=g, device="cuda")
    cache = Cache([n, 300], 1, 32, page, spare=40, k=[x, x[:300]], v=[x, x[:300]])
    mass = torch.rand((cache.pages, 1, page), generator=g, device="cuda")
    sums = torch.cat([mass[p] for p in cache.table[0].tolist()], 1)[0, :n]
    want = torch.cat((torch.tensor([0, 1], device="cuda"), sums[2:n - 10].topk(keep - 12).indices.sort().values + 2, torch.arange(n - 10, n, device="cuda")))
    for longest in (n, 5000):
        _, kept = evict(cache, mass.clone(), keep, 10, 2, longest)
        assert torch.equal(kept[0, 0].long(), want) and kept[1, 0, :301].tolist() == list(range(300)) + [-1]


@pytest.mark.parametrize("n", [9000, 10300, 11500, 12300, 13000])
def test_sums_that_nearly_fill_the_shared_memory_of_a_plain_launch(n):
    x = torch.zeros((n, 1, 32), device="cuda")
    cache = Cache([n], 1, 32, 64, spare=4, k=[x], v=[x])
    mass = torch.rand((cache.pages, 1, 64), device="cuda")
    sums = torch.cat([mass[p] for p in cache.table[0].tolist()], 1)[0, :n]
    _, kept = evict(cache, mass, 100, 0, 0)
    assert torch.equal(kept[0, 0].long(), sums.topk(100).indices.sort().values)


def test_a_page_of_two_requests_gets_the_weights_of_both():
    """One request twice in a call: every weight counts twice, whatever order they come in."""
    lens = [700, 700]
    cache = Cache(lens, 2, 64, 16, spare=90)
    cache.table[1] = cache.table[0]
    cache.k[1], cache.v[1] = cache.k[0], cache.v[0]
    cache.store(0, 0, cache.k[0], cache.v[0])
    for n in (1, 3):                                             # by the kernel itself, and by one of its own
        q = queries(n, 8, 64, torch.bfloat16)
        once, twice = torch.zeros((2, cache.pages, 2, 16), device="cuda")
        cache.attend(q, [n, 0], mass=once)
        out = cache.attend(torch.cat((q, q)), [n, n], mass=twice)
        assert torch.equal(out[:n], out[n:]) and torch.equal(twice, 2 * once)


def test_a_shared_page_is_not_written():
    """Two requests with the same pages, cut by different rows; the old pages stay as they were."""
    cache = Cache([64, 64], 2, 64, 16, spare=8)
    cache.table[1] = cache.table[0]
    cache.k[1], cache.v[1] = cache.k[0], cache.v[0]
    k0 = cache.k_cache.clone()
    mass = torch.rand((cache.pages, 2, 16), device="cuda")
    to, kept = evict(cache, mass, 30, 5, 1)
    old = cache.table[0].tolist()
    assert torch.equal(cache.k_cache[old], k0[old]) and torch.equal(kept[0], kept[1])


# ------------------------------------------------------------------ refusals (all by the host, before anything is launched)
def calls(**change):
    """Every entry point with good arguments but for the changed ones."""
    n, hq, hkv, dim, page = 2, 4, 2, 64, 16
    a = dict(hq=hq, q=queries(n, hq, dim, torch.bfloat16), out=queries(n, hq, dim, torch.bfloat16), k=queries(n, hkv, dim, torch.bfloat16), v=queries(n, hkv, dim, torch.bfloat16),
             k_cache=torch.zeros((6, hkv, kernels.int4_page_bytes(page, dim)), dtype=torch.uint8, device="cuda"), slots=i32([0, 1]), table=i32([[0, 1], [2, 3]]),
             req=i32([0, 1]), pos=i32([0, 1]), starts=i32([0, 1]), lens=i32([1, 1]), ctx=i32([20, 5]), most=1, longest=32, page=page, window=None, keep_first=0, sink=None,
             mass=torch.zeros((6, hkv, page), device="cuda"), to=i32([[4], [5]]), kept=i32([[[0] * 12] * hkv] * n), recent=2, first=1, span=128, tile=i32([0, 1]), zeros=i32([0, 0]),
             places=None)
    a["v_cache"] = a["k_cache"].clone()
    a["whole"], a["whole_v"] = torch.zeros((2, n, hkv, 32, dim), dtype=torch.bfloat16, device="cuda")
    a.update(change)
    places = (a["k_cache"], a["v_cache"])
    return dict(
        store=lambda: kernels.int4_store(a["k"], a["v"], *places, a["req"], a["pos"], a["slots"], a["table"], a["page"], mass=a["mass"]),
        read=lambda: kernels.int4_read(*places, a["k"], a["v"], a["req"], a["pos"], a["slots"], a["table"], a["page"]),
        expand=lambda: kernels.int4_expand(*places, a["whole"], a["whole_v"], a["slots"], a["table"], a["ctx"], a["page"]),
        decode=lambda: kernels.attn_decode_int4(a["q"], a["out"], *places, a["slots"], a["table"], a["starts"], a["lens"], a["ctx"], a["most"], a["longest"], a["page"], 0.125,
                                                a["window"], a["sink"], a["keep_first"], a["mass"]),
        prefill=lambda: kernels.attn_prefill_int4(a["q"], a["out"], *places, a["slots"], a["table"], a["tile"], a["zeros"], a["starts"], a["lens"], a["ctx"], a["longest"], a["page"],
                                                  0.125, a["window"], a["sink"], a["keep_first"], a["span"], a["places"]),
        evict=lambda: kernels.int4_evict(*places, a["mass"], a["slots"], a["table"], a["ctx"], a["to"], a["kept"], a["page"], a["longest"], a["recent"], a["first"]))


def test_good_arguments_are_taken():
    for call in calls().values():
        call()
    kernels.raise_if_kernel_gave_up()


EVERY = ("store", "read", "expand", "decode", "prefill", "evict")
BAD = [
    (EVERY, lambda: dict(page=12)), (EVERY, lambda: dict(page=8)), (EVERY, lambda: dict(page=0)), (EVERY, lambda: dict(page=-16)),
    (EVERY, lambda: dict(k_cache=torch.zeros((6, 2, 576), dtype=torch.int8, device="cuda"))),
    (EVERY, lambda: dict(k_cache=torch.zeros((7, 2, 576), dtype=torch.uint8, device="cuda"))),
    (EVERY, lambda: dict(v_cache=torch.zeros((6, 2, 577), dtype=torch.uint8, device="cuda"))),
    (EVERY, lambda: dict(k_cache=torch.zeros((6, 2, 1152), dtype=torch.uint8, device="cuda")[:, :, ::2])),
    (EVERY, lambda: dict(v_cache=torch.zeros((6, 2, 576), dtype=torch.uint8))),
    (EVERY, lambda: dict(table=i32([0, 1]))), (EVERY, lambda: dict(table=i32([[0, 1], [2, 3]]).long())), (EVERY, lambda: dict(table=torch.zeros((2, 2), dtype=torch.int32))),
    (EVERY, lambda: dict(table=i32([[0, 1, 2, 3], [2, 3, 4, 5]])[:, ::2])),
    (EVERY, lambda: dict(slots=i32([0, 1]).long())), (EVERY, lambda: dict(slots=torch.zeros(2, dtype=torch.int32))),
    (("expand", "decode", "prefill", "evict"), lambda: dict(slots=i32([0]))),
    (("store", "read"), lambda: dict(req=i32([0]))), (("store", "read"), lambda: dict(pos=i32([0, 1, 2]))),
    (("expand", "decode", "prefill", "evict"), lambda: dict(ctx=i32([20]))), (("decode", "prefill"), lambda: dict(starts=i32([0]))),
    (("store", "read"), lambda: dict(k=queries(2, 1, 64, torch.bfloat16), v=queries(2, 1, 64, torch.bfloat16))),           # another number of key heads
    (("store", "read"), lambda: dict(k=queries(2, 2, 32, torch.bfloat16), v=queries(2, 2, 32, torch.bfloat16))),           # another head size
    (("store", "read"), lambda: dict(v=queries(3, 2, 64, torch.bfloat16))), (("store", "read"), lambda: dict(v=queries(2, 2, 64, torch.float32))),
    (("store", "read"), lambda: dict(k=queries(2, 2, 64, torch.float16), v=queries(2, 2, 64, torch.float16))),
    (("store", "read"), lambda: dict(k=queries(2, 2, 64, torch.bfloat16).cpu())),
    (("store",), lambda: dict(k=queries(2, 2, 128, torch.bfloat16)[:, :, ::2])), (("read",), lambda: dict(k=queries(2, 4, 64, torch.bfloat16)[:, ::2])),
    (("expand",), lambda: dict(whole=torch.zeros((2, 2, 31, 64), dtype=torch.bfloat16, device="cuda"))),
    (("decode", "prefill"), lambda: dict(q=queries(2, 4, 64, torch.float16), out=queries(2, 4, 64, torch.float16))), (("decode", "prefill"), lambda: dict(out=queries(2, 4, 64, torch.float32))),
    (("decode", "prefill"), lambda: dict(q=queries(2, 3, 64, torch.bfloat16), out=queries(2, 3, 64, torch.bfloat16))),     # three query heads for two key heads
    (("decode", "prefill"), lambda: dict(q=queries(2, 4, 32, torch.bfloat16), out=queries(2, 4, 32, torch.bfloat16))),
    (("decode", "prefill"), lambda: dict(out=queries(3, 4, 64, torch.bfloat16))), (("decode", "prefill"), lambda: dict(q=queries(2, 8, 64, torch.bfloat16)[:, ::2])),
    (("decode",), lambda: dict(most=0)), (("decode", "prefill"), lambda: dict(longest=0)), (("evict",), lambda: dict(longest=0)),
    (("decode", "prefill"), lambda: dict(window=0)), (("decode", "prefill"), lambda: dict(keep_first=-1)), (("decode",), lambda: dict(sink=torch.zeros(3, device="cuda"))),
    (("store", "decode", "evict"), lambda: dict(mass=torch.zeros((6, 2, 8), device="cuda"))), (("store", "decode", "evict"), lambda: dict(mass=torch.zeros((5, 2, 16), device="cuda"))),
    (("store", "decode", "evict"), lambda: dict(mass=torch.zeros((6, 2, 16), dtype=torch.bfloat16, device="cuda"))),
    (("prefill",), lambda: dict(span=32)), (("prefill",), lambda: dict(q=queries(2, 4, 64, torch.float32), out=queries(2, 4, 64, torch.float32))), (("prefill",), lambda: dict(places=(i32([0]), i32([0])))),
    (("evict",), lambda: dict(to=i32([[4]]))), (("evict",), lambda: dict(kept=i32([[[0] * 20] * 2] * 2))), (("evict",), lambda: dict(kept=i32([[[0] * 12]] * 2))),
    (("evict",), lambda: dict(recent=-1)), (("evict",), lambda: dict(first=-1)), (("evict",), lambda: dict(recent=8, first=5)),
    (("evict",), lambda: dict(to=i32([[4], [5]]).long())), (("evict",), lambda: dict(kept=torch.zeros((2, 2, 12), device="cuda"))),
]


@pytest.mark.parametrize("case", range(len(BAD)))
def test_refusals(case):
    names, change = BAD[case]
    made = calls(**change())
    for name in names:
        with pytest.raises(KernelError):
            made[name]()


def test_planes_that_do_not_begin_on_16_bytes_are_refused():
    room = torch.zeros(6 * 2 * 576 + 16, dtype=torch.uint8, device="cuda")
    odd = room[8:8 + 6 * 2 * 576].view(6, 2, 576)
    made = calls(k_cache=odd)
    for name in EVERY:
        with pytest.raises(KernelError):
            made[name]()


# ------------------------------------------------------------------ together, and as programs run them
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_reply_with_eviction(dtype):
    """Tokens stored one by one, attended with their weights summed, and cut every few steps: the same as in 64 bits at every step."""
    hq, hkv, dim, page, keep = 8, 2, 64, 8, 40
    g = torch.Generator(device="cuda").manual_seed(6)
    pages = 40
    k_cache = torch.zeros((pages, hkv, kernels.int4_page_bytes(page, dim)), dtype=torch.uint8, device="cuda")
    v_cache, mass = torch.zeros_like(k_cache), torch.zeros((pages, hkv, page), device="cuda")
    free = list(range(pages))
    table = torch.full((1, 12), -1, dtype=torch.int32, device="cuda")
    slot, zero, one = i32([0]), i32([0]), i32([1])
    rows = [([], []) for _ in range(hkv)]                        # per key head: held keys and values
    sums = [[] for _ in range(hkv)]
    length = 0
    for step in range(90):
        k, v = torch.randn((2, 1, hkv, dim), generator=g, device="cuda").to(dtype)
        if length % page == 0:
            table[0, length // page] = free.pop()
        kernels.int4_store(k, v, k_cache, v_cache, zero, i32([length]), slot, table, page, mass=mass)
        for h in range(hkv):
            rows[h][0].append(plain.held(k)[0, h]); rows[h][1].append(plain.held(v)[0, h]); sums[h].append(0.0)
        length += 1
        q = (torch.randn((1, hq, dim), generator=g, device="cuda") * 1.5).to(dtype)
        out = torch.empty_like(q)
        kernels.attn_decode_int4(q, out, k_cache, v_cache, slot, table, zero, one, i32([length]), 1, length, page, dim ** -0.5, mass=mass)
        keys, values = (torch.stack([torch.stack(rows[h][i]) for h in range(hkv)]) for i in (0, 1))
        want, size, p = plain.attention(q, keys, values, dim ** -0.5, plain.seen(1, length))
        steps = torch.einsum("hnj,hjd->nhd", p, (values.unflatten(-1, (-1, 32)).abs().amax(-1) / 7).repeat_interleave(32, -1).repeat_interleave(hq // hkv, 0))
        assert ((out.double() - want).abs() <= bound(dtype, want, size, steps)).all(), step
        p = p.view(hkv, -1, length).sum(1)
        for h in range(hkv):
            sums[h] = [a + float(b) for a, b in zip(sums[h], p[h])]
        if length == keep + 8:
            to = i32([[free.pop() for _ in range(keep // page)]])
            kept = torch.empty((1, hkv, keep), dtype=torch.int32, device="cuda")
            kernels.int4_evict(k_cache, v_cache, mass, slot, table, i32([length]), to, kept, page, length, 8, 2)
            free += [p for p in table[0].tolist() if p >= 0]
            table[:] = -1
            table[0, :keep // page] = to[0]
            for h in range(hkv):
                stay = kept[0, h].tolist()
                # sums differ from the plain ones by roundings: the choice is theirs, and none that was left out is clearly larger
                left = [i for i in range(2, length - 8) if i not in stay]
                assert stay[:2] == [0, 1] and stay[-8:] == list(range(length - 8, length)) and len(set(stay)) == keep
                assert max(sums[h][i] for i in left) <= min(sums[h][i] for i in stay[2:-8]) + 1e-3
                rows[h] = tuple([x[i] for i in stay] for x in rows[h])
                sums[h] = [sums[h][i] for i in stay]
            length = keep
    kernels.raise_if_kernel_gave_up()


def test_captured_replayed_and_on_two_streams():
    """One capture of a whole turn replayed with other contents, beside the same calls on another stream."""
    hq, hkv, dim, page = 8, 2, 128, 16
    lens = [700, 60]
    cache, other = Cache(lens, hkv, dim, page, seed=1), Cache(lens, hkv, dim, page, seed=2)
    q = queries(2, hq, dim, torch.bfloat16)
    out = torch.empty_like(q)
    starts, ones = i32([0, 1]), i32([1, 1])
    mass = torch.zeros((cache.pages, hkv, page), device="cuda")
    k, v = torch.randn((2, 2, hkv, dim), device="cuda")
    req, pos = i32([0, 1]), i32([699, 59])

    def turn(c, q, out, mass):
        kernels.int4_store(k, v, c.k_cache, c.v_cache, req, pos, c.slots, c.table, page)
        kernels.attn_decode_int4(q, out, c.k_cache, c.v_cache, c.slots, c.table, starts, ones, c.ctx, 1, 1024, page, dim ** -0.5, mass=mass)

    turn(cache, q, out, mass)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turn(cache, q, out, mass)
    mass.zero_()
    plain_mass, plain_out = torch.zeros_like(mass), torch.empty_like(q)
    other_q, other_out, other_mass = queries(2, hq, dim, torch.bfloat16, seed=8), torch.empty_like(q), torch.zeros_like(mass)
    for i in range(4):
        q.copy_(queries(2, hq, dim, torch.bfloat16, seed=20 + i))
        k.copy_(torch.randn(k.shape, device="cuda")); v.copy_(torch.randn(v.shape, device="cuda"))
        cache.ctx.copy_(i32([700, 60 - i]))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            turn(other, other_q, other_out, other_mass)
        torch.cuda.synchronize()
        turn(cache, q, plain_out, plain_mass)
        assert torch.equal(out, plain_out) and torch.equal(mass, plain_mass)
        expected = torch.empty_like(q)
        kernels.attn_decode_int4(other_q, expected, other.k_cache, other.v_cache, other.slots, other.table, starts, ones, other.ctx, 1, 1024, page, dim ** -0.5)
        assert torch.equal(expected, other_out)
    kernels.raise_if_kernel_gave_up()


@pytest.mark.parametrize("dtype,span", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_prompts_and_cuts_captured_and_replayed(dtype, span):
    """A portion's attention, a weighed step and a cut in one capture, replayed with other contents, lengths and pages."""
    hq, hkv, dim, page = 8, 2, 64, 16
    cache = Cache([300, 180], hkv, dim, page, spare=20)
    q = queries(80, hq, dim, dtype)
    mass, kept = torch.zeros((cache.pages, hkv, page), device="cuda"), torch.empty((2, hkv, 64), dtype=torch.int32, device="cuda")
    to = i32(cache.free[:8]).view(2, 4)
    tiles = [(r, a) for r, n in ((0, 50), (1, 30)) for a in range(0, n, span)]
    lists = [i32(x) for x in ([r for r, _ in tiles], [a for _, a in tiles], [0, 50], [50, 30], [49, 79], [1, 1])]
    k_out, v_out = torch.empty((2, 2, hkv, 64, dim), device="cuda")

    def turn():
        out, last = torch.empty_like(q), torch.zeros_like(q)
        places = (cache.k_cache, cache.v_cache, cache.slots, cache.table)
        kernels.attn_prefill_int4(q, out, *places, *lists[:4], cache.ctx, 320, page, dim ** -0.5, span=span)
        kernels.attn_decode_int4(q, last, *places, lists[4], lists[5], cache.ctx, 1, 320, page, dim ** -0.5, mass=mass)
        kernels.int4_evict(cache.k_cache, cache.v_cache, mass, cache.slots, cache.table, cache.ctx, to, kept, page, 320, 8, 2)
        kernels.int4_expand(cache.k_cache, cache.v_cache, k_out, v_out, cache.slots, to, new, page)
        return out, last

    new = i32([64, 64])
    turn()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = turn()
    for i in range(3):
        q.copy_(queries(80, hq, dim, dtype, seed=30 + i))
        cache.ctx.copy_(i32([300 - 9 * i, 180 - i]))
        results = []
        for run in (lambda: (graph.replay(), held)[1], turn):
            mass.zero_()
            results.append([x.clone() for x in (*run(), mass, kept, k_out, v_out)])
        for a, b in zip(*results):
            assert torch.equal(a, b)
    kernels.raise_if_kernel_gave_up()


def test_far_places_pass_32_bits():
    """A pool of more than 2^31 bytes: the last page's rows are where they should be."""
    hkv, dim, page = 8, 128, 64
    bytes_ = hkv * kernels.int4_page_bytes(page, dim)
    pages = 2 ** 31 // bytes_ + 2
    k_cache = torch.empty((pages, hkv, bytes_ // hkv), dtype=torch.uint8, device="cuda")
    v_cache = torch.empty_like(k_cache)
    k, v = torch.randn((2, page, hkv, dim), device="cuda")
    table, where = i32([[pages - 1]]), (i32([0] * page), i32(list(range(page))), i32([0]))
    kernels.int4_store(k, v, k_cache, v_cache, *where, table, page)
    got_k, got_v = torch.empty((2, page, hkv, dim), device="cuda")
    kernels.int4_read(k_cache, v_cache, got_k, got_v, *where, table, page)
    assert torch.equal(got_k, plain.held(k).float()) and torch.equal(got_v, plain.held(v).float())
    q = queries(1, 32, dim, torch.bfloat16)
    out = torch.empty_like(q)
    kernels.attn_decode_int4(q, out, k_cache, v_cache, i32([0]), table, i32([0]), i32([1]), i32([page]), 1, page, page, dim ** -0.5)
    want, size, p = plain.attention(q, plain.held(k).transpose(0, 1), plain.held(v).transpose(0, 1), dim ** -0.5, plain.seen(1, page))
    assert ((out.double() - want).abs() <= bound(torch.bfloat16, want, size, plain.stepped(p, v))).all()
