"""Steps of a model whose cache is held in 4 bits, one by one: what a captured step launches, and every step's logits against 64 bits over the
rows that the cache really holds."""
import pytest
import torch

import plain_int4
from test_int4_cache import Launching
from test_int4_engine_gpu import RAW, model_of, stepper_of, tokens_of

pytestmark = pytest.mark.gpu


def read_out(stepper, key):
    """Keys and values that the cache holds of a request, of every layer: pairs of [kv_heads, rows, dim] in 64 bits."""
    from cisr_b200.ops import kernels

    cache, found = stepper.cache, []
    for entry in range(len(stepper.model.spec.run)):
        b = cache.binding(entry)
        n, mixer = cache.length(key), stepper.model.layers[entry].parts()["mixer"]
        k, v = torch.empty((2, 1, mixer.hkv, n, mixer.dim), device="cuda")
        one = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")
        group = cache.page_groups[cache.entry_group[entry][1]]
        table = torch.from_numpy(group.host_table[cache.slot(key)][None]).cuda()
        kernels.int4_expand(b.k, b.v, k, v, one(0), table, one(n), cache.page_size)
        found.append((k[0].double(), v[0].double()))
    return found


def on_held_rows(stepper, key, tokens, check_rows=True):
    """Logits [tokens, vocab] in 64 bits of the latest `tokens` of a request, whose rows are in the cache: with the keys and values that the cache
    holds, so that what is left are roundings.  Rounded to the model's type where the engine does.

    The tokens' own rows are checked: a held value is within half a step of what was stored, and that is within 2^-5 of the
    group's largest of the plain one (in float 2^-14), seven steps."""
    model, n = stepper.model, len(tokens)
    rounded = lambda x: x.to(model.dtype).double()
    norm = lambda x, part: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + RAW["rms_norm_eps"]) * part.weight.double()
    rows, first = stepper.cache.length(key), stepper.cache.seen(key) - n
    at = torch.arange(rows - n, rows, device="cuda")[:, None]
    j = torch.arange(rows, device="cuda")[None]
    x = model.embedding.table[torch.tensor(tokens, device="cuda")].double()
    for layer, (keys, values) in zip(model.layers, read_out(stepper, key)):
        mixer, ff, n1, n2 = (layer.parts()[p] for p in ("mixer", "feed_forward", "mixer_norm", "feed_forward_norm"))
        hq, hkv, dim = mixer.hq, mixer.hkv, mixer.dim
        qkv = (rounded(norm(x, n1)) @ mixer.qkv.double().T).view(n, hq + 2 * hkv, dim)
        inv = RAW["rope_theta"] ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
        angle = torch.arange(first, first + n, device="cuda", dtype=torch.float64)[:, None, None] * inv
        a, b = qkv[:, :hq + hkv, :dim // 2], qkv[:, :hq + hkv, dim // 2:]
        turned = rounded(torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1))
        for new, held in ((turned[:, hq:], keys), (rounded(qkv[:, hq + hkv:]), values)):
            top = new.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(n, hkv, dim // 32, 32).flatten(2)
            off = (held[:, rows - n:].transpose(0, 1) - new).abs()
            if check_rows:
                assert (off <= top / 14 + top * (2.0 ** -5 if model.dtype == torch.bfloat16 else 2.0 ** -14)).all(), float((off / top).max())
        ok = j <= at
        if mixer.window:
            ok &= at - j < mixer.window
        p = plain_int4.weights(turned[:, :hq], keys, dim ** -0.5, ok)
        mixed = torch.einsum("hnj,hjd->nhd", p, values.repeat_interleave(hq // hkv, 0))
        x = x + rounded(mixed.reshape(n, -1)) @ mixer.o.double().T
        gate, up = (rounded(norm(x, n2)) @ ff.gate_up.double().T).chunk(2, -1)
        x = x + rounded(torch.nn.functional.silu(gate) * up) @ ff.down.double().T
    return rounded(norm(x, model.final_norm)) @ model.head.weight.double().T


def logits_bound(dtype, layers=2):
    """Of the logits' spread.  bfloat16: seven places a layer and one behind are rounded, on both sides of numbers that are not quite the same: an
    independent rounding each, 2^-8 at most and 2^-8 / sqrt 3 in the mean square, which are added as if they all pointed one way.  float: as
    many places of 2^-16 (products of three bfloat16 parts and their sums), and an attention's scores as `bound` has them, 1.3e-4 a layer."""
    places = 7 * layers + 1
    return places * 2.0 ** -8 / 3 ** 0.5 if dtype == torch.bfloat16 else places * 2.0 ** -16 + layers * 1.3e-4


def check_step(stepper, got, portions):
    """A step's logits, all rows of all portions {key: tokens}: every one within the bound."""
    at = 0
    for key, tokens in portions.items():
        want = on_held_rows(stepper, key, tokens)
        off = (got[at:at + len(tokens)].double() - want).square().mean(-1).sqrt() / want.std()
        assert (off <= logits_bound(stepper.model.dtype, len(stepper.model.layers))).all(), (key, off.tolist())
        at += len(tokens)
    stepper.check_kernels()


def run_step(stepper, portions):
    from cisr_b200 import StepEntry

    return stepper.step([StepEntry(key, tokens, list(range(len(tokens)))) for key, tokens in portions.items()]).clone()


SHAPES = [("float32", 4, 2, 128), ("bfloat16", 4, 2, 256), ("bfloat16", 9, 3, 576), ("bfloat16", 4, 2, 384), ("bfloat16", 8, 2, 1024)]


@pytest.mark.parametrize("keep", [None, 600])
@pytest.mark.parametrize("dtype,heads,kv_heads,hidden", SHAPES)
def test_portions_of_every_length_in_one_step(dtype, heads, kv_heads, hidden, keep):
    """A long portion behind many rows, short and single ones beside it: by groups of like lengths, and straight over the pages, without and
    with keys that are weighed."""
    stepper = stepper_of(model_of(dtype, heads, kv_heads, hidden), n_pages=300, max_slots=8, keep=keep)
    before = dict(zip("abcdefgh", (400, 3, 90, 0, 33, 200, 1, 60)))
    for seed, (key, n) in enumerate(before.items()):
        stepper.create(key)
        if n:
            run_step(stepper, {key: tokens_of(n, seed)})
    for seed, lens in enumerate([(60, 40, 33, 70, 20, 1, 2, 32), (35, 1, 1, 1, 9, 33, 1, 150)]):
        portions = {key: tokens_of(n, 20 + 10 * seed + i) for i, (key, n) in enumerate(zip(before, lens))}
        check_step(stepper, run_step(stepper, portions), portions)
    stepper.cache.check()


@pytest.mark.parametrize("keep", [None, 64])
@pytest.mark.parametrize("dtype,n", [("bfloat16", 1), ("bfloat16", 3), ("float32", 2)])
def test_nothing_is_made_between_the_embedding_and_the_first_product(monkeypatch, dtype, n, keep):
    """A fused product looks its places up before it waits for the kernel ahead of it, which has to be one that does not write them."""
    from cisr_b200 import StepEntry
    from cisr_b200.ops import kernels

    stepper = stepper_of(model_of(dtype), graph=True, keep=keep)
    keys = [f"r{i}" for i in range(n)]
    for i, key in enumerate(keys):
        stepper.create(key)
        stepper.step([StepEntry(key, tokens_of(9 + i))])
    stepper.step([StepEntry(key, [i], [0]) for i, key in enumerate(keys)])
    graph, fresh = stepper.graphs.get(n, 12)
    assert not fresh
    with Launching() as mode:
        for name in ("embedding", "skinny_gemm", "gemm", "rope_store", "int4_store", "attn_decode_int4"):
            def logged(*args, _fn=getattr(kernels, name), _name=name, **kw):
                mode.seen.append(_name)
                return _fn(*args, **kw)
            monkeypatch.setattr(kernels, name, logged)
        graph._run(advance=False)
    torch.cuda.synchronize()
    monkeypatch.undo()
    begin = mode.seen.index("embedding") + 1
    between = mode.seen[begin:min(i for i, name in enumerate(mode.seen) if i >= begin and name in ("skinny_gemm", "gemm", "rope_store"))]
    assert between == [], mode.seen
    attend = [i for i, name in enumerate(mode.seen) if name == "attn_decode_int4"]
    assert attend and all(mode.seen[i - 1] == "int4_store" for i in attend), mode.seen       # it waits before it lets the attention start


@pytest.mark.parametrize("dtype,heads,kv_heads,hidden", SHAPES + [("bfloat16", 32, 8, 4096)])
@pytest.mark.parametrize("graph", [False, True])
def test_every_step_of_batches_of_changing_size(dtype, heads, kv_heads, hidden, graph):
    """Single tokens of one to eight requests by turns (captured steps of 1, 2, 4 and 8 rows, of two context sizes, that share their memory), a portion
    between them: every row of every step."""
    stepper = stepper_of(model_of(dtype, heads, kv_heads, hidden), n_pages=400, max_slots=8, graph=graph)
    keys = "abcdefgh"
    for i, key in enumerate(keys):
        stepper.create(key)
        portions = {key: tokens_of(5 + 35 * i, i)}
        check_step(stepper, run_step(stepper, portions), portions)
    turns = ["a", "abcdefgh", "cb", "abc", "h", "gfedcba", "bd", "a", "ah", "abcdefgh", "efg", "hg", "a"]
    for turn in range(2):
        for i, which in enumerate(turns):
            portions = {key: tokens_of(1, 100 * turn + 10 * i + j) for j, key in enumerate(which)}
            check_step(stepper, run_step(stepper, portions), portions)
            stepper.cache.check()
        portions = {"a": tokens_of(40, turn), "c": tokens_of(1, 7)}
        check_step(stepper, run_step(stepper, portions), portions)
    if graph:
        assert stepper.graphs.hits > 10 and {rows for rows, _ in stepper.graphs.graphs} == {1, 2, 4, 8}


@pytest.mark.parametrize("dtype,dim", [("float32", 32), ("bfloat16", 64), ("bfloat16", 128), ("bfloat16", 96)])
@pytest.mark.parametrize("graph", [False, True])
def test_every_step_of_a_layer_with_a_window(dtype, dim, graph):
    """One layer that sees 40 keys, whose pages go back as they are passed, and one that sees all."""
    from cisr_b200 import Model
    from test_toy_parts_gpu import W_CONFIG, register_windowed_toy

    register_windowed_toy()
    stepper = stepper_of(Model.from_config(dict(W_CONFIG, hidden_size=4 * dim, head_dim=dim, vocab_size=256), seed=5, dtype=dtype), n_pages=100, graph=graph)
    commit, late = stepper.cache.commit, []

    def commit_later(key, n):                                    # the rows of a step are looked at before passed pages go back
        stepper.cache.requests[key].length += n
        stepper.cache.requests[key].seen += n
        late.append((key, n))

    stepper.cache.commit = commit_later
    stepper.create("a"); stepper.create("b")
    steps = [{"a": n, "b": n // 3 + 1} for n in (100, 45, 3, 20, 52)] + [dict.fromkeys(("ab", "a", "ba")[i % 3], 1) for i in range(60)]
    for i, lens in enumerate(steps):
        portions = {key: tokens_of(n, 10 * i + j) for j, (key, n) in enumerate(lens.items())}
        check_step(stepper, run_step(stepper, portions), portions)
        while late:
            key, n = late.pop()
            stepper.cache.requests[key].length -= n
            stepper.cache.requests[key].seen -= n
            commit(key, n)
        stepper.cache.check()
    windowed = next(g for g in stepper.cache.page_groups if g.use.window)
    assert windowed.pool.n_used <= 2 * (40 // 8 + 1)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("chunk", [5, 48])
def test_every_step_of_requests_that_are_cut(dtype, graph, chunk):
    """Two requests that are cut again and again, alone and together: every step's logits are those of the rows that were held in it."""
    from cisr_b200.engine.step import Keep

    keep = Keep(rows=48, recent=12, first=2, slack=8)
    stepper = stepper_of(model_of(dtype, 4, 2, 256), keep=keep, graph=graph, n_pages=100)
    cuts = []
    cut = stepper._cut
    stepper._cut = lambda keys: cuts.append(list(keys))          # the rows of a step are looked at before it cuts
    stepper.create("a"); stepper.create("b")
    plan = [{"a": chunk, "b": 3}, {"a": chunk}, {"b": chunk, "a": 1}] + [{"a": 1, "b": 1}] * 20 + [{"a": 1}] * 9 + [{"b": chunk}] + [{"a": 1, "b": 1}] * 20
    sizes = []
    for i, lens in enumerate(plan):
        portions = {key: tokens_of(n, 1000 + 10 * i) for key, n in lens.items()}
        got = run_step(stepper, portions)
        check_step(stepper, got, portions)
        sizes.append(stepper.cache.length("a"))
        cut(cuts.pop())
        stepper.cache.check()
        assert all(stepper.cache.length(key) < keep.rows + keep.slack for key in portions)
    assert max(sizes) >= keep.rows + keep.slack and any(b < a for a, b in zip(sizes, sizes[1:]))


@pytest.mark.parametrize("keep", [None, 64])
@pytest.mark.parametrize("dtype,n", [("float32", 2), ("bfloat16", 1), ("bfloat16", 3)])
def test_tokens_that_the_device_chose(dtype, n, keep):
    """Steps that run one behind another without the host: each token is the largest logit of the rows that were held (or as good as it)."""
    from cisr_b200 import StepEntry

    stepper = stepper_of(model_of(dtype, 4, 2, 256), graph=True, keep=keep, n_pages=100)
    keys = [f"r{i}" for i in range(n)]
    for i, key in enumerate(keys):
        stepper.create(key)
        stepper.step([StepEntry(key, tokens_of(20 + i, i))])
    fed = {key: [i + 1] for i, key in enumerate(keys)}
    stepper.step([StepEntry(key, fed[key], [0]) for key in keys])
    first = stepper.last_tokens.tolist()
    chosen = stepper.decode_ahead(12).tolist()
    assert len(chosen) == 12
    stepper.check_kernels()
    for i, key in enumerate(keys):
        fed[key] += [first[i]] + [row[i] for row in chosen[:-1]]
        want = on_held_rows(stepper, key, fed[key])
        picked = want.gather(1, torch.tensor([[first[i]]] + [[row[i]] for row in chosen], device="cuda"))[:, 0]
        # a logit is off by several times what all are in the mean square
        assert (want.amax(-1) - picked <= 2 * 4 * logits_bound(stepper.model.dtype) * want.std()).all()
