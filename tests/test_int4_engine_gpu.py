"""A model whose cache is held in 4 bits, and one whose requests are cut down to the rows that attention has looked at most."""
import json
import subprocess
import sys

import pytest
import torch

import plain_int4
import plain_llama as pl
import tiny_models as tm

pytestmark = pytest.mark.gpu

RAW = {"architectures": ["LlamaForCausalLM"], "model_type": "llama", "hidden_act": "silu", "vocab_size": 256, "hidden_size": 128, "intermediate_size": 176,
       "num_hidden_layers": 2, "num_attention_heads": 4, "num_key_value_heads": 2, "rms_norm_eps": 1e-5, "rope_theta": 10000.0,
       "max_position_embeddings": 512, "tie_word_embeddings": True}


def model_of(dtype, heads=4, kv_heads=2, hidden=128, **more):
    from cisr_b200 import Model

    return Model.from_config({**RAW, "num_attention_heads": heads, "num_key_value_heads": kv_heads, "hidden_size": hidden, **more}, seed=3, dtype=dtype)


def tokens_of(n, seed=0):
    return torch.randint(0, 256, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


class Plain:
    """The same model in 64 bits with keys and values as 4 bits hold them: one sequence, token by token.  `keep` cuts it as the engine does, by
    weights of its own or by the places it is told."""

    def __init__(self, model):
        self.model = model
        t = lambda x: x.double()
        self.layers = [(l.parts()["mixer"], l.parts()["feed_forward"], l.parts()["mixer_norm"], l.parts()["feed_forward_norm"]) for l in model.layers]
        self.rows = [([], []) for _ in self.layers]
        self.t = t

    def norm(self, x, part):
        return x * torch.rsqrt(x.square().mean() + RAW["rms_norm_eps"]) * part.weight.double()

    def rounded(self, x):
        return x.to(self.model.dtype).double()

    def token(self, token, position):
        model = self.model
        x = model.embedding.table[token].double()
        for (mixer, ff, n1, n2), (keys, values) in zip(self.layers, self.rows):
            hq, hkv, dim = mixer.hq, mixer.hkv, mixer.dim
            h = self.rounded(self.norm(x, n1))
            qkv = (mixer.qkv.double() @ h).view(hq + 2 * hkv, dim)
            inv = RAW["rope_theta"] ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=x.device) / dim)
            cos, sin = (position * inv).cos(), (position * inv).sin()
            a, b = qkv[:hq + hkv, :dim // 2], qkv[:hq + hkv, dim // 2:]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
            q, k, v = self.rounded(turned[:hq]), self.rounded(turned[hq:]), self.rounded(qkv[hq + hkv:])
            keys.append(plain_int4.held(k)); values.append(plain_int4.held(v))
            ks, vs = torch.stack(keys, 1).repeat_interleave(hq // hkv, 0), torch.stack(values, 1).repeat_interleave(hq // hkv, 0)
            scores = torch.einsum("hd,hjd->hj", q, ks) * dim ** -0.5
            if mixer.window:
                scores[:, :max(0, len(keys) - mixer.window)] = -torch.inf
            p = torch.softmax(scores, -1)
            out = self.rounded(torch.einsum("hj,hjd->hd", p, vs).reshape(-1))
            x = x + mixer.o.double() @ out
            h = self.rounded(self.norm(x, n2))
            gate_up = ff.gate_up.double() @ h
            g, u = gate_up.chunk(2)
            x = x + ff.down.double() @ self.rounded(torch.nn.functional.silu(g) * u)
        return self.rounded(self.norm(x, model.final_norm)) @ model.head.weight.double().T


def stepper_of(model, **kw):
    from cisr_b200 import Stepper

    kw = {"n_pages": 64, "page_size": 8, "max_slots": 4, "cache": "int4", **kw}
    return Stepper(model, **kw)


@pytest.mark.parametrize("dtype,heads,kv_heads,hidden", [("float32", 4, 2, 128), ("bfloat16", 4, 2, 128), ("bfloat16", 6, 2, 384), ("float32", 2, 1, 256)])
@pytest.mark.parametrize("graph", [False, True])
def test_logits_are_those_of_a_cache_in_4_bits(dtype, heads, kv_heads, hidden, graph):
    """A prompt in one portion, and the same in small ones, then a reply, beside another request.

    The engine's keys and values differ from the plain ones by roundings, and a code that lies next to a border may then fall on its other
    side.  In bfloat16 a value x that is off by its last digit, 2^-8 x, crosses a border with the chance 2^-8 |x| / s, of codes up to 7 and some 3.2
    in the mean 1.2 %; each crossing is one step, so values are off by sqrt(0.012) steps, 3.4 % of their size of 3.2; keys put as much into
    the weights: 4.8 % of an attention's output, 6.8 % through two layers.  In float it is 2^-16 as often: 2e-4."""
    from cisr_b200 import StepEntry

    model = model_of(dtype, heads, kv_heads, hidden)
    prompt, reply = tokens_of(60, 1), tokens_of(20, 2)
    plain = Plain(model)
    want = torch.stack([plain.token(t, i) for i, t in enumerate(prompt + reply)])
    spread = want.std()
    results = []
    for portions in ([60], [7, 16, 1, 36]):
        stepper = stepper_of(model, graph=graph)
        stepper.create("a"); stepper.create("b")
        stepper.step([StepEntry("b", tokens_of(9, 5))])
        got, at = [], 0
        for n in portions:
            got.append(stepper.step([StepEntry("a", prompt[at:at + n], list(range(n))), StepEntry("b", tokens_of(1, at))]).clone())
            at += n
        for i, t in enumerate(reply):
            got.append(stepper.step([StepEntry("a", [t], [0]), StepEntry("b", [i], [0])])[:1].clone())
        stepper.check_kernels()
        got = torch.cat(got).double()
        off = (got - want).square().mean(-1).sqrt() / spread
        assert off.median() < (6.8e-2 if dtype == "bfloat16" else 2e-4), off
        results.append(got)
        stepper.release("a"); stepper.release("b")
        stepper.cache.check()
    assert ((results[0] - results[1]).square().mean(-1).sqrt() / spread).median() < (6.8e-2 if dtype == "bfloat16" else 2e-4)


@pytest.mark.parametrize("dtype,dim", [("float32", 32), ("bfloat16", 64), ("bfloat16", 96)])
@pytest.mark.parametrize("graph", [False, True])
def test_a_layer_with_a_window(dtype, dim, graph):
    """A layer that sees 40 keys, whose pages go back as they are passed, behind one that sees all."""
    from cisr_b200 import Model, StepEntry
    from test_toy_parts_gpu import W_CONFIG, register_windowed_toy

    register_windowed_toy()
    model = Model.from_config(dict(W_CONFIG, hidden_size=4 * dim, head_dim=dim, vocab_size=256), seed=5, dtype=dtype)
    prompt, reply = tokens_of(100, 1), tokens_of(60, 2)
    plain = Plain(model)
    want = torch.stack([plain.token(t, i) for i, t in enumerate(prompt + reply)])
    for portions in ([100], [45, 3, 52]):
        stepper = stepper_of(model, graph=graph)
        stepper.create("a")
        got, at = [], 0
        for n in portions:
            got.append(stepper.step([StepEntry("a", prompt[at:at + n], list(range(n)))]).clone())
            at += n
        for t in reply:
            got.append(stepper.step([StepEntry("a", [t], [0])]).clone())
            stepper.cache.check()
        stepper.check_kernels()
        windowed = next(g for g in stepper.cache.page_groups if g.use.window)
        assert windowed.pool.n_used <= 40 // 8 + 1
        off = (torch.cat(got).double() - want).square().mean(-1).sqrt() / want.std()
        assert off.median() < (6.8e-2 if dtype == "bfloat16" else 2e-4), off


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_engines_with_and_without_graphs(dtype):
    from cisr_b200 import Engine, Request

    model = model_of(dtype)
    outputs = []
    for kw in (dict(graph=False), dict(graph=True), dict(graph=False, policy="serial", token_budget=64, prefill_chunk=64)):
        engine = Engine.for_model(model, pages=64, page_size=8, max_active=3, cache="int4", **kw)
        for i, n in enumerate((5, 30, 17, 60)):
            engine.submit(Request(f"r{i}", tokens_of(n, i), max_new_tokens=12))
        outputs.append({r.key: r.generated for r in engine.run()})
        engine.stepper.cache.check()
        assert engine.stepper.cache.page_groups[0].pool.n_used == 0
        assert engine.stepper.cache.page_groups[0].storage.dtype == torch.uint8
    for other in outputs[1:]:        # sums run in other orders: a choice between near equals may differ, and then what follows it
        assert sum(outputs[0][k][0] == other[k][0] for k in other) >= 3
        assert all(len(v) == 12 for v in other.values())


def test_a_forked_request_goes_its_own_way():
    from cisr_b200 import StepEntry

    model = model_of("float32")
    stepper = stepper_of(model, keep=None)
    stepper.create("a")
    stepper.step([StepEntry("a", tokens_of(21))])
    stepper.fork("a", "b")
    one = stepper.step([StepEntry("a", [5], [0])]).clone()
    other = stepper.step([StepEntry("b", [9], [0])]).clone()
    again = stepper_of(model)
    again.create("c")
    again.step([StepEntry("c", tokens_of(21))])
    assert torch.allclose(again.step([StepEntry("c", [9], [0])]), other, atol=1e-3) and not torch.allclose(one, other, atol=1e-2)


@pytest.mark.parametrize("graph", [False, True])
def test_a_fork_of_a_request_that_is_cut(graph):
    """Source and copy run side by side with the same tokens, and are cut: each has its own numbers beside its keys, and they stay the same."""
    from cisr_b200 import StepEntry
    from cisr_b200.engine.step import Keep
    from cisr_b200.ops import kernels

    model = model_of("bfloat16")
    mixer = model.layers[0].mixer
    stepper = stepper_of(model, graph=graph, keep=Keep(rows=24, recent=8, first=2, slack=8))
    stepper.create("a")
    stepper.step([StepEntry("a", tokens_of(21))])
    stepper.fork("a", "b")
    group = stepper.cache.page_groups[0]
    for i, t in enumerate(tokens_of(40, 3)):
        logits = stepper.step([StepEntry(k, [t], [0]) for k in ("a", "b")])
        assert torch.equal(logits[0], logits[1])
        stepper.cache.check()
        n = stepper.cache.length("a")
        one, other = (torch.cat([group.mass[:, p] for p in stepper.cache.requests[k].tables[0]], -1)[..., :n] for k in ("a", "b"))
        assert torch.equal(one, other) and n < 32
        if i < 10:           # not cut yet: every query head has given one in all for each of the portion's latest tokens and each token since
            given = mixer.hq // mixer.hkv * (min(21, kernels.INT4_WEIGHED) + i + 1)
            assert ((one.double().sum(-1) - given).abs() < 1e-3 * given).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graph", [False, True])
def test_requests_that_are_cut(dtype, graph):
    """A reply far longer than the rows that stay: the cache's bookkeeping, places and weights are those of the same rows kept in 64 bits."""
    from cisr_b200 import StepEntry
    from cisr_b200.engine.step import Keep

    model = model_of(dtype)
    keep = Keep(rows=32, recent=12, first=2, slack=8)
    stepper = stepper_of(model, graph=graph, keep=keep)
    plain = Plain(model)
    stepper.create("a")
    prompt, reply = tokens_of(25, 1), tokens_of(70, 2)
    got = [stepper.step([StepEntry("a", prompt, list(range(25)))]).clone()]
    want = [plain.token(t, i) for i, t in enumerate(prompt)]
    cuts = 0
    for i, t in enumerate(reply):
        want.append(plain.token(t, 25 + i))
        group = stepper.cache.page_groups[0]
        before = [p for p in stepper.cache.requests["a"].tables[0]]
        got.append(stepper.step([StepEntry("a", [t], [0])])[:1].clone())
        stepper.cache.check()
        assert stepper.cache.seen("a") == 26 + i and stepper.cache.length("a") == len(plain.rows[0][0]) - (8 if len(plain.rows[0][0]) == 40 else 0)
        if len(plain.rows[0][0]) == 40:              # cut: the plain model takes over which rows stay, read out of the cache
            cuts += 1
            table = torch.tensor([stepper.cache.requests["a"].tables[0]], dtype=torch.int32, device="cuda")
            mixer = plain.layers[0][0]
            for layer, (k_cache, v_cache) in enumerate(group.planes):
                from cisr_b200.ops import kernels
                k, v = torch.empty((2, 1, mixer.hkv, 32, mixer.dim), device="cuda")
                one = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")
                kernels.int4_expand(k_cache, v_cache, k, v, one(0), table, one(32), 8)
                keys, values = plain.rows[layer]
                stay = []
                for h in range(mixer.hkv):
                    every = torch.stack([key[h] for key in keys])
                    near = (every[:, None] - k[0, h].double()[None]).square().sum(-1)
                    places = near.argmin(0).tolist()
                    assert places == sorted(places) and len(set(places)) == 32 and places[:2] == [0, 1] and places[-12:] == list(range(28, 40)), (layer, h, places)
                    stay.append(places)
                plain.rows[layer] = tuple([torch.stack([rows[stay[h][j]][h] for h in range(mixer.hkv)]) for j in range(32)] for rows in (keys, values))
    assert cuts == (25 + 70 - 32) // 8
    want, got = torch.stack(want), torch.cat(got).double()
    off = (got - want).square().mean(-1).sqrt() / want.std()
    assert off.median() < (3e-2 if dtype == "bfloat16" else 3e-4), off
    assert stepper.cache.page_groups[0].pool.peak <= 5 + 4 + 1


def test_an_engine_that_cuts():
    from cisr_b200 import Engine, Request

    model = model_of("bfloat16")
    for kw in (dict(graph=False), dict(graph=True), dict(graph=False, prefill_chunk=48, token_budget=64), dict(graph=True, reserve="lazy")):
        engine = Engine.for_model(model, pages=40, page_size=8, max_active=3, cache="int4", keep=48, **kw)
        for i, n in enumerate((5, 150, 17, 90)):
            engine.submit(Request(f"r{i}", tokens_of(n, i), max_new_tokens=120))
        done = engine.run()
        assert [len(r.generated) for r in done] == [120] * 4
        cache = engine.stepper.cache
        cache.check()
        assert cache.page_groups[0].pool.n_used == 0 and cache.page_groups[0].pool.peak <= 40
        assert all(len(t) == 0 for r in cache.requests.values() for t in r.tables.values())


def test_refusals():
    from cisr_b200 import Engine, Model

    model = model_of("float32")
    for kw, match in ((dict(cache="int8"), "int4"), (dict(cache="int4", page_size=12), "multiple of 8"), (dict(keep=32), "4 bits"),
                      (dict(cache="int4", keep=0), "cannot be cut")):
        with pytest.raises(ValueError, match=match):
            Engine.for_model(model, pages=8, **kw)
    with pytest.raises(ValueError, match="compute dtype only"):
        Engine.for_model(Model.from_config("tiny-a"), pages=8, cache="int4")       # head size 16
    with pytest.raises(ValueError, match="compute dtype only"):
        Engine.for_model(Model.from_config("ronolorn-small"), pages=8, cache="int4")


def test_the_command_line():
    for more in ([], ["--keep", "24", "--execution", "graph"]):
        done = subprocess.run([sys.executable, "-m", "cisr_b200", "--config", "smollm2-135m", "--tokens", "1,2,3,4", "--max-new-tokens", "40", "--cache", "int4", *more],
                              capture_output=True, text=True, timeout=300)
        assert done.returncode == 0, done.stderr[-2000:]
        assert len(json.loads(done.stdout)["requests"][0]["generated"]) == 40
