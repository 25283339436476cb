"""A cache held in 4 bits on the host (no GPU): sizes and refusals, the bookkeeping of requests that are cut, the engine's page arithmetic."""
import numpy as np
import pytest
import torch
import torch.utils._python_dispatch

from cisr_b200.cache import CacheManager, OutOfPages
from cisr_b200.config.spec import CacheUse
from cisr_b200.engine.scheduler import Engine, Request
from cisr_b200.engine.step import Keep
from cisr_b200.ops import kernels
from cisr_b200.ops.kernels import KernelError
from test_scheduler import VOCAB, choose

HELD = CacheUse("pages", kv_heads=2, head_dim=32, held="int4")


def manager(uses=(HELD, HELD), n_pages=12, page_size=8, max_slots=4, max_positions=96, weigh=True):
    return CacheManager(list(uses), n_pages, page_size, max_slots, max_positions, weigh=weigh)


def step(m, key, n):
    m.reserve([(key, n)])
    m.commit(key, n)


def test_the_bytes_of_a_page_and_sizes_that_are_refused():
    # 4 bits a value and 16 for 32 of them: 4.5
    for page in (8, 24, 64):
        for dim in (32, 64, 96, 128):
            assert kernels.int4_page_bytes(page, dim) * 8 == page * dim * 4.5
    for page in (0, -8, 4, 12, 63):
        with pytest.raises(KernelError, match="multiple of 8"):
            kernels.int4_page_bytes(page, 64)
    for dim in (0, 16, 48, 256):
        with pytest.raises(KernelError, match="head sizes 32, 64, 96, 128"):
            kernels.int4_page_bytes(16, dim)


def test_calls_on_the_cpu_are_refused():
    cache = torch.zeros((2, 1, kernels.int4_page_bytes(8, 32)), dtype=torch.uint8)
    x = torch.zeros((1, 1, 32))
    one = torch.zeros(1, dtype=torch.int32)
    table = torch.zeros((1, 1), dtype=torch.int32)
    mass = torch.zeros((2, 1, 8))
    kept = torch.zeros((1, 1, 4), dtype=torch.int32)
    for call in (lambda: kernels.int4_store(x, x, cache, cache, one, one, one, table, 8), lambda: kernels.int4_read(cache, cache, x, x, one, one, one, table, 8),
                 lambda: kernels.int4_expand(cache, cache, x[None], x[None], one, table, one, 8),
                 lambda: kernels.attn_decode_int4(x, x, cache, cache, one, table, one, one, one, 1, 8, 8, 1.0),
                 lambda: kernels.attn_prefill_int4(x, x, cache, cache, one, table, one, one, one, one, one, 8, 8, 1.0),
                 lambda: kernels.int4_evict(cache, cache, mass, one, table, one, table, kept, 8, 8, 1)):
        with pytest.raises(KernelError, match="CUDA device"):
            call()


def test_pages_in_4_bits_are_a_group_of_their_own():
    plain = CacheUse("pages", kv_heads=2, head_dim=32)
    m = manager((HELD, plain, HELD), weigh=False)
    assert [g.entries for g in m.page_groups] == [[0, 2], [1]]
    for use in (plain, CacheUse("pages", kv_heads=2, head_dim=32, held="int4", window=8)):
        with pytest.raises(ValueError, match="without a window"):
            manager((use,))
    with pytest.raises(ValueError, match="unknown form"):
        manager((CacheUse("pages", kv_heads=2, head_dim=32, held="int3"),), weigh=False)


def test_a_cut_request_goes_on_where_it_was():
    m = manager()
    m.create("a")
    step(m, "a", 30)
    old = list(m.requests["a"].tables[0])
    pages = m.plan_cut(["a"], 20)
    assert len(pages) == 1 and len(pages[0][0]) == 3 and not set(pages[0][0]) & set(old) and m.page_groups[0].pool.n_used == 7
    m.finish_cut(["a"], 20, pages)
    assert m.length("a") == 20 and m.seen("a") == 30 and m.requests["a"].tables[0] == pages[0][0] and m.page_groups[0].pool.n_used == 3
    where, page = m.drain_table_updates(0)
    table = np.full(m.width * 4, -1, np.int32)
    table[where] = page
    assert table.reshape(4, -1)[m.slot("a")].tolist() == pages[0][0] + [-1] * (m.width - 3)
    step(m, "a", 5)                  # four more fit the third page
    assert m.length("a") == 25 and m.seen("a") == 35 and len(m.requests["a"].tables[0]) == 4
    m.check()
    with pytest.raises(ValueError, match="context limit"):
        m.reserve([("a", 62)])       # positions count what was seen, not what is kept
    m.release("a")
    m.check()
    assert m.page_groups[0].pool.n_free == 12


def test_a_cut_that_finds_no_pages_changes_nothing():
    m = manager(n_pages=5)
    m.create("a")
    step(m, "a", 32)
    before = (list(m.requests["a"].tables[0]), m.page_groups[0].pool.n_free)
    assert m.plan_cut(["a"], 16) is None and not m.plan_free(1, 16) and m.plan_free(1, 8)
    assert (m.requests["a"].tables[0], m.page_groups[0].pool.n_free) == before and m.length("a") == 32
    m.check()


def test_a_fork_of_weighed_pages_gets_its_own():
    m = manager(n_pages=8)
    m.create("a")
    step(m, "a", 20)
    m.fork("a", "b")
    a, b = m.requests["a"].tables[0], m.requests["b"].tables[0]
    assert not set(a) & set(b) and m.drain_copies(0) == list(zip(a, b)) and m.length("b") == 20 and m.seen("b") == 20
    m.check()
    with pytest.raises(OutOfPages, match="3 wanted, 2 free"):
        m.fork("a", "c")
    assert "c" not in m.requests and len(m.free_slots) == 2
    m.release("a"); m.release("b")
    m.check()
    shared = manager(weigh=False)
    shared.create("a")
    step(shared, "a", 20)
    shared.fork("a", "b")
    assert shared.requests["a"].tables[0] == shared.requests["b"].tables[0]


class Launching(torch.utils._python_dispatch.TorchDispatchMode):
    """Names torch's operations that put something on the stream: all but views and new tensors."""
    QUIET = ("empty", "new_empty", "empty_like", "empty_strided", "unbind", "select", "slice", "view", "_unsafe_view", "as_strided", "transpose", "detach", "alias", "split", "t",
             "squeeze", "unsqueeze", "expand", "_reshape_alias", "chunk", "permute")

    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        name = func.overloadpacket.__name__
        if name not in self.QUIET:
            self.seen.append(name)
        return func(*args, **(kwargs or {}))


def test_a_steps_own_places_are_older_than_the_step():
    """The products look them up before they wait for the kernel ahead of them: no kernel of the step may write them, and what a captured step
    reads stays where it is when longer steps come."""
    from types import SimpleNamespace

    from cisr_b200.cache.manager import StepPlaces
    from cisr_b200.parts.attention import staged_rows

    places = StepPlaces(8, "cpu")
    with Launching() as mode:
        to = staged_rows(SimpleNamespace(n_tokens=5, device="cpu", shared={}), SimpleNamespace(places=places), 2, 32, torch.float32)
    assert mode.seen == [], mode.seen
    assert to.k.shape == to.v.shape == (1, 2, 5, 32) and to.page_size == 5 and to.block_table.tolist() == [[0]] and to.req_slot.tolist() == [0]
    assert to.positions.tolist() == [0, 1, 2, 3, 4] and to.token_req.tolist() == [0] * 5
    assert places(5)[0].data_ptr() == to.positions.data_ptr() and places(8)[0].data_ptr() == to.positions.data_ptr()
    rows, zeros = places(9)
    assert rows.tolist() == list(range(9)) and zeros.tolist() == [0] * 9 and places.lists[0][0].data_ptr() == to.positions.data_ptr()
    assert places(300)[0].tolist() == list(range(300)) and len(places.lists) == 3


def test_what_is_kept():
    assert Keep.of(64, 16) == Keep(64, 32, 4, 16) and Keep.of(4, 8) == Keep(4, 2, 1, 8) and Keep.of(1, 8) == Keep(1, 0, 0, 8)
    keep = Keep(10, 4, 6, 1)
    assert Keep.of(keep, 8) is keep
    for bad in ((0, 0, 0, 1), (8, 4, 5, 1), (8, -1, 0, 1), (8, 0, -1, 1), (8, 2, 2, 0)):
        with pytest.raises(ValueError, match="cannot be cut"):
            Keep(*bad)


class CuttingStepper:
    """The stepper's bookkeeping without its kernels."""

    def __init__(self, keep, pages, page_size, max_slots, max_positions):
        self.keep, self.cache, self.cuts, self.last_extras = keep, manager((HELD,), pages, page_size, max_slots, max_positions), 0, {}

    def create(self, key):
        self.cache.create(key)

    def release(self, key):
        self.cache.release(key)

    def step(self, entries, extra=None):
        self.cache.reserve([(e.key, len(e.tokens)) for e in entries])
        for e in entries:
            self.cache.commit(e.key, len(e.tokens))
        for e in entries:
            if self.cache.length(e.key) >= self.keep.rows + self.keep.slack:
                pages = self.cache.plan_cut([e.key], self.keep.rows)
                if pages is not None:
                    self.cache.finish_cut([e.key], self.keep.rows, pages)
                    self.cuts += 1
        self.cache.check()
        return np.zeros((sum(len(e.want) for e in entries), VOCAB), np.float32)


@pytest.mark.parametrize("reserve", ["full", "lazy"])
@pytest.mark.parametrize("pages,chunk", [(14, 8), (24, 5), (60, 16)])
def test_an_engine_needs_pages_for_the_rows_that_stay(reserve, pages, chunk):
    """Requests whose whole lives would not fit the pool run to their ends, each cut whenever it is time."""
    keep = Keep.of(32, 8)
    stepper = CuttingStepper(keep, pages, 8, 4, 400)
    engine = Engine(stepper, choose, VOCAB, 400, max_active=3, token_budget=32, prefill_chunk=chunk, reserve=reserve, keep=keep)
    for i, n in enumerate((5, 150, 33, 90, 200)):
        engine.submit(Request(f"r{i}", [1] * n, max_new_tokens=150))
    done = engine.run()
    assert [len(r.generated) for r in done] == [150] * 5 and stepper.cuts >= (5 + 150 + 33 + 90 + 200 + 5 * 149 - 5 * 40) // 8 // 2
    assert stepper.cache.page_groups[0].pool.n_used == 0


def test_a_request_that_never_fits_is_refused():
    """The rows that call for a cut, a portion more, and the cut's own pages are more than the pool has."""
    keep = Keep.of(64, 8)
    stepper = CuttingStepper(keep, 17, 8, 4, 400)
    engine = Engine(stepper, choose, VOCAB, 400, max_active=3, token_budget=32, prefill_chunk=8, keep=keep)
    with pytest.raises(ValueError, match="10 pages wanted, 9 exist"):
        engine.submit(Request("r", [1] * 200, max_new_tokens=100))
    engine.submit(Request("s", [1] * 20, max_new_tokens=10))
    assert len(engine.run()[-1].generated) == 10


def test_portions_go_in_groups_of_like_lengths():
    """A call writes every request's rows out at the length of its longest: at most half as much again as they have."""
    from cisr_b200.parts.attention import portion_groups

    assert portion_groups([1, 1, 2, 32], [5, 900, 40, 40], 32) == [] and portion_groups([], [], 32) == []
    assert portion_groups([100, 1, 60, 33], [1000, 9000, 900, 1000], 32) == [[0, 3, 2]]
    assert portion_groups([33] + [40] * 30 + [2] * 30, [100000] + [40] * 30 + [100000] * 30, 32) == [[0], list(range(1, 31))]
    rng = np.random.default_rng(3)
    for _ in range(200):
        n = int(rng.integers(1, 40))
        lens = rng.integers(0, 80, n).tolist()
        ends = [k + int(10 ** rng.uniform(0, 5)) for k in lens]
        groups = portion_groups(lens, ends, 32)
        assert sorted(r for g in groups for r in g) == [r for r, k in enumerate(lens) if k > 32]
        for g in groups:
            assert ends[g[0]] == max(ends[r] for r in g) and 2 * len(g) * ends[g[0]] <= 3 * sum(ends[r] for r in g)
