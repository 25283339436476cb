"""Steps of a model whose cache is held in 4 bits, one by one: what a captured step launches, and every step's logits against 64 bits over the
rows that the cache really holds."""
import pytest
import torch

from test_int4_cache import Launching
from test_int4_engine_gpu import model_of, stepper_of, tokens_of

pytestmark = pytest.mark.gpu


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
