"""Calls of more than 32 query rows a kv head in graphs, and plain calls of the same pool behind them."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_cache_int8 import filled, same
from tests.test_gpu_latent_graphs import Graph

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture(scope="module")
def dev():
    import relux_b200 as rb
    d = rb.Device(0)
    yield d
    d.close()


@pytest.mark.parametrize("int8", [True, False])
def test_plain_calls_behind_a_captured_prompt(dev, int8):
    """A long call on sequences out of order, captured; many plain ones on other sequences follow, and the graph's launches still run on its own."""
    rng = np.random.default_rng(1)
    H, Hkv, S, lens, ids = 32, 8, 40, [70, 41, 200], [2, 0]
    pool, cache = filled(dev, rng, lens, H, Hkv, 0, int8=int8)
    q = G.bf16(rng.standard_normal((2, S, H, D)))
    dq, out = dev.upload(q), dev.upload(np.zeros(q.shape, np.float32))
    call = lambda ids=ids: pool.decode(0, 2, dq, out, H, D, D ** -0.5, q_tokens=S, seq_ids=ids)  # noqa: E731
    call()
    want = out.download(q.shape, np.float32)
    for i, b in enumerate(ids):
        exact, bound = G.attend(cache.k[b], cache.v[b], q[i], lens[b] - S, G.causal(S), D ** -0.5)
        G.check(want[i], exact, bound)
    graph = Graph(dev, call)
    for _ in range(2):
        for _ in range(20):
            call([1, 2])
        out.zero()
        graph.launch()
        assert same(out.download(q.shape, np.float32), want)
    assert pool.status() == 0
    graph.free()
    dq.free()
    out.free()
    pool.destroy()
