"""A captured block keeps the scratch that it was captured with, when later calls of the same pool ask for more."""
import numpy as np
import pytest

from tests.test_gpu_block import D, H, HD, HKV, NAMES, Layer, dev, rows  # noqa: F401
from tests.test_gpu_latent_graphs import Graph
from tests.test_gpu_layer import build_gqa_pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["plain", "int8", "adapters", "both"])
def test_captured_blocks_keep_their_scratch(dev, kind):  # noqa: F811
    from relux_b200 import lib as L
    rng = np.random.default_rng(9)
    B = 3
    pool = build_gqa_pool(dev, np.random.default_rng(1), B, 1024, HKV, HD)
    layer = Layer(dev, rng, pool)
    more = dict(int8=layer.int8) if kind in ("int8", "both") else {}
    if kind in ("adapters", "both"):
        more.update(lora=layer.lora, rank=layer.rank, n_slots=layer.slots, adapter=[2, -1, 0])

    def world(S):
        dx, dr, out = dev.upload(rows(rng, B, S)), dev.upload(rows(rng, B, S)), dev.alloc(B * S * D * 4, L.DTYPE_F32)
        return lambda: pool.block_cached(0, B, dx, out, layer.dw, D, H, layer.dg, residual=dr, q_tokens=S, advance=False, **more), out, (B, S, D)
    small, out, shape = world(1)
    small()
    want = out.download(shape, np.float32)
    graph = Graph(dev, small)
    for S in (40, 700):      # each asks for more than the one before
        large, large_out, large_shape = world(S)
        large()
        first = large_out.download(large_shape, np.float32)
        assert np.isfinite(first).all()
        for _ in range(2):
            out.zero(), large_out.zero()
            graph.launch(), large(), graph.launch()
            assert np.array_equal(out.download(shape, np.float32).view(np.uint32), want.view(np.uint32))
            assert np.array_equal(large_out.download(large_shape, np.float32).view(np.uint32), first.view(np.uint32))
    assert pool.status() == 0
    graph.free()
    pool.destroy()
