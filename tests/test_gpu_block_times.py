"""What a pool's projection times say after blocks: the joint projections of a plain block are timed, those of a block with adapters or 8-bit weights, several launches, are not, and no older
call's time stands in for theirs."""
import numpy as np
import pytest

from tests.test_gpu_block import D, H, HD, HKV, Layer, dev  # noqa: F401
from tests.test_gpu_layer import build_gqa_pool

pytestmark = pytest.mark.gpu


def test_projection_times_of_blocks(dev):  # noqa: F811
    from relux_b200 import lib as L
    rng = np.random.default_rng(0)
    pool = build_gqa_pool(dev, np.random.default_rng(1), 2, 1024, HKV, HD)
    layer = Layer(dev, rng, pool)
    dx, out = dev.upload(rng.standard_normal((2, 1, D)).astype(np.float32)), dev.alloc(2 * D * 4, L.DTYPE_F32)
    plain = lambda: pool.block_cached(0, 2, dx, out, layer.dw, D, H)   # noqa: E731
    int8 = lambda: pool.block_cached(0, 2, dx, out, layer.dw, D, H, int8={"w_q": layer.int8["w_q"]})   # noqa: E731
    lora = lambda: pool.block_cached(0, 2, dx, out, layer.dw, D, H, lora={"w_k": layer.lora["w_k"]}, rank=16, n_slots=3, adapter=[0, -1])   # noqa: E731
    int8()
    ms, n = pool.mean_projection_ms(4)
    assert n == 0 and ms == 0
    plain()
    ms, n = pool.mean_projection_ms(1)
    assert n == 1 and 0 < ms < 5
    for call in (int8, lora):
        call()
        ms, n = pool.mean_projection_ms(1)
        assert n == 0 and ms == 0
    plain()
    for last, counted in ((1, 1), (2, 1), (4, 2), (5, 2)):
        ms, n = pool.mean_projection_ms(last)
        assert n == counted and 0 < ms < 5
    assert pool.status() == 0
    pool.destroy()


def test_untimed_blocks_take_no_slot(dev):  # noqa: F811
    """More calls than the ring of times holds, timed and untimed in turn: every time is its own call's, none counted from one whose slot it has inherited."""
    from relux_b200 import lib as L
    rng = np.random.default_rng(1)
    pool = build_gqa_pool(dev, np.random.default_rng(1), 1, 64, HKV, HD)
    layer = Layer(dev, rng, pool)
    dx, out = dev.upload(rng.standard_normal((1, 1, D)).astype(np.float32)), dev.alloc(D * 4, L.DTYPE_F32)
    for i in range(8192 + 40):
        pool.block_cached(0, 1, dx, out, layer.dw, D, H, advance=False, int8={"w_q": layer.int8["w_q"]} if i % 3 == 1 else None)
        if i % 2000 == 1999 or i > 8190:
            ms, n = pool.mean_projection_ms(1)
            assert n == (i % 3 != 1) and (not n or 0 < ms < 5)
    ms, n = pool.mean_projection_ms(9000)
    assert n == sum(i % 3 != 1 for i in range(40, 8232)) and 0 < ms < 1
    assert pool.status() == 0
    pool.destroy()
