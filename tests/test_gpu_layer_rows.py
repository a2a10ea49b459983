"""Layer steps and blocks of more rows than a grid's second dimension has blocks."""
import numpy as np
import pytest

from tests.test_gpu_block_sizes import HD, dev, make_pool  # noqa: F401
from tests.test_gpu_layer import make_gqa_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["layer", "block"])
def test_more_rows_than_a_grid_has_blocks(dev, oracle, kind):  # noqa: F811
    """66 000 rows, the same 50 sequences of 1320 tokens as in two calls of 25: the projections may be cut in another way, so that a sum's order differs (K = 128: below 2^-16 of a
    value), and with it a rounding to bf16 here or there, 2^-7 of the values' norm together."""
    from relux_b200 import lib as L
    rng = np.random.default_rng(2)
    B, S, D, H = 50, 1320, HD, 1
    w = {n: dev.upload(v) for n, v in make_gqa_weights(oracle, rng, D, H, 1).items()}
    x = rng.standard_normal((B, S, D)).astype(np.float32)
    dx, out, part = dev.upload(x), dev.alloc(x.nbytes, L.DTYPE_F32), dev.alloc(x.nbytes // 2, L.DTYPE_F32)
    pool = make_pool(dev, B, S, 1, False)
    for _ in range(B):
        pool.seq_alloc(S)
    call = lambda n, a, o, ids: (pool.forward_cached(0, n, a, o, w, D, H, q_tokens=S, seq_ids=ids) if kind == "layer" else   # noqa: E731
                                 pool.block_cached(0, n, a, o, w, D, H, q_tokens=S, seq_ids=ids))
    call(B, dx, out, None)
    got = out.download((B, S, D), np.float32)
    pool.set_len(0, np.zeros(B, np.int32))
    for half in range(2):
        ids = np.arange(B // 2, dtype=np.int32) + half * (B // 2)
        dpart = dev.upload(np.ascontiguousarray(x[ids]))
        call(B // 2, dpart, part, ids)
        want = part.download((B // 2, S, D), np.float32)
        assert np.linalg.norm(got[ids] - want) <= 2.0 ** -7 * np.linalg.norm(want)
        dpart.free()
    assert pool.status() == 0
    pool.destroy()
    for b in [dx, out, part] + list(w.values()):
        b.free()
