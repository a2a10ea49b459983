"""Adapters at the ends of what the call takes: more columns than a grid's second dimension has blocks, and sizes that it refuses."""
import numpy as np
import pytest

from tests.test_gpu_lora import dev, pool  # noqa: F401
from tests.test_gpu_norm_rows import get, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,shared", [([1], False), ([3, 14], False), ([20], True)])
def test_more_columns_than_blocks_of_a_grid(dev, pool, rows, shared):  # noqa: F811
    """65535 blocks of 256 columns and some: sampled columns, the first, the last and those around the limit among them."""
    from oracle import binding as orc
    from relux_b200 import lib as L
    rng = np.random.default_rng(sum(rows))
    N, K, rank, M = 65535 * 256 + 520, 8, 8, sum(rows)
    cols = np.unique(np.r_[0:8, 65535 * 256 - 8:65535 * 256 + 8, N - 8:N, rng.integers(0, N, 2000)])
    dx, x = put(dev, rng.standard_normal((M, K)), True)
    da, a = put(dev, rng.standard_normal((rank, K)) * K ** -0.5, True)
    b16 = orc.bf16_from_f32(np.tile(rng.standard_normal((4099, rank)).astype(np.float32), (N // 4099 + 1, 1))[:N])
    w16 = orc.bf16_from_f32(np.tile(rng.standard_normal((K, 4099)).astype(np.float32), (1, N // 4099 + 1))[:, :N].copy()) if shared else None
    db, dw = dev.upload(b16), dev.upload(w16) if shared else None
    out = dev.alloc(M * N * 4, L.DTYPE_F32)
    out.zero()
    adapter = [0] * len(rows)
    pool.matmul_lora(M, K, N, dx, dw, out, da, db, rank, 1, adapter, rows=rows)
    got = get(out, (M, N), False)[:, cols].astype(np.float64)
    b = orc.f32_from_bf16(np.ascontiguousarray(b16[cols])).astype(np.float64)
    x, a = x.astype(np.float64), a.astype(np.float64)
    want, size = (x @ a.T) @ b.T, (np.abs(x) @ np.abs(a).T) @ np.abs(b).T
    if shared:
        w = orc.f32_from_bf16(np.ascontiguousarray(w16[:, cols])).astype(np.float64)
        want, size = want + x @ w, size + np.abs(x) @ np.abs(w)
    assert (np.abs(got - want) <= size * (2.0 ** -16 + 2.0 ** -18)).all()
    for d in (dx, da, db, dw, out):
        if d is not None:
            d.free()


def test_sizes_past_2_30_are_refused(dev, pool):  # noqa: F811
    from relux_b200 import lib as L
    b = dev.alloc(1 << 12, L.DTYPE_BF16).ptr
    for more in (dict(k=(1 << 30) + 8), dict(n=(1 << 30) + 8), dict(k=(1 << 31) - 8), dict(n=(1 << 31) - 8)):
        with pytest.raises(L.ReluxCudaError) as e:
            pool.matmul_lora(**{**dict(m=1, k=64, n=64, x=b, w=b, out=b, lora_a=b, lora_b=b, rank=16, n_slots=1, adapter=[0], x_dtype=L.DTYPE_BF16, out_dtype=L.DTYPE_BF16), **more})
        assert e.value.code == L.ERR_UNSUPPORTED
