"""Forms of the adapters' call that its other tests do not reach: the projection's blocks of rows in turns behind groups of 16 rows, with tiles in several pieces that differ from row to row."""
import numpy as np
import pytest

from tests.test_gpu_lora import Case, dev, pool  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rank", [8, 64])
@pytest.mark.parametrize("K,N", [(2056, 1160), (4096, 392)])
@pytest.mark.parametrize("rows_each,B", [(33, 160), (80, 66), (7, 640)])
@pytest.mark.parametrize("x_bf16", [False, True])
def test_row_blocks_in_turns_of_many_requests(dev, pool, rows_each, B, K, N, rank, x_bf16):  # noqa: F811
    """Requests that fill their tiles to less than seven tenths, of more rows than the projection has blocks beside each other."""
    rng = np.random.default_rng(rows_each + K + rank)
    rows = np.full(B, rows_each) + rng.integers(-3, 4, B)
    c = Case(dev, rng, rows, rng.integers(-1, 5, B), K, N, rank, 5, x_bf16, not x_bf16)
    c.call(pool)
    c.check()
    c.free()
