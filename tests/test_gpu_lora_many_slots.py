"""Adapters at the ends of what the call takes: more slots than 16 bits number."""
import numpy as np
import pytest

from tests.test_gpu_lora import Case, dev, pool  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("adapter", [[32768, -1, 32799, 0], [32767]])
def test_rows_of_many_slots_keep_their_bits(dev, pool, adapter):  # noqa: F811
    """Up to 8 float32 rows keep 16 bits, however many slots there are."""
    rng = np.random.default_rng(len(adapter))
    c = Case(dev, rng, [1] * len(adapter), adapter, 264, 16, 8, 32800)
    c.call(pool)
    c.check()
    c.free()
