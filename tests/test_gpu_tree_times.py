"""The kernel times of calls whose streams are split: the join of the parts is in them."""
import ctypes as C

import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_cache_int8 import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
def test_the_join_is_part_of_the_time(int8):
    """One long sequence of one kv head: its parts are joined row by row, in several times what they take.  Of the time between two events around many
    calls, the rest (the append's launch, 5 us) is a small part."""
    import relux_b200 as rb
    from relux_b200 import lib as L
    dev = rb.Device(0)
    T, H, S, N = 50000, 32, 8, 40
    pool = make(dev, 1, T // 64 + 2, 1, int8=int8)
    rng = np.random.default_rng(0)
    x = dev.upload(rng.standard_normal((T, 1, G.D)).astype(np.float32))
    pool.append(0, x, x, 1, n_new=[T])
    q, out = dev.upload(rng.standard_normal((1, S, H, G.D)).astype(np.float32)), dev.alloc(S * H * G.D * 4, L.DTYPE_F32)
    call = lambda: pool.tree_verify(0, 1, q, out, x, x, H, G.D, G.D ** -0.5, np.arange(-1, S - 1))  # noqa: E731
    rt, stream, events, ms = C.CDLL("libcudart.so.12"), C.c_void_p(), [C.c_void_p(), C.c_void_p()], C.c_float()
    L.check(dev.lib.relux_cuda_stream(dev.h, C.byref(stream)))
    for e in events:
        assert rt.cudaEventCreate(C.byref(e)) == 0
    for _ in range(5):
        call()
    dev.sync()
    assert rt.cudaEventRecord(events[0], stream) == 0
    for _ in range(N):
        call()
    assert rt.cudaEventRecord(events[1], stream) == 0
    dev.sync()
    assert rt.cudaEventElapsedTime(C.byref(ms), *events) == 0
    times = pool.kernel_ms_list(N)
    assert len(times) == N and 0.6 * ms.value <= times.sum() <= 1.02 * ms.value, (times.sum(), ms.value)
    for e in events:
        rt.cudaEventDestroy(e)
    for b in (x, q, out):
        b.free()
    pool.destroy()
    dev.close()
