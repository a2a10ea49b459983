"""More than 32 query heads to a kv head over the 8-bit cache: such calls go to the tensor-core kernel whatever their number of tokens."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_cache_int8 import filled

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture(scope="module")
def dev():
    import relux_b200 as rb
    d = rb.Device(0)
    yield d
    d.close()


@pytest.mark.parametrize("H,Hkv", [(33, 1), (40, 1), (96, 2), (128, 1)])
@pytest.mark.parametrize("S", [1, 3, 17])
@pytest.mark.parametrize("lens", [[0, 63, 200], [1700]])
def test_decode_verify_and_step(dev, H, Hkv, S, lens):
    rng = np.random.default_rng(H + S)
    B = len(lens)
    pool, cache = filled(dev, rng, lens, H, Hkv, S + 1)
    k, v, q = G.rows(rng, B * S, Hkv), G.rows(rng, B * S, Hkv, "v"), G.bf16(rng.standard_normal((B, S, H, D)))
    out = np.empty((B, S, H, D), np.float32)
    outs = []
    pool.verify(0, B, q, out, k, v, H, D, D ** -0.5, S)
    outs.append(out.copy())
    pool.append(0, k, v, B, n_new=[S] * B)
    pool.decode(0, B, q, out, H, D, D ** -0.5, q_tokens=S)
    outs.append(out.copy())
    for b in range(B):
        cache.append(b, k[b * S:(b + 1) * S], v[b * S:(b + 1) * S])
        want, bound = G.attend(cache.k[b], cache.v[b], q[b], lens[b], G.causal(S), D ** -0.5)
        for name, o in zip(("verify", "decode"), outs):
            G.check(o[b], want, bound, "%s, sequence %d" % (name, b))
    out = np.empty((B, 1, H, D), np.float32)
    pool.step(0, B, k[:B], v[:B], np.ascontiguousarray(q[:, :1]), out, H, D, D ** -0.5)
    for b in range(B):
        cache.append(b, k[b:b + 1], v[b:b + 1])
        want, bound = G.attend(cache.k[b], cache.v[b], q[b, :1], lens[b] + S, G.causal(1), D ** -0.5)
        G.check(out[b], want, bound, "step, sequence %d" % b)
    assert pool.status() == 0
    pool.destroy()
