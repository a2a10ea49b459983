"""A block, or a layer step, that finds no memory for its output projection: nothing of it stays behind, and the next call is the one that it would have been."""
import numpy as np
import pytest

from tests.test_gpu_failed_step import _fill_memory
from tests.test_gpu_layer import build_gqa_pool, make_gqa_weights

pytestmark = pytest.mark.gpu
B, D, H, HKV, HD = 16, 1024, 8, 2, 128
NAMES = ("w_q", "w_k", "w_v", "w_o")


@pytest.fixture(scope="module")
def dev():
    import relux_b200 as rb
    d = rb.Device(0)
    yield d
    d.close()


class World:
    """A pool whose buffers have served a block of 8-bit projections; its output projection wants more."""

    def __init__(self, dev, oracle, kind, S):
        from relux_b200 import lib as L
        self.dev, self.kind, self.S = dev, kind, S
        rng = np.random.default_rng(5)
        self.pool = build_gqa_pool(dev, np.random.default_rng(1), B, 1024, HKV, HD)
        W = make_gqa_weights(oracle, rng, D, H, HKV)
        self.w, self.int8 = {n: dev.upload(v) for n, v in W.items()}, {}
        for n in NAMES:
            k, m = W[n].shape
            self.int8[n] = dev.alloc(k * m), dev.alloc(4 * m)
            self.pool.int8_weights(k, m, self.w[n], *self.int8[n])
        bf16 = lambda shape, std: dev.upload(oracle.bf16_from_f32(rng.standard_normal(shape, dtype=np.float32) * np.float32(std)))   # noqa: E731
        self.lora = {"w_o": (bf16((2, 64, D), D ** -0.5), bf16((2, D, 64), 0.1), None)}
        self.x, self.r = (rng.standard_normal((4, B * S, D), dtype=np.float32) for _ in range(2))
        self.dr, self.out = dev.alloc(B * S * D * 4, L.DTYPE_F32), dev.alloc(B * S * D * 4, L.DTYPE_F32)
        self.dx = dev.alloc(B * S * D * 4, L.DTYPE_F32)
        # the buffers of every other part of the call, the launch that sets lengths too
        self.load(0)
        self.pool.block_cached(0, B, self.dx, self.out, {}, D, H, residual=self.dr, residual_out=self.dr, int8=self.int8, q_tokens=S)
        self.pool.set_len(0, np.zeros(B, np.int32))

    def load(self, i):
        self.dx.upload(self.x[i])
        self.dr.upload(self.r[i])

    def step(self):
        """The call, with the residual in place; (result, residual)."""
        more = dict(int8={n: self.int8[n] for n in NAMES[:3]})
        if self.kind == "adapters":
            more.update(lora=self.lora, rank=64, n_slots=2, adapter=[i % 3 - 1 for i in range(B)])
        if self.kind == "host result":
            more["int8"] = self.int8
        out = np.empty((B * self.S, D), np.float32) if self.kind == "host result" else self.out
        self.pool.block_cached(0, B, self.dx, out, {"w_o": self.w["w_o"]}, D, H, residual=self.dr, residual_out=self.dr, q_tokens=self.S, **more)
        return out if self.kind == "host result" else self.out.download((B * self.S, D), np.float32)

    def lengths(self):
        return [self.pool.seq_len(0, s) for s in range(B)]

    def close(self):
        assert self.pool.status() == 0
        self.pool.destroy()
        for b in [self.dx, self.dr, self.out] + list(self.w.values()) + [x for v in self.int8.values() for x in v] + [x for x in self.lora["w_o"] if x]:
            b.free()


@pytest.mark.parametrize("S", [1, 40])
@pytest.mark.parametrize("kind", ["plain", "adapters", "host result"])
def test_block_without_memory(dev, oracle, kind, S):
    from relux_b200 import lib as L
    if kind != "plain" and S == 1:
        S = 17      # 16 rows ask for 0.6 MB: blocks of up to 1 MB may be left
    failing, other = World(dev, oracle, kind, S), World(dev, oracle, kind, S)
    failing.load(1)
    held = _fill_memory(dev)
    try:
        with pytest.raises(L.ReluxCudaError) as e:
            failing.step()
        assert e.value.code == L.ERR_OUT_OF_MEMORY
    finally:
        for b in held:
            b.free()
    assert failing.lengths() == [0] * B
    assert np.array_equal(failing.dr.download((B * S, D), np.float32), failing.r[1])      # the residual too
    for i in (1, 2):      # the device's lengths: where these rows land, and what they see
        if i == 2:
            failing.load(i)
        other.load(i)
        a, b = failing.step(), other.step()
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32)) and np.isfinite(a).all()
        assert np.array_equal(failing.dr.download((B * S, D), np.float32), other.dr.download((B * S, D), np.float32))
        assert failing.lengths() == other.lengths() == [i * S] * B
    for s in (0, B - 1):
        for x, y in zip(failing.pool.read_rows(0, s, 0, 2 * S), other.pool.read_rows(0, s, 0, 2 * S)):
            assert np.array_equal(x, y)
    failing.close(), other.close()


@pytest.mark.parametrize("kind", ["gqa", "mla"])
def test_layer_step_without_memory_for_its_result(dev, oracle, kind):
    """A first call has left its result on the device; a second one wants it on the host, and finds no room for it on the way there."""
    import relux_b200 as rb
    from relux_b200 import lib as L
    S, n_heads, d = 17, 8, 1024
    rng = np.random.default_rng(6)
    x = rng.standard_normal((3, B, S, d), dtype=np.float32)
    up = lambda k, m: dev.upload(oracle.bf16_from_f32(rng.standard_normal((k, m), dtype=np.float32) * np.float32(k ** -0.5)))   # noqa: E731
    if kind == "gqa":
        w = {n: up(d, m) for n, m in dict(w_q=d, w_k=HKV * HD, w_v=HKV * HD, w_o=d).items()}
        pools = [build_gqa_pool(dev, np.random.default_rng(1), B, 256, HKV, HD) for _ in range(2)]
    else:
        w = {n: up(k, m) for n, (k, m) in dict(w_q=(d, d), w_qr=(d, n_heads * 64), w_dkv=(d, 512), w_kr=(d, 64), w_uk=(512, d), w_uv=(512, d), w_o=(d, d)).items()}
        pools = [rb.Pool(dev, L.POOL_MLA, 1, B * 4, 64, B, 4, dC=512, dHR=64) for _ in range(2)]
        for p in pools:
            for _ in range(B):
                p.seq_alloc(256)
    dx, dout = dev.alloc(x[0].nbytes, L.DTYPE_F32), dev.alloc(x[0].nbytes, L.DTYPE_F32)

    def call(p, i):
        dx.upload(x[i])
        out = np.empty((B, S, d), np.float32)
        p.forward_cached(0, B, dx, out, w, d, n_heads, q_tokens=S)
        return out
    for p in pools:
        dx.upload(x[0])
        p.forward_cached(0, B, dx, dout, w, d, n_heads, q_tokens=S)
        p.set_len(0, np.full(B, S, np.int32))
    held = _fill_memory(dev)
    try:
        with pytest.raises(L.ReluxCudaError) as e:
            call(pools[0], 1)
        assert e.value.code == L.ERR_OUT_OF_MEMORY
    finally:
        for b in held:
            b.free()
    assert [pools[0].seq_len(0, s) for s in range(B)] == [S] * B
    for i in (1, 2):
        a, b = call(pools[0], i), call(pools[1], i)
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32)) and np.isfinite(a).all()
        assert [pools[0].seq_len(0, s) for s in range(B)] == [pools[1].seq_len(0, s) for s in range(B)] == [(i + 1) * S] * B
    for p in pools:
        assert p.status() == 0
        p.destroy()
    for b in list(w.values()) + [dx, dout]:
        b.free()
