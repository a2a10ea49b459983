"""Blocks at sizes, caches and orders that tests/test_gpu_block.py has not: d_model 4096, where projections of adapters are cut along K and take t as further columns; 8-bit weights over
an 8-bit cache; sequences in another order.

What is compared with: the same steps in numpy, in 64 bits but for what is rounded by definition (the norm's rows, quantised ones, cached rows).  Tolerances as derived in
tests/test_gpu_block.py: 2^-7 of a row's norm, 2^-6 where the output projection has 8-bit weights.  Over an 8-bit cache values that are d <= 2^-8.4 apart before a row is quantised are a step apart
behind it with probability d / step, and a row of 128 has its largest value near 2.7 of its standard deviation, step = 2.7 / 127 = 2^-5.55: sqrt(step d) = 2^-7 in the mean square, of V, and of K
times the scores, whose standard deviation is 2 where queries and keys have adapters: 2^-6 through the probabilities.  With 2^-6.6 of 8-bit output weights and 2^-8.4 of the rest 2^-5.6; 2^-5 is asked for."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_layer import make_gqa_weights
from tests.test_gpu_norm_rows import put

pytestmark = pytest.mark.gpu
HD = 128
NAMES = ("w_q", "w_k", "w_v", "w_o")


@pytest.fixture(scope="module")
def dev():
    import relux_b200 as rb
    d = rb.Device(0)
    yield d
    d.close()


def make_pool(dev, n_slots, capacity, Hkv, int8):
    import relux_b200 as rb
    from relux_b200 import lib as L
    per = (capacity + 63) // 64
    return rb.Pool(dev, L.POOL_GQA, 1, n_slots * per, 64, n_slots, per, num_kv_heads=Hkv, head_dim=HD, cache_int8=int8)


def rotate(x, start):
    half = HD // 2
    ang = (start + np.arange(x.shape[0]))[:, None, None] * (10000.0 ** (-2.0 * np.arange(half) / HD))
    out = np.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * np.cos(ang) - x[..., 1::2] * np.sin(ang)
    out[..., 1::2] = x[..., 1::2] * np.cos(ang) + x[..., 0::2] * np.sin(ang)
    return out


class Layer:
    def __init__(self, dev, rng, pool, D, H, Hkv, rank, slots):
        from oracle import binding as orc
        self.D, self.H, self.Hkv, self.rank, self.slots = D, H, Hkv, rank, slots
        W = make_gqa_weights(orc, rng, D, H, Hkv)
        self.w = {n: orc.f32_from_bf16(v) for n, v in W.items()}
        self.dw = {n: dev.upload(v) for n, v in W.items()}
        self.int8, self.w8, self.lora, self.ab = {}, {}, {}, {}
        for n in NAMES:
            k, m = W[n].shape
            self.int8[n] = dev.alloc(k * m), dev.alloc(4 * m)
            pool.int8_weights(k, m, self.dw[n], *self.int8[n])
            c, s = G.quantise(self.w[n].T)
            self.w8[n] = (c * s[:, None]).T
            da, a = put(dev, (rng.standard_normal((slots, rank, k)) * k ** -0.5).reshape(-1, k), True)
            db, b = put(dev, (rng.standard_normal((slots, m, rank)) * rank ** -0.5).reshape(-1, rank), True)
            self.lora[n], self.ab[n] = (da, db, None), (a.reshape(slots, rank, k), b.reshape(slots, m, rank))
        self.dg, self.g = put(dev, 1 + 0.2 * rng.standard_normal(D), True)

    def free(self):
        for v in list(self.dw.values()) + [x for t in (self.int8, self.lora) for v in t.values() for x in v if x] + [self.dg]:
            v.free()

    def project(self, y, n, int8, lora, adapter, S):
        y32 = y.astype(np.float32)
        y16 = G.bf16(y32)
        if n in int8:
            c, s = G.quantise(y32)
            out = (c * s[:, None].astype(np.float64)) @ self.w8[n].astype(np.float64)
        else:
            out = y16.astype(np.float64) @ self.w[n].astype(np.float64)
        if n in lora:
            a, b = self.ab[n]
            for i, s in enumerate(adapter):
                if s >= 0:
                    r = slice(i * S, (i + 1) * S)
                    out[r] += (y16[r].astype(np.float64) @ a[s].T) @ b[s].T
        return out

    def step(self, cache, order, x, r, int8, lora, adapter, held8):
        B, S, D = x.shape
        H, Hkv = self.H, self.Hkv
        h = (x + r).astype(np.float64).reshape(B * S, D)
        y = h / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-5) * self.g
        q, k, v = (self.project(y, n, int8, lora, adapter, S) for n in NAMES[:3])
        attn = np.zeros((B, S, H, HD))
        for b, seq in enumerate(order):
            rows = slice(b * S, (b + 1) * S)
            qb, kb, vb = q[rows].reshape(S, H, HD), k[rows].reshape(S, Hkv, HD), v[rows].reshape(S, Hkv, HD)
            start = cache[seq][0].shape[0]
            qb, kb = rotate(qb, start), rotate(kb, start)
            K, V = (np.concatenate([c, G.held(n.astype(np.float32), held8)]) for c, n in zip(cache[seq], (kb, vb)))
            cache[seq] = K, V
            for i in range(S):
                for hh in range(H):
                    s = K[:start + i + 1, hh // (H // Hkv)].astype(np.float64) @ qb[i, hh] / np.sqrt(HD)
                    p = np.exp(s - s.max())
                    attn[b, i, hh] = p @ V[:start + i + 1, hh // (H // Hkv)] / p.sum()
        return self.project(attn.reshape(B * S, H * HD), "w_o", int8, lora, adapter, S).reshape(B, S, D)


@pytest.mark.parametrize("B,S", [(3, 1), (20, 1), (5, 9), (2, 150)])
@pytest.mark.parametrize("int8,lora,held8", [(NAMES, (), True), ((), NAMES, False), (NAMES, NAMES, True), (("w_q", "w_o"), ("w_k", "w_o"), False)])
def test_wide_layers_in_another_order(dev, B, S, int8, lora, held8):
    """d_model 4096, 32 heads on 8, adapters of rank 64 in 3 slots; sequences in an order of their own, two of the pool's not named."""
    rng = np.random.default_rng(B * 10 + S)
    D, H, Hkv, slots = 4096, 32, 8, 3
    pool = make_pool(dev, B + 2, 512, Hkv, held8)
    for _ in range(B + 2):
        pool.seq_alloc(512)
    layer = Layer(dev, rng, pool, D, H, Hkv, 64, slots)
    order = rng.permutation(B + 2)[:B].astype(np.int32)
    cache = {int(s): (np.zeros((0, Hkv, HD), np.float32),) * 2 for s in order}
    adapter = [int(a) for a in rng.integers(-1, slots, B)]
    adapter[0] = 0
    bound = 2.0 ** (-5 if held8 else -6 if "w_o" in int8 else -7)
    for _ in range(2):
        x, r = (G.bf16(rng.standard_normal((B, S, D)).astype(np.float32)) for _ in range(2))
        dx, dr, out = dev.upload(x), dev.upload(r), dev.alloc(B * S * D * 4, 0)
        pool.block_cached(0, B, dx, out, {n: v for n, v in layer.dw.items() if n not in int8}, D, H, layer.dg, residual=dr, residual_out=dr,
                          int8={n: layer.int8[n] for n in int8}, lora={n: layer.lora[n] for n in lora}, rank=64, n_slots=slots,
                          adapter=adapter if lora else None, q_tokens=S, seq_ids=order)
        want = layer.step(cache, [int(s) for s in order], x, r, int8, lora, adapter, held8)
        got = out.download((B, S, D), np.float32)
        assert np.array_equal(dr.download((B, S, D), np.float32), x + r)
        for b in range(B):
            assert np.linalg.norm(got[b] - want[b]) <= bound * np.linalg.norm(want[b]), b
        for b in (dx, dr, out):
            b.free()
    assert pool.status() == 0
    pool.destroy()
    layer.free()
