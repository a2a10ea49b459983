"""The attention half of a block in one call: residual, norm, projections with 8-bit weights and adapters, RoPE, append, attention, output projection.

Without either the call is relux_rmsnorm and relux_gqa_forward_cached, bit for bit.  With them it is compared with the same steps in numpy, in 64 bits but for what is rounded by
definition (the norm's rows, quantised ones, cached rows).  What the numpy steps do not round is rounded seven times on the way (rows, queries, probabilities, attention's rows, adapters' t, P
V's and the output's operands), each by at most 2^-8 of a value, 2^-9.8 in the mean square: the result's norm is off by less than 2.7 times that, 2^-8.4; 2^-7 is asked for.
Where the output projection has 8-bit weights, attention's rows are quantised, and values that are d apart before that are a whole step apart behind it with probability
d / step: the mean square of the difference is step * mean |d|, not d^2.  A row of 1024 has its largest value near 3.3 of its standard deviation, step = 3.3 / 127 = 2^-5.3,
mean |d| <= 2^-8.4: 2^-6.85 of the row's norm, and with what comes behind it below 2^-6.6; 2^-6 is asked for."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_latent_graphs import Graph
from tests.test_gpu_layer import build_gqa_pool, make_gqa_weights
from tests.test_gpu_norm_rows import put

pytestmark = pytest.mark.gpu
D, H, HKV, HD = 1024, 8, 2, 128
NAMES = ("w_q", "w_k", "w_v", "w_o")


@pytest.fixture(scope="module")
def dev():
    import relux_b200 as rb
    d = rb.Device(0)
    yield d
    d.close()


class Layer:
    """Device weights of a layer in all forms, and their values."""

    def __init__(self, dev, rng, pool, rank=16, slots=3):
        from oracle import binding as orc
        self.rank, self.slots = rank, slots
        W = make_gqa_weights(orc, rng, D, H, HKV)
        self.w = {n: orc.f32_from_bf16(v).astype(np.float64) for n, v in W.items()}
        self.dw = {n: dev.upload(v) for n, v in W.items()}
        self.int8, self.w8, self.lora, self.ab = {}, {}, {}, {}
        for n in NAMES:
            k, m = W[n].shape
            codes, scales = dev.alloc(k * m), dev.alloc(4 * m)
            pool.int8_weights(k, m, self.dw[n], codes, scales)
            c, s = G.quantise(orc.f32_from_bf16(W[n]).T)
            self.int8[n], self.w8[n] = (codes, scales), (c.astype(np.float64) * s[:, None]).T
            da, a = put(dev, (rng.standard_normal((slots, rank, k)) * k ** -0.5).reshape(-1, k), True)
            db, b = put(dev, (rng.standard_normal((slots, m, rank)) * rank ** -0.5).reshape(-1, rank), True)
            f = (0.5 + rng.random(slots)).astype(np.float32)
            self.lora[n], self.ab[n] = (da, db, dev.upload(f)), (a.reshape(slots, rank, k).astype(np.float64), b.reshape(slots, m, rank).astype(np.float64), f)
        self.dg, self.g = put(dev, 1 + 0.2 * rng.standard_normal(D), True)

    def project(self, y, n, int8, lora, adapter, S):
        """y [B * S, k], the norm's rows in 64 bits (bf16 or 8-bit ones are made here)."""
        y32 = y.astype(np.float32)
        y16 = G.bf16(y32).astype(np.float64)
        if n in int8:
            c, s = G.quantise(y32)
            out = (c.astype(np.float64) * s[:, None]) @ self.w8[n]
        else:
            out = y16 @ self.w[n]
        if n in lora:
            a, b, f = self.ab[n]
            for i, s in enumerate(adapter):
                if s >= 0:
                    r = slice(i * S, (i + 1) * S)
                    out[r] += float(f[s]) * (y16[r] @ a[s].T) @ b[s].T
        return out

    def step(self, cache, x, residual, int8, lora, adapter, rope):
        B, S, _ = x.shape
        h = (x + residual if residual is not None else x).astype(np.float64).reshape(B * S, D)
        y = h / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-5) * self.g
        q, k, v = (self.project(y, n, int8, lora, adapter, S) for n in NAMES[:3])
        attn = np.zeros((B, S, H, HD))
        for b in range(B):
            r = slice(b * S, (b + 1) * S)
            qb, kb, vb = q[r].reshape(S, H, HD), k[r].reshape(S, HKV, HD), v[r].reshape(S, HKV, HD)
            start = cache[b][0].shape[0]
            qb, kb = rope(qb, start), rope(kb, start)
            K, V = (np.concatenate([c, G.bf16(n.astype(np.float32))]) for c, n in zip(cache[b], (kb, vb)))
            cache[b] = (K, V)
            for i in range(S):
                for hh in range(H):
                    s = K[:start + i + 1, hh // (H // HKV)].astype(np.float64) @ qb[i, hh] / np.sqrt(HD)
                    p = np.exp(s - s.max())
                    attn[b, i, hh] = p @ V[:start + i + 1, hh // (H // HKV)] / p.sum()
        return h.reshape(B, S, D), self.project(attn.reshape(B * S, H * HD), "w_o", int8, lora, adapter, S).reshape(B, S, D)


def rotate(x, start):
    half = HD // 2
    pos = (start + np.arange(x.shape[0]))[:, None, None]
    ang = pos * (10000.0 ** (-2.0 * np.arange(half) / HD))
    out = np.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * np.cos(ang) - x[..., 1::2] * np.sin(ang)
    out[..., 1::2] = x[..., 1::2] * np.cos(ang) + x[..., 0::2] * np.sin(ang)
    return out


def rows(rng, B, S):
    return G.bf16(rng.standard_normal((B, S, D)).astype(np.float32))


@pytest.mark.parametrize("x_bf16", [False, True])
@pytest.mark.parametrize("B,S,residual", [(1, 1, True), (3, 2, True), (4, 1, False), (2, 70, True)])
def test_a_block_is_a_norm_and_a_layer(dev, B, S, residual, x_bf16):
    from relux_b200 import lib as L
    rng = np.random.default_rng(B + S)
    pools = [build_gqa_pool(dev, np.random.default_rng(1), B, 256, HKV, HD) for _ in range(2)]
    layer = Layer(dev, rng, pools[0])
    h = dev.alloc(B * S * D * 4, L.DTYPE_F32)
    y = dev.alloc(B * S * D * 4, L.DTYPE_F32)
    sums = [dev.alloc(B * S * D * 4, L.DTYPE_F32) for _ in range(2)]
    for _ in range(2):
        dx, x = put(dev, rows(rng, B, S).reshape(-1, D), x_bf16)
        dr, r = put(dev, rows(rng, B, S).reshape(-1, D), False)
        out = [np.empty((B, S, D), np.float32) for _ in range(2)]
        pools[0].block_cached(0, B, dx, out[0], layer.dw, D, H, layer.dg, residual=dr if residual else None, residual_out=sums[0] if residual else None, q_tokens=S)
        pools[1].rmsnorm(B * S, D, dx, layer.dg, 1e-5, residual=dr if residual else None, residual_out=sums[1] if residual else None, out=y, residual_dtype=0, out_dtype=0)
        pools[1].forward_cached(0, B, y, out[1], layer.dw, D, H, q_tokens=S)
        assert np.array_equal(out[0].view(np.uint32), out[1].view(np.uint32)) and np.isfinite(out[0]).all()
        if residual:
            got = [s.download((B * S, D), np.float32) for s in sums]
            assert np.array_equal(got[0], x + r) and np.array_equal(got[0], got[1])
    for b in range(B):
        k, v = (p.read_rows(0, b, 0, 2 * S) for p in pools)
        assert np.array_equal(k[0], v[0]) and np.array_equal(k[1], v[1])
    for p in pools:
        assert p.status() == 0
        p.destroy()
    for b in [h, y] + sums:
        b.free()


@pytest.mark.parametrize("B,S,slots_of", [(1, 1, [1]), (5, 1, [2, -1, 0, 2, 1]), (3, 6, [-1, 2, 2]), (3, 90, [1, 0, -1])])
@pytest.mark.parametrize("int8,lora", [(NAMES, ()), ((), NAMES), (NAMES, NAMES), (("w_k", "w_o"), ("w_q", "w_v"))])
def test_projections_of_every_kind(dev, B, S, slots_of, int8, lora):
    rng = np.random.default_rng(B * 10 + S)
    pool = build_gqa_pool(dev, np.random.default_rng(1), B, 512, HKV, HD)
    layer = Layer(dev, rng, pool)
    cache = [(np.zeros((0, HKV, HD), np.float32),) * 2 for _ in range(B)]
    for step in range(2):
        x, r = rows(rng, B, S), rows(rng, B, S)
        dx, dr = dev.upload(x), dev.upload(r)
        out = dev.alloc(B * S * D * 4, 0)
        pool.block_cached(0, B, dx, out, {n: v for n, v in layer.dw.items() if n not in int8}, D, H, layer.dg, residual=dr, residual_out=dr,
                          int8={n: layer.int8[n] for n in int8}, lora={n: layer.lora[n] for n in lora}, rank=layer.rank, n_slots=layer.slots,
                          adapter=slots_of if lora else None, q_tokens=S)
        h, want = layer.step(cache, x, r, int8, lora, slots_of, rotate)
        got = out.download((B, S, D), np.float32)
        assert np.array_equal(dr.download((B, S, D), np.float32), (x + r))
        for b in range(B):      # every request by itself
            assert np.linalg.norm(got[b] - want[b]) <= 2.0 ** (-6 if "w_o" in int8 else -7) * np.linalg.norm(want[b]), (step, b)
        for b in (dx, dr, out):
            b.free()
    assert pool.status() == 0
    pool.destroy()


def test_blocks_in_a_graph_and_not_advancing(dev):
    """Rows left past the cursor (a verify); the call captured, launched twice on the same lengths: the same bits."""
    from relux_b200 import lib as L
    rng = np.random.default_rng(3)
    B, S = 3, 4
    pool = build_gqa_pool(dev, np.random.default_rng(1), B, 256, HKV, HD)
    layer = Layer(dev, rng, pool)
    dx, dr, out = dev.upload(rows(rng, B, S)), dev.upload(rows(rng, B, S)), dev.alloc(B * S * D * 4, L.DTYPE_F32)
    call = lambda: pool.block_cached(0, B, dx, out, layer.dw, D, H, layer.dg, residual=dr, int8={"w_v": layer.int8["w_v"]},  # noqa: E731
                                     lora={"w_q": layer.lora["w_q"], "w_o": layer.lora["w_o"]}, rank=layer.rank, n_slots=layer.slots, adapter=[0, -1, 2], q_tokens=S,
                                     advance=False)
    call()
    want = out.download((B, S, D), np.float32)
    graph = Graph(dev, call)
    for _ in range(2):
        out.zero()
        graph.launch()
        assert np.array_equal(out.download((B, S, D), np.float32).view(np.uint32), want.view(np.uint32))
    assert [pool.seq_len(0, b) for b in range(B)] == [0] * B and pool.status() == 0
    graph.free()
    pool.destroy()


def test_refusals_leave_the_cache_as_it_was(dev):
    from relux_b200 import lib as L
    rng = np.random.default_rng(4)
    pool = build_gqa_pool(dev, np.random.default_rng(1), 2, 64, HKV, HD)
    layer = Layer(dev, rng, pool)
    dx, out = dev.upload(rows(rng, 2, 1)), dev.alloc(2 * D * 4, L.DTYPE_F32)
    lora = dict(lora=layer.lora, rank=16, n_slots=3, adapter=[0, 1])

    def refused(code, **kw):
        a = dict(layer=0, n_seqs=2, x=dx, out=out, weights=layer.dw, d_model=D, num_heads=H, norm_weight=layer.dg)
        a.update(kw)
        with pytest.raises(L.ReluxCudaError) as e:
            pool.block_cached(**a)
        assert e.value.code == code and pool.seq_len(0, 0) == 0
    refused(L.ERR_INVALID_ARG, **{**lora, "adapter": [0, 3]})
    refused(L.ERR_INVALID_ARG, **{**lora, "adapter": None})
    refused(L.ERR_INVALID_ARG, **{**lora, "n_slots": 0})
    refused(L.ERR_UNSUPPORTED, **{**lora, "rank": 20})
    refused(L.ERR_INVALID_ARG, eps=-1.0)
    refused(L.ERR_INVALID_ARG, residual_out=out)
    refused(L.ERR_INVALID_ARG, weights={n: layer.dw[n] for n in NAMES[:3]})
    refused(L.ERR_INVALID_ARG, int8={"w_q": (layer.int8["w_q"][0], None)})
    refused(L.ERR_INVALID_ARG, lora={"w_q": (layer.lora["w_q"][0], None, None)}, rank=16, n_slots=3, adapter=[0, 1])
    refused(L.ERR_INVALID_ARG, norm_weight=layer.dg.ptr + 4)
    refused(L.ERR_INVALID_ARG, out=out.ptr + 4)
    refused(L.ERR_INVALID_ARG, x=dx.ptr + 4, x_dtype=0)
    with pytest.raises(L.ReluxCudaError):
        pool.tune(L.TUNE_GEMM_GENERIC, 1)
        try:
            pool.block_cached(0, 2, dx, out, layer.dw, D, H)
        finally:
            pool.tune(L.TUNE_GEMM_GENERIC, -1)
    with pytest.raises(TypeError):
        pool.block_cached(0, 2, dx, out, layer.dw, D, H, residual=np.zeros((2, D), np.float32))
    with pytest.raises(ValueError):
        pool.block_cached(0, 2, dx, out, layer.dw, D, H, adapter=[0])
    pool.block_cached(0, 2, dx, out, layer.dw, D, H)
    assert pool.seq_len(0, 0) == 1
    pool.destroy()
