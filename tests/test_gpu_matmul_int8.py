"""Products of 8-bit rows with 8-bit weights: whole sums in 64 bits, then the two products and the rounding of the rule, so that every result is known bit for bit."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_latent_graphs import Graph

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    import relux_b200 as rb
    d = rb.Device(0)
    yield d
    d.close()


@pytest.fixture(scope="module")
def pool(dev):
    import relux_b200 as rb
    from relux_b200 import lib as L
    p = rb.Pool(dev, L.POOL_GQA, 1, 1, num_kv_heads=1, head_dim=128)
    yield p
    assert p.status() == 0
    p.destroy()


def operands(rng, M, K, N):
    return (rng.integers(-127, 128, (M, K)).astype(np.int8), np.exp2(rng.standard_normal(M)).astype(np.float32),
            rng.integers(-127, 128, (N, K)).astype(np.int8), np.exp2(rng.standard_normal(N) - 8).astype(np.float32))


def plain(a, sa, w, sw, bf16):
    total = (a.astype(np.float64) @ w.astype(np.float64).T)      # below 2^53: exact
    with np.errstate(all="ignore"):
        c = (total.astype(np.float32) * sa[:, None]).astype(np.float32) * sw
    return G.bf16(c) if bf16 else c


def same(got, want):
    return np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(got)].view(np.uint32), want[~np.isnan(want)].view(np.uint32))


class Case:
    def __init__(self, dev, a, sa, w, sw, bf16):
        from relux_b200 import lib as L
        self.shape, self.bf16 = (a.shape[0], a.shape[1], w.shape[0]), bf16
        self.d = [dev.upload(x) for x in (a, sa, w, sw)]
        M, _, N = self.shape
        self.out = dev.alloc((M + 1) * N * (2 if bf16 else 4), L.DTYPE_BF16 if bf16 else L.DTYPE_F32)
        self.clear(dev)

    def clear(self, dev):
        from relux_b200 import lib as L
        L.check(dev.lib.relux_cuda_memset(dev.h, self.out.ptr, 0xFF, self.out.nbytes))

    def call(self, pool):
        pool.matmul_int8(*self.shape, *self.d, self.out)

    def get(self):
        """The result; the row behind it is as it was."""
        from oracle import binding as orc
        M, _, N = self.shape
        raw = self.out.download((M + 1, N), np.uint16 if self.bf16 else np.uint32)
        assert (raw[M] == raw.dtype.type(-1 & (0xFFFF if self.bf16 else 0xFFFFFFFF))).all()
        return orc.f32_from_bf16(np.ascontiguousarray(raw[:M])) if self.bf16 else raw[:M].view(np.float32)

    def free(self):
        for b in self.d + [self.out]:
            b.free()


@pytest.mark.parametrize("M", [1, 2, 16, 17, 33, 64, 65, 128, 129, 200, 256, 257, 300, 513, 1100])
@pytest.mark.parametrize("K,N", [(16, 8), (48, 136), (144, 120), (1040, 1288), (4096, 512), (528, 4104)])
def test_products(dev, pool, M, K, N):
    rng = np.random.default_rng(M + K + N)
    ops = operands(rng, M, K, N)
    for bf16 in (False, True):
        c = Case(dev, *ops, bf16)
        c.call(pool)
        assert same(c.get(), plain(*ops, bf16))
        c.free()


@pytest.mark.parametrize("M,K,N", [(1, 16384, 4096), (60, 4096, 16384), (300, 8192, 4096), (2500, 1024, 6144), (4100, 512, 2048)])
def test_larger_products(dev, pool, M, K, N):
    rng = np.random.default_rng(M)
    ops = operands(rng, M, K, N)
    c = Case(dev, *ops, True)
    for _ in range(2):      # the second finds the first's counters and pieces
        c.clear(dev)
        c.call(pool)
        assert same(c.get(), plain(*ops, True))
    c.free()


def test_the_largest_sums(dev, pool):
    """All codes -128 at the longest K: the sum is 2^14 K, just below 2^31."""
    K, N, M = 131056, 8, 17
    a, w = np.full((M, K), -128, np.int8), np.full((N, K), -128, np.int8)
    ops = (a, np.ones(M, np.float32), w, np.ones(N, np.float32))
    c = Case(dev, *ops, False)
    c.call(pool)
    assert (c.get() == np.float32(16384.0 * K)).all()
    c.free()


def test_rows_of_nan(dev, pool):
    """A row or a column whose scale is NaN, codes zeros: NaN in that row and column, nowhere else."""
    rng = np.random.default_rng(3)
    a, sa, w, sw = operands(rng, 70, 256, 136)
    a[5], sa[5], w[100], sw[100] = 0, np.nan, 0, np.nan
    c = Case(dev, a, sa, w, sw, False)
    c.call(pool)
    got = c.get()
    assert same(got, plain(a, sa, w, sw, False)) and np.isnan(got[5]).all() and np.isnan(got[:, 100]).all() and np.isnan(got).sum() == 70 + 136 - 1
    c.free()


def test_many_calls_without_waiting_and_graphs(dev, pool):
    """Calls of different sizes one behind another share the pieces' memory and the counters; captured ones, launched between them, too; and plain launches."""
    from relux_b200 import lib as L
    rng = np.random.default_rng(4)
    ops = [operands(rng, *s) for s in [(1, 4096, 1024), (40, 2048, 4096), (200, 4096, 640), (300, 2048, 1288)]]
    cases = [Case(dev, *o, False) for o in ops]
    want = [plain(*o, False) for o in ops]
    cases[0].call(pool)
    graph = Graph(dev, lambda: [c.call(pool) for c in cases[:2]])
    for chained in (1, 0):
        pool.tune(L.TUNE_CHAINED_LAUNCHES, chained)
        for c in cases:
            c.clear(dev)
        for _ in range(5):
            for c in cases:
                c.call(pool)
            graph.launch()
        for c, x in zip(cases, want):
            assert same(c.get(), x)
    pool.tune(L.TUNE_CHAINED_LAUNCHES, -1)
    graph.free()
    for c in cases:
        c.free()


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("K,N", [(16, 8), (80, 72), (272, 200), (1024, 640)])
def test_weights(dev, pool, bf16, K, N):
    from oracle import binding as orc
    from relux_b200 import lib as L
    rng = np.random.default_rng(K)
    w = (rng.standard_normal((K, N)) * np.exp2(rng.standard_normal(N))).astype(np.float32)
    w[:, 1], w[3, 2], w[5, 4] = 0, np.nan, np.inf
    bits = orc.bf16_from_f32(w)
    d = dev.upload(bits if bf16 else w)
    codes, scales = dev.alloc(N * K), dev.alloc(4 * N)
    L.check(dev.lib.relux_cuda_memset(dev.h, codes.ptr, 0x55, codes.nbytes))
    pool.int8_weights(K, N, d, codes, scales)
    want, s = G.quantise((orc.f32_from_bf16(bits) if bf16 else w).T)
    assert np.array_equal(codes.download((N, K), np.int8), want)
    got = scales.download(N, np.float32)
    assert same(got, s) and np.isnan(got[2]) and np.isnan(got[4])
    for b in (d, codes, scales):
        b.free()


def test_norm_then_product(dev, pool):
    """As a layer uses them, many times without waiting: the residual's sum, the norm in 8 bits, the projection.  The product is that of the numbers the norm has written."""
    from relux_b200 import lib as L
    rng = np.random.default_rng(8)
    M, K, N = 50, 2048, 1544
    x, r = (rng.standard_normal((M, K)).astype(np.float32) for _ in range(2))
    _, _, w, sw = operands(rng, M, K, N)
    dx, dr, dw, dsw = (dev.upload(v) for v in (x, r, w, sw))
    h, codes, scales, out = dev.alloc(4 * M * K, 0), dev.alloc(M * K), dev.alloc(4 * M), dev.alloc(4 * M * N, L.DTYPE_F32)
    for _ in range(20):
        L.check(dev.lib.relux_cuda_memset(dev.h, codes.ptr, 1, codes.nbytes))
        pool.rmsnorm(M, K, dx, None, 1e-5, residual=dr, residual_out=h, codes=codes, scales=scales)
        pool.matmul_int8(M, K, N, codes, scales, dw, dsw, out)
    c, s = codes.download((M, K), np.int8), scales.download(M, np.float32)
    assert same(out.download((M, N), np.float32), plain(c, s, w, sw, False))
    y = (x.astype(np.float64) + r)
    y /= np.sqrt((y * y).mean(-1, keepdims=True) + 1e-5)
    assert (np.abs(c * s[:, None].astype(np.float64) - y) <= s[:, None] * 0.5 + np.abs(y) * 2.0 ** -16).all()
    for b in (dx, dr, dw, dsw, h, codes, scales, out):
        b.free()


def test_refusals(dev, pool):
    from relux_b200 import lib as L
    b = dev.alloc(1 << 20, L.DTYPE_F32)

    def refused(code, **kw):
        a = dict(m=2, k=64, n=64, a=b, a_scales=b, w=b, w_scales=b, out=b)
        a.update(kw)
        with pytest.raises(L.ReluxCudaError) as e:
            pool.matmul_int8(**a)
        assert e.value.code == code
    for n in ("m", "k", "n"):
        refused(L.ERR_INVALID_ARG, **{n: 0})
    for n in ("a", "a_scales", "w", "w_scales"):
        refused(L.ERR_INVALID_ARG, **{n: None})
        refused(L.ERR_INVALID_ARG, **{n: b.ptr + 8})
    refused(L.ERR_INVALID_ARG, out=b.ptr, out_dtype=3)
    refused(L.ERR_UNSUPPORTED, k=72)
    refused(L.ERR_UNSUPPORTED, n=60)
    refused(L.ERR_UNSUPPORTED, k=131072, a=b.ptr, w=b.ptr, out=b.ptr, out_dtype=0)
    b.free()
