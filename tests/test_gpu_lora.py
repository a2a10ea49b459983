"""A shared projection with the low-rank adapters of many requests, against the sums in 64 bits.

Tolerances: sums of K products in float32, one rounding each at most, K 2^-24 of the sum of the magnitudes.  float32 rows are rounded to bf16 (by definition, so the oracle
does), but in calls of few rows or without a shared projection, which keep two bf16 halves of them, 2^-16 of a value, as t is kept in every call; the rank's sum has as many
roundings as products; a bf16 result 2^-8."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_latent_graphs import Graph
from tests.test_gpu_norm_rows import get, put

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


class Case:
    def __init__(self, dev, rng, rows, adapter, K, N, rank, slots, x_bf16=False, out_bf16=False, factors=True, shared=True):
        from relux_b200 import lib as L
        self.dev, self.rows, self.adapter, self.K, self.N, self.rank, self.slots = dev, np.asarray(rows, np.int32), np.asarray(adapter, np.int32), K, N, rank, slots
        self.M, self.x_bf16, self.out_bf16 = int(self.rows.sum()), x_bf16, out_bf16
        x = rng.standard_normal((self.M, K)).astype(np.float32)
        self.dx, self.x = put(dev, x, x_bf16)
        self.dw, self.w = put(dev, rng.standard_normal((K, N)) * K ** -0.5, True) if shared else (None, None)
        self.da, self.a = put(dev, (rng.standard_normal((slots, rank, K)) * K ** -0.5).reshape(-1, K), True)
        self.db, self.b = put(dev, (rng.standard_normal((slots, N, rank)) * rank ** -0.5).reshape(-1, rank), True)
        self.a, self.b = self.a.reshape(slots, rank, K), self.b.reshape(slots, N, rank)
        self.factors = (0.5 + rng.random(slots)).astype(np.float32) if factors else None
        self.df = dev.upload(self.factors) if factors else None
        self.out = dev.alloc((self.M + 1) * N * (2 if out_bf16 else 4), L.DTYPE_BF16 if out_bf16 else L.DTYPE_F32)
        self.clear()

    def clear(self, byte=0xFF):
        from relux_b200 import lib as L
        L.check(self.dev.lib.relux_cuda_memset(self.dev.h, self.out.ptr, byte, self.out.nbytes))

    def call(self, pool, accumulate=False):
        pool.matmul_lora(self.M, self.K, self.N, self.dx, self.dw, self.out, self.da, self.db, self.rank, self.slots, self.adapter, rows=self.rows, factors=self.df,
                         accumulate=accumulate)

    def plain(self, before=None):
        """(result, its bound) in 64 bits."""
        x = self.x.astype(np.float64)
        whole = self.w is None or (self.M <= 8 and self.M * self.rank <= 256)
        if not whole:
            x = G.bf16(self.x).astype(np.float64)
        half = 2.0 ** -16 if whole and not self.x_bf16 else 0
        u = 2.0 ** -24
        out, bound = np.zeros((self.M, self.N)), np.zeros((self.M, self.N))
        if before is not None:
            out += before
        with np.errstate(all="ignore"):
            if self.w is not None:
                out += x @ self.w.astype(np.float64)
                bound += ((self.K + 8) * u + half) * (np.abs(x) @ np.abs(self.w).astype(np.float64))
            at = 0
            for n, s in zip(self.rows, self.adapter):
                if s >= 0:
                    r = slice(at, at + n)
                    a, b = self.a[s].astype(np.float64), self.b[s].astype(np.float64)
                    f = 1.0 if self.factors is None else float(self.factors[s])
                    out[r] += f * ((x[r] @ a.T) @ b.T)
                    bound[r] += f * (((self.K + 2 * self.rank + 16) * u + 2.0 ** -16 + half) * ((np.abs(x[r]) @ np.abs(a).T) @ np.abs(b).T))
                at += n
            bound += np.abs(out) * (2.0 ** -22 + (2.0 ** -8 if self.out_bf16 else 0))
        return out, bound

    def get(self):
        got = get(self.out, (self.M + 1, self.N), self.out_bf16)
        assert np.isnan(got[self.M]).all()      # the row behind the last is as it was
        return got[:self.M].astype(np.float64)

    def check(self):
        out, bound = self.plain()
        assert (np.abs(self.get() - out) <= bound).all()

    def free(self):
        for b in (self.dx, self.dw, self.da, self.db, self.df, self.out):
            if b is not None:
                b.free()


def requests(rng, B, S, slots):
    rows = rng.integers(0, S + 1, B) if S > 1 else np.ones(B, int)
    rows[0] = max(rows[0], 1)
    return rows, rng.integers(-1, slots, B)


@pytest.mark.parametrize("rank", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("B,S,K,N,slots", [(1, 1, 8, 8, 1), (1, 1, 4096, 1024, 3), (20, 1, 264, 392, 7), (64, 1, 2048, 520, 64), (7, 5, 1000, 264, 3), (3, 90, 520, 1288, 4),
                                           (5, 400, 328, 136, 3), (200, 9, 72, 200, 20)])
@pytest.mark.parametrize("x_bf16,out_bf16", [(False, False), (True, True), (False, True)])
def test_adapters(dev, pool, rank, B, S, K, N, slots, x_bf16, out_bf16):
    rng = np.random.default_rng(rank + B + K)
    rows, adapter = requests(rng, B, S, slots)
    c = Case(dev, rng, rows, adapter, K, N, rank, slots, x_bf16, out_bf16, factors=B != 7)
    c.call(pool)
    c.check()
    c.free()


@pytest.mark.parametrize("M", [1, 40, 700, 3000])
def test_one_adapter_and_none(dev, pool, M):
    rng = np.random.default_rng(M)
    for adapter in (0, -1):
        for x_bf16 in (False, True):
            c = Case(dev, rng, [M], [adapter], 512, 640, 16, 1, x_bf16)
            c.call(pool)
            c.check()
            c.free()


def test_more_requests_than_a_launch_takes(dev, pool):
    """2500 requests of a row each, neighbours never alike: lists of several launches."""
    rng = np.random.default_rng(9)
    B = 2500
    c = Case(dev, rng, np.ones(B, int), np.arange(B) % 5 - 1, 136, 200, 16, 4)
    c.call(pool)
    c.check()
    c.free()


def test_row_blocks_in_turns(dev, pool):
    """So many rows that the projection's blocks of rows come in turns: pieces differ from row to row."""
    rng = np.random.default_rng(10)
    c = Case(dev, rng, [2900, 1, 1999, 300], [1, 0, -1, 2], 1032, 1160, 32, 3, True, True)
    c.call(pool)
    c.check()
    c.free()


@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("shared", [False, True])
def test_added_to_what_is_there(dev, pool, shared, out_bf16):
    rng = np.random.default_rng(11)
    rows, adapter = requests(rng, 12, 6, 4)
    c = Case(dev, rng, rows, adapter, 264, 392, 16, 4, out_bf16=out_bf16, shared=shared)
    before = G.bf16(rng.standard_normal((c.M, c.N)).astype(np.float32))
    from oracle import binding as orc
    c.out.upload(orc.bf16_from_f32(before) if out_bf16 else before)
    c.call(pool, accumulate=True)
    out, bound = c.plain(before)
    assert (np.abs(c.get() - out) <= bound + np.abs(before) * 2.0 ** -23).all()
    if not shared:      # without: rows of no adapter are zeros
        c.clear()
        c.call(pool)
        c.check()
    c.free()


def test_infinities_and_nan_stay_with_their_request(dev, pool):
    rng = np.random.default_rng(12)
    c = Case(dev, rng, [1] * 30, [i % 4 - 1 for i in range(30)], 264, 392, 16, 3, True)
    from oracle import binding as orc
    c.a[1, 3, 7], c.b[1, 100, 2], c.b[2, 5, :] = np.nan, np.inf, np.inf
    c.da.upload(orc.bf16_from_f32(c.a)), c.db.upload(orc.bf16_from_f32(c.b))
    c.x[4, 9] = np.nan      # the first adapter's... request 4 has none
    c.x[5, 9] = np.inf
    c.dx.upload(orc.bf16_from_f32(c.x))
    c.call(pool)
    got = c.get()
    out, bound = c.plain()
    fine = np.isfinite(out)
    assert (np.isfinite(got) == fine).all() and (np.abs(got - out)[fine] <= bound[fine]).all()
    ids = np.asarray(c.adapter)
    assert fine[(ids <= 0) & (np.arange(30) != 4) & (np.arange(30) != 5)].all() and not fine[ids == 1].any() and not fine[4].any()
    assert not fine[ids == 2][:, 5].any() and np.delete(fine[(ids == 2)], 5, axis=1).all()
    c.free()


# requests of a row each, few and so few that float32 rows are split; requests whose tiles are nearly full, with rows past their ends
FORMS = [([1] * 4, [0, 1, 2, -1], True), ([1] * 4, [-1, 2, 1, 0], False), ([1] * 12, [0, 1, 2, -1] * 3, True), ([1] * 8, [0, 1, 2, -1] * 2, False), ([250, 128, 380, 90], [0, 1, 2, -1], True), ([90, 380, 128, 250], [2, -1, 1, 0], False),
         ([1, 2, 0, 7, 5, 3, 1, 11], [0, 1, 2, -1] * 2, True), ([9, 1, 60, 20, 3], [2, -1, 1, 0, 2], False)]


@pytest.mark.parametrize("rows,adapter,x_bf16", FORMS)
@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("K,N,rank", [(264, 392, 16), (2048, 520, 8), (520, 1288, 32)])
def test_added_in_every_form(dev, pool, rows, adapter, x_bf16, out_bf16, K, N, rank):
    from oracle import binding as orc
    rng = np.random.default_rng(16)
    c = Case(dev, rng, rows, adapter, K, N, rank, 3, x_bf16, out_bf16)
    before = G.bf16(rng.standard_normal((c.M, c.N)).astype(np.float32))
    c.out.upload(orc.bf16_from_f32(before) if out_bf16 else before)
    c.call(pool, accumulate=True)
    out, bound = c.plain(before)
    assert (np.abs(c.get() - out) <= bound + np.abs(before) * 2.0 ** -23).all()
    c.free()


@pytest.mark.parametrize("rows,adapter,x_bf16", FORMS)
@pytest.mark.parametrize("K,rank", [(264, 16), (264, 8), (2056, 16), (2056, 64)])
def test_infinities_and_nan_in_every_form(dev, pool, rows, adapter, x_bf16, K, rank):
    """The second adapter and a row of the third's hold NaN, a column of the third an infinity: what the formula leaves finite is."""
    from oracle import binding as orc
    rng = np.random.default_rng(17)
    c = Case(dev, rng, rows, adapter, K, 392, rank, 3, x_bf16)
    c.a[1, 3, 7], c.b[2, 5, :] = np.nan, np.inf
    c.da.upload(orc.bf16_from_f32(c.a)), c.db.upload(orc.bf16_from_f32(c.b))
    ids = np.repeat(np.asarray(adapter), rows)
    bad = np.flatnonzero(ids == 2)[-1]
    c.x[bad, 9], c.x[np.flatnonzero(ids == -1)[0], 8] = np.inf, np.nan
    c.dx.upload(orc.bf16_from_f32(c.x) if x_bf16 else c.x)
    c.call(pool)
    got, (out, bound) = c.get(), c.plain()
    fine = np.isfinite(out)
    assert fine[ids == 0].all() and not fine[ids == 1].any() and not fine[bad].any()
    assert (np.isfinite(got) == fine).all() and (np.abs(got - out)[fine] <= bound[fine]).all()
    c.free()


@pytest.mark.parametrize("M,rank", [(1, 8), (1, 16), (2, 16), (1, 32), (4, 8), (3, 8)])
@pytest.mark.parametrize("K,N", [(8, 8), (72, 136), (1032, 520), (4096, 4736), (4096, 4744), (16384, 1024)])
@pytest.mark.parametrize("x_bf16", [False, True])
def test_a_few_rows(dev, pool, M, rank, K, N, x_bf16):
    rng = np.random.default_rng(M * rank + K)
    c = Case(dev, rng, [1] * M, [i % 4 for i in range(M)], K, N, rank, 4, x_bf16, x_bf16)
    for _ in range(3):
        c.call(pool)
    c.check()
    c.free()


@pytest.mark.parametrize("adapter", [[0, 1], [1, 0], [-1, 1], [0, -1], [0, 0]])
@pytest.mark.parametrize("x_bf16", [False, True])
def test_two_rows_added_beside_nan(dev, pool, adapter, x_bf16):
    """The second adapter is NaN throughout: rows of the other, or of none, are as if it were not there."""
    from oracle import binding as orc
    rng = np.random.default_rng(18)
    c = Case(dev, rng, [1, 1], adapter, 1032, 520, 8, 2, x_bf16)
    c.a[1], c.b[1] = np.nan, np.nan
    c.da.upload(orc.bf16_from_f32(c.a)), c.db.upload(orc.bf16_from_f32(c.b))
    before = G.bf16(rng.standard_normal((2, 520)).astype(np.float32))
    c.out.upload(before)
    c.call(pool, accumulate=True)
    out, bound = c.plain(before)
    got, fine = c.get(), np.asarray(adapter) != 1
    assert np.isnan(got[~fine]).all() and (np.abs(got - out)[fine] <= (bound + np.abs(before) * 2.0 ** -23)[fine]).all()
    c.free()


@pytest.mark.parametrize("M,slots,rank", [(17, 1, 8), (17, 40, 128), (33, 3, 64), (40, 15, 16), (64, 64, 32), (100, 2, 128), (128, 128, 128), (128, 30, 8), (65, 48, 64)])
@pytest.mark.parametrize("K,N", [(2048, 8), (2056, 1288), (4096, 136)])
@pytest.mark.parametrize("x_bf16", [False, True])
def test_few_rows_of_long_k(dev, pool, M, slots, rank, K, N, x_bf16):
    rng = np.random.default_rng(M + slots + K)
    for adapter in (rng.integers(-1, slots, M), rng.permutation(M) % (slots + 1) - 1, np.full(M, -1)):
        c = Case(dev, rng, [1] * M, adapter, K, N, rank, slots, x_bf16, not x_bf16)
        for _ in range(2):
            c.call(pool)
        c.check()
        c.free()


@pytest.mark.parametrize("K,rank,slots", [(520, 32, 5), (2056, 32, 5), (4096, 128, 24)])
def test_rows_alone_and_among_others(dev, pool, K, rank, slots):
    """A request's rows are the same bits whatever other requests' adapters are."""
    rng = np.random.default_rng(13)
    c = Case(dev, rng, [1] * 24, [0] * 24, K, 392, rank, slots)
    c.call(pool)
    alone = c.get()
    c.adapter = rng.integers(-1, slots, 24).astype(np.int32)
    c.adapter[[3, 17]] = 0
    c.call(pool)
    assert np.array_equal(c.get()[[3, 17]], alone[[3, 17]])
    c.free()


def test_calls_without_waiting_and_in_graphs(dev, pool):
    """Calls of several sizes share their workspace; a captured one keeps its places, and reads what its slots hold at the launch."""
    from oracle import binding as orc
    from relux_b200 import lib as L
    rng = np.random.default_rng(14)
    cases = [Case(dev, rng, rows, ad, K, N, r, 6, xb) for rows, ad, K, N, r, xb in
             [([1], [2], 1024, 520, 16, False), ([1] * 40, list(rng.integers(-1, 6, 40)), 264, 1032, 8, True), ([300, 5, 77], [3, -1, 5], 520, 264, 64, False),
              ([1] * 40, list(rng.integers(-1, 6, 40)), 2056, 1032, 32, True), ([1] * 20, list(rng.integers(-1, 6, 20)), 4096, 264, 128, False)]]
    for c in cases:
        c.call(pool)
    graph = Graph(dev, lambda: [c.call(pool) for c in cases])
    large = Case(dev, rng, [900, 100], [0, 5], 1024, 2048, 128, 6)
    for chained in (1, 0):
        pool.tune(L.TUNE_CHAINED_LAUNCHES, chained)
        for c in cases:
            c.clear()
        for _ in range(4):
            for c in cases + [large]:
                c.call(pool)
        for c in cases + [large]:
            c.check()
    pool.tune(L.TUNE_CHAINED_LAUNCHES, -1)
    for c in cases:
        c.db.upload(orc.bf16_from_f32(c.b * 2))
        c.b = c.b * 2
        c.clear()
    graph.launch()
    for c in cases:
        c.check()
    graph.free()
    for c in cases + [large]:
        c.free()


def test_beside_an_8_bit_projection(dev, pool):
    """The norm's rows twice, in 8 bits for the shared projection and as bf16 for the adapters, which are added to its result."""
    from relux_b200 import lib as L
    rng = np.random.default_rng(15)
    rows, adapter = requests(rng, 10, 4, 3)
    c = Case(dev, rng, rows, adapter, 512, 392, 16, 3, True, shared=False)
    M, K, N = c.M, c.K, c.N
    h0 = dev.upload(rng.standard_normal((M, K)).astype(np.float32))
    dw = dev.upload((rng.standard_normal((K, N)) * K ** -0.5).astype(np.float32))
    codes, scales, w, sw = dev.alloc(M * K), dev.alloc(4 * M), dev.alloc(K * N), dev.alloc(4 * N)
    pool.int8_weights(K, N, dw, w, sw)
    pool.rmsnorm(M, K, h0, None, 1e-5, out=c.dx, codes=codes, scales=scales)
    pool.matmul_int8(M, K, N, codes, scales, w, sw, c.out)
    base = c.get()
    c.call(pool, accumulate=True)
    c.x = get(c.dx, (M, K), True)
    out, bound = c.plain(base)
    assert (np.abs(c.get() - out) <= bound + np.abs(base) * 2.0 ** -23).all()
    assert L.OK == pool.status()
    for b in (h0, dw, codes, scales, w, sw):
        b.free()
    c.free()


def test_refusals(dev, pool):
    from relux_b200 import lib as L
    b = dev.alloc(1 << 20, L.DTYPE_BF16)

    def refused(code, **kw):
        a = dict(m=2, k=64, n=64, x=b, w=b, out=b, lora_a=b, lora_b=b, rank=16, n_slots=2, adapter=[0, 1])
        a.update(kw)
        with pytest.raises(L.ReluxCudaError) as e:
            pool.matmul_lora(**a)
        assert e.value.code == code
    for n in ("m", "k", "n", "n_slots"):
        refused(L.ERR_INVALID_ARG, **{n: 0})
    for n in ("lora_a", "lora_b"):
        refused(L.ERR_INVALID_ARG, **{n: None})
    for n in ("w", "lora_a", "lora_b", "factors"):
        refused(L.ERR_INVALID_ARG, **{n: b.ptr + 8})
    refused(L.ERR_INVALID_ARG, adapter=[0, 2])
    refused(L.ERR_INVALID_ARG, adapter=[0, -2])
    refused(L.ERR_INVALID_ARG, adapter=[0, 1, 1])
    refused(L.ERR_INVALID_ARG, adapter=[])
    refused(L.ERR_INVALID_ARG, rows=[1, 2])
    refused(L.ERR_INVALID_ARG, rows=[3, -1])
    refused(L.ERR_UNSUPPORTED, k=60)
    refused(L.ERR_UNSUPPORTED, n=60)
    refused(L.ERR_UNSUPPORTED, rank=24)
    refused(L.ERR_UNSUPPORTED, m=(1 << 30) + 8, rows=[1 << 30, 8], x=b.ptr, out=b.ptr, x_dtype=L.DTYPE_BF16, out_dtype=L.DTYPE_BF16)
    b.free()
