"""float32 rows that keep 16 bits in calls of every size, against the sums in 64 bits of the rows as they are.

Tolerances: two bf16 halves hold a value within 2^-16 of it; that and K roundings of the sum, of the magnitudes' sum.  t keeps 16 bits more.  A bf16 result 2^-8."""
import ctypes as C

import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_latent_graphs import Graph
from tests.test_gpu_lora import Case, dev, pool  # noqa: F401
from tests.test_gpu_lora_infinities import FORMS, K_A, K_W, COL_B, COL_W, N, spread, upload, with_infinities

pytestmark = pytest.mark.gpu


class Whole(Case):
    def call(self, pool, accumulate=False):  # noqa: F811
        pool.matmul_lora(self.M, self.K, self.N, self.dx, self.dw, self.out, self.da, self.db, self.rank, self.slots, self.adapter, rows=self.rows, factors=self.df,
                         accumulate=accumulate, x_halves=True)

    def plain(self, before=None):
        x, half, u = self.x.astype(np.float64), 2.0 ** -16, 2.0 ** -24
        out, bound = x @ self.w.astype(np.float64), ((self.K + 16) * u + half) * (np.abs(x) @ np.abs(self.w).astype(np.float64))
        if before is not None:
            out = out + before
        ids = np.repeat(self.adapter, self.rows)
        for s in range(self.slots):
            r = ids == s
            a, b, f = self.a[s].astype(np.float64), self.b[s].astype(np.float64), 1.0 if self.factors is None else float(self.factors[s])
            out[r] += f * ((x[r] @ a.T) @ b.T)
            bound[r] += f * (((self.K + 2 * self.rank + 16) * u + 2 * half) * ((np.abs(x[r]) @ np.abs(a).T) @ np.abs(b).T))
        return out, bound + np.abs(out) * (2.0 ** -22 + (2.0 ** -8 if self.out_bf16 else 0))


SIZES = [([1] * 9, 264, 392, 16), ([1] * 64, 2056, 1288, 16), ([1] * 24, 4096, 264, 128), ([3, 1, 60, 0, 20, 7], 520, 136, 8), ([80] * 4, 1000, 520, 32), ([250, 128, 380, 90], 520, 1288, 64),
         ([1] * 700, 264, 392, 32), ([33] * 160, 2056, 1160, 8), ([2900, 1, 1999, 300], 1032, 1160, 16), ([9] * 1300, 136, 72, 16)]


@pytest.mark.parametrize("rows,K,n,rank", SIZES, ids=str)
@pytest.mark.parametrize("out_bf16", [False, True])
def test_rows_keep_16_bits(dev, pool, rows, K, n, rank, out_bf16):  # noqa: F811
    rng = np.random.default_rng(sum(rows) + K)
    c = Whole(dev, rng, rows, rng.integers(-1, 5, len(rows)), K, n, rank, 5, False, out_bf16)
    c.call(pool)
    c.check()
    if not out_bf16:      # and what it is for: rows rounded to bf16 are 50 times as far off
        out, _ = c.plain()
        whole = np.linalg.norm(c.get() - out)
        Case.call(c, pool)
        assert np.linalg.norm(c.get() - out) > 50 * whole
    c.free()


def test_a_row_is_the_same_whatever_the_batch(dev, pool):  # noqa: F811
    """The rows that a call of eight has in 16 bits: within both calls' sums of each other when more rows join, where rounded rows are 2^-9 away."""
    rng = np.random.default_rng(5)
    c = Whole(dev, rng, [1] * 40, [i % 4 - 1 for i in range(40)], 520, 264, 16, 3)
    out, bound = c.plain()
    for n in (8, 9, 40):
        c.rows, c.adapter, c.M = np.ones(n, np.int32), np.asarray([i % 4 - 1 for i in range(n)], np.int32), n
        c.clear()
        c.call(pool)
        assert (np.abs(c.get() - out[:n]) <= bound[:n]).all()
    c.free()


@pytest.mark.parametrize("rows", [[1] * 20, [250, 128, 380, 90]], ids=str)
def test_added_and_in_a_graph(dev, pool, rows):  # noqa: F811
    rng = np.random.default_rng(6)
    c = Whole(dev, rng, rows, [i % 4 - 1 for i in range(len(rows))], 520, 392, 16, 3)
    before = G.bf16(rng.standard_normal((c.M, c.N)).astype(np.float32))
    c.out.upload(before)
    c.call(pool, accumulate=True)
    out, bound = c.plain(before)
    assert (np.abs(c.get() - out) <= bound + np.abs(before) * 2.0 ** -23).all()
    graph = Graph(dev, lambda: c.call(pool))
    other = Whole(dev, rng, [700, 900], [0, 2], 1032, 520, 64, 3)
    for _ in range(2):
        c.clear()
        other.call(pool)
        graph.launch()
        other.check(), c.check()
    graph.free()
    c.free(), other.free()


@pytest.mark.parametrize("rows,adapter,K,rank", [f for f in FORMS if sum(f[0]) > 8])
def test_infinities_keep_their_sign(dev, pool, rows, adapter, K, rank):  # noqa: F811
    rng = np.random.default_rng(sum(rows) + K + rank)
    c = Whole(dev, rng, rows, adapter, K, N, rank, 3)
    spread(c)
    c.w[K_W, COL_W] = 0
    c.a[1, 3, K_A], c.b[2, COL_B, 2] = 0, 0
    out, bound = with_infinities(c, True, True, True)
    c.w[K_W, COL_W] = np.inf
    c.a[1, 3, K_A], c.b[2, COL_B, 2] = np.inf, -np.inf
    upload(c)
    c.call(pool)
    got, fine = c.get(), np.isfinite(out)
    assert np.array_equal(np.isnan(got), np.isnan(out)) and (got[np.isinf(out)] == out[np.isinf(out)]).all()
    assert (np.abs(got[fine] - out[fine]) <= bound[fine]).all()
    c.free()


def test_bf16_rows_do_not_care(dev, pool):  # noqa: F811
    rng = np.random.default_rng(7)
    c = Case(dev, rng, [250, 40], [0, 1], 264, 392, 16, 2, True)
    c.call(pool)
    want = c.get()
    c.clear()
    Whole.call(c, pool)
    assert np.array_equal(c.get(), want)
    c.free()


def test_refusals(dev, pool):  # noqa: F811
    from relux_b200 import lib as L
    b = dev.alloc(1 << 12, L.DTYPE_F32).ptr
    with pytest.raises(L.ReluxCudaError) as e:
        pool.matmul_lora((1 << 29) + 8, 64, 64, b, b, b, b, b, 16, 1, [0], rows=[(1 << 29) + 8], x_dtype=L.DTYPE_F32, out_dtype=L.DTYPE_F32, x_halves=True)
    assert e.value.code == L.ERR_UNSUPPORTED
    a = L.MatmulLoraArgs(m=1, k=64, n=64, rank=16, n_slots=1, n_seqs=1, x_halves=2, x=b, w=b, lora_a=b, lora_b=b, adapter=np.zeros(1, np.int32).ctypes.data, out=b)
    assert pool.lib.relux_matmul_lora(pool.h, C.byref(a)) == L.ERR_INVALID_ARG
