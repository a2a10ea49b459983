"""Infinities in the weights and in the adapters, by sign: whatever form a call takes, a result is an infinity of the formula's sign, or NaN, exactly where the formula is.

The formula of a result with infinities is known without sums: the finite part, plus a signed infinity for every infinite product (two of opposite signs: NaN).  Finite results
are within the tolerances of tests/test_gpu_lora.py."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_lora import Case, dev, pool  # noqa: F401

pytestmark = pytest.mark.gpu

# every form of the call: one launch, few rows, columns of the projection, groups of 16 rows with and without explicit lists, tiles of one request; each with bf16 and float32 rows
FORMS = [([1], [1], 264, 16), ([1, 1], [1, 2], 520, 8), ([1] * 6, [1, 2, 0, -1, 2, 1], 264, 32), ([1] * 16, [1, 2, 0, -1] * 4, 264, 16), ([1] * 20, [1, 2, 0, -1] * 5, 264, 16),
         ([1] * 24, [1, 2, 0, -1] * 6, 2056, 64), ([80, 90, 70, 75], [1, 2, -1, 0], 264, 16), ([1] * 700, [i % 4 - 1 for i in range(700)], 264, 32),
         ([250, 128, 380, 90], [1, 2, 0, -1], 264, 16), ([250, 128, 380, 90], [1, 2, 0, -1], 520, 64), ([250, 128, 380, 90], [1, 2, 0, -1], 2056, 8)]
N, K_W, COL_W, K_A, COL_B = 392, 11, 17, 7, 5


def spread(c):
    """Values that bf16 holds, that it does not, and whose rest is of the other sign, of both signs, in the two places that meet an infinity."""
    some = np.array([1.0, -1.0, 1.003, -1.003, 1.0077, -1.0077, 0.3, -0.3], np.float32)
    at = np.arange(c.M)
    c.x[:, K_W], c.x[:, K_A] = some[at % 8], some[(at // 3) % 8]
    if c.x_bf16:
        c.x = G.bf16(c.x)


def upload(c):
    from oracle import binding as orc
    c.da.upload(orc.bf16_from_f32(c.a)), c.db.upload(orc.bf16_from_f32(c.b))
    c.dx.upload(orc.bf16_from_f32(c.x) if c.x_bf16 else c.x)
    if c.w is not None:
        c.dw.upload(orc.bf16_from_f32(c.w))


def with_infinities(c, in_w, in_a, in_b):
    """(result, bound): infinities as they are placed by the caller's flags."""
    finite, bound = c.plain()
    t = np.zeros((c.M, c.rank))
    ids = np.repeat(np.asarray(c.adapter), c.rows)
    for s in range(c.slots):
        t[ids == s] = c.x[ids == s].astype(np.float64) @ c.a[s].astype(np.float64).T * float(c.factors[s])
    out, inf = finite.copy(), np.inf
    with np.errstate(all="ignore"):
        if in_w:
            out[:, COL_W] += np.sign(c.x[:, K_W]) * inf
        if in_a:     # the sum of adapter 1 that it is in, and with it every column
            r = ids == 1
            out[r] += np.sign(c.x[r, K_A])[:, None] * np.sign(c.b[1, :, 3])[None] * inf
        if in_b:     # one column of adapter 2
            r = ids == 2
            out[r, COL_B] += -np.sign(t[r, 2]) * inf
    return out, bound


@pytest.mark.parametrize("rows,adapter,K,rank", FORMS)
@pytest.mark.parametrize("x_bf16", [False, True])
@pytest.mark.parametrize("shared", [True, False])
def test_infinities_keep_their_sign(dev, pool, rows, adapter, K, rank, x_bf16, shared):  # noqa: F811
    rng = np.random.default_rng(sum(rows) + K + rank)
    c = Case(dev, rng, rows, adapter, K, N, rank, 3, x_bf16, shared=shared)
    spread(c)
    places = dict(in_w=shared, in_a=True, in_b=True)
    # the finite part of what meets an infinity is that of a zero
    if shared:
        c.w[K_W, COL_W] = 0
    c.a[1, 3, K_A], c.b[2, COL_B, 2] = 0, 0
    out, bound = with_infinities(c, **places)
    if shared:
        c.w[K_W, COL_W] = np.inf
    c.a[1, 3, K_A], c.b[2, COL_B, 2] = np.inf, -np.inf
    upload(c)
    c.call(pool)
    got, fine = c.get(), np.isfinite(out)
    assert not fine.all()
    assert np.array_equal(np.isnan(got), np.isnan(out))
    assert (got[np.isinf(out)] == out[np.isinf(out)]).all()
    assert (np.abs(got - out)[fine] <= bound[fine]).all()
    c.free()


@pytest.mark.parametrize("rows,adapter,K,rank", FORMS)
@pytest.mark.parametrize("x_bf16", [False, True])
def test_zeros_beside_infinities_are_nan(dev, pool, rows, adapter, K, rank, x_bf16):  # noqa: F811
    """Zero times an infinity is NaN in the formula, in every form."""
    rng = np.random.default_rng(sum(rows) + K + rank + 1)
    c = Case(dev, rng, rows, adapter, K, N, rank, 3, x_bf16)
    c.x[:, K_W] = 0
    c.w[K_W, COL_W] = 0
    out, bound = c.plain()
    c.w[K_W, COL_W] = np.inf
    upload(c)
    c.call(pool)
    got, other = c.get(), np.arange(N) != COL_W
    assert np.isnan(got[:, COL_W]).all()
    assert (np.abs(got - out)[:, other] <= bound[:, other]).all()
    c.free()


@pytest.mark.parametrize("rows,adapter,K,rank", FORMS)
@pytest.mark.parametrize("x_bf16", [False, True])
def test_rows_of_an_infinity(dev, pool, rows, adapter, K, rank, x_bf16):  # noqa: F811
    """A row that holds an infinity and has no adapter: infinities of the weights' signs in every column; other rows are not touched."""
    if -1 not in adapter:
        adapter = [-1] + adapter[1:]
    rng = np.random.default_rng(sum(rows) + K + rank + 2)
    c = Case(dev, rng, rows, adapter, K, N, rank, 3, x_bf16)
    row = int(np.flatnonzero(np.repeat(np.asarray(adapter), rows) == -1)[-1])
    out, bound = c.plain()
    c.x[row, 9] = -np.inf
    out[row] = -np.sign(c.w[9].astype(np.float64)) * np.inf
    upload(c)
    c.call(pool)
    got, other = c.get(), np.arange(c.M) != row
    assert (got[row] == out[row]).all()
    assert (np.abs(got - out)[other] <= bound[other]).all()
    c.free()


@pytest.mark.parametrize("rows,adapter,K,rank", FORMS)
def test_products_that_vanish(dev, pool, rows, adapter, K, rank):  # noqa: F811
    """Values and factors whose product is below the smallest float32, of both signs, and zeros of both signs: the adapter's part is nothing, and not NaN."""
    rng = np.random.default_rng(sum(rows) + K + rank + 3)
    c = Case(dev, rng, rows, adapter, K, N, rank, 3, False)
    c.factors[:] = 1e-20, -1e-20, 1e-20
    c.df.upload(c.factors)
    c.x *= np.float32(1e-28)
    c.x[:, ::5], c.x[:, 1::5] = 0.0, -0.0
    c.dx.upload(c.x)
    c.call(pool)
    got = c.get()
    out, _ = c.plain()
    size = np.abs(c.x).astype(np.float64) @ np.abs(c.w).astype(np.float64)
    assert np.isfinite(got).all() and (np.abs(got - out) <= size * 2.0 ** -8).all()
    c.free()
