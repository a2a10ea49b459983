"""Rows whose offsets pass 2^32: sampled rows, the last among them, against the formulas; all other rows are of zeros or of one repeated block."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_lora import dev, pool  # noqa: F401
from tests.test_gpu_matmul_int8 import same
from tests.test_gpu_norm_rows import BF16, REL, plain as norm_plain

pytestmark = pytest.mark.gpu


class Big:
    """Device memory of zeros with a few rows filled in."""

    def __init__(self, dev, rows, d, dtype):  # noqa: F811
        self.d, self.dtype, self.row_bytes = d, dtype, d * np.dtype(dtype).itemsize
        self.buf = dev.alloc(rows * self.row_bytes)
        self.buf.zero()
        self.ptr, self.free = self.buf.ptr, self.buf.free

    def set(self, i, a):
        self.buf.upload(np.ascontiguousarray(a, self.dtype), i * self.row_bytes)

    def row(self, i):
        return self.buf.download(self.d, self.dtype, i * self.row_bytes)


def sampled(rng, n, border):
    """Rows on both sides of a border, the first and the last."""
    return sorted({0, 1, n - 1, n - 2, border, border - 1, min(border + 1, n - 1), *(int(i) for i in rng.integers(0, n, 6))})


@pytest.mark.parametrize("n,d", [((1 << 32) // 32768 + 33, 32768), ((1 << 32) // 128 + 333, 128)])
def test_norm_and_8_bit_rows(dev, pool, n, d):  # noqa: F811
    from oracle import binding as orc
    from relux_b200 import lib as L
    rng = np.random.default_rng(d)
    x, out = (Big(dev, n, d, np.uint16) for _ in range(2))
    codes, scales = Big(dev, n, d, np.int8), dev.alloc(4 * n)
    at = sampled(rng, n, (1 << 32) // d)
    rows = orc.f32_from_bf16(orc.bf16_from_f32(rng.standard_normal((len(at), d)).astype(np.float32)))
    for i, r in zip(at, rows):
        x.set(i, orc.bf16_from_f32(r))
    pool.rmsnorm(n, d, x.ptr, None, 1e-5, out=out.ptr, codes=codes.ptr, scales=scales, dtype=L.DTYPE_BF16)
    _, y = norm_plain(rows, None, None, 1e-5)
    s = scales.download(n, np.float32)
    for i, want in zip(at, y):
        got = orc.f32_from_bf16(out.row(i)).astype(np.float64)
        assert (np.abs(got - want) <= np.abs(want) * (REL + BF16)).all(), i
        assert (np.abs(codes.row(i) * float(s[i]) - want) <= s[i] * 0.5 + np.abs(want) * 2.0 ** -16).all(), i
    pool.int8_rows(n, d, x.ptr, codes.ptr, scales, dtype=L.DTYPE_BF16)
    s = scales.download(n, np.float32)
    for i, r in zip(at, rows):
        want, scale = G.quantise(r)
        assert np.array_equal(codes.row(i), want) and s[i] == scale, i
    others = np.delete(np.arange(n), at)
    assert not s[others].any()
    for b in (x, out, codes, scales):
        b.free()


@pytest.mark.parametrize("M,K,N", [((1 << 32) // 65536 + 77, 65536, 8), ((1 << 32) // 16384 + 99, 16, 16384)])
def test_8_bit_products(dev, pool, M, K, N):  # noqa: F811
    """Operand rows, then result rows, past 2^32."""
    from relux_b200 import lib as L
    rng = np.random.default_rng(K)
    a, out = Big(dev, M, K, np.int8), Big(dev, M, N, np.float32)
    w, sw, sa = rng.integers(-127, 128, (N, K)).astype(np.int8), np.exp2(rng.standard_normal(N)).astype(np.float32), np.exp2(rng.standard_normal(M)).astype(np.float32)
    dw, dsw, dsa = (dev.upload(v) for v in (w, sw, sa))
    at = sampled(rng, M, (1 << 32) // max(K, N))
    rows = rng.integers(-127, 128, (len(at), K)).astype(np.int8)
    for i, r in zip(at, rows):
        a.set(i, r)
    pool.matmul_int8(M, K, N, a.ptr, dsa, dw, dsw, out.ptr, out_dtype=L.DTYPE_F32)
    for i, r in zip(at, rows):
        want = ((r.astype(np.float64) @ w.astype(np.float64).T).astype(np.float32) * sa[i]).astype(np.float32) * sw
        assert same(out.row(i), want), i
    assert not out.row(at[-1] - 5 if at[-1] - 5 not in at else 2).any()
    for b in (a, out, dw, dsw, dsa):
        b.free()


# tiles of one request, rows and then results past 2^32; more rows than there are such tiles for, in few requests and, without a projection, in many; results of those
LORA = [(130600, 32896, 8, 3, True), (130600, 16, 32896, 3, True), ((1 << 32) // 16384 + 99, 16384, 16, 2, True), ((1 << 32) // 16384 + 99, 16384, 8, 4000, False),
        ((1 << 32) // 16384 + 99, 16, 16384, 5000, True)]


@pytest.mark.parametrize("M,K,N,B,shared", LORA)
@pytest.mark.parametrize("x_bf16", [True, False])
def test_adapters(dev, M, K, N, B, shared, x_bf16):  # noqa: F811
    from oracle import binding as orc
    import relux_b200 as rb
    from relux_b200 import lib as L
    pool = rb.Pool(dev, L.POOL_GQA, 1, 1, num_kv_heads=1, head_dim=128)      # its own: what a call of this size needs goes with it
    rng = np.random.default_rng(K + B)
    rank, slots = 8, 3
    x, out = Big(dev, M, K, np.uint16 if x_bf16 else np.float32), Big(dev, M, N, np.uint16)
    bf16 = lambda a: orc.f32_from_bf16(orc.bf16_from_f32(np.ascontiguousarray(a, np.float32)))   # noqa: E731
    w, la, lb = bf16(rng.standard_normal((K, N)) * K ** -0.5), bf16(rng.standard_normal((slots * rank, K)) * K ** -0.5), bf16(rng.standard_normal((slots * N, rank)))
    dw, da, db = (dev.upload(orc.bf16_from_f32(v)) for v in (w, la, lb))
    cuts = np.sort(rng.choice(M - 1, B - 1, replace=False)) + 1
    each = np.diff(np.r_[0, cuts, M]).astype(np.int32)
    adapter = (np.arange(B) % (slots + 1) - 1).astype(np.int32)
    of_row = np.repeat(adapter, each)
    at = sampled(rng, M, (1 << 32) // max(K, N))
    rows = bf16(rng.standard_normal((len(at), K)))
    for i, r in zip(at, rows):
        x.set(i, orc.bf16_from_f32(r) if x_bf16 else r)
    pool.matmul_lora(M, K, N, x.ptr, dw if shared else None, out.ptr, da, db, rank, slots, adapter, rows=each, x_dtype=L.DTYPE_BF16 if x_bf16 else L.DTYPE_F32,
                     out_dtype=L.DTYPE_BF16)
    for i, r in zip(at, rows.astype(np.float64)):
        want, size = (r @ w, np.abs(r) @ np.abs(w)) if shared else (np.zeros(N), np.zeros(N))
        s = of_row[i]
        if s >= 0:
            a, b = la[s * rank:(s + 1) * rank].astype(np.float64), lb[s * N:(s + 1) * N].astype(np.float64)
            want, size = want + (r @ a.T) @ b.T, size + (1 + 2.0 ** 8 / K) * ((np.abs(r) @ np.abs(a).T) @ np.abs(b).T)
        # sums of K products in float32; t in 16 bits: 2^8 / K times K 2^-24
        assert (np.abs(orc.f32_from_bf16(out.row(i)) - want) <= np.abs(want) * 2.0 ** -8 + size * (K + 40) * 2.0 ** -24).all(), i
    assert pool.status() == 0
    pool.destroy()
    for b in (x, out, dw, da, db):
        b.free()
