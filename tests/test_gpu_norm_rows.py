"""The norm with the residual's addition and rows in 8 bits, against the formula in 64 bits.

Tolerances, in units of u = 2^-24 (half a step of float32, relative): a sum of squares is taken over at most 32 products a thread, one rounding each, and ten
levels of a tree: 42 u of positive terms, half of that in the root; the root is two units in the last place off, 4 u; mean and eps 3 u, halved; the sum h one, the two
products two.  Together below 32 u = 2^-19.  A bf16 result is rounded once more, 2^-8 (half of finfo.eps)."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_latent_graphs import Graph

pytestmark = pytest.mark.gpu
REL, BF16 = 2.0 ** -19, 2.0 ** -8


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


def activations(rng, n, d):
    x = rng.standard_normal((n, d)) * np.exp2(rng.standard_normal((n, 1)))
    x[:, 5::61] *= 8
    return x.astype(np.float32)


def put(dev, x, bf16):
    """(device buffer, the values it holds as float32)."""
    from oracle import binding as orc
    if not bf16:
        return dev.upload(np.ascontiguousarray(x, np.float32)), np.asarray(x, np.float32)
    bits = orc.bf16_from_f32(np.ascontiguousarray(x, np.float32))
    return dev.upload(bits), orc.f32_from_bf16(bits)


def get(buf, shape, bf16):
    from oracle import binding as orc
    return orc.f32_from_bf16(buf.download(shape, np.uint16)) if bf16 else buf.download(shape, np.float32)


def plain(x, r, w, eps):
    """(h in float32 as it is added, y in 64 bits of the same h in 64 bits)."""
    with np.errstate(all="ignore"):
        h32 = x if r is None else x + r
        h = x.astype(np.float64) if r is None else x.astype(np.float64) + r
        y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
        return h32, y if w is None else y * w


@pytest.mark.parametrize("n,d", [(1, 8), (3, 24), (33, 128), (511, 128), (7, 136), (2, 256), (5, 264), (1, 4096), (40, 4104), (3, 8192), (2, 8200), (3, 16384), (2, 16400),
                                 (2, 32768), (700, 1000)])
@pytest.mark.parametrize("xb,rb,wb,ob", [(True, True, True, True), (False, False, False, False), (True, False, True, True), (False, True, False, True), (True, None, None, False),
                                         (False, None, True, False)])
def test_norm(dev, pool, n, d, xb, rb, wb, ob):
    from relux_b200 import lib as L
    rng = np.random.default_rng(n * 7 + d)
    dx, x = put(dev, activations(rng, n, d), xb)
    dr, r = put(dev, activations(rng, n, d), rb) if rb is not None else (None, None)
    dw, w = put(dev, 1 + 0.3 * rng.standard_normal(d), wb) if wb is not None else (None, None)
    out = dev.alloc(n * d * (2 if ob else 4), L.DTYPE_BF16 if ob else L.DTYPE_F32)
    h = dev.alloc(n * d * (2 if rb else 4), L.DTYPE_BF16 if rb else L.DTYPE_F32) if rb is not None else None
    pool.rmsnorm(n, d, dx, dw, 1e-5, residual=dr, residual_out=h, out=out)
    h32, y = plain(x, r, w, 1e-5)
    got = get(out, (n, d), ob).astype(np.float64)
    # h is 2^-24 of itself off, so y near a cancelled h too: relative to |x| + |r| there
    size = np.abs(y) if r is None else (np.abs(x) + np.abs(r)) * np.abs(y) / np.maximum(np.abs(h32), 1e-30)
    bound = np.abs(y) * (REL + (BF16 if ob else 0)) + size * 2.0 ** -23
    assert (np.abs(got - y) <= bound).all()
    if h is not None:
        want = G.bf16(h32) if rb else h32
        assert np.array_equal(get(h, (n, d), rb).view(np.uint32), want.view(np.uint32))
    for b in (dx, dr, dw, out, h):
        if b is not None:
            b.free()


@pytest.mark.parametrize("n,d", [(1, 16), (35, 128), (9, 144), (4, 1008), (3, 4096), (70, 2048), (2, 12304), (2, 32768)])
@pytest.mark.parametrize("bf16", [True, False])
def test_rows_in_8_bits(dev, pool, n, d, bf16):
    """Of rows as they are: the rule, bit for bit.  Behind a norm: numbers within half a step of the formula's value, and the norm's error."""
    rng = np.random.default_rng(n + d)
    x = activations(rng, n, d)
    if n > 2:
        x[0] = 0
        x[1] *= np.float32(1e-39) / np.abs(x[1]).max()
        x[2] *= np.float32(1e-30)
    dx, x = put(dev, x, bf16)
    codes, scales, out = dev.alloc(n * d), dev.alloc(4 * n), dev.alloc(4 * n * d, 0)
    pool.int8_rows(n, d, dx, codes, scales)
    want, s = G.quantise(x)
    assert np.array_equal(codes.download((n, d), np.int8), want)
    assert np.array_equal(scales.download(n, np.float32).view(np.uint32), s.view(np.uint32))
    dw, w = put(dev, 1 + 0.3 * rng.standard_normal(d), True)
    pool.rmsnorm(n, d, dx, dw, 1e-5, out=out, out_dtype=0, codes=codes, scales=scales)
    y32 = out.download((n, d), np.float32)
    want, s = G.quantise(y32)      # both results of one call hold the same y
    assert np.array_equal(codes.download((n, d), np.int8), want)
    assert np.array_equal(scales.download(n, np.float32).view(np.uint32), s.view(np.uint32))
    for b in (dx, dw, codes, scales, out):
        b.free()


def test_infinities_and_nan_stay_in_their_rows(dev, pool):
    rng = np.random.default_rng(2)
    n, d = 40, 128
    x = activations(rng, n, d)
    x[3, 7], x[11, 100], x[20, 0] = np.nan, np.inf, -np.inf
    x[30] = 3e30        # its squares pass float32's range: the norm's row is zeros
    dx, x = put(dev, x, False)
    codes, scales, out = dev.alloc(n * d), dev.alloc(4 * n), dev.alloc(4 * n * d, 0)
    pool.rmsnorm(n, d, dx, None, 1e-5, out=out, codes=codes, scales=scales)
    got, s, c = out.download((n, d), np.float32), scales.download(n, np.float32), codes.download((n, d), np.int8)
    bad = np.isin(np.arange(n), [3, 11, 20])
    assert np.isnan(got[3]).all() and np.isnan(got[11, 100]) and np.isnan(got[20, 0])
    assert np.isnan(s[bad]).all() and (c[bad] == 0).all()
    assert (got[30] == 0).all() and s[30] == 0 and (c[30] == 0).all()
    ok = ~bad & (np.arange(n) != 30)
    _, y = plain(x[ok], None, None, 1e-5)
    assert (np.abs(got[ok] - y) <= np.abs(y) * (REL + 2.0 ** -23)).all() and np.isfinite(s[ok]).all()
    pool.int8_rows(n, d, dx, codes, scales)
    s = scales.download(n, np.float32)
    assert np.isnan(s[bad]).all() and np.isfinite(s[~bad]).all() and (codes.download((n, d), np.int8)[bad] == 0).all()
    for b in (dx, codes, scales, out):
        b.free()


@pytest.mark.parametrize("bf16", [True, False])
def test_in_place_and_in_a_graph(dev, pool, bf16):
    """Residual updated in place, the norm written over x; the same captured and launched again; rows behind the last one are left as they were."""
    rng = np.random.default_rng(5)
    n, d = 6, 2056
    e = 2 if bf16 else 4
    x0, r0 = (np.concatenate([activations(rng, n, d), np.full((1, d), 7, np.float32)]) for _ in range(2))
    dx, x = put(dev, x0, bf16)
    dr, r = put(dev, r0, bf16)
    dw, w = put(dev, 1 + 0.3 * rng.standard_normal(d), True)
    call = lambda: pool.rmsnorm(n, d, dx, dw, 1e-5, residual=dr, residual_out=dr, out=dx)  # noqa: E731
    call()
    for k in range(3):
        h32, y = plain(x[:n], r[:n], w, 1e-5)
        got, h = get(dx, (n + 1, d), bf16), get(dr, (n + 1, d), bf16)
        assert np.array_equal(h[:n], G.bf16(h32) if bf16 else h32)
        size = (np.abs(x[:n]) + np.abs(r[:n])) * np.abs(y) / np.maximum(np.abs(h32), 1e-30)
        assert (np.abs(got[:n] - y) <= np.abs(y) * (REL + (BF16 if bf16 else 0)) + size * 2.0 ** -23).all()
        assert (got[n] == 7).all() and (h[n] == 7).all()
        x, r = got, h
        if k == 0:
            graph = Graph(dev, call)
        graph.launch()
    graph.free()
    assert e and pool.status() == 0
    for b in (dx, dr, dw):
        b.free()


def test_refusals(dev, pool):
    from relux_b200 import lib as L
    b = dev.alloc(1 << 16, L.DTYPE_F32)

    def refused(code, **kw):
        a = dict(n_rows=2, d=64, x=b, out=b)
        a.update(kw)
        with pytest.raises(L.ReluxCudaError) as e:
            pool.rmsnorm(**a)
        assert e.value.code == code
    refused(L.ERR_INVALID_ARG, n_rows=0)
    refused(L.ERR_INVALID_ARG, d=0)
    refused(L.ERR_INVALID_ARG, eps=-1.0)
    refused(L.ERR_INVALID_ARG, eps=float("nan"))
    refused(L.ERR_INVALID_ARG, out=None)
    refused(L.ERR_INVALID_ARG, residual_out=b)
    refused(L.ERR_INVALID_ARG, codes=b)
    refused(L.ERR_INVALID_ARG, scales=b)
    refused(L.ERR_INVALID_ARG, x=b.ptr + 4, dtype=0)
    refused(L.ERR_INVALID_ARG, out_dtype=2, out=b.ptr)
    refused(L.ERR_UNSUPPORTED, d=60)
    refused(L.ERR_UNSUPPORTED, d=32776, n_rows=1, x=b.ptr, out=b.ptr, dtype=0)
    refused(L.ERR_UNSUPPORTED, d=72, codes=b, scales=b)
    for kw in (dict(d=24), dict(d=32784, x=b.ptr, codes=b.ptr)):
        with pytest.raises(L.ReluxCudaError):
            pool.int8_rows(**{**dict(n_rows=1, d=16, x=b, codes=b, scales=b, dtype=0), **kw})
    with pytest.raises(L.ReluxCudaError):
        pool.int8_weights(24, 8, b, b, b)
    with pytest.raises(L.ReluxCudaError):
        pool.int8_weights(16, 12, b, b, b)
    b.free()
