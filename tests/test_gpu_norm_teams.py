"""Narrow rows, so many that a team takes four of them: sizes with rows and lanes left over, in both types, and as 8-bit rows.  Tolerances as in tests/test_gpu_norm_rows.py."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_norm_rows import BF16, REL, activations, dev, get, plain, pool, put  # noqa: F401

pytestmark = pytest.mark.gpu
SIZES = [(20441, 128), (40003, 72), (9703, 256), (303106, 8), (77781, 24), (13999, 176)]


@pytest.mark.parametrize("n,d", SIZES)
@pytest.mark.parametrize("xb,rb,wb,ob", [(True, True, True, True), (False, False, False, False), (True, False, True, False), (False, None, None, True)])
def test_four_rows_a_team(dev, pool, n, d, xb, rb, wb, ob):  # noqa: F811
    from relux_b200 import lib as L
    rng = np.random.default_rng(n + d)
    dx, x = put(dev, activations(rng, n, d), xb)
    dr, r = put(dev, activations(rng, n, d), rb) if rb is not None else (None, None)
    dw, w = put(dev, 1 + 0.3 * rng.standard_normal(d), wb) if wb is not None else (None, None)
    out = dev.alloc((n + 1) * d * (2 if ob else 4), L.DTYPE_BF16 if ob else L.DTYPE_F32)
    h = dev.alloc((n + 1) * d * (2 if rb else 4), L.DTYPE_BF16 if rb else L.DTYPE_F32) if rb is not None else None
    for b in (out, h):
        if b is not None:
            L.check(dev.lib.relux_cuda_memset(dev.h, b.ptr, 0xFF, b.nbytes))
    pool.rmsnorm(n, d, dx, dw, 1e-5, residual=dr, residual_out=h, out=out)
    h32, y = plain(x, r, w, 1e-5)
    got = get(out, (n + 1, d), ob).astype(np.float64)
    assert np.isnan(got[n]).all()      # the row behind the last is as it was
    size = np.abs(y) if r is None else (np.abs(x) + np.abs(r)) * np.abs(y) / np.maximum(np.abs(h32), 1e-30)
    assert (np.abs(got[:n] - y) <= np.abs(y) * (REL + (BF16 if ob else 0)) + size * 2.0 ** -23).all()
    if h is not None:
        held = get(h, (n + 1, d), rb)
        assert np.array_equal(held[:n].view(np.uint32), (G.bf16(h32) if rb else h32).view(np.uint32)) and np.isnan(held[n]).all()
    for b in (dx, dr, dw, out, h):
        if b is not None:
            b.free()


@pytest.mark.parametrize("n,d", [s for s in SIZES if s[1] % 16 == 0])
@pytest.mark.parametrize("bf16", [True, False])
def test_four_rows_a_team_in_8_bits(dev, pool, n, d, bf16):  # noqa: F811
    from relux_b200 import lib as L
    rng = np.random.default_rng(n + d + 1)
    x = activations(rng, n, d)
    x[[0, n - 2]], x[5, 3], x[n - 1, d - 1] = 0, np.nan, np.inf
    dx, x = put(dev, x, bf16)
    dw, w = put(dev, 1 + 0.3 * rng.standard_normal(d), True)
    codes, scales, out = dev.alloc((n + 1) * d), dev.alloc(4 * (n + 1)), dev.alloc(4 * n * d, 0)
    for norm in (False, True):
        for b in (codes, scales):
            L.check(dev.lib.relux_cuda_memset(dev.h, b.ptr, 0x55, b.nbytes))
        if norm:
            pool.rmsnorm(n, d, dx, dw, 1e-5, out=out, out_dtype=0, codes=codes, scales=scales)
            want, s = G.quantise(out.download((n, d), np.float32))
        else:
            pool.int8_rows(n, d, dx, codes, scales)
            want, s = G.quantise(x)
        c, got = codes.download((n + 1, d), np.int8), scales.download(n + 1, np.float32)
        assert np.array_equal(c[:n], want) and (c[n] == 0x55).all() and got[n:].view(np.uint32)[0] == 0x55555555
        bad = np.isnan(s)
        assert np.array_equal(np.isnan(got[:n]), bad) and bad[5] and bad[n - 1] and bad.sum() == 2
        assert np.array_equal(got[:n][~bad].view(np.uint32), s[~bad].view(np.uint32))
    for b in (dx, dw, codes, scales, out):
        b.free()
