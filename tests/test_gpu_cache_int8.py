"""The 8-bit grouped-query cache: rows bit for bit by its rule, attention within a bound derived from its roundings (tests/gqa_plain.py)."""
import numpy as np
import pytest

from tests import gqa_plain as G

pytestmark = pytest.mark.gpu
D, PAGE = 128, 64


@pytest.fixture(scope="module")
def dev():
    import relux_b200 as rb
    d = rb.Device(0)
    yield d
    d.close()


def make(dev, B, per, Hkv, seed=0, layers=1, int8=True, spare=3, max_seqs=None):
    import relux_b200 as rb
    from relux_b200 import lib as L
    n = max_seqs or B
    pool = rb.Pool(dev, L.POOL_GQA, layers, n * per + spare, PAGE, n, per, num_kv_heads=Hkv, head_dim=D, cache_int8=int8)
    pool.set_tables(np.random.default_rng(seed).permutation(n * per + spare)[:n * per].astype(np.int32).reshape(n, per))
    return pool


def read(pool, dev, layer, tok0, n, f32=True, seq_ids=None):
    """(K, V) by relux_gqa_read_kv, as float32."""
    from oracle import binding as orc
    from relux_b200 import lib as L
    shape = (int(np.sum(n)), pool.prm.gqa_num_kv_heads, D)
    if layer < 0:
        shape = (pool.prm.num_layers,) + shape
    bufs = [dev.alloc(max(1, int(np.prod(shape))) * (4 if f32 else 2), L.DTYPE_F32 if f32 else L.DTYPE_BF16) for _ in range(2)]
    pool.read_kv(layer, len(n), bufs[0], bufs[1], tok0, n, seq_ids=seq_ids)
    got = [b.download(shape, np.float32 if f32 else np.uint16) for b in bufs]
    for b in bufs:
        b.free()
    return got if f32 else [orc.f32_from_bf16(x) for x in got]


def bufs_dtype(f32):
    from relux_b200 import lib as L
    return L.DTYPE_F32 if f32 else L.DTYPE_BF16


def orc_f32(bits):
    from oracle import binding as orc
    return orc.f32_from_bf16(bits)


def same(a, b):
    return np.array_equal(np.asarray(a, np.float32).view(np.uint32), np.asarray(b, np.float32).view(np.uint32))


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("head_major", [True, False])
@pytest.mark.parametrize("Hkv", [1, 3, 8])
def test_rows_are_quantised_by_the_rule(dev, f32, head_major, Hkv):
    from oracle import binding as orc
    from relux_b200 import lib as L
    rng = np.random.default_rng(Hkv + 10 * f32)
    B, per = 4, 3
    pool = make(dev, B, per, Hkv)
    ids, cache = np.array([2, 0, 3], np.int32), G.Cache(B, Hkv, True)
    for n_new in ([1, 1, 1], [0, 70, 5], [63, 2, 128], [1, 9, 1]):
        parts = []
        for which in "kv":
            xs = [G.rows(rng, n, Hkv, which) for n in n_new]
            if not f32:
                xs = [G.bf16(x) for x in xs]
            parts.append(xs)
        for j, b in enumerate(ids):
            cache.append(b, parts[0][j], parts[1][j])
        flat = [np.concatenate([(x.transpose(1, 0, 2) if head_major else x).reshape(-1, D) for x in xs]) for xs in parts]
        if not f32:
            flat = [orc.bf16_from_f32(x) for x in flat]
        pool.append(0, flat[0], flat[1], 3, seq_ids=ids, n_new=n_new, layout=L.LAYOUT_HEAD_MAJOR if head_major else L.LAYOUT_TOKEN_MAJOR)
    n = np.array([len(cache.k[b]) for b in ids], np.int32)
    k, v = read(pool, dev, 0, None, n, seq_ids=ids)
    assert same(k, np.concatenate([cache.k[b] for b in ids])) and same(v, np.concatenate([cache.v[b] for b in ids]))
    k, v = read(pool, dev, 0, [3, 64, 0], n - [3, 64, 0], f32=False, seq_ids=ids)
    assert same(k, G.bf16(np.concatenate([cache.k[b][t:] for b, t in zip(ids, (3, 64, 0))])))
    k, v = pool.read_rows(0, 0, 1, 20)
    assert same(orc.f32_from_bf16(v), G.bf16(cache.v[0][1:21]))
    assert pool.status() == 0
    pool.destroy()


def test_rows_of_special_values(dev):
    Hkv = 2
    x = np.zeros((9, Hkv, D), np.float32)
    x[1, 0, 7] = -3.5                      # one value
    x[2, 1] = 1e-37                        # too small for a scale
    x[3, 0, 3], x[3, 0, 4] = 1e-45, 2e-36  # a subnormal number beside a small one
    x[4, 0, 9] = np.inf
    x[5, 1, 127] = np.nan
    x[6, 0] = np.float32(3.3e38)
    x[7, 1] = np.arange(D) - 63.5          # ties
    x[8, 1, 0], x[8, 1, 1:] = 127, 2.5
    pool = make(dev, 1, 1, Hkv)
    pool.append(0, x, x[::-1].copy(), 1, n_new=[9])
    k, v = read(pool, dev, 0, None, [9])
    want = G.held(x, True)
    assert np.array_equal(np.isnan(k), np.isnan(want)) and same(np.nan_to_num(k), np.nan_to_num(want))
    assert np.isnan(k[4, 0]).all() and not np.isnan(k[4, 1]).any() and np.isnan(k[5, 1]).all()
    assert k[8, 1, 1] == 2 and (k[2] == 0).all()          # 2.5 lies between 2 and 3
    assert same(np.nan_to_num(v), np.nan_to_num(G.held(x[::-1], True)))
    pool.destroy()


@pytest.mark.parametrize("f32", [True, False])
def test_read_kv_to_any_multiple_of_16(dev, f32):
    """Places that are multiples of 16 bytes only; what lies before and behind them stays."""
    rng = np.random.default_rng(5)
    lens, Hkv, es = [130, 61], 3, 4 if f32 else 2
    pool, _ = filled(dev, rng, lens, Hkv, Hkv, 0, int8=True)
    want = read(pool, dev, 0, [1, 0], [129, 61], f32=True)
    n = int(np.prod(want[0].shape))
    for at_k, at_v in ((16, 16), (0, 48), (16, 32)):
        bufs = [dev.upload(np.full(n * es // 4 + 32, 0x7B7B7B7B, np.uint32)) for _ in range(2)]
        pool.read_kv(0, 2, bufs[0].ptr + at_k, bufs[1].ptr + at_v, [1, 0], [129, 61], dtype=bufs_dtype(f32))
        for b, at, w in zip(bufs, (at_k, at_v), want):
            raw = b.download((n * es + 128,), np.uint8)
            assert (raw[:at] == 0x7B).all() and (raw[at + n * es:] == 0x7B).all()
            got = raw[at:at + n * es].view(np.float32 if f32 else np.uint16).reshape(w.shape)
            assert same(got, w) if f32 else same(orc_f32(got), G.bf16(w))
            b.free()
    pool.destroy()


@pytest.mark.parametrize("int8", [True, False])
def test_read_kv_of_every_layer(dev, int8):
    rng = np.random.default_rng(3)
    L_, B, Hkv = 3, 300, 2                 # more sequences than one launch carries
    pool = make(dev, B, 2, Hkv, layers=L_, int8=int8)
    n = rng.integers(0, 80, B).astype(np.int32)
    k = [G.rows(rng, int(n.sum()), Hkv) for _ in range(L_)]
    v = [G.rows(rng, int(n.sum()), Hkv, "v") for _ in range(L_)]
    for l in range(L_):
        pool.append(l, k[l], v[l], B, n_new=n)
    gk, gv = read(pool, dev, -1, None, n)
    assert same(gk, G.held(np.stack(k), int8)) and same(gv, G.held(np.stack(v), int8))
    gk, gv = read(pool, dev, 1, None, n, f32=False)
    assert same(gk, G.bf16(G.held(k[1], int8)))
    pool.destroy()


def filled(dev, rng, lens, H, Hkv, extra, int8=True, seed=1):
    B = len(lens)
    per = (max(lens) + extra + PAGE - 1) // PAGE + 1
    pool, cache = make(dev, B, per, Hkv, seed=seed, int8=int8), G.Cache(B, Hkv, int8)
    if sum(lens):
        k, v = [G.rows(rng, n, Hkv) for n in lens], [G.rows(rng, n, Hkv, "v") for n in lens]
        pool.append(0, np.concatenate(k), np.concatenate(v), B, n_new=lens)
        for b in range(B):
            cache.append(b, k[b], v[b])
    return pool, cache


HEADS = [(32, 8), (8, 8), (12, 4), (32, 1), (64, 8)]


@pytest.mark.parametrize("H,Hkv", HEADS)
@pytest.mark.parametrize("lens", [[1], [63, 64, 65, 1], [700, 128, 2, 129], [5000]])
def test_decode(dev, H, Hkv, lens):
    rng = np.random.default_rng(sum(lens) + H)
    pool, cache = filled(dev, rng, lens, H, Hkv, 0)
    B = len(lens)
    q = G.bf16(rng.standard_normal((B, 1, H, D)))
    out = np.empty((B, 1, H, D), np.float32)
    pool.decode(0, B, q, out, H, D, D ** -0.5)
    for b in range(B):
        want, bound = G.attend(cache.k[b], cache.v[b], q[b], lens[b] - 1, G.causal(1), D ** -0.5)
        G.check(out[b], want, bound, "sequence %d" % b)
    assert pool.status() == 0
    pool.destroy()


@pytest.mark.parametrize("scale_of_q", [1.0, 1e-30, 3e30, 0.0])
def test_queries_of_any_size(dev, scale_of_q):
    """Queries become binary16 behind a power of two: none overflows, none is lost."""
    rng = np.random.default_rng(8)
    H, Hkv, lens = 16, 4, [100, 3]
    pool, cache = filled(dev, rng, lens, H, Hkv, 0)
    q = (rng.standard_normal((2, 1, H, D)) * scale_of_q).astype(np.float32)
    q[..., :4] *= 1e-3
    scale = D ** -0.5 if scale_of_q == 0 else float(np.float32(D ** -0.5 / scale_of_q))
    out = np.empty((2, 1, H, D), np.float32)
    pool.decode(0, 2, q, out, H, D, scale)
    for b in range(2):
        # a query's value is off by 2^-11 of itself, or, below 2^-28 of its row's largest, by 2^-39 of that
        want, bound = G.attend(cache.k[b], cache.v[b], q[b], lens[b] - 1, G.causal(1), scale, q_rounding=2.0 ** -11)
        G.check(out[b], want, bound, "sequence %d" % b)
    pool.destroy()


@pytest.mark.parametrize("S", [2, 4, 5, 8, 33, 100, 257])
@pytest.mark.parametrize("H,Hkv", [(32, 8), (12, 4), (64, 8)])
@pytest.mark.parametrize("lens", [[0, 1, 62], [640, 61]])
def test_verify_and_prompt_chunks(dev, S, H, Hkv, lens):
    from oracle import binding as orc
    rng = np.random.default_rng(S + H + len(lens))
    pool, cache = filled(dev, rng, lens, H, Hkv, S)
    B = len(lens)
    k, v = G.rows(rng, B * S, Hkv), G.rows(rng, B * S, Hkv, "v")
    q = G.bf16(rng.standard_normal((B, S, H, D)))
    out, out16 = np.empty((B, S, H, D), np.float32), np.empty((B, S, H, D), np.uint16)
    pool.verify(0, B, q, out, k, v, H, D, D ** -0.5, S)
    assert [pool.seq_len(0, b) for b in range(B)] == lens
    pool.append(0, k, v, B, n_new=[S] * B)
    pool.decode(0, B, orc.bf16_from_f32(q), out16, H, D, D ** -0.5, q_tokens=S)
    for b in range(B):
        cache.append(b, k[b * S:(b + 1) * S], v[b * S:(b + 1) * S])
        want, bound = G.attend(cache.k[b], cache.v[b], q[b], lens[b], G.causal(S), D ** -0.5)
        G.check(out[b], want, bound, "verify, sequence %d" % b)
        G.check(orc.f32_from_bf16(out16[b]), want, bound, "decode, sequence %d" % b, bf16_out=True)
        gk, gv = read(pool, dev, 0, [0], [lens[b] + S], seq_ids=[b])
        assert same(gk, cache.k[b]) and same(gv, cache.v[b])
    assert pool.status() == 0
    pool.destroy()


@pytest.mark.parametrize("S", [1, 3, 40])
def test_no_mask(dev, S):
    """causal = 0: every query sees every row."""
    rng = np.random.default_rng(S)
    H, Hkv, lens = 16, 2, [S, 130]
    pool, cache = filled(dev, rng, lens, H, Hkv, 0)
    q = G.bf16(rng.standard_normal((2, S, H, D)))
    out = np.empty((2, S, H, D), np.float32)
    pool.decode(0, 2, q, out, H, D, D ** -0.5, q_tokens=S, causal=False)
    for b in range(2):
        want, bound = G.attend(cache.k[b], cache.v[b], q[b], lens[b], np.zeros((S, 0), bool), D ** -0.5)
        G.check(out[b], want, bound, "sequence %d" % b)
    pool.destroy()


def test_steps_of_a_batch(dev):
    """Fused steps, sequences named out of order, one of them resting: rows and outputs as by append and decode."""
    rng = np.random.default_rng(5)
    H, Hkv, lens = 32, 8, [63, 10, 200, 0]
    pool, cache = filled(dev, rng, lens, H, Hkv, 8)
    ids = np.array([3, 0, 2], np.int32)
    for _ in range(4):
        k, v, q = G.rows(rng, 3, Hkv), G.rows(rng, 3, Hkv, "v"), G.bf16(rng.standard_normal((3, 1, H, D)))
        out = np.empty((3, 1, H, D), np.float32)
        pool.step(0, 3, k, v, q, out, H, D, D ** -0.5, seq_ids=ids)
        for j, b in enumerate(ids):
            cache.append(b, k[j:j + 1], v[j:j + 1])
            n = len(cache.k[b])
            want, bound = G.attend(cache.k[b], cache.v[b], q[j], n - 1, G.causal(1), D ** -0.5)
            G.check(out[j], want, bound, "sequence %d" % b)
            assert pool.seq_len(0, int(b)) == n
            gk, _ = read(pool, dev, 0, [0], [n], seq_ids=[b])
            assert same(gk, cache.k[b])
    assert pool.seq_len(0, 1) == 10
    pool.destroy()


def test_what_no_query_sees_is_harmless(dev):
    """Rows of NaN past the cursor, and in pages that another sequence has left."""
    rng = np.random.default_rng(6)
    H, Hkv, lens, S = 32, 8, [50, 64, 130], 2
    pool, cache = filled(dev, rng, lens, H, Hkv, 70)
    bad = np.full((3 * 66, Hkv, D), np.nan, np.float32)
    bad[::2] = np.inf
    pool.append(0, bad, bad, 3, n_new=[66] * 3, advance=False)
    q, out = G.bf16(rng.standard_normal((3, S, H, D))), np.empty((3, S, H, D), np.float32)
    k, v = G.rows(rng, 3 * S, Hkv), G.rows(rng, 3 * S, Hkv, "v")
    k[1], v[3] = np.nan, np.inf            # the second draft of sequence 0, and of sequence 1: their first queries do not see them
    pool.verify(0, 3, q, out, k, v, H, D, D ** -0.5, S)
    for b in range(3):
        cache.append(b, k[b * S:(b + 1) * S], v[b * S:(b + 1) * S])
        seen = 1 if b < 2 else 2
        want, bound = G.attend(cache.k[b][:lens[b] + seen], cache.v[b][:lens[b] + seen], q[b][:seen], lens[b], G.causal(seen), D ** -0.5)
        G.check(out[b][:seen], want, bound, "sequence %d" % b)
    assert np.isnan(out[0, 1]).all() and np.isnan(out[1, 1]).all()
    pool.destroy()


def test_many_sequences(dev):
    """More sequences than the launch carries as arguments."""
    rng = np.random.default_rng(7)
    H, Hkv, B = 8, 2, 300
    lens = [int(x) for x in rng.integers(1, 100, B)]
    pool, cache = filled(dev, rng, lens, H, Hkv, 0)
    q, out = G.bf16(rng.standard_normal((B, 1, H, D))), np.empty((B, 1, H, D), np.float32)
    pool.decode(0, B, q, out, H, D, D ** -0.5)
    for b in range(B):
        want, bound = G.attend(cache.k[b], cache.v[b], q[b], lens[b] - 1, G.causal(1), D ** -0.5)
        G.check(out[b], want, bound, "sequence %d" % b)
    pool.destroy()


@pytest.mark.parametrize("calls", [(1, 2), (20, 1)])
def test_a_layer_step(dev, calls):
    """relux_gqa_forward_cached on an 8-bit pool: its attention over the rows that the pool holds afterwards; of a step and of a prompt."""
    from oracle import binding as orc
    rng = np.random.default_rng(9)
    H, Hkv, lens, dm = 2, 1, [90, 0], 256
    pool, cache = filled(dev, rng, lens, H, Hkv, 24)
    w = {n: orc.bf16_from_f32(rng.standard_normal((dm, c)).astype(np.float32) * dm ** -0.5) for n, c in (("w_q", dm), ("w_k", D), ("w_v", D), ("w_o", dm))}
    dw = {n: dev.upload(x) for n, x in w.items()}
    f = {n: orc.f32_from_bf16(x).astype(np.float64) for n, x in w.items()}
    for S in calls:
        before = [pool.seq_len(0, b) for b in range(2)]
        x, out = rng.standard_normal((2, S, dm)).astype(np.float32), np.empty((2, S, dm), np.float32)
        pool.forward_cached(0, 2, x, out, dw, dm, H, q_tokens=S, rope=False)
        xb = G.bf16(x).astype(np.float64)
        for b in range(2):
            gk, gv = read(pool, dev, 0, [0], [before[b] + S], seq_ids=[b])
            # queries are rounded to bf16 by the projection: 2^-8 of each
            want, bound = G.attend(gk, gv, (xb[b] @ f["w_q"]).reshape(S, H, D), before[b], G.causal(S), D ** -0.5, q_rounding=2.0 ** -8)
            bound = bound + (np.abs(want) + bound) * 2.0 ** -8          # the output projection's operand is bf16
            G.check(out[b], want.reshape(S, dm) @ f["w_o"], bound.reshape(S, dm) @ np.abs(f["w_o"]) + 1e-5, "S=%d, sequence %d" % (S, b))
            # the new rows: projections in float32, then the rule; half a step of the scale and the projection's own rounding
            new = (xb[b] @ f["w_v"]).reshape(S, Hkv, D)
            step = np.abs(new).max(-1, keepdims=True) / 127
            assert (np.abs(gv[before[b]:] - new) <= step * 0.51 + 1e-4).all()
    pool.destroy()
    for x in dw.values():
        x.free()


def test_file_round_trip(dev, tmp_path):
    rng = np.random.default_rng(10)
    pool, cache = filled(dev, rng, [77], 8, 2, 0)
    pool.save_file(0, str(tmp_path / "c"), 100)
    other = make(dev, 1, 2, 2, int8=False)
    other.load_file(0, str(tmp_path / "c"), 100, [77])
    k, v = read(other, dev, 0, None, [77])
    assert same(k, G.bf16(cache.k[0])) and same(v, G.bf16(cache.v[0]))
    back = make(dev, 1, 2, 2)
    back.load_file(0, str(tmp_path / "c"), 100, [77])
    k, v = read(back, dev, 0, None, [77])
    assert same(k, G.held(G.bf16(cache.k[0]), True))
    for p in (pool, other, back):
        p.destroy()


def test_refusals(dev):
    import ctypes as C
    import relux_b200 as rb
    from relux_b200 import lib as L
    for kw, code in ((dict(kind=L.POOL_MLA, dC=64, dHR=16), L.ERR_UNSUPPORTED), (dict(kind=L.POOL_GQA, num_kv_heads=2, head_dim=64), L.ERR_UNSUPPORTED),
                     (dict(kind=L.POOL_GQA, num_kv_heads=2, head_dim=128, page_tokens=32), L.ERR_UNSUPPORTED),
                     (dict(kind=L.POOL_GQA, num_kv_heads=2, head_dim=128, reference_compat=True), L.ERR_INVALID_ARG)):
        kw = dict(kw)
        with pytest.raises(L.ReluxCudaError) as e:
            rb.Pool(dev, kw.pop("kind"), 1, 4, kw.pop("page_tokens", 64), 1, 4, cache_int8=True, **kw)
        assert e.value.code == code
    pool = make(dev, 2, 2, 2)
    x = np.ones((2, 2, D), np.float32)
    pool.append(0, x, x, 2)
    q, out = np.ones((2, 1, 4, D), np.float32), np.empty((2, 1, 4, D), np.float32)
    launches = dev.launch_count()

    def refused(code, f, *a, **kw):
        with pytest.raises(L.ReluxCudaError) as e:
            f(*a, **kw)
        assert e.value.code == code, str(e.value)

    refused(L.ERR_UNSUPPORTED, pool.decode, 0, 2, q, out, 4, D, 0.1, mode=L.ATTN_REFERENCE)
    refused(L.ERR_INVALID_ARG, pool.decode, 0, 2, q, out, 4, D, 0.1, mode=L.ATTN_REFERENCE_FAITHFUL)
    dq, do = dev.upload(q), dev.alloc(out.nbytes, L.DTYPE_F32)
    refused(L.ERR_UNSUPPORTED, pool.decode_noalloc, 0, 2, dq, do, 4, D, 0.1)
    refused(L.ERR_OVERFLOW, pool.append, 0, np.ones((2 * 128, 2, D), np.float32), np.ones((2 * 128, 2, D), np.float32), 2, n_new=[128, 128])
    refused(L.ERR_INVALID_ARG, pool.read_kv, 1, 2, dq, do, None, [1, 1], dtype=L.DTYPE_F32)
    refused(L.ERR_INVALID_ARG, pool.read_kv, 0, 2, dq.ptr + 8, do.ptr, None, [1, 1], dtype=L.DTYPE_F32)
    refused(L.ERR_INVALID_ARG, pool.read_kv, 0, 2, dq.ptr, do.ptr, [127, 0], [2, 1], dtype=L.DTYPE_F32)
    refused(L.ERR_INVALID_ARG, pool.read_kv, 0, 2, dq.ptr, do.ptr, [-1, 0], [2, 1], dtype=L.DTYPE_F32)
    refused(L.ERR_INVALID_ARG, pool.read_kv, 0, 2, dq.ptr, do.ptr, None, [-1, 1], dtype=L.DTYPE_F32)
    refused(L.ERR_INVALID_ARG, pool.read_kv, 0, 2, dq.ptr, do.ptr, None, [1, 1], seq_ids=[1, 1], dtype=L.DTYPE_F32)
    refused(L.ERR_INVALID_ARG, pool.read_kv, 0, 2, dq.ptr, do.ptr, None, [1, 1], dtype=7)
    args = L.ReadKvArgs(layer=0, n_seqs=2, n_tokens=np.ones(2, np.int32).ctypes.data, k=dq.ptr, v=do.ptr)
    args.reserved[1] = 1
    assert pool.lib.relux_gqa_read_kv(pool.h, C.byref(args)) == L.ERR_INVALID_ARG
    assert pool.lib.relux_gqa_read_kv(pool.h, None) == L.ERR_INVALID_ARG
    mla = rb.Pool(dev, L.POOL_MLA, 1, 2, PAGE, 1, 2, dC=64, dHR=16)
    mla.seq_alloc(10)
    refused(L.ERR_INVALID_ARG, mla.read_kv, 0, 1, dq.ptr, do.ptr, None, [1], dtype=L.DTYPE_F32)
    assert dev.launch_count() == launches
    pool.decode(0, 2, q, out, 4, D, 0.1)      # the pool still serves
    assert np.abs(out - 1).max() < 0.01 and pool.status() == 0
    mla.destroy()
    pool.destroy()
    dq.free()
    do.free()
