"""Infinities and NaN in calls of more than 32 query rows a kv head (drafted trees, verifies over the 8-bit cache): they reach the outputs of who sees them, and no
others, however the streams of a call fall into ranges."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_cache_int8 import filled

pytestmark = pytest.mark.gpu
D, PAGE = 128, 64


@pytest.fixture(scope="module")
def dev():
    import relux_b200 as rb
    d = rb.Device(0)
    yield d
    d.close()


def short_streams(dev, int8, H, S, tree):
    """Streams of one tile, several to a range: the flags of a piece are of that piece alone.  Every ninth sequence has a NaN or an infinity among the values of one
    of its new rows, every eleventh one among those of a cached row, of one kv head each."""
    rng = np.random.default_rng(S + H)
    B, Hkv, g = 160, 8, H // 8
    lens = [int(x) for x in rng.integers(1, 128 - S, B)]
    pool, cache = filled(dev, rng, [0] * B, H, Hkv, 128, int8=int8)
    k0, v0 = [G.rows(rng, n, Hkv) for n in lens], [G.rows(rng, n, Hkv, "v") for n in lens]
    k, v = G.rows(rng, B * S, Hkv).reshape(B, S, Hkv, D), G.rows(rng, B * S, Hkv, "v").reshape(B, S, Hkv, D)
    cached, new = {}, {}
    for b in range(B):
        if b % 11 == 5:
            cached[b] = int(rng.integers(Hkv))
            v0[b][int(rng.integers(lens[b])), cached[b], int(rng.integers(D))] = np.inf
        if b % 9 == 4:
            new[b] = int(rng.integers(S)), int(rng.integers(Hkv))
            v[b, new[b][0], new[b][1], int(rng.integers(D))] = np.nan if b % 2 else -np.inf
    pool.append(0, np.concatenate(k0), np.concatenate(v0), B, n_new=lens)
    parents = np.stack([G.random_tree(rng, S) for _ in range(B)])
    q, out = G.bf16(rng.standard_normal((B, S, H, D))), np.empty((B, S, H, D), np.float32)
    outs = []
    for _ in range(3):
        out[...] = 7
        args = (0, B, q, out, k.reshape(-1, Hkv, D), v.reshape(-1, Hkv, D), H, D, D ** -0.5)
        if tree:
            pool.tree_verify(*args, parents)
        else:
            pool.verify(*args, S)
        outs.append(out.copy())
    for b in range(B):
        see = G.ancestors(parents[b], S, S) if tree else G.causal(S)
        bad = np.zeros((S, H), bool)
        if b in cached:
            bad[:, cached[b] * g:(cached[b] + 1) * g] = True
        if b in new:
            bad[see[:, new[b][0]], new[b][1] * g:(new[b][1] + 1) * g] = True
        with np.errstate(invalid="ignore"):
            K, V = (np.concatenate([G.held(x, int8), G.held(y, int8)]) for x, y in ((k0[b], k[b]), (v0[b], v[b])))
        want, bound = G.attend(K, np.nan_to_num(V, posinf=0, neginf=0), q[b], lens[b], see, D ** -0.5)
        for o in outs:
            # an infinity that is seen may stay one in its dim; over the 8-bit cache, and of a drafted row, the whole head is NaN
            assert not np.isfinite(o[b]).all(-1)[bad].any(), "sequence %d" % b
            G.check(o[b][~bad], want[~bad], bound[~bad], "sequence %d" % b)
    assert pool.status() == 0
    pool.destroy()


@pytest.mark.parametrize("H,S", [(32, 12), (32, 25), (64, 40)])
@pytest.mark.parametrize("tree", [True, False])
def test_short_streams_of_the_8_bit_cache(dev, H, S, tree):
    short_streams(dev, True, H, S, tree)


@pytest.mark.parametrize("H,S", [(32, 12), (32, 25), (64, 40)])
def test_short_streams_of_the_bf16_cache(dev, H, S):
    short_streams(dev, False, H, S, True)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("S", [4, 12, 25, 64])
@pytest.mark.parametrize("lens", [[2048], [100] * 40, [1500] * 40])
def test_a_nan_among_queries_reaches_their_output(dev, int8, S, lens):
    """Streams that one range has, and streams that are cut: the row of the NaN is NaN, and no other."""
    rng = np.random.default_rng(S + len(lens))
    B, H, Hkv = len(lens), 32, 8
    pool, cache = filled(dev, rng, lens, H, Hkv, S, int8=int8)
    parents = G.random_tree(rng, S)
    k, v, q = G.rows(rng, B * S, Hkv), G.rows(rng, B * S, Hkv, "v"), G.bf16(rng.standard_normal((B, S, H, D)))
    bad = np.zeros((B, S, H), bool)
    for b in range(B):
        s, h = int(rng.integers(S)), int(rng.integers(H))
        bad[b, s, h] = True
        q[b, s, h, int(rng.integers(D))] = np.nan
    see, out = G.ancestors(parents, S, S), np.full((B, S, H, D), 7, np.float32)
    for tree in (True, False) if int8 or S <= 8 else (True,):
        if tree:
            pool.tree_verify(0, B, q, out, k, v, H, D, D ** -0.5, parents)
        else:
            pool.verify(0, B, q, out, k, v, H, D, D ** -0.5, S)
        assert np.isnan(out[bad]).all() and np.isfinite(out[~bad]).all()
        for b in range(0, B, 13):
            K, V = (np.concatenate([c[b], G.held(x[b * S:(b + 1) * S], int8)]) for c, x in ((cache.k, k), (cache.v, v)))
            want, bound = G.attend(K, V, np.nan_to_num(q[b]), lens[b], see if tree else G.causal(S), D ** -0.5)
            G.check(out[b][~bad[b]], want[~bad[b]], bound[~bad[b]], "sequence %d" % b)
    pool.destroy()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("S", [3, 12, 25, 64])
def test_a_nan_key_that_is_all_of_a_part(dev, int8, S):
    """The tile of the new rows by itself is a part of its stream in some of these calls, and a query sees one row there, whose key is NaN."""
    rng = np.random.default_rng(S)
    H, Hkv = 32, 8
    for n in range(8, 23):
        pool, _ = filled(dev, rng, [128 * n], H, Hkv, S, int8=int8)
        k, v, q = G.rows(rng, S, Hkv), G.rows(rng, S, Hkv, "v"), G.bf16(rng.standard_normal((1, S, H, D)))
        k[0, :, 5] = np.nan
        out = np.full((1, S, H, D), 7, np.float32)
        pool.tree_verify(0, 1, q, out, k, v, H, D, D ** -0.5, np.full(S, -1))      # only roots
        assert np.isnan(out[0, 0]).all() and np.isfinite(out[0, 1:]).all(), n
        if int8 or S <= 8:
            pool.verify(0, 1, q, out, k, v, H, D, D ** -0.5, S)                     # the first draft, which all see
            assert np.isnan(out).all(), n
        pool.destroy()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("S", [6, 12, 16, 25, 64])
@pytest.mark.parametrize("lens", [[700], [90, 128, 0], [300] * 40])
def test_whatever_stands_in_rows_past_the_nodes(dev, int8, S, lens):
    """Queries of a padded batch may be anything: their outputs are zeros, and nobody else's change."""
    rng = np.random.default_rng(S + len(lens))
    B, H, Hkv = len(lens), 32, 8
    pool, cache = filled(dev, rng, lens, H, Hkv, S, int8=int8)
    nodes = [int(x) for x in rng.integers(0, S, B)]
    n, parents = sum(nodes), G.random_tree(rng, S)
    k, v, q = G.rows(rng, n, Hkv), G.rows(rng, n, Hkv, "v"), G.bf16(rng.standard_normal((B, S, H, D)))
    want, at = [], 0
    for b, m in enumerate(nodes):
        K, V = (np.concatenate([c[b], G.held(y[at:at + m], int8)]) for c, y in ((cache.k, k), (cache.v, v)))
        want.append(G.attend(K, V, q[b, :m], lens[b], G.ancestors(parents, m, S)[:m, :m], D ** -0.5) if b < 4 else None)
        at += m
    for fill in (0.0, np.inf, -np.inf, np.nan, 3e38):
        x = q.copy()
        for b in range(B):
            x[b, nodes[b]:] = G.bf16(np.float32(fill)) * (np.sign(q[b, nodes[b]:]) if fill == 3e38 else 1)
        out = np.full((B, S, H, D), 7, np.float32)
        pool.tree_verify(0, B, x, out, k, v, H, D, D ** -0.5, parents, n_nodes=nodes)
        for b, m in enumerate(nodes):
            assert (out[b, m:] == 0).all(), fill
            if want[b] and m:
                G.check(out[b, :m], *want[b], "sequence %d, %g" % (b, fill))
    assert pool.status() == 0
    pool.destroy()


@pytest.mark.parametrize("S", [1, 4, 12, 25, 64])
@pytest.mark.parametrize("scale", [1e-8, 1e-30])
def test_queries_of_zeros_under_a_small_scale(dev, S, scale):
    """Over the 8-bit cache a query comes with a factor that holds the softmax scale: it must not vanish, or a hidden score, minus infinity, becomes NaN."""
    rng = np.random.default_rng(S)
    H, Hkv, lens = 32, 8, [100, 7]
    pool, cache = filled(dev, rng, lens, H, Hkv, S)
    k, v = G.rows(rng, 2 * S, Hkv), G.rows(rng, 2 * S, Hkv, "v")
    q = G.bf16(rng.standard_normal((2, S, H, D)))
    q[:, :, ::2] = 0
    q[:, :, 1] = 1e-38
    out = np.empty((2, S, H, D), np.float32)
    for tree in (False, True):
        if tree:
            pool.tree_verify(0, 2, q, out, k, v, H, D, scale, np.arange(-1, S - 1))
        else:
            pool.verify(0, 2, q, out, k, v, H, D, scale, S)
        for b in range(2):
            K, V = (np.concatenate([c[b], G.held(x[b * S:(b + 1) * S], True)]) for c, x in ((cache.k, k), (cache.v, v)))
            want, bound = G.attend(K, V, q[b], lens[b], G.causal(S), scale, q_rounding=2.0 ** -8)
            G.check(out[b], want, bound, "sequence %d" % b)
    pool.destroy()
