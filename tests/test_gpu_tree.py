"""Drafted trees over the grouped-query caches: attention within a bound derived from its roundings (tests/gqa_plain.py), commits bit for bit, and rounds of
both as a serving loop makes them."""
import ctypes as C

import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_cache_int8 import filled, make, read, same

pytestmark = pytest.mark.gpu
D, PAGE = 128, 64


@pytest.fixture(scope="module")
def dev():
    import relux_b200 as rb
    d = rb.Device(0)
    yield d
    d.close()


def tree_case(dev, rng, lens, nodes, S, H, Hkv, int8, one_tree=False, kv_f32=True, q_dtype="f32", out_bf16=False, what=""):
    from oracle import binding as orc
    B = len(lens)
    pool, cache = filled(dev, rng, lens, H, Hkv, S, int8=int8)
    parents = G.random_tree(rng, S) if one_tree else np.stack([G.random_tree(rng, S, roots=int(rng.integers(1, 5))) for _ in range(B)])
    n = int(np.sum(nodes))
    k, v = G.rows(rng, n, Hkv), G.rows(rng, n, Hkv, "v")
    q = G.bf16(rng.standard_normal((B, S, H, D)))
    out = np.full((B, S, H, D), 7, np.uint16 if out_bf16 else np.float32)
    conv = (lambda x: x) if kv_f32 else orc.bf16_from_f32
    if not kv_f32:
        k, v = G.bf16(k), G.bf16(v)
    pool.tree_verify(0, B, q if q_dtype == "f32" else orc.bf16_from_f32(q), out, conv(k), conv(v), H, D, D ** -0.5, parents, n_nodes=nodes)
    got = orc.f32_from_bf16(out) if out_bf16 else out
    at = 0
    for b in range(B):
        kk, vv = G.held(k[at:at + nodes[b]], int8), G.held(v[at:at + nodes[b]], int8)
        at += nodes[b]
        see = G.ancestors(parents if one_tree else parents[b], nodes[b], S)[:, :nodes[b]]
        K, V = np.concatenate([cache.k[b], kk]), np.concatenate([cache.v[b], vv])
        m = nodes[b]
        if m:
            want, bound = G.attend(K, V, q[b][:m], lens[b], see[:m], D ** -0.5)
            G.check(got[b][:m], want, bound, "%s sequence %d" % (what, b), bf16_out=out_bf16)
        assert (got[b][m:] == 0).all()
        assert pool.seq_len(0, b) == lens[b]
        if m:
            gk, gv = read(pool, dev, 0, [lens[b]], [m], seq_ids=[b])
            assert same(gk, kk) and same(gv, vv)
    assert pool.status() == 0
    pool.destroy()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,Hkv", [(32, 8), (8, 8), (12, 4), (64, 8), (32, 1)])
@pytest.mark.parametrize("S", [1, 2, 7, 16, 33, 64])
def test_tree(dev, int8, H, Hkv, S):
    rng = np.random.default_rng(S * 100 + H + Hkv + int8)
    tree_case(dev, rng, [0, 63, 130], [S, max(1, S - 3), S], S, H, Hkv, int8)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lens", [[1], [64], [65, 127, 128, 129], [60], [191], [3000, 5], [0, 0]])
def test_lengths_around_pages(dev, int8, lens):
    rng = np.random.default_rng(sum(lens) + int8)
    for S in (5, 40):
        tree_case(dev, rng, lens, [S] * len(lens), S, 16, 4, int8, what="S=%d" % S)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("kv_f32,q_dtype,out_bf16", [(True, "bf16", True), (False, "f32", False), (False, "bf16", True)])
def test_types(dev, int8, kv_f32, q_dtype, out_bf16):
    rng = np.random.default_rng(4)
    for S in (6, 50):
        tree_case(dev, rng, [100, 64], [S, S // 2], S, 32, 8, int8, kv_f32=kv_f32, q_dtype=q_dtype, out_bf16=out_bf16)


@pytest.mark.parametrize("int8", [False, True])
def test_one_tree_for_all_and_sequences_without_nodes(dev, int8):
    rng = np.random.default_rng(5)
    for S, H in ((9, 8), (40, 32)):
        tree_case(dev, rng, [10, 0, 200, 64], [S, 0, 1, S - 1], S, H, 4, int8, one_tree=True)
        tree_case(dev, rng, [10, 0, 200, 64], [0, 0, 0, 0], S, H, 4, int8)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("S", [3, 30])
def test_many_sequences(dev, int8, S):
    rng = np.random.default_rng(6 + S)
    B = 270
    lens = [int(x) for x in rng.integers(0, 70, B)]
    tree_case(dev, rng, lens, [int(x) for x in rng.integers(1, S + 1, B)], S, 8, 2, int8)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,S", [(8, 6), (32, 20)])
def test_a_chain_is_a_verify(dev, int8, H, S):
    """A tree of one branch sees what relux_gqa_verify's causal mask sees."""
    rng = np.random.default_rng(7)
    Hkv, lens = 4, [100, 33]
    pool, cache = filled(dev, rng, lens, H, Hkv, S, int8=int8)
    k, v, q = G.rows(rng, 2 * S, Hkv), G.rows(rng, 2 * S, Hkv, "v"), G.bf16(rng.standard_normal((2, S, H, D)))
    a, b = np.empty((2, S, H, D), np.float32), np.empty((2, S, H, D), np.float32)
    pool.verify(0, 2, q, a, k, v, H, D, D ** -0.5, S)
    pool.tree_verify(0, 2, q, b, k, v, H, D, D ** -0.5, np.arange(-1, S - 1))
    for i in range(2):
        K, V = (np.concatenate([c[i], G.held(x[i * S:(i + 1) * S], int8)]) for c, x in ((cache.k, k), (cache.v, v)))
        want, bound = G.attend(K, V, q[i], lens[i], G.causal(S), D ** -0.5)
        G.check(a[i], want, bound, "verify")
        G.check(b[i], want, bound, "tree")
    pool.destroy()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,S", [(8, 8), (32, 24)])
def test_infinities_and_nan_reach_who_sees_them(dev, int8, H, S):
    rng = np.random.default_rng(8)
    Hkv, lens = 4, [70, 64, 0]
    pool, cache = filled(dev, rng, lens, H, Hkv, 80, int8=int8)
    stale = np.full((3 * 70, Hkv, D), np.nan, np.float32)
    stale[1::2] = -np.inf
    pool.append(0, stale, stale, 3, n_new=[70] * 3, advance=False)     # what an older draft left
    parents = np.array([-1, -1, 0, 0, 1, 2, 2, 4] + [7] * (S - 8), np.int32)
    k, v = G.rows(rng, 3 * S, Hkv), G.rows(rng, 3 * S, Hkv, "v")
    q = G.bf16(rng.standard_normal((3, S, H, D)))
    # node 2 of the first sequence has a NaN among its keys, node 1 of the second an infinity among its values (one kv head each), of the third nobody
    k[2, 1, 5] = np.nan
    v[S + 1, 2, 9] = -np.inf
    out = np.empty((3, S, H, D), np.float32)
    pool.tree_verify(0, 3, q, out, k, v, H, D, D ** -0.5, parents)
    see, g = G.ancestors(parents, S, S), H // Hkv
    with np.errstate(invalid="ignore"):
        for b, (node, head) in enumerate(((2, 1), (1, 2), (None, None))):
            K, V = (np.concatenate([c[b], G.held(x[b * S:(b + 1) * S], int8)]) for c, x in ((cache.k, k), (cache.v, v)))
            fine = np.ones((S, H), bool)
            if node is not None:
                fine[see[:, node], head * g:(head + 1) * g] = False
                assert np.isnan(out[b][~fine]).all()
                K, V = np.nan_to_num(K, posinf=0, neginf=0), np.nan_to_num(V, posinf=0, neginf=0)
            want, bound = G.attend(K, V, q[b], lens[b], see, D ** -0.5)
            G.check(out[b][fine], want[fine], bound[fine], "sequence %d" % b)
    pool.destroy()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("layer", [-1, 1])
def test_commit_moves_the_path(dev, int8, layer):
    rng = np.random.default_rng(9)
    L_, B, Hkv, S = 3, 5, 3, 64
    lens = [0, 50, 64, 127, 200]
    pool = make(dev, B, 6, Hkv, layers=L_, int8=int8)
    paths = [[0, 1, 2], [3, 5, 6, 7, 9, 40, 63], [], list(range(64)), [63]]
    k = [[G.rows(rng, n + S, Hkv) for n in lens] for _ in range(L_)]
    v = [[G.rows(rng, n + S, Hkv, "v") for n in lens] for _ in range(L_)]
    for l in range(L_):
        pool.append(l, np.concatenate([x[:n] for x, n in zip(k[l], lens)]), np.concatenate([x[:n] for x, n in zip(v[l], lens)]), B, n_new=lens)
        pool.append(l, np.concatenate([x[n:] for x, n in zip(k[l], lens)]), np.concatenate([x[n:] for x, n in zip(v[l], lens)]), B, n_new=[S] * B, advance=False)
    ids = np.array([4, 1, 0, 3, 2], np.int32)
    path = np.full((B, 64), -7, np.int32)
    for i, b in enumerate(ids):
        path[i, :len(paths[b])] = paths[b]
    pool.tree_commit(layer, path, [len(paths[b]) for b in ids], seq_ids=ids)
    for l in range(L_):
        moved = layer < 0 or l == layer
        for b in range(B):
            n = lens[b] + (len(paths[b]) if moved else 0)
            assert pool.seq_len(l, b) == n
            gk, gv = read(pool, dev, l, [0], [lens[b] + S], seq_ids=[b])
            for got, rows_ in ((gk, k[l][b]), (gv, v[l][b])):
                want = G.held(rows_, int8)
                if moved:
                    want[lens[b]:n] = want[lens[b] + np.asarray(paths[b], int)]
                assert same(got, want), (l, b)
    # the lengths of the device are the host's: an append lands behind the path
    x = G.rows(rng, B, Hkv)
    pool.append(1, x, x, B)
    for b in range(B):
        gk, _ = read(pool, dev, 1, [lens[b] + len(paths[b])], [1], seq_ids=[b])
        assert same(gk, G.held(x[b:b + 1], int8))
    assert pool.status() == 0
    pool.destroy()


@pytest.mark.parametrize("D_,P", [(64, 16), (128, 64), (72, 7)])
def test_commit_and_read_of_other_shapes(dev, D_, P):
    """Pools that tree attention does not take: pages of other sizes, other head widths."""
    import relux_b200 as rb
    from relux_b200 import lib as L
    from oracle import binding as orc
    rng = np.random.default_rng(D_)
    Hkv, n, S = 3, 20, 30
    pool = rb.Pool(dev, L.POOL_GQA, 1, 12, P, 1, 12, num_kv_heads=Hkv, head_dim=D_)
    pool.set_tables(rng.permutation(12).astype(np.int32)[None])
    x = rng.standard_normal((n + S, Hkv, D_)).astype(np.float32)
    pool.append(0, x[:n], x[:n], 1, n_new=[n])
    pool.append(0, x[n:], x[n:], 1, n_new=[S], advance=False)
    pool.tree_commit(0, [[2, 3, 29]], [3])
    bufs = [dev.alloc((n + 3) * Hkv * D_ * 2) for _ in range(2)]
    pool.read_kv(0, 1, bufs[0], bufs[1], None, [n + 3])
    want = orc.bf16_from_f32(x[list(range(n)) + [n + 2, n + 3, n + 29]])
    for b in bufs:
        assert np.array_equal(b.download(want.shape, np.uint16), want)
        b.free()
    pool.destroy()


@pytest.mark.parametrize("int8", [False, True])
def test_rounds_of_drafting(dev, int8):
    """A serving loop: prompt, then rounds of tree, commit and one plain step, on two layers; all lengths and outputs by the plain form."""
    rng = np.random.default_rng(11)
    H, Hkv, B, S, L_ = 32, 8, 3, 25, 2
    prompt = [40, 130, 7]
    pool = make(dev, B, 6, Hkv, layers=L_, int8=int8)
    caches = [G.Cache(B, Hkv, int8) for _ in range(L_)]
    for l in range(L_):
        k, v = [G.rows(rng, n, Hkv) for n in prompt], [G.rows(rng, n, Hkv, "v") for n in prompt]
        pool.append(l, np.concatenate(k), np.concatenate(v), B, n_new=prompt)
        for b in range(B):
            caches[l].append(b, k[b], v[b])
    for _ in range(3):
        parents = np.stack([G.random_tree(rng, S, 4) for _ in range(B)])
        drafts = []
        for l in range(L_):
            k, v = G.rows(rng, B * S, Hkv).reshape(B, S, Hkv, D), G.rows(rng, B * S, Hkv, "v").reshape(B, S, Hkv, D)
            q, out = G.bf16(rng.standard_normal((B, S, H, D))), np.empty((B, S, H, D), np.float32)
            pool.tree_verify(l, B, q, out, k.reshape(-1, Hkv, D), v.reshape(-1, Hkv, D), H, D, D ** -0.5, parents)
            drafts.append((k, v))
            for b in range(B):
                K, V = (np.concatenate([c, G.held(x[b], int8)]) for c, x in ((caches[l].k[b], k), (caches[l].v[b], v)))
                want, bound = G.attend(K, V, q[b], len(caches[l].k[b]), G.ancestors(parents[b], S, S), D ** -0.5)
                G.check(out[b], want, bound, "layer %d sequence %d" % (l, b))
        path, n = np.zeros((B, S), np.int32), np.zeros(B, np.int32)
        for b in range(B):
            j, up = int(rng.integers(0, S)), []
            while j >= 0:
                up.append(j)
                j = int(parents[b, j])
            path[b, :len(up)], n[b] = up[::-1], len(up)
        pool.tree_commit(-1, path, n)
        for l, (k, v) in enumerate(drafts):
            for b in range(B):
                caches[l].append(b, k[b, path[b, :n[b]]], v[b, path[b, :n[b]]])
        for l in range(L_):
            k, v, q = G.rows(rng, B, Hkv), G.rows(rng, B, Hkv, "v"), G.bf16(rng.standard_normal((B, 1, H, D)))
            out = np.empty((B, 1, H, D), np.float32)
            pool.step(l, B, k, v, q, out, H, D, D ** -0.5)
            for b in range(B):
                caches[l].append(b, k[b:b + 1], v[b:b + 1])
                m = len(caches[l].k[b])
                assert pool.seq_len(l, b) == m
                want, bound = G.attend(caches[l].k[b], caches[l].v[b], q[b], m - 1, G.causal(1), D ** -0.5)
                G.check(out[b], want, bound, "step, layer %d sequence %d" % (l, b))
    assert pool.status() == 0
    pool.destroy()


def test_pipelined_and_device_calls_agree(dev):
    from relux_b200 import lib as L
    from oracle import binding as orc
    rng = np.random.default_rng(12)
    H, Hkv, S, lens = 16, 4, 12, [100, 20]
    for int8 in (False, True):
        pool, _ = filled(dev, rng, lens, H, Hkv, S, int8=int8)
        parents = np.stack([G.random_tree(rng, S) for _ in lens])
        k, v, q = G.rows(rng, 2 * S, Hkv), G.rows(rng, 2 * S, Hkv, "v"), G.bf16(rng.standard_normal((2, S, H, D)))
        a = np.empty((2, S, H, D), np.float32)
        pool.tree_verify(0, 2, q, a, k, v, H, D, D ** -0.5, parents)
        pins = [dev.pinned(x.shape, np.float32) for x in (q, k, v, a)]
        for p, x in zip(pins, (q, k, v)):
            p.array[...] = x
        pool.tree_verify(0, 2, pins[0].array, pins[3].array, pins[1].array, pins[2].array, H, D, D ** -0.5, parents, pipelined=True)
        pool.wait_output(0)
        assert same(pins[3].array, a)
        bufs = [dev.upload(x) for x in (q, k, v)] + [dev.alloc(a.nbytes, L.DTYPE_F32)]
        pool.tree_verify(0, 2, bufs[0], bufs[3], bufs[1], bufs[2], H, D, D ** -0.5, parents)
        assert same(bufs[3].download(a.shape, np.float32), a)
        qh, oh = np.ascontiguousarray(q.transpose(0, 2, 1, 3)), np.empty((2, H, S, D), np.float32)
        kh, vh = (np.ascontiguousarray(x.reshape(2, S, Hkv, D).transpose(0, 2, 1, 3)) for x in (k, v))
        pool.tree_verify(0, 2, qh, oh, kh, vh, H, D, D ** -0.5, parents, kv_layout=L.LAYOUT_HEAD_MAJOR, q_layout=L.LAYOUT_HEAD_MAJOR,
                         out_layout=L.LAYOUT_HEAD_MAJOR)
        assert same(oh.transpose(0, 2, 1, 3), a)
        dev.sync()
        for x in bufs:
            x.free()
        for p in pins:
            p.close()
        pool.destroy()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,S", [(8, 6), (32, 20), (64, 40)])
def test_a_captured_call_runs_again(dev, int8, H, S):
    """Append of uneven sequences and a tree's verify in a graph, launched twice, with other calls of the pool between; two such graphs share its workspaces."""
    from oracle import binding as orc
    from relux_b200 import lib as L
    from tests.test_gpu_latent_graphs import Graph
    rng = np.random.default_rng(S + int8)
    Hkv, lens, n_new = 4, [100, 20, 301], [3, 1, 2]
    pool, cache = filled(dev, rng, lens, H, Hkv, S + 8, int8=int8)
    parents = np.stack([G.random_tree(rng, S) for _ in lens])
    up = lambda x: dev.upload(orc.bf16_from_f32(x))  # noqa: E731
    calls = []
    for ids in ([0, 1, 2], [2, 0]):
        n = [n_new[b] for b in ids]
        k, v, q = G.rows(rng, S * len(ids), Hkv), G.rows(rng, S * len(ids), Hkv, "v"), G.bf16(rng.standard_normal((len(ids), S, H, D)))
        bufs = [up(x) for x in (q, k, v, k[:sum(n)], v[:sum(n)])] + [dev.upload(np.full(q.shape, np.nan, np.float32))]

        def call(ids=ids, n=n, bufs=bufs):
            m = len(ids)
            pool.append(0, bufs[3], bufs[4], m, seq_ids=ids, n_new=n, advance=False)
            pool.tree_verify(0, m, bufs[0], bufs[5], bufs[1], bufs[2], H, D, D ** -0.5, parents[ids], seq_ids=ids)
        calls.append((call, bufs, ids, q, k, v))
    want = []
    for call, bufs, ids, q, k, v in calls:
        call()
        want.append(bufs[5].download(q.shape, np.float32))
        see = [G.ancestors(parents[b], S, S) for b in ids]
        for i, b in enumerate(ids):
            K, V = (np.concatenate([c, G.held(G.bf16(x[i * S:(i + 1) * S]), int8)]) for c, x in ((cache.k[b], k), (cache.v[b], v)))
            exact, bound = G.attend(K, V, q[i], lens[b], see[i], D ** -0.5)
            G.check(want[-1][i], exact, bound)
    graphs = [Graph(dev, c[0]) for c in calls]
    for _ in range(2):
        for (call, bufs, ids, q, k, v), g, w in zip(calls, graphs, want):
            bufs[5].zero()
            g.launch()
            assert same(bufs[5].download(q.shape, np.float32), w)
    assert pool.status() == 0
    for g in graphs:
        g.free()
    for c in calls:
        for b in c[1]:
            b.free()
    pool.destroy()


def test_two_handles_and_pools_in_turn(dev):
    """The same calls on two pools of each of two handles, none waited for in between, are each other's equals."""
    import relux_b200 as rb
    rng = np.random.default_rng(3)
    H, Hkv, S, lens = 32, 8, 24, [500, 70]
    other = rb.Device(0)
    parents = np.stack([G.random_tree(rng, S) for _ in lens])
    k, v, q = G.rows(rng, 2 * S, Hkv), G.rows(rng, 2 * S, Hkv, "v"), G.bf16(rng.standard_normal((2, S, H, D)))
    for int8 in (False, True):
        pools = [filled(d, np.random.default_rng(4), lens, H, Hkv, S, int8=int8)[0] for d in (dev, other, dev, other)]
        outs = [np.empty((2, S, H, D), np.float32) for _ in pools]
        for _ in range(3):
            for p, o in zip(pools, outs):
                p.tree_verify(0, 2, q, o, k, v, H, D, D ** -0.5, parents)
        dev.sync()
        other.sync()
        assert np.isfinite(outs[0]).all() and all(same(o, outs[0]) for o in outs[1:])
        for p in pools:
            assert p.status() == 0
            p.destroy()
    other.close()


def test_refusals(dev):
    import relux_b200 as rb
    from relux_b200 import lib as L
    H, Hkv, S = 8, 4, 5
    pool = make(dev, 2, 2, Hkv, int8=False)
    x = np.ones((2 * 100, Hkv, D), np.float32)
    pool.append(0, x, x, 2, n_new=[100, 100])
    q, out, kv = np.ones((2, S, H, D), np.float32), np.empty((2, S, H, D), np.float32), np.ones((2 * S, Hkv, D), np.float32)
    par = np.arange(-1, S - 1)
    launches = dev.launch_count()

    def refused(code, f, *a, **kw):
        with pytest.raises(L.ReluxCudaError) as e:
            f(*a, **kw)
        assert e.value.code == code, str(e.value)

    base = (0, 2, q, out, kv, kv, H, D, 0.1)
    for bad in ([0, 0, 1, 2, 3], [-1, 1, 0, 0, 0], [-1, -2, 0, 0, 0], [-1, 0, 3, 0, 0]):
        refused(L.ERR_INVALID_ARG, pool.tree_verify, *base, bad)
        refused(L.ERR_INVALID_ARG, pool.tree_verify, *base, [list(par), bad])
    refused(L.ERR_INVALID_ARG, pool.tree_verify, *base, par, n_nodes=[6, 4])
    refused(L.ERR_INVALID_ARG, pool.tree_verify, *base, par, n_nodes=[-1, 4])
    refused(L.ERR_INVALID_ARG, pool.tree_verify, *base, par, seq_ids=[1, 1])
    refused(L.ERR_INVALID_ARG, pool.tree_verify, *base, par, seq_ids=[0, 2])
    refused(L.ERR_INVALID_ARG, pool.tree_verify, 1, 2, q, out, kv, kv, H, D, 0.1, par)
    refused(L.ERR_INVALID_ARG, pool.tree_verify, 0, 2, q, out, kv, kv, 6, D, 0.1, par)
    refused(L.ERR_INVALID_ARG, pool.tree_verify, 0, 2, q, out, kv, kv, H, 64, 0.1, par)
    refused(L.ERR_INVALID_ARG, pool.tree_verify, 0, 2, q, out, kv, kv, H, D, 0.0, par)
    refused(L.ERR_UNSUPPORTED, pool.tree_verify, *base, par, mode=L.ATTN_REFERENCE)
    wide = np.ones((2, 65, H, D), np.float32)
    refused(L.ERR_UNSUPPORTED, pool.tree_verify, 0, 2, wide, wide, np.ones((130, Hkv, D), np.float32), np.ones((130, Hkv, D), np.float32), H, D, 0.1, np.full(65, -1))
    big = np.ones((2, 64, H, D), np.float32)
    refused(L.ERR_OVERFLOW, pool.tree_verify, 0, 2, big, big.copy(), np.ones((128, Hkv, D), np.float32), np.ones((128, Hkv, D), np.float32), H, D, 0.1, np.full(64, -1))
    at = L.AttnArgs(layer=0, n_seqs=2, q_tokens=S, num_heads=H, head_dim=D, scale=0.1, q=q.ctypes.data, out=out.ctypes.data)
    n_new = np.full(2, S, np.int32)
    ap = L.AppendArgs(layer=0, n_seqs=2, n_new=n_new.ctypes.data, a=kv.ctypes.data, b=kv.ctypes.data)
    par32 = np.ascontiguousarray(par, np.int32)

    def raw(**kw):
        t, a, e = L.TreeArgs(parents=par32.ctypes.data, n_trees=1), L.AttnArgs.from_buffer_copy(at), L.AppendArgs.from_buffer_copy(ap)
        for name, value in kw.items():
            which, field = name.split("__")
            setattr({"t": t, "a": a, "e": e}[which], field, value)
        return pool.lib.relux_gqa_tree_verify(pool.h, C.byref(a), C.byref(e), C.byref(t))

    for kw in (dict(t__parents=None), dict(t__n_trees=0), dict(t__n_trees=3), dict(a__extra_tokens=S), dict(e__advance=1), dict(e__n_seqs=1), dict(e__a=None),
               dict(a__q=None), dict(e__dtype=9), dict(e__layout=9), dict(e__flags=8), dict(a__flags=8), dict(a__q_tokens=0), dict(a__num_heads=0),
               dict(a__n_seqs=0, e__n_seqs=0)):
        assert raw(**kw) == L.ERR_INVALID_ARG, kw
    ids = np.array([0, 1], np.int32)
    assert raw(a__seq_ids=ids.ctypes.data) == L.ERR_INVALID_ARG
    for args in ((None, C.byref(ap), C.byref(L.TreeArgs())), (C.byref(at), None, C.byref(L.TreeArgs())), (C.byref(at), C.byref(ap), None)):
        assert pool.lib.relux_gqa_tree_verify(pool.h, *args) == L.ERR_INVALID_ARG
    for other in (rb.Pool(dev, L.POOL_GQA, 1, 4, 32, 1, 4, num_kv_heads=4, head_dim=D), rb.Pool(dev, L.POOL_GQA, 1, 4, PAGE, 1, 4, num_kv_heads=4, head_dim=64),
                  rb.Pool(dev, L.POOL_GQA, 1, 4, PAGE, 1, 4, num_kv_heads=4, head_dim=D, reference_compat=True)):
        other.seq_alloc(100)
        hd = other.prm.gqa_head_dim
        one = np.ones((1, S, H, hd), np.float32)
        refused(L.ERR_UNSUPPORTED, other.tree_verify, 0, 1, one, one.copy(), np.ones((S, 4, hd), np.float32), np.ones((S, 4, hd), np.float32), H, hd, 0.1, par)
        other.destroy()
    mla = rb.Pool(dev, L.POOL_MLA, 1, 2, PAGE, 1, 2, dC=64, dHR=16)
    mla.seq_alloc(10)
    refused(L.ERR_INVALID_ARG, mla.tree_verify, 0, 1, q[:1], out[:1], kv, kv, H, D, 0.1, par)
    refused(L.ERR_INVALID_ARG, mla.tree_commit, 0, [[0]], [1])
    mla.destroy()
    # commits
    refused(L.ERR_INVALID_ARG, pool.tree_commit, 1, [[0], [0]], [1, 1])
    for bad in ([1, 1, 2], [2, 1, 3], [-1, 0, 1], [0, 1, 64]):
        refused(L.ERR_INVALID_ARG, pool.tree_commit, 0, [[0, 1, 2], bad], [3, 3])
    refused(L.ERR_INVALID_ARG, pool.tree_commit, 0, [[0, 1], [0, 1]], [2, 3])
    refused(L.ERR_INVALID_ARG, pool.tree_commit, 0, [[0, 1], [0, 1]], [2, -1])
    refused(L.ERR_OVERFLOW, pool.tree_commit, 0, [[0], [28]], [1, 1])
    refused(L.ERR_INVALID_ARG, pool.tree_commit, 0, [[0], [0]], [1, 1], seq_ids=[0, 0])
    assert pool.lib.relux_gqa_tree_commit(pool.h, None) == L.ERR_INVALID_ARG
    assert dev.launch_count() == launches and [pool.seq_len(0, b) for b in range(2)] == [100, 100]
    pool.tree_verify(*base, par)          # the pool still serves
    assert np.abs(out - 1).max() < 0.01 and pool.status() == 0
    pool.destroy()
