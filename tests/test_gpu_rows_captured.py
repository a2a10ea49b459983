"""Calls of more than 32 query rows a kv head in graphs, and plain calls of the same pool behind them."""
import numpy as np
import pytest

from tests import gqa_plain as G
from tests.test_gpu_cache_int8 import filled, same
from tests.test_gpu_latent_graphs import Graph

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture(scope="module")
def dev():
    import relux_b200 as rb
    d = rb.Device(0)
    yield d
    d.close()


@pytest.mark.parametrize("int8", [True, False])
def test_plain_calls_behind_a_captured_prompt(dev, int8):
    """A long call on sequences out of order, captured; many plain ones on other sequences follow, and the graph's launches still run on its own."""
    rng = np.random.default_rng(1)
    H, Hkv, S, lens, ids = 32, 8, 40, [70, 41, 200], [2, 0]
    pool, cache = filled(dev, rng, lens, H, Hkv, 0, int8=int8)
    q = G.bf16(rng.standard_normal((2, S, H, D)))
    dq, out = dev.upload(q), dev.upload(np.zeros(q.shape, np.float32))
    call = lambda ids=ids: pool.decode(0, 2, dq, out, H, D, D ** -0.5, q_tokens=S, seq_ids=ids)  # noqa: E731
    call()
    want = out.download(q.shape, np.float32)
    for i, b in enumerate(ids):
        exact, bound = G.attend(cache.k[b], cache.v[b], q[i], lens[b] - S, G.causal(S), D ** -0.5)
        G.check(want[i], exact, bound)
    graph = Graph(dev, call)
    for _ in range(2):
        for _ in range(20):
            call([1, 2])
        out.zero()
        graph.launch()
        assert same(out.download(q.shape, np.float32), want)
    assert pool.status() == 0
    graph.free()
    dq.free()
    out.free()
    pool.destroy()


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("S", [6, 12, 64])
def test_workspaces_that_grow_behind_a_capture(dev, int8, S):
    """A tree's call in a graph, float32 queries and head-major outputs, so that they are converted in workspaces too; then plain calls of forty times its size,
    which need larger ones; then the graph's launches."""
    from relux_b200 import lib as L
    rng = np.random.default_rng(S)
    B, H, Hkv, few = 40, 32, 8, 2
    lens = [int(x) for x in rng.integers(150, 300, B)]
    pool, cache = filled(dev, rng, lens, H, Hkv, S, int8=int8)
    parents = G.random_tree(rng, S)
    k, v, q = G.rows(rng, B * S, Hkv), G.rows(rng, B * S, Hkv, "v"), G.bf16(rng.standard_normal((B, S, H, D)))

    def case(m):
        return [dev.upload(x) for x in (q[:m], k[:m * S], v[:m * S], np.zeros((m, H, S, D), np.float32))]

    def call(m, b):
        pool.tree_verify(0, m, b[0], b[3], b[1], b[2], H, D, D ** -0.5, parents, out_layout=L.LAYOUT_HEAD_MAJOR)

    small, large = case(few), case(B)
    call(few, small)
    want = small[3].download((few, H, S, D), np.float32)
    for b in range(few):
        K, V = (np.concatenate([c[b], G.held(x[b * S:(b + 1) * S], int8)]) for c, x in ((cache.k, k), (cache.v, v)))
        exact, bound = G.attend(K, V, q[b], lens[b], G.ancestors(parents, S, S), D ** -0.5)
        G.check(want[b].transpose(1, 0, 2), exact, bound)
    graph = Graph(dev, lambda: call(few, small))
    call(B, large)
    dev.sync()
    spoil = [dev.upload(np.full(1 << m, np.nan, np.float32)) for m in range(12, 24)]      # in whatever is free now
    for _ in range(2):
        small[3].zero()
        graph.launch()
        assert same(small[3].download(want.shape, np.float32), want)
        call(B, large)
    assert all(np.isnan(s.download((1 << m,), np.float32)).all() for m, s in zip(range(12, 24), spoil))
    assert pool.status() == 0
    graph.free()
    for x in small + large + spoil:
        x.free()
    pool.destroy()


@pytest.mark.parametrize("mode", [0, 1])     # cudaStreamCaptureModeGlobal, ThreadLocal: no call that allocates may be seen by the capture
def test_a_prompt_captured_in_a_strict_mode(dev, mode):
    import ctypes as C
    from relux_b200 import lib as L
    rng = np.random.default_rng(2)
    H, Hkv, S, lens, ids = 16, 4, 24, [50, 90, 30], [2, 1]
    pool, _ = filled(dev, rng, lens, H, Hkv, 0)
    q = G.bf16(rng.standard_normal((2, S, H, D)))
    dq, out = dev.upload(q), dev.upload(np.zeros(q.shape, np.float32))
    call = lambda: pool.decode(0, 2, dq, out, H, D, D ** -0.5, q_tokens=S, seq_ids=ids)  # noqa: E731
    call()
    want = out.download(q.shape, np.float32)
    rt, stream, graph, ready = C.CDLL("libcudart.so.12"), C.c_void_p(), C.c_void_p(), C.c_void_p()
    L.check(dev.lib.relux_cuda_stream(dev.h, C.byref(stream)))
    assert rt.cudaStreamBeginCapture(stream, mode) == 0
    call()
    assert rt.cudaStreamEndCapture(stream, C.byref(graph)) == 0 and rt.cudaGraphInstantiate(C.byref(ready), graph, C.c_ulonglong(0)) == 0
    out.zero()
    assert rt.cudaGraphLaunch(ready, stream) == 0
    assert same(out.download(q.shape, np.float32), want)
    assert rt.cudaGraphExecDestroy(ready) == 0 and rt.cudaGraphDestroy(graph) == 0
    dq.free()
    out.free()
    pool.destroy()


@pytest.mark.parametrize("int8", [True, False])
def test_a_captured_commit_and_read_back(dev, int8):
    """Commits in a graph go by the lengths that the device has: a second launch commits the next nodes behind the first one's."""
    from tests.test_gpu_cache_int8 import read
    rng = np.random.default_rng(4)
    Hkv, S, lens = 3, 64, [50, 127, 3]
    pool, cache = filled(dev, rng, lens, Hkv, Hkv, S, int8=int8)
    k, v = G.rows(rng, 3 * S, Hkv), G.rows(rng, 3 * S, Hkv, "v")
    pool.append(0, k, v, 3, n_new=[S] * 3, advance=False)
    ids, path, n = np.array([2, 0], np.int32), np.array([[1, 4, 5, 20], [0, 3, 0, 0]], np.int32), np.array([4, 2], np.int32)
    bufs = [dev.upload(np.zeros((8, Hkv, D), np.float32)) for _ in range(2)]

    def call():
        pool.tree_commit(0, path, n, seq_ids=ids)
        pool.read_kv(0, 2, bufs[0], bufs[1], [3, 50], [6, 2], seq_ids=ids)

    graph = Graph(dev, call)
    pool.set_len(0, [50, 3], seq_ids=[0, 2])          # the host's lengths know of the captured call; the device's have not moved
    want = [[np.concatenate([G.held(x[b * S:(b + 1) * S], int8)]) for x in (k, v)] for b in range(3)]
    at = {0: 0, 2: 0}
    for _ in range(2):
        graph.launch()
        for b, p, m in ((2, path[0], 4), (0, path[1], 2)):
            for w in want[b]:
                w[at[b]:at[b] + m] = w[at[b] + p[:m]]
            at[b] += m
        for i, buf in enumerate(bufs):
            assert same(buf.download((8, Hkv, D), np.float32), np.concatenate([want[2][i][:6], want[0][i][:2]]))
    for b in range(3):
        gk, gv = read(pool, dev, 0, [lens[b]], [S], seq_ids=[b])
        assert same(gk, want[b][0]) and same(gv, want[b][1])
    x = G.rows(rng, 2, Hkv)
    pool.append(0, x, x, 2, seq_ids=[0, 2])           # by the device's lengths
    for i, b in enumerate((0, 2)):
        gk, _ = read(pool, dev, 0, [lens[b] + at[b]], [1], seq_ids=[b])
        assert same(gk, G.held(x[i:i + 1], int8))
    assert pool.status() == 0
    graph.free()
    for b in bufs:
        b.free()
    pool.destroy()
