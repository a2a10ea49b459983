"""What the Python calls of trees and of the read-back refuse by themselves, and the argument structs, without a GPU."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def pool():
    import __graft_entry__ as g
    g.build()
    import relux_b200 as rb
    from relux_b200 import lib as L
    p = rb.Pool.__new__(rb.Pool)
    p.lib, p.h, p.kind = L.load(), None, L.POOL_GQA
    p.prm = L.PoolParams(kind=L.POOL_GQA, num_layers=2, gqa_num_kv_heads=2, gqa_head_dim=128)
    return p


def test_struct_layouts(tmp_path):
    from relux_b200 import lib as L
    fields = [("relux_read_kv_args", L.ReadKvArgs), ("relux_tree_args", L.TreeArgs), ("relux_tree_commit_args", L.TreeCommitArgs)]
    lines = "".join('printf("%%zu ", sizeof(%s)); ' % n + "".join('printf("%%zu ", offsetof(%s, %s)); ' % (n, f[0]) for f in s._fields_) for n, s in fields)
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "relux_cuda.h"\nint main(void){ %s return 0; }\n' % lines)
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert got == [x for _, s in fields for x in [C.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]]


def test_shapes_are_checked(pool):
    x = np.zeros((2, 3, 4, 128), np.float32)
    with pytest.raises(ValueError):
        pool.tree_verify(0, 2, x, x, x, x, 4, 128, 0.1, np.zeros((3, 3), np.int32))
    with pytest.raises(ValueError):
        pool.tree_verify(0, 2, x, x, x, x, 4, 128, 0.1, np.zeros((1, 1, 3), np.int32))
    with pytest.raises(ValueError):
        pool.tree_verify(0, 2, x, x, x, x, 4, 128, 0.1, [-1, 0, 1], n_nodes=[3])
    with pytest.raises(ValueError):
        pool.tree_commit(0, [[0, 1]], [2, 1])
    with pytest.raises(ValueError):
        pool.tree_commit(0, [0, 1], [2])
    with pytest.raises(ValueError):
        pool.tree_commit(0, [[0], [1]], [1, 1], seq_ids=[0])
    with pytest.raises(TypeError):
        pool.read_kv(0, 1, x, x, None, [1])
    with pytest.raises(ValueError):
        pool.read_kv(0, 2, 16, 16, None, [1], dtype=0)


def test_bad_handles(pool):
    from relux_b200 import lib as L
    assert pool.lib.relux_gqa_read_kv(None, None) == L.ERR_BAD_HANDLE
    assert pool.lib.relux_gqa_tree_verify(None, None, None, None) == L.ERR_BAD_HANDLE
    assert pool.lib.relux_gqa_tree_commit(None, None) == L.ERR_BAD_HANDLE


def test_the_plain_form_of_the_tests():
    """The 64-bit attention that the GPU tests compare with, against a softmax written out; a tree that is a chain is the causal mask."""
    from tests import gqa_plain as G
    rng = np.random.default_rng(0)
    K, V, q = (rng.standard_normal(s) for s in ((7, 2, 128), (7, 2, 128), (3, 4, 128)))
    assert np.array_equal(G.ancestors([-1, 0, 1], 3, 3), G.causal(3))
    out, bound = G.attend(K, V, q, 4, G.causal(3), 0.1)
    for i in range(3):
        for h in range(4):
            e = np.exp([q[i, h] @ K[t, h // 2] * 0.1 for t in range(5 + i)])
            assert np.allclose(out[i, h], (e[:, None] * V[:5 + i, h // 2]).sum(0) / e.sum())
    assert (bound > 0).all()
    c, s = G.quantise(np.array([[0.0] * 127 + [1e-37], [2.5] * 127 + [127.0], [np.inf] * 128], np.float32))
    assert s[0] == 0 and np.isnan(s[2]) and c[1, 0] == 2 and c[1, 127] == 127 and (c[2] == 0).all()
