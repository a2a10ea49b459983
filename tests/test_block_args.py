"""What the Python call of a block refuses by itself, without a GPU: host arrays where the device's memory is meant, and buffers that are too short."""
import numpy as np
import pytest

from tests.test_more_args import buffer

B, S, D, H, HKV, RANK, SLOTS = 3, 2, 512, 4, 2, 16, 5
COLS = dict(w_q=D, w_k=256, w_v=256, w_o=D)


@pytest.fixture(scope="module")
def pool():
    import __graft_entry__ as g
    g.build()
    import relux_b200 as rb
    from relux_b200 import lib as L
    p = rb.Pool.__new__(rb.Pool)
    p.lib, p.h, p.kind = L.load(), None, L.POOL_GQA
    p.prm = L.PoolParams(kind=L.POOL_GQA, num_layers=1, gqa_num_kv_heads=HKV, gqa_head_dim=128)
    return p


def arguments():
    m = B * S
    return dict(layer=0, n_seqs=B, q_tokens=S, d_model=D, num_heads=H, x=buffer(m * D * 4, 0), out=buffer(m * D * 4, 0), norm_weight=buffer(2 * D, 1),
                residual=buffer(m * D * 4, 0), residual_out=buffer(m * D * 4, 0), weights={n: buffer(2 * D * c, 1) for n, c in COLS.items()},
                int8={n: (buffer(D * c, 1), buffer(4 * c, 0)) for n, c in COLS.items()},
                lora={n: (buffer(2 * SLOTS * RANK * D, 1), buffer(2 * SLOTS * RANK * c, 1), buffer(4 * SLOTS, 0)) for n, c in COLS.items()}, rank=RANK, n_slots=SLOTS,
                adapter=[0, -1, 4], seq_ids=[2, 0, 1])


def changed(args, path, f):
    """The arguments with what lies at `path` (a name, then a projection, then a place) replaced by f of it."""
    out = dict(args)
    if len(path) == 1:
        out[path[0]] = f(args[path[0]])
        return out
    group = dict(args[path[0]])
    if len(path) == 2:
        group[path[1]] = f(group[path[1]])
    else:
        t = list(group[path[1]])
        t[path[2]] = f(t[path[2]])
        group[path[1]] = tuple(t)
    out[path[0]] = group
    return out


DEVICE = ([("norm_weight",), ("residual",), ("residual_out",)] + [("weights", n) for n in COLS] + [("int8", n, i) for n in COLS for i in range(2)] +
          [("lora", n, i) for n in COLS for i in range(3)])


def test_complete_arguments_reach_the_library(pool):
    from relux_b200 import lib as L
    for more in ({}, dict(int8=None), dict(lora=None, adapter=None), dict(residual=None, residual_out=None), dict(norm_weight=None, seq_ids=None)):
        with pytest.raises(L.ReluxCudaError) as e:
            pool.block_cached(**{**arguments(), **more})
        assert e.value.code == L.ERR_BAD_HANDLE


@pytest.mark.parametrize("path", DEVICE, ids=str)
def test_host_arrays(pool, path):
    host = np.zeros(1 << 16, np.float32)
    with pytest.raises(TypeError):
        pool.block_cached(**changed(arguments(), path, lambda b: host))


@pytest.mark.parametrize("path", DEVICE + [("x",), ("out",)], ids=str)
def test_short_buffers(pool, path):
    with pytest.raises(ValueError):
        pool.block_cached(**changed(arguments(), path, lambda b: buffer(b.nbytes - 1, b.dtype_flag)))


def test_a_residual_of_the_other_type(pool):
    """residual_out is of the residual's type: a bf16-sized buffer beside a float32 residual is too short."""
    with pytest.raises(ValueError):
        pool.block_cached(**{**arguments(), "residual_out": buffer(B * S * D * 2, 1)})


def test_host_inputs_and_results_by_shape(pool):
    x, out = np.zeros((B, S, D), np.float32), np.zeros((B, S, D), np.float32)
    from relux_b200 import lib as L
    with pytest.raises(L.ReluxCudaError):
        pool.block_cached(**{**arguments(), "x": x, "out": out})
    for more in (dict(x=x[:2]), dict(out=out[:, :1]), dict(out=np.zeros((B, S, D), np.uint16)), dict(x=np.zeros((D, S, B), np.float32).T), dict(out=np.zeros((D, S, B), np.float32).T)):
        with pytest.raises((ValueError, TypeError)):
            pool.block_cached(**{**arguments(), "x": x, "out": out, **more})


def test_lists_of_another_length(pool):
    for more in (dict(seq_ids=[0, 1]), dict(adapter=[0, 1]), dict(seq_ids=[[0], [1], [2]])):
        with pytest.raises(ValueError):
            pool.block_cached(**{**arguments(), **more})
