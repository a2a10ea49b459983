"""What the Python calls of the norm and of 8-bit products refuse by themselves, and the argument structs, without a GPU."""
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
    return p


def buffer(nbytes, flag):
    import relux_b200 as rb
    b = rb.DeviceBuffer.__new__(rb.DeviceBuffer)
    b.ptr, b.nbytes, b.dtype_flag, b.free = 4096, nbytes, flag, lambda: None
    return b


def structs():
    from relux_b200 import lib as L
    return [("relux_rmsnorm_args", L.RmsnormArgs), ("relux_int8_rows_args", L.Int8RowsArgs), ("relux_int8_weights_args", L.Int8WeightsArgs),
            ("relux_matmul_int8_args", L.MatmulInt8Args), ("relux_matmul_lora_args", L.MatmulLoraArgs),
            ("relux_block_projection", L.BlockProjection), ("relux_gqa_block_args", L.GqaBlockArgs)]


def test_struct_layouts(tmp_path):
    fields = structs()
    lines = "".join('printf("%%zu ", sizeof(%s)); ' % n + "".join('printf("%%zu ", offsetof(%s, %s)); ' % (n, f[0]) for f in s._fields_) for n, s in fields)
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "relux_cuda.h"\nint main(void){ %s return 0; }\n' % lines)
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert got == [x for _, s in fields for x in [C.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]]


def test_host_arrays_and_short_buffers(pool):
    host, f32, bf16 = np.zeros((2, 64), np.float32), buffer(2 * 64 * 4, 0), buffer(2 * 64 * 2, 1)
    with pytest.raises(TypeError):
        pool.rmsnorm(2, 64, f32, out=host)
    with pytest.raises(TypeError):
        pool.rmsnorm(2, 64, host, out=f32)
    for kw in (dict(n_rows=3), dict(d=128), dict(residual=buffer(255, 1)), dict(weight=buffer(127, 1)), dict(out=buffer(511, 0)), dict(codes=buffer(127, 1)),
               dict(scales=buffer(7, 0))):
        with pytest.raises(ValueError):
            pool.rmsnorm(**{**dict(n_rows=2, d=64, x=f32, out=f32), **kw})
    with pytest.raises(ValueError):
        pool.int8_rows(2, 64, bf16, buffer(127, 1), buffer(8, 0))
    with pytest.raises(ValueError):
        pool.int8_weights(64, 2, bf16, buffer(128, 1), buffer(7, 0))
    with pytest.raises(ValueError):
        pool.matmul_int8(2, 64, 8, buffer(128, 1), buffer(8, 0), buffer(511, 1), buffer(32, 0), f32)
    with pytest.raises(ValueError):
        pool.matmul_int8(2, 64, 80, buffer(128, 1), buffer(8, 0), buffer(64 * 80, 1), buffer(320, 0), f32)


def test_a_bad_handle(pool):
    from relux_b200 import lib as L
    f32 = buffer(512, 0)
    with pytest.raises(L.ReluxCudaError) as e:
        pool.rmsnorm(2, 64, f32, out=f32)
    assert e.value.code == L.ERR_BAD_HANDLE
