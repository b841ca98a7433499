"""Rows beyond what one launch can have threads for - fewer than 2^32 - go into several, each with its part (no GPU: launches on a stand-in for
the runtime)."""
import ctypes as C

import launch_recorder
import pytest


def calls(rec, name, *args):
    rc, launches = rec.of(name, *args)
    return [rc, launches]


def norm(rec, rows, cols):
    return calls(rec, "sg_rmsnorm_fp8_rows", rec.A, None, None, None, rec.B, rec.D, rec.S, C.c_float(1e-5), rows, cols, None)


def pack(rec, n, k):
    return calls(rec, "sg_int4_pack", rec.A, rec.B, None, rec.D, n, k, 128, 0, k // 2, None)


def product(rec, m, n, k, group):
    return calls(rec, "sg_int4_gemm", rec.A, rec.B, rec.D, m, n, k, group, 0, None)


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return launch_recorder.build(tmp_path_factory.mktemp("fake"))


def grid_of(fake, function, *args):
    rc, launches = launch_recorder.scenario(fake, "test_launch_limits", function, *args)
    assert rc == 0
    for kernel, grid, threads, _ in launches:
        assert grid * threads < 2 ** 32, (kernel, grid, threads)
    return sum(grid for _, grid, _, _ in launches), len(launches)


@pytest.mark.parametrize("rows,cols,of_workgroup", [(2 ** 26 + 5, 528, 1), (2 ** 27 + 9, 512, 8), (2 ** 22 + 1, 9000 * 16, 1), (2 ** 31 - 1, 16, 64),
                                                   (2 ** 24, 4096, 1)])
def test_norm(fake, rows, cols, of_workgroup):
    grid, launches = grid_of(fake, "norm", rows, cols)
    assert -(-rows // of_workgroup) <= grid <= -(-rows // of_workgroup) + launches


def test_norm_is_one_launch_up_to_there(fake):
    assert grid_of(fake, "norm", 20000, 8192) == (20000, 1)
    assert grid_of(fake, "norm", 2 ** 20, 4096) == (2 ** 20, 1)


@pytest.mark.parametrize("n,k", [(16 * 2 ** 20 + 3, 8192), (2 ** 31 - 1, 128)])
def test_pack(fake, n, k):
    grid, launches = grid_of(fake, "pack", n, k)
    need = -(-n // 16) * (k // 128)
    assert need <= 4 * grid <= need + 4 * launches
    assert grid_of(fake, "pack", 57344, 8192)[1] == 1


@pytest.mark.parametrize("m,n,k,group", [(2 ** 30, 16, 32, 32), (2 ** 29 + 77, 128, 128, 128), (2 ** 31 - 1, 4, 32, 32)])
def test_product(fake, m, n, k, group):
    grid, launches = grid_of(fake, "product", m, n, k, group)
    assert launches > 1 and grid * 64 >= m
    assert grid_of(fake, "product", 8192, 28672, 8192, 64)[1] == 1
