"""Calls that the 8-bit operators refuse, and calls with nothing to do. A refused call enqueues nothing and does not look into its context, so
both kinds are checked without a GPU, on a context of zeros and addresses that are never read."""
import ctypes as C

import pytest

import bmapi

F32, BF16 = 0, 1
A = 1 << 20   # an aligned address


@pytest.fixture(scope="module")
def lib():
    lib = C.CDLL(bmapi.LIB_PATH)
    vp, ci, cf = C.c_void_p, C.c_int, C.c_float
    lib.bmc_quantize_rows_q8.argtypes = [vp, ci, vp, ci, vp, vp, ci, ci, ci]
    lib.bmc_rmsnorm_q8.argtypes = [vp, ci, vp, ci, vp, vp, ci, vp, ci, ci, vp, ci, vp, ci, ci, cf]
    lib.bmc_swiglu_q8.argtypes = [vp, ci, vp, ci, vp, vp, vp, ci, ci, ci]
    lib.bmc_matmul_q8.argtypes = [vp, ci, vp, ci, vp, ci, vp, vp, vp, vp, ci, ci, ci, ci]
    return lib


CTX = C.create_string_buffer(1 << 16)


def call(lib, name, good, **changes):
    args = dict(good, **changes)
    ctx = args.pop("ctx", C.addressof(CTX))
    return getattr(lib, "bmc_" + name)(ctx, *args.values())


ROWS = dict(dtype=F32, q=A, ldq=64, scale=A, x=A, ldx=64, rows=0, C=64)
NORM = dict(dtype=F32, q=A, ldq=64, scale=A, sum=A, lds=64, x=2 * A, ldx=64, add_dtype=BF16, add=3 * A, lda=64, w=A, rows=0, C=64, eps=1e-5)
SWIGLU = dict(dtype=BF16, q=A, ldq=64, scale=A, gate=A, up=A + 128, ldgu=128, rows=0, H=64)
MATMUL = dict(dtype=F32, out=A, ldo=32, q=A, ldq=64, scale=A, w=A, wscale=A, residual=2 * A, ldr=32, BT=0, C=64, OC=32)


@pytest.mark.parametrize("name,good", [("quantize_rows_q8", ROWS), ("rmsnorm_q8", NORM), ("swiglu_q8", SWIGLU), ("matmul_q8", MATMUL)])
def test_nothing_to_do(lib, name, good):
    assert call(lib, name, good) == 0
    assert call(lib, name, good, ctx=None) == -100


@pytest.mark.parametrize("rc,change", [
    (-1, dict(dtype=2)), (-1, dict(dtype=-1)), (-1, dict(q=None)), (-1, dict(scale=None)), (-1, dict(x=None)), (-1, dict(rows=-1)), (-1, dict(C=0)),
    (-1, dict(C=-3)), (-1, dict(C=57345, ldq=60000, ldx=60000)), (-1, dict(ldq=63)), (-1, dict(ldx=63)), (-3, dict(scale=A + 2)), (-3, dict(x=A + 2)),
    (-3, dict(dtype=BF16, x=A + 1)), (0, dict(dtype=BF16, x=A + 2)), (0, dict(C=57344, ldq=57344, ldx=57344)), (0, dict(q=A + 1))])
def test_quantize_rows(lib, rc, change):
    assert call(lib, "quantize_rows_q8", ROWS, **change) == rc


@pytest.mark.parametrize("rc,change", [
    (-1, dict(dtype=3)), (-1, dict(add_dtype=2)), (0, dict(add_dtype=2, add=None)), (-1, dict(w=None)), (-1, dict(lda=63)), (0, dict(lda=0, add=None)),
    (-1, dict(lds=63)), (0, dict(lds=0, sum=None)), (-1, dict(C=0)), (-1, dict(rows=-7)), (-3, dict(w=A + 1)), (-3, dict(add=A + 1)),
    (-3, dict(sum=A + 2)), (-1, dict(sum=2 * A, lds=80)), (0, dict(sum=2 * A)), (-1, dict(sum=3 * A)), (0, dict(sum=3 * A, add_dtype=F32)),
    (-1, dict(sum=3 * A, add_dtype=F32, lds=72))])
def test_rmsnorm(lib, rc, change):
    assert call(lib, "rmsnorm_q8", NORM, **change) == rc


@pytest.mark.parametrize("rc,change", [(-1, dict(gate=None)), (-1, dict(up=None)), (-1, dict(ldgu=63)), (-1, dict(H=0)), (-1, dict(rows=-1)),
                                       (-3, dict(up=A + 1)), (-3, dict(gate=A + 1)), (-1, dict(dtype=7))])
def test_swiglu(lib, rc, change):
    assert call(lib, "swiglu_q8", SWIGLU, **change) == rc


@pytest.mark.parametrize("rc,change", [
    (-1, dict(dtype=2)), (-1, dict(BT=-1)), (-1, dict(OC=-1)), (-1, dict(C=0)), (-1, dict(C=131072, ldq=131072)), (0, dict(C=131056, ldq=131056)),
    (-1, dict(ldq=48)), (-1, dict(ldo=31)), (-1, dict(ldr=31)), (0, dict(ldr=0, residual=None)), (-1, dict(out=None)), (-1, dict(q=None)),
    (-1, dict(scale=None)), (-1, dict(w=None)), (-1, dict(wscale=None)), (-2, dict(C=56)), (-2, dict(ldq=72)), (-3, dict(q=A + 8)), (-3, dict(w=A + 1)),
    (-3, dict(scale=A + 2)), (-3, dict(wscale=A + 2)), (-3, dict(out=A + 2)), (0, dict(dtype=BF16, out=A + 2)), (-3, dict(residual=A + 1)),
    (-1, dict(residual=A, ldr=40)), (0, dict(residual=A)), (0, dict(BT=5, OC=0, ldo=0, residual=None))])
def test_matmul(lib, rc, change):
    assert call(lib, "matmul_q8", MATMUL, **change) == rc


def test_session_mode(lib):
    lib.bmx_model_set_act_quant.argtypes = [C.c_void_p, C.c_int]
    lib.bm_create_model.restype = C.c_void_p
    lib.bm_create_model.argtypes = [C.c_void_p, C.c_void_p]
    lib.bm_destroy_model.argtypes = [C.c_void_p]
    a = bmapi.make_arch("tiny")
    m = lib.bm_create_model(None, C.byref(a))
    assert m
    assert [lib.bmx_model_set_act_quant(m, b) for b in (8, 0, 4, 1, -8, 16)] == [0, 0, -1, -1, -1, -1]
    assert lib.bmx_model_set_act_quant(None, 8) == -1
    lib.bm_destroy_model(m)
