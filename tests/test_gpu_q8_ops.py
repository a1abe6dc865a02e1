"""The 8-bit activation operators (bmc_quantize_rows_q8, bmc_rmsnorm_q8, bmc_swiglu_q8, bmc_matmul_q8) against their definitions in
64 bits.

Tolerances. u = 2^-24 is half a step of fp32, 2^-8 half a step of bf16. A row value v that the kernel has with relative error t gives a
scale with relative error t + u, a reciprocal with one more u and a quotient with one more: the code is the nearest integer to a quotient
that is off by at most 127 (2 t + 4 u), so |code * scale - v| <= (1/2 + 127 (2 t + 4 u)) * scale.
  rows   t = 0
  norm   the sum's addition u, the sum of squares (a thread adds at most C / 32 of them in a row, then trees: C / 32 + 16 roundings, of which
         the root takes half, plus two each for the square's own), mean, eps, root, reciprocal and two products: t = (C / 64 + 20) u
  swiglu the exponential's argument is off by 2 |g| u absolutely and the exponential by 4 u; four more roundings: t = (2 |g| + 12) u
  product: conversion of the sum, product of the scales, their product: 3 u of the product; u of the sum with the residual; the store."""
import ctypes as C
import subprocess
import sys

import numpy as np
import pytest

from bmcapi import BMC_BF16, BMC_F32, Backend, bf16_round

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [BMC_F32, BMC_BF16]


@pytest.fixture(scope="module")
def be(product):
    b = Backend(product)
    yield b
    b.close()


@pytest.fixture(autouse=True)
def _free(be):
    yield
    assert be.lib.bmc_sync(be.ctx) == 0
    for p in be.bufs:
        be.lib.bmc_free(be.ctx, p)
    be.bufs.clear()


def rng_of(*key):
    return np.random.default_rng([int(k) for k in key])


def values(rng, rows, cols, dtype, std=1.0):
    x = (rng.standard_normal((rows, cols)) * std).astype(np.float32)
    x[:, ::64] *= 20.0
    return bf16_round(x) if dtype == BMC_BF16 else x


def put_rows(be, x, dtype, ld, shift=0):
    """x at a leading dimension of its own, `shift` elements behind an aligned address; the gaps hold NaN."""
    rows, cols = x.shape
    flat = np.full(shift + rows * ld, np.nan, np.float32)
    flat[shift:shift + rows * ld].reshape(rows, ld)[:, :cols] = x
    return be.put(flat, dtype) + shift * (2 if dtype == BMC_BF16 else 4)


def put_bytes(be, a):
    a = np.ascontiguousarray(a)
    p = be.alloc(a.nbytes)
    assert be.lib.bmc_upload(be.ctx, p, a.ctypes.data, a.nbytes) == 0 and be.lib.bmc_sync(be.ctx) == 0
    return p


def filled(be, n, byte):
    p = be.alloc(n)
    assert be.lib.bmc_memset(be.ctx, p, byte, n) == 0
    return p


def check_codes(codes, scale, v, t):
    """codes and scales of rows against the 64-bit values v, known to the kernel within the relative error t."""
    top = np.abs(v).max(1)
    t_row = np.max(np.broadcast_to(t, v.shape), axis=1)
    ref = top / 127.0
    assert np.all(np.abs(scale - ref) <= (t_row + 2 * U) * ref), np.max(np.abs(scale - ref) / np.maximum(ref, 1e-300))
    assert np.abs(codes.astype(np.int32)).max(initial=0) <= 127
    off = np.abs(codes * scale.astype(np.float64)[:, None] - v)
    bound = (0.5 + 127 * (2 * t + 4 * U)) * np.maximum(scale, ref)[:, None]
    assert np.all(off <= bound), (off / np.maximum(ref, 1e-300)[:, None]).max()
    some = ref > 0
    assert np.all(np.abs(codes[some].astype(np.int32)).max(1) == 127)   # the largest value of a row has the largest code


ROW_SHAPES = [(1, 1), (1, 16), (3, 5), (2, 31), (5, 33), (64, 960), (7, 964), (9, 1000), (4, 1024), (33, 576), (5, 1032), (6, 2560), (3, 2563), (2, 4096),
              (3, 4099), (2, 8192), (2, 8200), (1, 12345), (2, 16384), (1, 16392), (2, 32768), (1, 40000), (1, 57344), (700, 960), (1500, 130)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", ROW_SHAPES)
@pytest.mark.parametrize("gap,shift", [(0, 0), (16, 0), (3, 1)])
def test_quantize_rows(be, dtype, rows, cols, gap, shift):
    x = values(rng_of(rows, cols, gap), rows, cols, dtype)
    ldq, ldx = cols + (gap + 15) // 16 * 16, cols + gap
    dx, dq, ds = put_rows(be, x, dtype, ldx, shift), filled(be, rows * ldq + 64, 0x55), filled(be, rows * 4 + 64, 0x55)
    assert be.lib.bmc_quantize_rows_q8(be.ctx, dtype, dq, ldq, ds, dx, ldx, rows, cols) == 0
    q = be.get(dq, (rows * ldq + 64,), np_dtype=np.int8)
    check_codes(q[:rows * ldq].reshape(rows, ldq)[:, :cols], be.get(ds, (rows,)), x.astype(np.float64), 0.0)
    assert np.all(q[rows * ldq:] == 0x55) and np.all(q[:rows * ldq].reshape(rows, ldq)[:, cols:] == 0x55)   # gaps and what lies behind
    assert np.all(be.get(ds, (rows * 4 + 64,), np_dtype=np.uint8)[rows * 4:] == 0x55)


def norm_ref(x, add, w, eps):
    s = x.astype(np.float64) + (0 if add is None else add.astype(np.float64))
    return s, s / np.sqrt(np.mean(s * s, axis=1, keepdims=True) + eps) * w.astype(np.float64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("add_dtype", [None] + DTYPES)
@pytest.mark.parametrize("rows,cols", ROW_SHAPES)
def test_rmsnorm(be, dtype, add_dtype, rows, cols):
    rng = rng_of(rows, cols, dtype, 7)
    gap = cols % 3 * 8
    x, w = values(rng, rows, cols, dtype), (1 + 0.2 * rng.standard_normal(cols)).astype(np.float32)
    add = None if add_dtype is None else values(rng, rows, cols, add_dtype, 0.5)
    lds = cols + gap
    dx, dw = put_rows(be, x, dtype, cols + gap), be.put(w)
    da = None if add is None else put_rows(be, add, add_dtype, cols + 2 * gap)
    dq, ds, dsum = be.alloc(rows * cols), be.alloc(rows * 4), filled(be, rows * lds * 4 + 64, 0xFF)   # 0xFFFF.. is a NaN in both types
    assert be.lib.bmc_rmsnorm_q8(be.ctx, dtype, dq, cols, ds, dsum, lds, dx, cols + gap, add_dtype or 0, da, cols + 2 * gap, dw, rows, cols, 1e-5) == 0
    s, v = norm_ref(x, add, w, 1e-5)
    check_codes(be.get(dq, (rows, cols), np_dtype=np.int8), be.get(ds, (rows,)), v, (cols / 64 + 20) * U)
    got = be.get(dsum, (rows, lds), dtype)
    assert np.all(np.isnan(got[:, cols:]))
    assert np.all(np.abs(got[:, :cols] - s) <= (U if dtype == BMC_F32 else U + 2.0 ** -8) * np.abs(s))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [33, 65, 71, 72, 1537, 4093, 16385, 16391])
@pytest.mark.parametrize("shift", [0, 1, 6, 15])
def test_rows_that_start_inside_a_vector(be, dtype, cols, shift):
    """Contiguous rows from the same element on in every operand: each row starts at another element of a vector. Eight rows see them all."""
    rows, rng = 8, rng_of(cols, shift, dtype, 5)
    x, a, w = values(rng, rows, cols, dtype), values(rng, rows, cols, dtype, 0.5), (1 + 0.2 * rng.standard_normal(cols)).astype(np.float32)
    dx, da, dw = put_rows(be, x, dtype, cols, shift), put_rows(be, a, dtype, cols, shift), be.put(w)
    n, size = rows * cols, 2 if dtype == BMC_BF16 else 4
    for norm in (True, False):
        dq, ds, dsum = filled(be, n + 64, 0x55), filled(be, (rows + 1) * 4, 0x55), filled(be, (n + 64) * size, 0x55)
        if norm:
            assert be.lib.bmc_rmsnorm_q8(be.ctx, dtype, dq + shift, cols, ds, dsum + shift * size, cols, dx, cols, dtype, da, cols, dw, rows, cols, 1e-5) == 0
            s, v = norm_ref(x, a, w, 1e-5)
            raw = be.get(dsum, ((n + 64) * size,), np_dtype=np.uint8)
            assert np.all(raw[:shift * size] == 0x55) and np.all(raw[(shift + n) * size:] == 0x55)
            got = be.get(dsum + shift * size, (rows, cols), dtype)
            assert np.all(np.abs(got - s) <= (U if dtype == BMC_F32 else U + 2.0 ** -8) * np.abs(s))
        else:
            assert be.lib.bmc_quantize_rows_q8(be.ctx, dtype, dq + shift, cols, ds, dx, cols, rows, cols) == 0
            v = x.astype(np.float64)
        q, sc = be.get(dq, (n + 64,), np_dtype=np.int8), be.get(ds, (rows + 1,))
        assert np.all(q[:shift] == 0x55) and np.all(q[shift + n:] == 0x55) and sc[rows:].view(np.int32)[0] == 0x55555555
        check_codes(q[shift:shift + n].reshape(rows, cols), sc[:rows], v, (cols / 64 + 20) * U if norm else 0.0)

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [33, 960, 4100, 40000])
def test_rmsnorm_sum_in_place_and_left_out(be, dtype, cols):
    rows, rng = 9, rng_of(cols, dtype, 3)
    x, a, w = values(rng, rows, cols, dtype), values(rng, rows, cols, dtype), np.ones(cols, np.float32)
    got = []
    for where in ("own", "x", "add", None):
        dx, da, dw = be.put(x, dtype), be.put(a, dtype), be.put(w)
        dq, ds, own = be.alloc(rows * cols), be.alloc(rows * 4), be.alloc(rows * cols * 4)
        dsum = {"own": own, "x": dx, "add": da, None: None}[where]
        assert be.lib.bmc_rmsnorm_q8(be.ctx, dtype, dq, cols, ds, dsum, cols, dx, cols, dtype, da, cols, dw, rows, cols, 1e-5) == 0
        got.append((be.get(dq, (rows, cols), np_dtype=np.int8), be.get(ds, (rows,)), None if dsum is None else be.get(dsum, (rows, cols), dtype)))
        if where != "x":
            assert np.array_equal(be.get(dx, (rows, cols), dtype), x)
        if where != "add":
            assert np.array_equal(be.get(da, (rows, cols), dtype), a)
    for q, s, t in got[1:]:
        assert np.array_equal(q, got[0][0]) and np.array_equal(s, got[0][1]) and (t is None or np.array_equal(t, got[0][2]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", ROW_SHAPES)
def test_swiglu(be, dtype, rows, cols):
    rng = rng_of(rows, cols, dtype, 11)
    gu = values(rng, rows, 2 * cols, dtype, 1.5)
    if cols >= 4:
        gu[0, :4] = bf16_round(np.array([-90.0, 90.0, 0.0, -30.0], np.float32))
    d = be.put(gu, dtype)
    dq, ds = be.alloc(rows * cols), be.alloc(rows * 4)
    up = d + cols * (2 if dtype == BMC_BF16 else 4)
    assert be.lib.bmc_swiglu_q8(be.ctx, dtype, dq, cols, ds, d, up, 2 * cols, rows, cols) == 0
    g, u = gu[:, :cols].astype(np.float64), gu[:, cols:].astype(np.float64)
    check_codes(be.get(dq, (rows, cols), np_dtype=np.int8), be.get(ds, (rows,)), g / (1 + np.exp(-g)) * u, (2 * np.abs(g) + 12) * U)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(6000, 1001), (5000, 1535), (2500, 4099), (1300, 9003), (4000, 2048), (3000, 1536)])
def test_many_rows(be, dtype, rows, cols):
    """Enough rows that a thread holds as many values as it may; odd widths, whose rows start anywhere inside a vector. The unused operands of one
    operator are those of another: rows as x, norm with an addend of either type, SwiGLU of two matrices."""
    rng = rng_of(rows, cols, dtype, 21)
    x, a = values(rng, rows, cols, dtype), values(rng, rows, cols, dtype, 0.5)
    w = (1 + 0.2 * rng.standard_normal(cols)).astype(np.float32)
    dx, da, dw = be.put(x, dtype), be.put(a, dtype), be.put(w)
    dq, ds, dsum = filled(be, rows * cols + 64, 0x55), be.alloc(rows * 4), filled(be, rows * cols * 4 + 64, 0xFF)
    e = 2 if dtype == BMC_BF16 else 4

    def codes():
        q = be.get(dq, (rows * cols + 64,), np_dtype=np.int8)
        assert np.all(q[rows * cols:] == 0x55)
        return q[:rows * cols].reshape(rows, cols), be.get(ds, (rows,))

    assert be.lib.bmc_quantize_rows_q8(be.ctx, dtype, dq, cols, ds, dx, cols, rows, cols) == 0
    check_codes(*codes(), x.astype(np.float64), 0.0)
    assert be.lib.bmc_rmsnorm_q8(be.ctx, dtype, dq, cols, ds, dsum, cols, dx, cols, dtype, da, cols, dw, rows, cols, 1e-5) == 0
    s, v = norm_ref(x, a, w, 1e-5)
    check_codes(*codes(), v, (cols / 64 + 20) * U)
    raw = be.get(dsum, (rows * cols * e + 64,), np_dtype=np.uint8)
    assert np.all(raw[rows * cols * e:] == 0xFF)
    assert np.all(np.abs(be.get(dsum, (rows, cols), dtype) - s) <= (U if dtype == BMC_F32 else U + 2.0 ** -8) * np.abs(s))
    assert be.lib.bmc_swiglu_q8(be.ctx, dtype, dq, cols, ds, da, dx, cols, rows, cols) == 0
    g, u = a.astype(np.float64), x.astype(np.float64)
    check_codes(*codes(), g / (1 + np.exp(-g)) * u, (2 * np.abs(g) + 12) * U)
    other = values(rng, rows, cols, BMC_F32 + BMC_BF16 - dtype, 0.5)
    assert be.lib.bmc_rmsnorm_q8(be.ctx, dtype, dq, cols, ds, dx, cols, dx, cols, BMC_F32 + BMC_BF16 - dtype, be.put(other, BMC_F32 + BMC_BF16 - dtype), cols, dw, rows, cols, 1e-5) == 0
    check_codes(*codes(), norm_ref(x, other, w, 1e-5)[1], (cols / 64 + 20) * U)


@pytest.mark.parametrize("cols", [40, 961, 5000, 50000])
def test_rows_that_cannot_be_scaled(be, cols):
    """Zeros, subnormal scales, the largest finite values, infinities and NaN, one kind a row."""
    x = np.ones((8, cols), np.float32)
    x[0] = 0.0
    x[1] = 1e-38
    x[2] = 3.0e38
    x[3, cols - 1] = np.inf
    x[4, 0] = -np.inf
    x[5, cols // 2] = np.nan
    x[6] = -0.0
    x[7] = 2e-36
    dx, dq, ds = be.put(x), filled(be, 8 * cols, 0x11), be.alloc(32)
    assert be.lib.bmc_quantize_rows_q8(be.ctx, BMC_F32, dq, cols, ds, dx, cols, 8, cols) == 0
    q, s = be.get(dq, (8, cols), np_dtype=np.int8), be.get(ds, (8,))
    assert np.all(q[[0, 1, 3, 4, 5, 6]] == 0) and np.all(q[[2, 7]] == 127)
    assert np.array_equal(s[[0, 1, 6]], np.zeros(3, np.float32)) and np.all(np.isnan(s[[3, 4, 5]]))
    assert np.allclose(s[[2, 7]], x[[2, 7], 0] / 127, rtol=3 * U)
    # the norm: a row of zeros stays zero; a sum of squares that overflows, an infinity and a NaN give NaN
    dw = be.put(np.ones(cols, np.float32))
    assert be.lib.bmc_rmsnorm_q8(be.ctx, BMC_F32, dq, cols, ds, None, 0, dx, cols, 0, None, 0, dw, 8, cols, 1e-5) == 0
    q, s = be.get(dq, (8, cols), np_dtype=np.int8), be.get(ds, (8,))
    assert np.all(np.isnan(s[[2, 3, 4, 5]])) and np.all(q[[0, 2, 3, 4, 5, 6]] == 0) and s[0] == 0 and s[6] == 0
    # SwiGLU: as up, the same rows; an infinite gate is no number either. silu(1) * 2e-36 / 127 = 1.151e-38 lies below the smallest normal
    # number, 1.175e-38: row 7 is stored as zeros here
    gate = np.ones((8, cols), np.float32)
    gate[6, 0] = -np.inf
    both = be.put(np.concatenate([gate, x], axis=1))
    assert be.lib.bmc_swiglu_q8(be.ctx, BMC_F32, dq, cols, ds, both, both + 4 * cols, 2 * cols, 8, cols) == 0
    q, s = be.get(dq, (8, cols), np_dtype=np.int8), be.get(ds, (8,))
    assert np.all(np.isnan(s[[3, 4, 5]])) and s[0] == 0 and s[7] == 0 and np.all(q[[0, 1, 3, 4, 5, 7]] == 0) and np.all(q[2] == 127)
    assert np.isnan(s[6])


# ---- product ---------------------------------------------------------------------------------------------------------------------------
def product_case(be, dtype, M, K, N, residual=False, ldq=None, ldo=None, ldr=None, shift=0, extreme=False, key=0):
    rng = rng_of(M, K, N, key)
    ldq, ldo, ldr = ldq or K, ldo or N, ldr or N
    q = rng.integers(-128, 128, (M, K)).astype(np.int8) if not extreme else np.full((M, K), -128, np.int8)
    w = rng.integers(-128, 128, (N, K)).astype(np.int8) if not extreme else np.full((N, K), -128, np.int8)
    sa, sw = rng.uniform(0.01, 0.3, M).astype(np.float32), rng.uniform(1e-4, 1e-2, N).astype(np.float32)
    qp = np.full((M, ldq), 99, np.int8)
    qp[:, :K] = q
    dq, dw = put_bytes(be, qp), put_bytes(be, w)
    dsa, dsw = be.put(sa), be.put(sw)
    r = values(rng, M, N, dtype, 3.0) if residual else None
    dr = put_rows(be, r, dtype, ldr, shift) if residual else None
    e = 2 if dtype == BMC_BF16 else 4
    dout = filled(be, (shift + M * ldo) * e + 64, 0xFF)
    assert be.lib.bmc_matmul_q8(be.ctx, dtype, dout + shift * e, ldo, dq, ldq, dsa, dw, dsw, dr, ldr, M, K, N) == 0
    raw = be.get(dout, ((shift + M * ldo) * e + 64,), np_dtype=np.uint8)
    assert np.all(raw[: shift * e] == 0xFF) and np.all(raw[(shift + M * ldo) * e:] == 0xFF)
    out = be.get(dout + shift * e, (M, ldo), dtype)
    assert np.all(np.isnan(out[:, N:]))
    prod = (q.astype(np.float64) @ w.astype(np.float64).T) * sa.astype(np.float64)[:, None] * sw.astype(np.float64)
    ref = prod + (0 if r is None else r.astype(np.float64))
    bound = 3.01 * U * np.abs(prod) + (1.01 * U if residual else 0) * np.abs(ref) + (1.001 * 2.0 ** -8 * np.abs(ref) if dtype == BMC_BF16 else 0)
    off = np.abs(out[:, :N] - ref)
    assert np.all(off <= bound), (np.argwhere(off > bound)[:4], off.max(), np.abs(ref).max())


SMALL = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 96, 100, 127, 128, 129, 160, 255, 256, 257, 300, 511, 700]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", SMALL)
def test_product_tokens(be, dtype, M):
    product_case(be, dtype, M, 960, 200, residual=M % 2 == 1)


@pytest.mark.parametrize("N", [1, 2, 5, 31, 32, 33, 64, 127, 128, 129, 255, 256, 257, 960, 1600, 5120])
@pytest.mark.parametrize("M", [1, 5, 40, 200, 1300])
def test_product_channels(be, M, N):
    product_case(be, BMC_F32 if N % 2 else BMC_BF16, M, 576, N)


@pytest.mark.parametrize("K", [16, 32, 48, 112, 128, 144, 240, 256, 272, 384, 512, 960, 1536, 2560, 4096, 4112, 11008])
@pytest.mark.parametrize("M", [1, 4, 24, 130, 400])
def test_product_reduction(be, M, K):
    product_case(be, BMC_BF16 if K % 32 else BMC_F32, M, K, 136, residual=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 960, 1600), (6, 2560, 960), (64, 960, 5120), (64, 2560, 960), (512, 960, 1600), (2048, 960, 5120), (3000, 1536, 1001),
                                   (4099, 2048, 2048), (2500, 128, 2500), (5000, 16, 3000)])
def test_product_model_shapes(be, dtype, M, K, N):
    product_case(be, dtype, M, K, N, residual=N % 2 == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 240, 70), (5, 960, 333), (50, 480, 130), (300, 976, 520), (1100, 960, 2000)])
@pytest.mark.parametrize("gap,shift", [(16, 0), (1, 3), (8, 1)])
def test_product_strides(be, dtype, M, K, N, gap, shift):
    product_case(be, dtype, M, K, N, residual=True, ldq=K + 32, ldo=N + gap, ldr=N + 2 * gap + 1, shift=shift)


@pytest.mark.parametrize("M", [1, 3, 20, 150, 1200])
def test_product_largest_sums(be, M):
    """Every code -128 at the largest K: the sum is 2147221504, 262144 below overflow."""
    product_case(be, BMC_F32, M, 131056, 70 if M < 1000 else 520, extreme=True)


@pytest.mark.parametrize("M", [2, 30, 200, 1200])
def test_product_residual_in_place_and_repeated(be, M):
    """out may be the residual; the integer sum makes repeated calls bit-equal."""
    K, N = 960, 640
    rng = rng_of(M, 5)
    q, w = rng.integers(-127, 128, (M, K)).astype(np.int8), rng.integers(-127, 128, (N, K)).astype(np.int8)
    r = rng.standard_normal((M, N)).astype(np.float32)
    dq, dw, ds, dsw = put_bytes(be, q), put_bytes(be, w), be.put(np.full(M, 0.01, np.float32)), be.put(np.full(N, 0.02, np.float32))
    got = []
    for _ in range(4):
        dr, dout = be.put(r), be.alloc(M * N * 4)
        assert be.lib.bmc_matmul_q8(be.ctx, BMC_F32, dout, N, dq, K, ds, dw, dsw, dr, N, M, K, N) == 0
        assert be.lib.bmc_matmul_q8(be.ctx, BMC_F32, dr, N, dq, K, ds, dw, dsw, dr, N, M, K, N) == 0
        got += [be.get(dout, (M, N)), be.get(dr, (M, N))]
    for g in got[1:]:
        assert np.array_equal(g, got[0])


@pytest.mark.parametrize("M", [1, 40, 400])
def test_product_of_rows_without_a_scale(be, M):
    """A token whose scale is NaN has NaN products, one with scale 0 has zeros, and no other token sees either."""
    K, N = 480, 150
    rng = rng_of(M, 9)
    q, w = rng.integers(-127, 128, (M, K)).astype(np.int8), rng.integers(-127, 128, (N, K)).astype(np.int8)
    sa = np.full(M, 0.01, np.float32)
    sa[0] = np.nan
    q[0] = 0
    if M > 1:
        sa[M // 2] = 0.0
    dout = be.alloc(M * N * 4)
    assert be.lib.bmc_matmul_q8(be.ctx, BMC_F32, dout, N, put_bytes(be, q), K, be.put(sa), put_bytes(be, w), be.put(np.full(N, 0.02, np.float32)), None, 0, M, K, N) == 0
    out = be.get(dout, (M, N))
    assert np.all(np.isnan(out[0]))
    if M > 1:
        assert np.all(out[M // 2] == 0) and not np.isnan(out[1:]).any()


def test_offsets_beyond_32_bits(be):
    """Rows 2^30 elements apart: the third one starts 8 GB (fp32) behind the first."""
    ld, cols, rows = 1 << 30, 1000, 3
    rng = rng_of(17)
    x = values(rng, rows, cols, BMC_F32)
    dx = be.alloc(((rows - 1) * ld + cols) * 4)
    dq, ds = be.alloc((rows - 1) * ld + 1008), be.alloc(16)
    for r in range(rows):
        row = np.ascontiguousarray(x[r])
        assert be.lib.bmc_upload(be.ctx, dx + r * ld * 4, row.ctypes.data, cols * 4) == 0 and be.lib.bmc_sync(be.ctx) == 0
    assert be.lib.bmc_quantize_rows_q8(be.ctx, BMC_F32, dq, ld, ds, dx, ld, rows, cols) == 0
    codes = np.stack([be.get(dq + r * ld, (1008,), np_dtype=np.int8) for r in range(rows)])
    check_codes(codes[:, :cols], be.get(ds, (rows,)), x.astype(np.float64), 0.0)
    assert not codes[:, cols:].any()
    # the product reads those rows in place (the eight codes behind the row are zero) and writes rows as far apart
    w = rng.integers(-127, 128, (64, 1008)).astype(np.int8)
    sw = np.full(64, 0.01, np.float32)
    assert be.lib.bmc_matmul_q8(be.ctx, BMC_F32, dx, ld, dq, ld, ds, put_bytes(be, w), be.put(sw), None, 0, rows, 1008, 64) == 0
    out = np.stack([be.get(dx + r * ld * 4, (64,)) for r in range(rows)])
    ref = (codes.astype(np.float64) @ w.astype(np.float64).T) * be.get(ds, (rows,)).astype(np.float64)[:, None] * np.float64(sw[0])
    assert np.all(np.abs(out - ref) <= 3.01 * U * np.abs(ref))


def test_the_largest_number_of_rows(be):
    """2^31 - 1 rows of one column: every row is its own largest value."""
    rows = 2 ** 31 - 1
    dx, dq, ds = filled(be, rows * 4, 0x3F), filled(be, rows + 1, 0x55), filled(be, rows * 4, 0xFF)
    last = np.array([-2.0, 0.0, 1e30], np.float32)
    assert be.lib.bmc_upload(be.ctx, dx + (rows - 3) * 4, last.ctypes.data, 12) == 0
    assert be.lib.bmc_quantize_rows_q8(be.ctx, BMC_F32, dq, 1, ds, dx, 1, rows, 1) == 0
    assert be.lib.bmc_sync(be.ctx) == 0
    assert list(be.get(dq + rows - 4, (5,), np_dtype=np.int8)) == [127, -127, 0, 127, 0x55]
    value = np.frombuffer(b"\x3f" * 4, np.float32).astype(np.float64)[0]
    ref = np.array([value, 2.0, 0.0, 1e30]) / 127.0
    assert np.all(np.abs(be.get(ds + (rows - 4) * 4, (4,)) - ref) <= 2 * U * ref)
    for first in (0, 2 ** 30 - 2, 2 ** 30 + 12345):
        assert np.all(be.get(dq + first, (4,), np_dtype=np.int8) == 127)
        assert np.all(np.abs(be.get(ds + first * 4, (4,)) - value / 127.0) <= 2 * U * value / 127.0)

# ---- together --------------------------------------------------------------------------------------------------------------------------
def mlp_inputs(rows, D, H, key=1):
    rng = rng_of(rows, D, H, key)
    x, a = values(rng, rows, D, BMC_F32), values(rng, rows, D, BMC_BF16, 0.3)
    w = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    wgu, wdn = (rng.standard_normal((2 * H, D)) * D ** -0.5).astype(np.float32), (rng.standard_normal((D, H)) * H ** -0.5).astype(np.float32)
    return x, a, w, wgu, wdn


class Mlp:
    """norm with the residual's addition -> gate | up product -> SwiGLU -> down product with the residual, weights quantised on the device."""

    def __init__(self, be, rows, D, H, key=1):
        self.be, self.rows, self.D, self.H = be, rows, D, H
        self.host = x, a, w, wgu, wdn = mlp_inputs(rows, D, H, key)
        self.x, self.a, self.w = be.put(x), be.put(a, BMC_BF16), be.put(w)
        self.gu_q, self.gu_s, self.dn_q, self.dn_s = be.alloc(2 * H * D), be.alloc(8 * H), be.alloc(D * H), be.alloc(4 * D)
        for src, q, s, oc, c in ((be.put(wgu), self.gu_q, self.gu_s, 2 * H, D), (be.put(wdn), self.dn_q, self.dn_s, D, H)):
            assert be.lib.bmc_quantize_rows_q8(be.ctx, BMC_F32, q, c, s, src, c, oc, c) == 0
        self.q, self.s, self.sum = be.alloc(rows * D), be.alloc(rows * 4), be.alloc(rows * D * 4)
        self.gu, self.hq, self.hs, self.out = be.alloc(rows * 4 * H), be.alloc(rows * H), be.alloc(rows * 4), be.alloc(rows * D * 4)

    def run(self):
        lib, ctx, n, D, H = self.be.lib, self.be.ctx, self.rows, self.D, self.H
        assert lib.bmc_rmsnorm_q8(ctx, BMC_F32, self.q, D, self.s, self.sum, D, self.x, D, BMC_BF16, self.a, D, self.w, n, D, 1e-5) == 0
        assert lib.bmc_matmul_q8(ctx, BMC_BF16, self.gu, 2 * H, self.q, D, self.s, self.gu_q, self.gu_s, None, 0, n, D, 2 * H) == 0
        assert lib.bmc_swiglu_q8(ctx, BMC_BF16, self.hq, H, self.hs, self.gu, self.gu + 2 * H, 2 * H, n, H) == 0
        assert lib.bmc_matmul_q8(ctx, BMC_F32, self.out, D, self.hq, H, self.hs, self.dn_q, self.dn_s, self.sum, D, n, H, D) == 0

    def reference(self):
        def to8(v):
            s = np.abs(v).max(1, keepdims=True) / 127
            return np.rint(v / s) * s
        x, a, w, wgu, wdn = (h.astype(np.float64) for h in self.host)
        s, v = norm_ref(x, a, w, 1e-5)
        gu = to8(v) @ to8(wgu).T
        g, u = gu[:, :self.H], gu[:, self.H:]
        return s, s + to8(g / (1 + np.exp(-g)) * u) @ to8(wdn).T


@pytest.mark.parametrize("rows", [1, 5, 64, 333])
def test_gated_mlp_of_8_bit_products(be, rows):
    """The four operators in a row: each stage against its definition on what the stage before it left on the device, to that stage's own bound,
    and the whole chain against a chain in 64 bits. The latter's bound, on a row's 2-norm relative to the branch: gate | up are stored in bf16
    (2^-8, about 2^-9 in the mean, each), so v is off by d = 0.25 % of its size; a code then falls on the other side of a tie with probability
    d / step and moves by a step, which makes sqrt(step * d) = sqrt(0.1 * 0.0025) = 1.6 % where the row's largest value is 12 times the mean
    size (step = 12 / 127). A tie that falls the other way in the first norm moves gate | up by one step of x in about sqrt(15) * 60 steps
    (fifteen channels of 960 hold most of the row), 0.4 %, and so v's codes by sqrt(0.1 * 0.004) = 2 %. 5 % bounds their sum."""
    D, H = 960, 2560
    m = Mlp(be, rows, D, H)
    m.run()
    _, _, w, _, _ = m.host
    s, v = norm_ref(m.host[0], m.host[1], w, 1e-5)
    total = be.get(m.sum, (rows, D))
    assert np.all(np.abs(total - s) <= U * np.abs(s))
    q, qs = be.get(m.q, (rows, D), np_dtype=np.int8), be.get(m.s, (rows,))
    check_codes(q, qs, v, (D / 64 + 20) * U)
    gu = be.get(m.gu, (rows, 2 * H), BMC_BF16)
    exact = (q.astype(np.float64) @ be.get(m.gu_q, (2 * H, D), np_dtype=np.int8).T.astype(np.float64)) * np.outer(qs, be.get(m.gu_s, (2 * H,))).astype(np.float64)
    assert np.all(np.abs(gu - exact) <= (4 * U + 1.001 * 2.0 ** -8) * np.abs(exact))
    hq, hs = be.get(m.hq, (rows, H), np_dtype=np.int8), be.get(m.hs, (rows,))
    g, u = gu[:, :H].astype(np.float64), gu[:, H:].astype(np.float64)
    check_codes(hq, hs, g / (1 + np.exp(-g)) * u, (2 * np.abs(g) + 12) * U)
    branch = (hq.astype(np.float64) @ be.get(m.dn_q, (D, H), np_dtype=np.int8).T.astype(np.float64)) * np.outer(hs, be.get(m.dn_s, (D,))).astype(np.float64)
    out = be.get(m.out, (rows, D))
    assert np.all(np.abs(out - (total + branch)) <= 4 * U * np.abs(branch) + 1.01 * U * np.abs(total + branch))
    s, ref = m.reference()
    assert np.all(np.linalg.norm(out - ref, axis=1) <= 0.05 * np.linalg.norm(ref - s, axis=1))
    first = be.get(m.out, (rows, 960))
    m.run()
    assert np.array_equal(be.get(m.out, (rows, 960)), first)   # nothing in the chain depends on an order that changes


def test_two_captured_chains_and_an_eager_one(be):
    """Two chains captured into the context's two graphs, replayed in turn on changed inputs, with an eager chain between them."""
    chains = [Mlp(be, 40, 576, 1536, key=k) for k in (1, 2, 3)]
    for m in chains:
        m.run()
    want = [be.get(m.out, (m.rows, m.D)) for m in chains]
    for slot in (0, 1):
        assert be.lib.bmc_graph_select(C.c_void_p(be.ctx), slot) == 0
        assert be.lib.bmc_graph_begin(C.c_void_p(be.ctx)) == 0
        chains[slot].run()
        assert be.lib.bmc_graph_end(C.c_void_p(be.ctx)) == 0
    twice = []
    for scale in (1.0, 0.5):
        for m in chains:
            x = (m.host[0] * np.float32(scale)).astype(np.float32)
            assert be.lib.bmc_upload(be.ctx, m.x, x.ctypes.data, x.nbytes) == 0
            assert be.lib.bmc_memset(be.ctx, m.out, 0xFF, m.rows * m.D * 4) == 0 and be.lib.bmc_sync(be.ctx) == 0
        for slot in (0, 1):
            be.lib.bmc_graph_select(C.c_void_p(be.ctx), slot)
            assert be.lib.bmc_graph_launch(C.c_void_p(be.ctx)) == 0
            if slot == 0:
                chains[2].run()
        twice.append([be.get(m.out, (m.rows, m.D)) for m in chains])
    for got, w in zip(twice[0], want):
        assert np.array_equal(got, w)
    for m, got in zip(chains, twice[1]):
        m.run()
        assert np.array_equal(be.get(m.out, (m.rows, m.D)), got)


def test_side_stream(be):
    """On the context's second stream, beside work of the same operators on the first."""
    a, b = Mlp(be, 300, 576, 1536, key=4), Mlp(be, 7, 576, 1536, key=5)
    a.run(), b.run()
    want = [be.get(m.out, (m.rows, m.D)) for m in (a, b)]
    for m in (a, b):
        assert be.lib.bmc_memset(be.ctx, m.out, 0xFF, m.rows * m.D * 4) == 0
    ctx = C.c_void_p(be.ctx)
    assert be.lib.bmc_side_begin(ctx) == 0
    b.run()
    ticket = be.lib.bmc_side_end(ctx)
    a.run()
    assert ticket >= 0 and be.lib.bmc_side_wait(ctx, ticket) == 0
    for m, w in zip((a, b), want):
        assert np.array_equal(be.get(m.out, (m.rows, m.D)), w)


FIRST_USE_IN_A_CAPTURE = """
import ctypes as C, sys
import numpy as np
sys.path.insert(0, "bare.metal_b200"); sys.path.insert(0, "tests")
import bmapi, bmcapi, test_gpu_q8_ops as t
be = bmcapi.Backend(bmapi.load_product())
rng = np.random.default_rng(1)
ctx = C.c_void_p(be.ctx)
todo = []
for M, K, N in ((1, 960, 200), (24, 2560, 130), (600, 960, 1600), (5000, 2048, 1600)):
    q, w = rng.integers(-128, 128, (M, K)).astype(np.int8), rng.integers(-128, 128, (N, K)).astype(np.int8)
    dq, dw, ds, dn, out = t.put_bytes(be, q), t.put_bytes(be, w), be.put(np.full(M, 0.5, np.float32)), be.put(np.full(N, 0.25, np.float32)), be.alloc(M * N * 4)
    todo.append((M, K, N, q, w, dq, dw, ds, dn, out))
x = rng.standard_normal((40, 960)).astype(np.float32)
dx, cq, cs = be.put(x), be.alloc(40 * 960), be.alloc(160)
assert be.lib.bmc_graph_begin(ctx) == 0
for M, K, N, q, w, dq, dw, ds, dn, out in todo:
    assert be.lib.bmc_matmul_q8(be.ctx, 0, out, N, dq, K, ds, dw, dn, None, 0, M, K, N) == 0
assert be.lib.bmc_quantize_rows_q8(be.ctx, 0, cq, 960, cs, dx, 960, 40, 960) == 0
assert be.lib.bmc_graph_end(ctx) == 0
for _ in range(2):
    assert be.lib.bmc_graph_launch(ctx) == 0
assert be.lib.bmc_sync(be.ctx) == 0
for M, K, N, q, w, dq, dw, ds, dn, out in todo:
    got = be.get(out, (M, N))
    want = (q.astype(np.float64) @ w.astype(np.float64).T) * 0.125
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * np.abs(want)), (M, K, N)
t.check_codes(be.get(cq, (40, 960), np_dtype=np.int8), be.get(cs, (40,)), x.astype(np.float64), 0.0)
"""


def test_first_use_in_a_capture():
    """A process whose first call of every kernel is being captured."""
    r = subprocess.run([sys.executable, "-c", FIRST_USE_IN_A_CAPTURE], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


FIRST_USE_BY_THREADS = """
import sys, threading
import numpy as np
sys.path.insert(0, "bare.metal_b200"); sys.path.insert(0, "tests")
import bmapi, bmcapi, test_gpu_q8_ops as t
lib = bmapi.load_product()
backends = [bmcapi.Backend(lib) for _ in range(4)]
rng = np.random.default_rng(2)
shapes = ((24, 2560, 130), (600, 960, 1600), (5000, 2048, 1600), (3, 960, 200))
q = {K: rng.integers(-128, 128, (5000, K)).astype(np.int8) for K in (960, 2048, 2560)}
w = {K: rng.integers(-128, 128, (1600, K)).astype(np.int8) for K in q}
x = rng.standard_normal((3, 20000)).astype(np.float32)
got, failed, gate = {}, [], threading.Barrier(4)
def work(i):
    try:
        be = backends[i]
        dq, dw = {K: t.put_bytes(be, q[K]) for K in q}, {K: t.put_bytes(be, w[K]) for K in w}
        ds, dn = be.put(np.full(5000, 0.5, np.float32)), be.put(np.full(1600, 0.25, np.float32))
        outs = [be.alloc(M * N * 4) for M, K, N in shapes]
        dx, cq, cs = be.put(x), be.alloc(x.size), be.alloc(12)
        gate.wait()
        for _ in range(8):
            for (M, K, N), out in zip(shapes, outs):
                assert lib.bmc_matmul_q8(be.ctx, 0, out, N, dq[K], K, ds, dw[K], dn, None, 0, M, K, N) == 0
            assert lib.bmc_quantize_rows_q8(be.ctx, 0, cq, 20000, cs, dx, 20000, 3, 20000) == 0
        assert lib.bmc_sync(be.ctx) == 0
        got[i] = [be.get(out, (M, N)) for (M, K, N), out in zip(shapes, outs)] + [be.get(cq, x.shape, np_dtype=np.int8), be.get(cs, (3,))]
    except BaseException as e:
        failed.append(e)
        gate.abort()
threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
[th.start() for th in threads]
[th.join() for th in threads]
assert not failed, failed
for r in got.values():
    for (M, K, N), out in zip(shapes, r):
        want = (q[K][:M].astype(np.float64) @ w[K][:N].astype(np.float64).T) * 0.125
        assert np.all(np.abs(out - want) <= 2.0 ** -24 * np.abs(want)), (M, K, N)
    t.check_codes(r[4], r[5], x.astype(np.float64), 0.0)
"""


def test_first_use_by_threads_with_contexts_of_their_own():
    """Four threads whose first calls meet, each on its own context's stream: every plan of the product beside the others."""
    r = subprocess.run([sys.executable, "-c", FIRST_USE_BY_THREADS], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
