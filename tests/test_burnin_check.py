"""The comparison of a diagnostic's sampled outputs with the host's: one wrong sample is enough, wherever it comes."""
import ctypes
import math

import numpy as np
import pytest

from kubernetes_amd.deviceplugin.burnin import BurnIn, BurnInResult
from kubernetes_amd.ops import hip_kernels as hk

SIZE = 96
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def lib():
    try:
        return hk.load()
    except hk.HIPError:
        pytest.skip("the library is not built")


def row(seed):
    """bf16 bits of SIZE values, their codes and scales, and what these stand for."""
    r = np.random.default_rng(seed)
    x = ((r.uniform(-1, 1, SIZE) * 2.0 ** r.integers(-3, 3, SIZE)).astype(np.float32).view(np.uint32) & 0xFFFF0000).view(np.float32)
    x[32:64] = 0
    x[33] = -0.0
    blocks = x.astype(np.float64).reshape(-1, 32)
    top = np.abs(blocks).max(1)
    s = np.where(top > 0, np.frexp(top)[1] - 1 - 2 + 127, 0).astype(np.uint8)
    w = np.abs(blocks) / 2.0 ** (s.astype(float) - 127)[:, None]
    grid = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
    d = np.abs(np.minimum(w, 6)[:, :, None] - grid)
    near = d == d.min(2, keepdims=True)
    code = np.where(near[:, :, ::2].any(2), 2 * near[:, :, ::2].argmax(2), 2 * near[:, :, 1::2].argmax(2) + 1)
    value = np.where(np.signbit(blocks), -1, 1) * grid[code] * 2.0 ** (s.astype(float) - 127)[:, None]
    code = (code + 8 * np.signbit(blocks)).astype(np.uint8).reshape(-1)
    return (x.view(np.uint32) >> 16).astype(np.uint16), code[::2] | code[1::2] << 4, s, value.reshape(-1)


def sample(lib, a, b, got, worst, size=SIZE):
    args = [v.ctypes.data_as(ctypes.c_void_p) for v in (*a[:3], *b[:3])]
    assert lib.kamd_diag_mfma_fp4_sample(*args, size, got, ctypes.byref(worst)) == 0


def wrong(kind, a, b, got):
    """A sample with something wrong, and the least error that it has to give."""
    x, q, s, v = (m.copy() for m in a)
    if kind == "nan":
        return a, b, NAN, INF
    if kind == "infinity":
        return a, b, -INF, INF
    if kind == "value":
        return a, b, got + 100.0, 0.1
    if kind == "code":
        q[5] ^= 0x10
    elif kind == "sign of zero":
        q[16] ^= 0x80
    elif kind == "scale":
        s[2] += 1
    elif kind == "scale of NaN":
        s[0] = 255
        return (x, q, s, v), b, got, INF
    elif kind == "input that is not finite":
        x[3] = 0x7F80
    return (x, q, s, v), b, got, 1.0


KINDS = ["nan", "infinity", "value", "code", "sign of zero", "scale", "scale of NaN", "input that is not finite"]


def test_right_samples_pass(lib):
    worst = ctypes.c_double(0)
    for seed in range(20):
        a, b = row(seed), row(100 + seed)
        sample(lib, a, b, float(a[3] @ b[3]), worst)
        sample(lib, b, a, float(a[3] @ b[3]), worst)
    # the output is rounded to 32 bits once
    assert worst.value <= 2.0 ** -24


@pytest.mark.parametrize("at", [0, 4, 8])
@pytest.mark.parametrize("kind", KINDS)
def test_one_wrong_sample_stays(lib, kind, at):
    worst = ctypes.c_double(0)
    for seed in range(9):
        a, b = row(seed), row(100 + seed)
        got, least = float(a[3] @ b[3]), 0.0
        if seed == at:
            a, b, got, least = wrong(kind, a, b, got)
        before = worst.value
        sample(lib, a, b, got, worst)
        assert worst.value >= max(before, least)
    r = BurnInResult(ok=False, tflops=1400.0, hbm_gbps=6000.0, fp8_tflops=2800.0, fp4_tflops=4000.0, fp4_rel_err=worst.value)
    assert "relative error" in BurnIn(min_fp4_tflops=2000.0).judge(r)


@pytest.mark.parametrize("kinds", [("code", "nan", "value"), ("nan", "code"), ("scale", "value", "nan"), ("nan", "nan")])
def test_wrong_samples_do_not_hide_each_other(lib, kinds):
    worst = ctypes.c_double(0)
    for seed, kind in enumerate(kinds):
        a, b = row(seed), row(100 + seed)
        a, b, got, _ = wrong(kind, a, b, float(a[3] @ b[3]))
        sample(lib, a, b, got, worst)
    a, b = row(50), row(51)
    sample(lib, a, b, float(a[3] @ b[3]), worst)
    assert worst.value == INF and not math.isnan(worst.value)


def test_sample_refuses_sizes(lib):
    a, b = row(1), row(2)
    args = [v.ctypes.data_as(ctypes.c_void_p) for v in (*a[:3], *b[:3])]
    worst = ctypes.c_double(0)
    for size in (0, -32, 31, 33):
        assert lib.kamd_diag_mfma_fp4_sample(*args, size, 0.0, ctypes.byref(worst)) == -1
    assert lib.kamd_diag_mfma_fp4_sample(None, *args[1:], SIZE, 0.0, ctypes.byref(worst)) == -1 and worst.value == 0


# ---------------------------------------------------------------------------
# the bf16 and fp8 products and vector_add

def wide_row(seed, fp8):
    """Bits of SIZE values and the values."""
    r = np.random.default_rng(seed)
    if fp8:   # e4m3: the codes of 1.0 to 1.875 and their negatives
        bits = (0x38 + r.integers(0, 8, SIZE) + 0x80 * r.integers(0, 2, SIZE)).astype(np.uint8)
        return bits, (1 + (bits & 7) / 8.0) * np.where(bits & 0x80, -1, 1)
    bits = (r.uniform(-1, 1, SIZE).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    return bits, (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


@pytest.mark.parametrize("at", [0, 4, 8, None])
@pytest.mark.parametrize("wrong_output", [NAN, INF, -INF, 1e6])
@pytest.mark.parametrize("fp8", [0, 1])
def test_wide_sample(lib, fp8, wrong_output, at):
    worst = ctypes.c_double(0)
    for seed in range(9):
        (a, va), (b, vb) = wide_row(seed, fp8), wide_row(100 + seed, fp8)
        got = wrong_output if seed == at else float(va @ vb)
        lib.kamd_diag_mfma_sample(a.ctypes.data_as(ctypes.c_void_p), b.ctypes.data_as(ctypes.c_void_p), SIZE, fp8, got,
                                  ctypes.byref(worst))
    if at is None:
        assert worst.value <= 2.0 ** -24
    else:
        assert worst.value == INF if wrong_output != 1e6 else 1e3 < worst.value < 1e6
        r = BurnInResult(ok=False, tflops=1400.0, hbm_gbps=6000.0, fp8_tflops=2800.0)
        r.mfma_rel_err, r.fp8_rel_err = (0.0, worst.value) if fp8 else (worst.value, 0.0)
        assert "relative error" in BurnIn().judge(r)


@pytest.mark.parametrize("at", [0, 500, 999, None])
@pytest.mark.parametrize("wrong_output", [NAN, INF, 1e6])
def test_vector_add_error(lib, wrong_output, at):
    r = np.random.default_rng(1)
    a, b = r.uniform(0, 1, 1000).astype(np.float32), r.uniform(0, 1, 1000).astype(np.float32)
    c = a + b
    if at is not None:
        c[at] = wrong_output
    got = lib.kamd_diag_vector_add_error(*(v.ctypes.data_as(ctypes.c_void_p) for v in (a, b, c)), 1000)
    if at is None:
        assert got == 0
    else:
        assert got == INF if wrong_output != 1e6 else got > 1e5
        assert "vector_add" in BurnIn().judge(BurnInResult(ok=False, vadd_err=got, tflops=1400.0, hbm_gbps=6000.0, fp8_tflops=2800.0))
