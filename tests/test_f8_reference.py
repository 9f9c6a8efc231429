"""The 8-bit tests' own reference, on the CPU: the formats against published values, the encoder against every code and tie,
and what the library's 8-bit entry points answer before it is initialised."""
import ctypes

import numpy as np
import pytest

import f8_reference as ref
from backup_1_amd import capi


def test_formats_hold_the_published_values():
    # OCP 8-bit floating point specification: largest, smallest normal, smallest subnormal
    t = ref.TABLE[capi.E4M3]
    assert t[0x7E] == 448 and t[0x08] == 2.0 ** -6 and t[0x01] == 2.0 ** -9 and np.isnan(t[0x7F]) and np.isnan(t[0xFF]) and t[0xBC] == -1.5
    t = ref.TABLE[capi.E5M2]
    assert t[0x7B] == 57344 and t[0x04] == 2.0 ** -14 and t[0x01] == 2.0 ** -16 and np.isinf(t[0x7C]) and np.isnan(t[0x7D]) and t[0xBE] == -1.5


@pytest.mark.parametrize("fmt", [capi.E4M3, capi.E5M2])
def test_encoder(fmt):
    t = ref.TABLE[fmt]
    codes = np.flatnonzero(np.isfinite(t)).astype(np.uint8)
    assert np.array_equal(ref.encode(t[codes], fmt), codes)
    grid = t[:128][np.isfinite(t[:128])]
    mid = (grid[1:] + grid[:-1]) / 2
    tie = ref.encode(mid, fmt)
    assert np.all(tie % 2 == 0) and np.all(np.abs(tie.astype(int) - np.arange(mid.size) - 0.5) == 0.5)
    assert np.array_equal(ref.encode(np.nextafter(mid, 0), fmt), np.arange(mid.size))
    assert np.array_equal(ref.encode(-np.nextafter(mid, np.inf), fmt), (np.arange(mid.size) + 1) | 0x80)


@pytest.mark.parametrize("fmt", [capi.E4M3, capi.E5M2])
@pytest.mark.parametrize("scale", [capi.SCALE_F32, capi.SCALE_E8M0])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantisation_is_within_half_a_step(fmt, scale, block_rows):
    x = np.random.RandomState(1).randn(150, 300).astype(np.float32)
    codes, s = ref.quantize(x, fmt, scale, block_rows)
    back = ref.dequantize(codes, fmt, s, block_rows)
    full = ref.spread(ref.scale_values(s), 150, 300, block_rows)
    half, tiny = (2.0 ** -4, 2.0 ** -10) if fmt == capi.E4M3 else (2.0 ** -3, 2.0 ** -17)
    assert np.all(np.abs(back - x) <= np.maximum(np.abs(x) * half, tiny * full) * (1 + 1e-6))
    assert np.nanmax(np.abs(ref.TABLE[fmt][codes])) <= ref.LARGEST[fmt] * 1.0
    if scale == capi.SCALE_F32:
        assert np.abs(ref.TABLE[fmt][codes]).max() == ref.LARGEST[fmt]


def test_entry_points_refuse_before_init():
    import torch  # noqa: F401
    L = capi.lib()
    if L.decx_hip_is_init():
        pytest.skip("library already initialised in this process")
    for end in ("", "_async"):
        assert getattr(L, "decx_hip_f8_quantize" + end)(None, 8, 0, 1, 8, 1, 0, 0, None, 8, None, 8, None, 0, None, 0) == 0x01
        assert getattr(L, "decx_hip_f8gemm" + end)(None, 8, 0, None, 8, None, 8, 0, None, 8, 1, 0, None, 0, None, 8, 0, 8, 8, 8) == 0x01
        assert getattr(L, "decx_hip_rmsnorm_f8" + end)(None, 8, None, 0, None, 0.0, 0, 1, 8, None, 0, None, None, 0, None, 0, None, 0, 0, 0) == 0x01
        assert getattr(L, "decx_hip_rmsnorm_backward" + end)(None, 8, None, None, None, 8, None, 0, 0, 1, 8, None, 8, None, None, 0) == 0x01
        assert "initialized first" in capi.last_error()


def test_packed_calls_refuse_like_the_others():
    L = capi.lib()
    if L.decx_hip_is_init():
        pytest.skip("library already initialised in this process")
    words = (ctypes.c_int64 * 20)()
    for call in range(4):
        assert L.decx_hip_f8_call(call, ctypes.addressof(words), 0) == 0x01 and L.decx_hip_f8_call(call, ctypes.addressof(words), 1) == 0x01
    assert L.decx_hip_f8_call(4, ctypes.addressof(words), 0) == 0x0b and L.decx_hip_f8_call(0, None, 0) == 0x0d
    with pytest.raises(capi.DecxHipError):
        capi.f8gemm(16, 8, 0, 16, 8, 16, 8, 0, 16, 8, 1, 0, 16, 8, 0, 1, 1, 1)


def test_workspace_query_is_host_only():
    assert capi.rmsnorm_backward_workspace(1, 100) == 400
    assert capi.rmsnorm_backward_workspace(0, 100) == 0 and capi.rmsnorm_backward_workspace(5, -1) == 0
    for M in (1, 2, 100, 511, 512, 513, 5000, 100000):
        need = capi.rmsnorm_backward_workspace(M, 8192)
        assert 0 < need <= min(M, 512) * 8192 * 4 and need % (8192 * 4) == 0
