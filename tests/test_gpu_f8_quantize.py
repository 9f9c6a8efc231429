"""decx_hip_f8_quantize: codes and scales are defined bit for bit, so everything here is compared for equality."""
import numpy as np
import pytest

import f8_reference as ref
from backup_1_amd import capi, workloads
from f8_reference import Pitched

pytestmark = pytest.mark.gpu
TYPES = (capi.F32, capi.F16, capi.BF16)


def values(M, K, kind, seed):
    x = workloads.normal((M, K), seed).astype(np.float32)
    x[:, ::7] *= 30.0
    x[:, ::11] *= 1e-3
    return ref.to_type(x, kind)


def run(x, kind, fmt, scale, block_rows, both=True, rows=True, pitch=(0, 0, 0), lead=(0, 0, 0)):
    """(codes, scales, codes of the transpose, its scales); pitches and offsets of X, the codes, the scales"""
    M, K = x.shape
    kb, mb = -(-K // 128), -(-M // 128)
    st = np.float32 if scale == capi.SCALE_F32 else np.uint8
    dx = Pitched(x, K + pitch[0], lead[0])
    q = Pitched.empty(M, K, np.uint8, pitch=K + pitch[1], lead=lead[1]) if rows else None
    s = Pitched.empty(kb, M if block_rows == 1 else mb, st, pitch=(M if block_rows == 1 else mb) + pitch[2], lead=lead[2]) if rows else None
    qt = Pitched.empty(K, M, np.uint8, pitch=M + pitch[1], lead=lead[1]) if both else None
    t = Pitched.empty(mb, K if block_rows == 1 else kb, st, pitch=(K if block_rows == 1 else kb) + pitch[2], lead=lead[2]) if both else None
    p = lambda b: (b.ptr, b.ld) if b is not None else (None, 0)  # noqa: E731
    capi.f8_quantize(dx.ptr, dx.ld, kind, M, K, block_rows, fmt, scale, *p(q), *p(s), *p(qt), *p(t))
    dx.result()
    return [b.result() if b is not None else None for b in (q, s, qt, t)]


def check(x, kind, fmt, scale, block_rows, got):
    v = ref.from_type(x, kind)
    for (codes, scales), w in ((got[:2], v), (got[2:], v.T)):
        if codes is None:
            continue
        want_codes, want_scales = ref.quantize(w, fmt, scale, block_rows)
        assert np.array_equal(scales, want_scales)
        assert np.array_equal(codes, want_codes)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: ref.TYPE_NAMES[k])
@pytest.mark.parametrize("fmt,scale", [(capi.E4M3, capi.SCALE_F32), (capi.E4M3, capi.SCALE_E8M0), (capi.E5M2, capi.SCALE_F32), (capi.E5M2, capi.SCALE_E8M0)])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("both", [False, True])
def test_every_kind(gpu, kind, fmt, scale, block_rows, both):
    x = values(150, 300, kind, 3)
    check(x, kind, fmt, scale, block_rows, run(x, kind, fmt, scale, block_rows, both))


@pytest.mark.parametrize("M,K", [(1, 1), (1, 7), (1, 128), (1, 129), (1, 4096), (2, 1000), (15, 127), (16, 512), (17, 513), (127, 128), (128, 129),
                                 (129, 255), (300, 8), (1000, 1), (513, 1030)])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("both", [False, True])
def test_sizes(gpu, M, K, block_rows, both):
    x = values(M, K, capi.BF16, M + K)
    check(x, capi.BF16, capi.E4M3, capi.SCALE_F32, block_rows, run(x, capi.BF16, capi.E4M3, capi.SCALE_F32, block_rows, both))


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: ref.TYPE_NAMES[k])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_any_pitch_and_alignment(gpu, kind, block_rows):
    x = values(140, 270, kind, 8)
    for pitch, lead in (((1, 3, 5), (1, 1, 1)), ((2, 13, 2), (3, 5, 7)), ((242, 16, 0), (8, 16, 4))):
        check(x, kind, capi.E4M3, capi.SCALE_E8M0, block_rows, run(x, kind, capi.E4M3, capi.SCALE_E8M0, block_rows, True, True, pitch, lead))


def test_transpose_alone(gpu):
    x = values(200, 333, capi.F16, 4)
    for block_rows in (1, 128):
        got = run(x, capi.F16, capi.E5M2, capi.SCALE_F32, block_rows, True, rows=False)
        check(x, capi.F16, capi.E5M2, capi.SCALE_F32, block_rows, got)


@pytest.mark.parametrize("scale", [capi.SCALE_F32, capi.SCALE_E8M0])
@pytest.mark.parametrize("fmt", [capi.E4M3, capi.E5M2])
def test_borders_of_the_scale_and_of_the_grid(gpu, fmt, scale):
    """Blocks whose largest value is exactly, just below and just above a power of two times the format's largest; values on
    the ties of the grid, below its smallest step, signed zeros; blocks of zeros and of values below 2^-100; the largest and
    the smallest fp32."""
    top = np.float32(ref.LARGEST[fmt])
    x = np.zeros((12, 128), np.float32)
    for i, p in enumerate((-60, 0, 100 if fmt == capi.E4M3 else 90)):
        a = np.float32(top * 2.0 ** p)
        x[3 * i, :3] = a, -a / 3, a / 7
        x[3 * i + 1, :3] = np.nextafter(a, np.float32(0)), a / 5, 0
        x[3 * i + 2, :3] = np.nextafter(a, np.float32(np.inf)), a / 5, -0.0
    grid = ref.TABLE[fmt][:120].astype(np.float32)
    x[9, 0] = top
    x[9, 1:120] = (grid[1:] + grid[:-1]) / 2 * np.where(np.arange(119) % 2, 1, -1)          # every tie
    x[9, 120:124] = grid[1] / 2, grid[1] / 2 * 1.001, -grid[1] / 2, grid[1] / 4
    x[10, :4] = 1e-45, -1e-38, 2.0 ** -101, -0.0
    x[11, :3] = 3.4028235e38, -3.4028235e38, 1e-45
    check(x, capi.F32, fmt, scale, 1, run(x, capi.F32, fmt, scale, 1))
    check(np.zeros((130, 130), np.float32), capi.F32, fmt, scale, 128, run(np.zeros((130, 130), np.float32), capi.F32, fmt, scale, 128))


@pytest.mark.parametrize("scale", [capi.SCALE_F32, capi.SCALE_E8M0])
@pytest.mark.parametrize("fmt", [capi.E4M3, capi.E5M2])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_nan_and_infinity_stay_in_their_block(gpu, fmt, scale, block_rows):
    x = values(200, 400, capi.F32, 9)
    x[3, 140], x[150, 300] = np.nan, -np.inf
    q, s, qt, t = run(x, capi.F32, fmt, scale, block_rows)
    clean = np.where(np.isfinite(x), x, 0.0).astype(np.float32)
    for codes, scales, w, c in ((q, s, x, clean), (qt, t, x.T, clean.T)):
        bad = ref.spread(block_amax_bad(w, block_rows), w.shape[0], w.shape[1], block_rows)
        with np.errstate(invalid="ignore"):
            v = ref.TABLE[fmt][codes] * ref.spread(ref.scale_values(scales), w.shape[0], w.shape[1], block_rows)
        assert np.all(np.isnan(v[bad]) | np.isinf(v[bad])), "a finite value out of a block with NaN or infinity"
        assert np.all(np.isnan(v[~np.isfinite(w)]))
        want = ref.dequantize(*ref.quantize(c, fmt, scale, block_rows)[:1], fmt, ref.quantize(c, fmt, scale, block_rows)[1], block_rows)
        assert np.array_equal(v[~bad], want[~bad])


def block_amax_bad(x, block_rows):
    return ref.block_amax(np.where(np.isfinite(x), 0.0, 1.0), block_rows).T > 0


def test_same_bits_again(gpu):
    x = values(300, 1000, capi.BF16, 2)
    a, b = (run(x, capi.BF16, capi.E4M3, capi.SCALE_F32, 1) for _ in range(2))
    assert all(np.array_equal(p, q) for p, q in zip(a, b))


def test_refusals(gpu):
    L = capi.lib()
    d = capi.DeviceBuffer(1 << 16)
    ok = [d.ptr, 64, capi.F32, 32, 64, 1, capi.E4M3, capi.SCALE_F32, d.ptr + 16384, 64, d.ptr + 32768, 32, None, 0, None, 0]

    def refused(code, **change):
        names = ["X", "ldx", "type", "M", "K", "block_rows", "format", "scale", "Q", "ldq", "S", "lds", "Qt", "ldqt", "St", "ldst"]
        args = [change.get(n, v) for n, v in zip(names, ok)]
        assert L.decx_hip_f8_quantize(*args) == code and capi.last_error().strip(), change

    assert L.decx_hip_f8_quantize(*ok) == 0
    refused(0x0d, X=None)
    refused(0x0d, Q=None)
    refused(0x0d, S=None)
    refused(0x0d, Qt=d.ptr + 40000, ldqt=32)
    refused(0x03, M=0)
    refused(0x03, K=-1)
    refused(0x0b, type=3)
    refused(0x0b, format=2)
    refused(0x0b, scale=-1)
    refused(0x0d, block_rows=64)
    refused(0x0d, ldx=63)
    refused(0x0d, ldq=63)
    refused(0x0d, lds=31)
    refused(0x0d, Qt=d.ptr + 40000, ldqt=31, St=d.ptr + 50000, ldst=64)
    refused(0x0d, Qt=d.ptr + 40000, ldqt=32, St=d.ptr + 50000, ldst=63)
    refused(0x0d, X=d.ptr + 2)
    refused(0x0d, X=d.ptr + 1, type=capi.F16)
    refused(0x0d, S=d.ptr + 32769)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: ref.TYPE_NAMES[k])
@pytest.mark.parametrize("K", range(1, 18))
def test_each_short_row(gpu, kind, K):
    x = values(9, K, kind, 60 + K)
    for block_rows in (1, 128):
        check(x, kind, capi.E4M3, capi.SCALE_F32, block_rows, run(x, kind, capi.E4M3, capi.SCALE_F32, block_rows, True, True, (3, 1, 0), (1, 1, 0)))
    check(x, kind, capi.E5M2, capi.SCALE_E8M0, 1, run(x, kind, capi.E5M2, capi.SCALE_E8M0, 1, False))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_matrix_larger_than_the_caches(gpu, block_rows):
    """104 MB of fp32, where fewer workgroups share a unit: 5 copies of 1024 rows give 5 copies of their codes and scales."""
    M, K, times = 1024, 5080, 5
    x = values(M, K, capi.F32, 95)
    got = run(np.tile(x, (times, 1)), capi.F32, capi.E4M3, capi.SCALE_F32, block_rows)
    rows = got[1].shape[1] // times
    want = ref.quantize(x, capi.E4M3, capi.SCALE_F32, block_rows)
    assert np.array_equal(got[0], np.tile(want[0], (times, 1))) and np.array_equal(got[1], np.tile(want[1], (1, times))) and rows == want[1].shape[1]
    want = ref.quantize(x.T.copy(), capi.E4M3, capi.SCALE_F32, block_rows)
    assert np.array_equal(got[2], np.tile(want[0], (1, times))) and np.array_equal(got[3], np.tile(want[1], (times, 1)))
