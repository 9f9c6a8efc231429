"""decx_hip_rmsnorm_f8 and decx_hip_rmsnorm_backward against 64-bit arithmetic; the gradient also against differences."""
import numpy as np
import pytest

import f8_reference as ref
from backup_1_amd import capi, workloads
from f8_reference import Pitched

pytestmark = pytest.mark.gpu
TYPES = (capi.F32, capi.F16, capi.BF16)
EPS = 1e-5
# A sum over a row: at most 32 terms in a thread, 6 steps over the lanes, 15 over the waves, a rounding in each product; in
# steps of 2^-24 of the sum of the magnitudes
SUM = 60 * 2.0 ** -24


def inputs(M, K, kind, seed):
    x = workloads.normal((M, K), seed).astype(np.float32)
    x[:, ::13] *= 15.0
    r = workloads.normal((M, K), seed + 1).astype(np.float32) * 2
    w = 1 + 0.2 * workloads.normal((K,), seed + 2).astype(np.float32)
    return [ref.to_type(v, kind) for v in (x, r, w)]


def run(x, r, w, kind, fmt=capi.E4M3, scale=capi.SCALE_F32, eps=EPS, want="HsYQ", inplace=None, pitch=0, lead=0):
    M, K = x.shape
    st = np.float32 if scale == capi.SCALE_F32 else np.uint8
    kw = dict(pitch=K + pitch, lead=lead)
    dx, dw = Pitched(x, **kw), Pitched(w, lead=lead)
    dr = Pitched(r, **kw) if r is not None else None
    H = (dx if inplace == "x" else dr if inplace == "r" else Pitched.empty(M, K, x.dtype, **kw)) if "H" in want else None
    Y = Pitched.empty(M, K, x.dtype, **kw) if "Y" in want else None
    rstd = Pitched.empty(1, M, np.float32) if "s" in want else None
    Q = Pitched.empty(M, K, np.uint8, **kw) if "Q" in want else None
    S = Pitched.empty(-(-K // 128), M, st, pitch=M + pitch, lead=lead) if "Q" in want else None
    p = lambda b: (b.ptr, b.ld) if b is not None else (None, 0)  # noqa: E731
    capi.rmsnorm_f8(dx.ptr, dx.ld, *p(dr), dw.ptr, eps, kind, M, K, *p(H), p(rstd)[0], *p(Y), *p(Q), *p(S), fmt, scale)
    return {n: b.result() if b is not None else None for n, b in (("H", H), ("Y", Y), ("rstd", rstd), ("Q", Q), ("S", S))}


def check(x, r, w, kind, got, fmt=capi.E4M3, scale=capi.SCALE_F32, eps=EPS):
    M, K = x.shape
    h = x
    if r is not None:                                            # fp32 holds the sum of two 16-bit values to one rounding
        h = ref.to_type(ref.from_type(x, kind).astype(np.float32) + ref.from_type(r, kind).astype(np.float32), kind)
    if got["H"] is not None:
        assert np.array_equal(got["H"].view(np.uint8), h.view(np.uint8))
    v = ref.from_type(h, kind)
    rstd = 1 / np.sqrt((v * v).mean(1) + eps)
    if got["rstd"] is not None:                                  # half of the sum's error, then division, addition, root, division
        assert np.all(np.abs(got["rstd"][0] - rstd) <= rstd * (SUM / 2 + 4 * 2.0 ** -24))
    y = v * rstd[:, None] * ref.from_type(w, kind)
    off = np.abs(y) * (SUM / 2 + 6 * 2.0 ** -24)                 # and two products
    if got["Y"] is not None:
        err = np.abs(ref.from_type(got["Y"], kind) - y)
        assert np.all(err <= off + np.abs(y) * ref.HALF_STEP[kind] * 1.001 + (2.0 ** -25 if kind == capi.F16 else 0))
    if got["Q"] is not None:
        s = ref.scale_values(got["S"]).T                         # [row][block]
        amax = np.maximum(ref.block_amax(y, 1), 2.0 ** -100)
        least = amax / ref.LARGEST[fmt]
        if scale == capi.SCALE_F32:
            assert np.all(np.abs(s - least) <= least * (SUM / 2 + 8 * 2.0 ** -24))
        else:                                                    # the least power of two, up to the error of amax at its border
            assert np.all((s >= least * (1 - 1e-5)) & (s < 2 * least * (1 + 1e-5)))
        full = ref.spread(s.T, M, K, 1)
        codes = ref.TABLE[fmt][got["Q"]]
        # half a step of the grid at the value, or half its smallest step, and the errors of y and of 1 / s
        half, tiny = (2.0 ** -4, 2.0 ** -10) if fmt == capi.E4M3 else (2.0 ** -3, 2.0 ** -17)
        assert np.all(np.abs(codes * full - y) <= np.maximum(np.abs(y) * half, tiny * full) * (1 + 1e-5) + off + np.abs(y) * 3 * 2.0 ** -24)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: ref.TYPE_NAMES[k])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 100), (1, 4096), (3, 129), (5, 512), (4, 513), (17, 1500), (9, 2048), (9, 2049), (3, 4097), (3, 8192), (2, 8200),
                                 (2, 16384), (2, 16385), (1, 32768), (300, 384)])
def test_sizes_and_types(gpu, kind, M, K):
    x, r, w = inputs(M, K, kind, M + K)
    check(x, r, w, kind, run(x, r, w, kind))
    check(x, None, w, kind, run(x, None, w, kind))


@pytest.mark.parametrize("fmt", [capi.E4M3, capi.E5M2])
@pytest.mark.parametrize("scale", [capi.SCALE_F32, capi.SCALE_E8M0])
def test_formats_and_scales(gpu, fmt, scale):
    x, r, w = inputs(33, 700, capi.BF16, 4)
    check(x, r, w, capi.BF16, run(x, r, w, capi.BF16, fmt, scale), fmt, scale)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: ref.TYPE_NAMES[k])
def test_pitches_alignment_and_results_left_out(gpu, kind):
    x, r, w = inputs(20, 333, kind, 6)
    for want in ("HsYQ", "H", "s", "Y", "Q", "HQ", "sY"):
        for pitch, lead in ((0, 0), (1, 1), (11, 3), (64, 16)):
            check(x, r, w, kind, run(x, r, w, kind, want=want, pitch=pitch, lead=lead))


def test_sum_written_over_an_input(gpu):
    x, r, w = inputs(30, 900, capi.F16, 7)
    for where in ("x", "r"):
        check(x, r, w, capi.F16, run(x, r, w, capi.F16, inplace=where))


def test_rows_of_zeros_and_rows_that_are_not_finite(gpu):
    x, r, w = inputs(6, 300, capi.F32, 8)
    x[1] = r[1] = 0
    x[2, 299], x[4, 5] = np.nan, np.inf
    got = run(x, r, w, capi.F32)
    good = [0, 1, 3, 5]
    check(x[good], r[good], w, capi.F32, {n: (v[:, good] if n in ("rstd", "S") else v[good]) for n, v in got.items()})
    assert np.isnan(got["rstd"][0, 2]) and got["rstd"][0, 4] == 0
    assert np.all(np.isnan(got["Y"][2])) and np.isnan(got["Y"][4, 5]) and np.all(np.isnan(got["S"][:, 2]))
    zero = run(np.zeros((2, 50), np.float32), None, w[:50], capi.F32, eps=0.0)          # no eps: 0 * infinity
    assert np.all(np.isnan(zero["Y"])) and np.all(np.isinf(zero["rstd"])) and np.all(np.isnan(zero["S"]))


def backward(h, w, rstd, dy, dr, kind, want_dw=True, inplace=None, pitch=0, lead=0):
    M, K = h.shape
    kw = dict(pitch=K + pitch, lead=lead)
    dH, dW, dS, dY = Pitched(h, **kw), Pitched(w, lead=lead), Pitched(rstd), Pitched(dy, **kw)
    dR = Pitched(dr, **kw) if dr is not None else None
    dX = {"h": dH, "y": dY, "r": dR}[inplace] if inplace else Pitched.empty(M, K, h.dtype, **kw)
    need = capi.rmsnorm_backward_workspace(M, K)
    work = Pitched(np.full((1, need), 0xFF, np.uint8))           # NaNs: nothing in it may matter; the guard behind it is checked
    dw = Pitched.empty(1, K, np.float32, lead=lead) if want_dw else None
    capi.rmsnorm_backward(dH.ptr, dH.ld, dW.ptr, dS.ptr, dY.ptr, dY.ld, dR.ptr if dR else None, dR.ld if dR else 0, kind, M, K, dX.ptr, dX.ld,
                          dw.ptr if dw else None, work.ptr if dw else None, need if dw else 0)
    work.result()
    return dX.result(), dw.result()[0] if dw else None


def gradient64(h, w, rstd, dy, dr):
    n = h * rstd[:, None]
    g = dy * w
    dx = rstd[:, None] * (g - n * (g * n).mean(1, keepdims=True)) + dr
    size = rstd[:, None] * (np.abs(g) + np.abs(n) * np.abs(g * n).mean(1, keepdims=True))
    return dx, size, (dy * n).sum(0), np.abs(dy * n).sum(0)


def check_backward(h, w, rstd, dy, dr, kind, got, M):
    dx, dw = got
    f = lambda a: ref.from_type(a, kind)  # noqa: E731
    d = f(dr) if dr is not None else np.zeros(h.shape)
    want, size, want_w, size_w = gradient64(f(h), f(w), rstd.astype(np.float64), f(dy), d)
    err = np.abs(f(dx) - want)
    # the row's sum, and at most 8 roundings of one element's way; the addition of dr; the rounding to the type
    assert np.all(err <= size * (SUM + 8 * 2.0 ** -24) + (size + np.abs(d)) * 2.0 ** -23 + np.abs(want) * ref.HALF_STEP[kind] * 1.001 +
                  (2.0 ** -25 if kind == capi.F16 else 0))
    if dw is not None:                                           # in order: a workgroup's rows, every 16th workgroup, the 16
        assert np.all(np.abs(dw - want_w) <= size_w * (M + 20) * 2.0 ** -24)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: ref.TYPE_NAMES[k])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 300), (7, 129), (33, 512), (600, 513), (1100, 200), (512, 100), (511, 65), (513, 33), (512, 4100), (50, 1500), (20, 2049), (600, 4097), (3, 8200), (5, 16385),
                                 (2, 32768)])
def test_gradient(gpu, kind, M, K):
    h, dy, w = inputs(M, K, kind, M + 2 * K)
    dr = ref.to_type(workloads.normal((M, K), 77), kind)
    rstd = (1 / np.sqrt((ref.from_type(h, kind) ** 2).mean(1) + EPS)).astype(np.float32)
    check_backward(h, w, rstd, dy, dr, kind, backward(h, w, rstd, dy, dr, kind), M)
    check_backward(h, w, rstd, dy, None, kind, backward(h, w, rstd, dy, None, kind, want_dw=False), M)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: ref.TYPE_NAMES[k])
def test_gradient_in_place_and_any_pitch(gpu, kind):
    h, dy, w = inputs(40, 333, kind, 9)
    dr = ref.to_type(workloads.normal((40, 333), 78), kind)
    rstd = (1 / np.sqrt((ref.from_type(h, kind) ** 2).mean(1) + EPS)).astype(np.float32)
    plain = backward(h, w, rstd, dy, dr, kind)
    for where in ("h", "y", "r", None):
        for pitch, lead in ((0, 0), (3, 1), (51, 16)):
            got = backward(h, w, rstd, dy, dr, kind, inplace=where, pitch=pitch, lead=lead)
            # dX bit for bit; dW's parts may be added in another order where dX lies over an input
            assert np.array_equal(got[0].view(np.uint8), plain[0].view(np.uint8))
            check_backward(h, w, rstd, dy, dr, kind, got, 40)


def test_gradient_against_differences(gpu):
    """Of sum(dy * y + dr * h) by each of some inputs and weights: central differences in 64 bits are exact to 1e-7 here."""
    M, K = 4, 70
    x, r, w = [ref.from_type(v, capi.F32) for v in inputs(M, K, capi.F32, 10)]
    dy, dr = workloads.normal((M, K), 11).astype(np.float32), workloads.normal((M, K), 12).astype(np.float32)

    def loss(h, w):
        return float((dy * h / np.sqrt((h * h).mean(1, keepdims=True) + EPS) * w).sum() + (dr * h).sum())

    h = (x + r).astype(np.float32).astype(np.float64)
    rstd = (1 / np.sqrt((h * h).mean(1) + EPS)).astype(np.float32)
    dx, dw = backward(h.astype(np.float32), w.astype(np.float32), rstd, dy, dr, capi.F32)
    step = 1e-4
    for m, k in ((0, 0), (1, 13), (2, 69), (3, 31), (0, 26)):
        e = np.zeros((M, K))
        e[m, k] = step
        assert abs((loss(h + e, w) - loss(h - e, w)) / (2 * step) - dx[m, k]) < 2e-5
    for k in (0, 13, 69):
        e = np.zeros(K)
        e[k] = step
        assert abs((loss(h, w + e) - loss(h, w - e)) / (2 * step) - dw[k]) < 2e-5


def test_same_bits_again(gpu):
    h, dy, w = inputs(700, 1000, capi.BF16, 13)
    rstd = (1 / np.sqrt((ref.from_type(h, capi.BF16) ** 2).mean(1) + EPS)).astype(np.float32)
    a, b = (backward(h, w, rstd, dy, None, capi.BF16) for _ in range(2))
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    p, q = (run(h, dy, w, capi.BF16) for _ in range(2))
    assert all(np.array_equal(p[n].view(np.uint8), q[n].view(np.uint8)) for n in p)


def test_refusals(gpu):
    L = capi.lib()
    d = capi.DeviceBuffer(1 << 18)
    at = [d.ptr + (i << 14) for i in range(16)]
    names = ["X", "ldx", "R", "ldr", "W", "eps", "type", "M", "K", "H", "ldh", "rstd", "Y", "ldy", "Q", "ldq", "S", "lds", "format", "scale"]
    ok = [at[0], 64, at[1], 64, at[2], 1e-5, capi.F32, 32, 64, at[3], 64, at[4], at[5], 64, at[6], 64, at[7], 32, 0, 0]

    def refused(code, **change):
        assert L.decx_hip_rmsnorm_f8(*[change.get(n, v) for n, v in zip(names, ok)]) == code and capi.last_error().strip(), change

    d.fill(0)
    assert L.decx_hip_rmsnorm_f8(*ok) == 0
    refused(0x0d, X=None)
    refused(0x0d, W=None)
    refused(0x0d, H=None, Y=None, Q=None, rstd=None)
    refused(0x0d, S=None)
    refused(0x03, M=0)
    refused(0x03, K=0)
    refused(0x0d, K=32769, ldx=40000, ldr=40000, ldh=40000, ldy=40000, ldq=40000)
    refused(0x0b, type=9)
    refused(0x0b, format=2)
    refused(0x0b, scale=2)
    refused(0x0d, eps=-1.0)
    refused(0x0d, eps=float("nan"))
    for n in ("ldx", "ldr", "ldh", "ldy", "ldq"):
        refused(0x0d, **{n: 63})
    refused(0x0d, lds=31)
    refused(0x0d, H=at[3] + 2)
    refused(0x0d, rstd=at[4] + 1)
    refused(0x0d, S=at[7] + 2)

    names = ["H", "ldh", "W", "rstd", "dY", "lddy", "dR", "lddr", "type", "M", "K", "dX", "lddx", "dW", "work", "bytes"]
    need = capi.rmsnorm_backward_workspace(32, 64)
    ok = [at[0], 64, at[1], at[2], at[3], 64, at[4], 64, capi.F32, 32, 64, at[5], 64, at[6], at[7], need]

    def refused(code, **change):
        assert L.decx_hip_rmsnorm_backward(*[change.get(n, v) for n, v in zip(names, ok)]) == code and capi.last_error().strip(), change

    assert need >= 64 * 4 and L.decx_hip_rmsnorm_backward(*ok) == 0
    for n in ("H", "W", "rstd", "dY", "dX", "work"):
        refused(0x0d, **{n: None})
    refused(0x0d, bytes=need - 1)
    refused(0x0d, work=at[7] + 1)
    refused(0x03, M=-1)
    refused(0x03, K=0)
    refused(0x0d, K=32769, ldh=40000, lddy=40000, lddr=40000, lddx=40000)
    refused(0x0b, type=-1)
    for n in ("ldh", "lddy", "lddr", "lddx"):
        refused(0x0d, **{n: 63})
    refused(0x0d, dW=at[6] + 2)
    refused(0x0d, dX=at[5] + 1)


def test_weights_whose_product_with_the_row_overflows(gpu):
    x = ref.to_type(workloads.normal((5, 200), 40).astype(np.float32) * np.float32(2.0 ** 60), capi.BF16)
    w = ref.to_type(workloads.normal((1, 200), 41).astype(np.float32) * np.float32(2.0 ** 80), capi.BF16)      # h * w beyond 2^128, y is not
    check(x, None, w, capi.BF16, run(x, None, w, capi.BF16))


@pytest.mark.parametrize("call", ["quantize", "f8gemm", "norm", "backward"])
def test_integers_beyond_an_int_are_refused(gpu, call):
    d, far = capi.DeviceBuffer(64), 1 << 32
    with pytest.raises(capi.DecxHipError) as e:
        if call == "quantize":
            capi.f8_quantize(d.ptr, 16, 0, 1, far + 1, 1, 0, 0, d.ptr, 16, d.ptr, 1)
        elif call == "f8gemm":
            capi.f8gemm(d.ptr, 16, 0, d.ptr, 1, d.ptr, 16, 0, d.ptr, 1, 128, 0, d.ptr, 1, 0, 1, 1, far + 1)
        elif call == "norm":
            capi.rmsnorm_f8(d.ptr, far + 16, None, 0, d.ptr, 1e-5, 0, 1, 1, d.ptr, 16, None, None, 0, None, 0, None, 0)
        else:
            capi.rmsnorm_backward(d.ptr, 16, d.ptr, d.ptr, d.ptr, 16, None, 0, 0, 1, 1, d.ptr, far + 16, None, None, 0)
    assert e.value.code == 0x0d and "no int" in str(e.value)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: ref.TYPE_NAMES[k])
@pytest.mark.parametrize("M,K", [(3, 9001), (5, 20001), (300, 16400), (1030, 40)])
def test_gradient_of_long_rows_in_place(gpu, kind, M, K):
    """Rows that a workgroup of 1024 holds: results over each input, the sums of several rows a workgroup; the same bits as apart."""
    h, dy, w = inputs(M, K, kind, 21)
    dr = ref.to_type(workloads.normal((M, K), 79), kind)
    rstd = (1 / np.sqrt((ref.from_type(h, kind) ** 2).mean(1) + EPS)).astype(np.float32)
    plain = backward(h, w, rstd, dy, dr, kind)
    check_backward(h, w, rstd, dy, dr, kind, plain, M)
    for where in ("h", "y", "r"):
        got = backward(h, w, rstd, dy, dr, kind, inplace=where, pitch=5)
        assert np.array_equal(got[0].view(np.uint8), plain[0].view(np.uint8))
        check_backward(h, w, rstd, dy, dr, kind, got, M)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: ref.TYPE_NAMES[k])
@pytest.mark.parametrize("K", range(1, 18))
def test_each_short_row(gpu, kind, K):
    x, r, w = inputs(5, K, kind, 200 + K)
    check(x, r, w, kind, run(x, r, w, kind, pitch=3, lead=1))
    rstd = (1 / np.sqrt((ref.from_type(x, kind) ** 2).mean(1) + EPS)).astype(np.float32)
    check_backward(x, w, rstd, r, None, kind, backward(x, w, rstd, r, None, kind, pitch=1, lead=1), 5)


@pytest.mark.parametrize("kind,M,K,times", [(capi.BF16, 700, 8192, 6), (capi.F16, 900, 8192, 10), (capi.F32, 500, 8190, 9)])
def test_inputs_larger_than_the_caches(gpu, kind, M, K, times):
    """More than 96 MiB, where loads and workgroups a unit are chosen otherwise: some rows against 64 bits, the same rows again and
    again in the same bits."""
    x, r, w = inputs(M, K, kind, 90)
    big = lambda a: np.tile(a, (times, 1))  # noqa: E731
    got = run(big(x), big(r), w, kind)
    first = {n: (v[:, :M] if n in ("rstd", "S") else v[:M]) for n, v in got.items()}
    check(x, r, w, kind, first)
    for n, v in got.items():
        want = np.tile(first[n], (1, times)) if n in ("rstd", "S") else big(first[n])
        assert np.array_equal(v.view(np.uint8), want.view(np.uint8)), n
    rstd = first["rstd"][0]
    dx, dw = backward(big(x), w, np.tile(rstd, times), big(r), big(r), kind)
    check_backward(x, w, rstd, r, r, kind, (dx[:M], None), M)
    assert np.array_equal(dx.view(np.uint8), big(dx[:M]).view(np.uint8))
    _, _, want_w, size_w = gradient64(ref.from_type(x, kind), ref.from_type(w, kind), rstd.astype(np.float64), ref.from_type(r, kind), 0.0)
    assert np.all(np.abs(dw - times * want_w) <= times * size_w * (times * M + 20) * 2.0 ** -24)


@pytest.mark.parametrize("kind", [capi.F32, capi.BF16], ids=lambda k: ref.TYPE_NAMES[k])
@pytest.mark.parametrize("power,eps", [(70, EPS), (122, EPS), (64, 0.0), (63, EPS), (-64, 0.0), (-80, 0.0), (-110, 0.0), (-80, EPS), (-61, 1e-37)])
@pytest.mark.parametrize("M,K", [(3, 7), (4, 300), (3, 1500), (2, 4100), (2, 9000), (2, 20000)])
def test_rows_whose_squares_leave_fp32(gpu, kind, power, eps, M, K):
    """Finite rows whose squares overflow or lose their bits, beside an ordinary row: the bounds are those of ordinary rows."""
    x, r = (workloads.normal((M, K), s).astype(np.float32) * np.float32(2.0 ** power) for s in (50, 51))
    x[0], r[0] = workloads.normal((K,), 52), 0
    x, r, w = ref.to_type(x, kind), ref.to_type(r, kind), ref.to_type(1 + 0.2 * workloads.normal((1, K), 53), kind)
    got = run(x, r, w, kind, eps=eps)
    check(x, r, w, kind, got, eps=eps)
    if abs(power) <= 80:                                         # the gradient by that rstd; beyond, dx leaves the types' normal range
        dy = ref.to_type(workloads.normal((M, K), 54), kind)
        check_backward(got["H"], w, got["rstd"][0], dy, None, kind, backward(got["H"], w, got["rstd"][0], dy, None, kind), M)


def test_rows_at_the_ends_of_fp32(gpu):
    """Rows of the largest finite values, whose rstd is subnormal (half its step is 2^-22 of it, within the bounds); rows whose
    rstd no fp32 holds."""
    x = np.where(workloads.normal((2, 600), 55) > 0, np.float32(3e38), np.float32(-2e38)).astype(np.float32)
    w = np.ones((1, 600), np.float32)
    got = run(x, None, w, capi.F32, eps=0.0)
    check(x, None, w, capi.F32, got, eps=0.0)
    least = run(np.full((1, 600), 1e-44, np.float32), None, w, capi.F32, eps=0.0)
    assert np.all(np.isinf(least["rstd"]))
