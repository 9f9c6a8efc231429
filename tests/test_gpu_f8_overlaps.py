"""The 8-bit operators where their operands lie over each other: what decx_hip.h allows gives the same bits as apart, the rest is
refused before anything is launched."""
import numpy as np
import pytest

import f8_reference as ref
from backup_1_amd import capi, workloads
from f8_reference import Pitched

pytestmark = pytest.mark.gpu
M, K, N = 32, 64, 48
EPS = 1e-5


@pytest.fixture(scope="module")
def at(gpu):
    """Sixteen places 16 KiB apart in one block of zeros: each holds any operand of these sizes."""
    d = capi.DeviceBuffer(1 << 18)
    d.fill(0)
    places = [d.ptr + (i << 14) for i in range(16)]
    yield places
    del d


def refused(call, names, args, **change):
    with pytest.raises(capi.DecxHipError) as e:
        call(*[change.get(n, v) for n, v in zip(names, args)])
    assert e.value.code == 0x0d and "lies over" in str(e.value), change


def test_quantise(at):
    X, Q, S, Qt, St = at[:5]
    names = ["X", "ldx", "type", "M", "K", "block_rows", "fmt", "scale", "Q", "ldq", "S", "lds", "Qt", "ldqt", "St", "ldst"]
    args = [X, K, capi.F32, M, K, 1, 0, capi.SCALE_F32, Q, K, S, M, Qt, M, St, K]
    capi.f8_quantize(*args)
    for change in ({"Q": X}, {"Q": X + 4 * K * M - 1}, {"S": X}, {"Qt": X + 8}, {"St": X + 4 * (K * M - 1)}, {"Q": S}, {"Q": Qt}, {"Qt": Q + K * M - 1}, {"S": St}, {"St": Q}):
        refused(capi.f8_quantize, names, args, **change)


def test_quantise_into_columns_of_the_sources_own_matrix(gpu):
    """X is the left half of a matrix, the codes lie in its right half: their spans meet, their bytes do not."""
    x = workloads.normal((50, 136), 5).astype(np.float32)
    both = np.zeros((50, 272), np.float32)
    both[:, :136] = x
    d, s = Pitched(both), Pitched.empty(2, 50, np.float32)
    capi.f8_quantize(d.ptr, 272, capi.F32, 50, 136, 1, 0, 0, d.ptr + 136 * 4, 272 * 4, s.ptr, 50)
    got = d.result()
    codes, scales = ref.quantize(x, capi.E4M3, capi.SCALE_F32, 1)
    assert np.array_equal(got[:, :136], x) and np.array_equal(got[:, 136:].copy().view(np.uint8)[:, :136], codes) and np.array_equal(s.result(), scales)


def test_product(at):
    A, SA, B, SB, C, D = at[:6]
    names = ["A", "lda", "fa", "SA", "ldsa", "B", "ldb", "fb", "SB", "ldsb", "b_rows", "scale", "D", "ldd", "type", "M", "N", "K", "C", "ldc"]
    args = [A, K, 0, SA, M, B, K, 0, SB, 1, 128, 0, D, N, capi.F32, M, N, K, C, N]
    capi.f8gemm(*args)
    for change in ({"D": A}, {"D": SA}, {"D": B}, {"D": SB}, {"D": A + K * M - 4}, {"D": C, "ldd": N + 4}, {"D": C + 4}, {"D": C + 4 * N}, {"D": C - 4}):
        refused(capi.f8gemm, names, args, **change)
    capi.f8gemm(*[{"D": C}.get(n, v) for n, v in zip(names, args)])
    capi.f8gemm(*[{"D": C, "ldd": N + 4, "M": 1}.get(n, v) for n, v in zip(names, args)])          # one row has no pitch


def test_norm(at):
    X, R, W, H, rstd, Y, Q, S = at[:8]
    names = ["X", "ldx", "R", "ldr", "W", "eps", "type", "M", "K", "H", "ldh", "rstd", "Y", "ldy", "Q", "ldq", "S", "lds"]
    args = [X, K, R, K, W, EPS, capi.F32, M, K, H, K, rstd, Y, K, Q, K, S, M]
    capi.rmsnorm_f8(*args)
    for change in ({"H": X, "ldh": K + 8}, {"H": X + 4 * K}, {"H": R + 4}, {"H": W}, {"rstd": X}, {"rstd": W}, {"rstd": R + 4 * K * M - 4}, {"Y": H}, {"Y": W}, {"Y": X + 4 * K},
                   {"Q": X}, {"Q": R}, {"S": X}, {"S": rstd}, {"Q": Y}, {"S": Q}, {"H": X, "Y": X}):
        refused(capi.rmsnorm_f8, names, args, **change)


def test_gradient(at):
    H, W, rstd, dY, dR, dX, dW, work = at[:8]
    need = capi.rmsnorm_backward_workspace(M, K)
    names = ["H", "ldh", "W", "rstd", "dY", "lddy", "dR", "lddr", "type", "M", "K", "dX", "lddx", "dW", "work", "bytes"]
    args = [H, K, W, rstd, dY, K, dR, K, capi.F32, M, K, dX, K, dW, work, need]
    assert need <= 1 << 14
    capi.rmsnorm_backward(*args)
    for change in ({"dW": W}, {"dW": H}, {"dW": dY}, {"dW": dR}, {"dW": dX}, {"dW": rstd}, {"dX": W}, {"dX": rstd}, {"dX": H, "lddx": K + 8}, {"dX": dY + 4 * K}, {"dX": dR - 4},
                   {"dX": H + 4}, {"work": W}, {"work": dY + 4}, {"work": dX}, {"work": dW}, {"work": rstd}):
        refused(capi.rmsnorm_backward, names, args, **change)
    capi.rmsnorm_backward(*[{"dX": H, "lddx": K + 8, "M": 1}.get(n, v) for n, v in zip(names, args)])


@pytest.mark.parametrize("kind", (capi.F32, capi.F16, capi.BF16), ids=lambda k: ref.TYPE_NAMES[k])
@pytest.mark.parametrize("M,K", [(5, 64), (30, 333), (7, 5), (3, 9000), (2, 20001)])
def test_norm_over_its_inputs(gpu, kind, M, K):
    """y over x or r, with h over the other one: the bits of a call with places of their own."""
    x, r, w = (ref.to_type(workloads.normal(shape, seed).astype(np.float32), kind) for shape, seed in (((M, K), 1), ((M, K), 2), ((1, K), 3)))
    dw = Pitched(w)

    def run(H, X, R, Y):
        capi.rmsnorm_f8(X.ptr, X.ld, R.ptr, R.ld, dw.ptr, EPS, kind, M, K, H.ptr, H.ld, None, Y.ptr, Y.ld, None, 0, None, 0)
        return H.result().view(np.uint8), Y.result().view(np.uint8)

    place = lambda v: Pitched(v, pitch=K + 3, lead=1)  # noqa: E731
    empty = lambda: Pitched.empty(M, K, x.dtype, pitch=K + 3, lead=1)  # noqa: E731
    want = run(empty(), place(x), place(r), empty())
    for h_over, y_over in (("x", "r"), ("r", "x"), (None, "x"), (None, "r")):
        d = {"x": place(x), "r": place(r), None: empty()}
        got = run(d[h_over], d["x"], d["r"], d[y_over])
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), (h_over, y_over)
