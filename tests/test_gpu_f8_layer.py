"""The 8-bit operators together, as a layer of a model uses them: two products with the norm before and the ReLU between,
its whole backward pass, the same captured into a graph, and operands that lie further apart than 32 bits reach."""
import ctypes

import numpy as np
import pytest

import f8_reference as ref
from backup_1_amd import capi, workloads
from f8_reference import Pitched

pytestmark = pytest.mark.gpu
EPS = 1e-5


class Layer:
    """out = relu(norm(x + r) W1^T) W2^T and the gradients of sum(out * g) by x + r, the norm's weight, W1 and W2.  Weights are
    quantised in squares, activations and gradients along the contraction of the product that reads them."""

    def __init__(self, M, K, F, kind, scale, seed=1):
        self.M, self.K, self.F, self.kind, self.scale = M, K, F, kind, scale
        st = np.float32 if scale == capi.SCALE_F32 else np.uint8
        n = lambda rows, cols, s, f: workloads.normal((rows, cols), seed + s).astype(np.float32) * np.float32(f)  # noqa: E731
        self.x, self.r = ref.to_type(n(M, K, 0, 1), kind), ref.to_type(n(M, K, 1, 1), kind)
        self.w = ref.to_type(1 + n(1, K, 2, 0.1), kind)
        self.w1, self.w2 = n(F, K, 3, K ** -0.5), n(K, F, 4, F ** -0.5)
        self.g = n(M, K, 5, 1)
        self.d = {}
        for name in ("x", "r", "w", "w1", "w2", "g"):
            self.d[name] = Pitched(getattr(self, name))
        up = lambda v: -(-v // 16) * 16  # noqa: E731

        def new(name, rows, cols, dtype):
            self.d[name] = Pitched.empty(rows, cols, dtype, pitch=up(cols))

        def coded(name, rows, cols, block_rows=1):
            new(name, rows, cols, np.uint8)
            new("s_" + name, -(-cols // 128), rows if block_rows == 1 else -(-rows // 128), st)

        wide = ref.NP_TYPE[kind]
        new("h", M, K, wide), new("rstd", 1, M, np.float32), new("y", M, K, wide)
        coded("qy", M, K), coded("qyt", K, M)
        coded("qw1", F, K, 128), coded("qw1t", K, F, 128), coded("qw2", K, F, 128), coded("qw2t", F, K, 128)
        for name in ("a", "da", "dpre"):
            self.d[name] = Pitched.empty(M, F, np.float32)       # dense: the ReLU family walks consecutive floats
        self.d["act"], self.d["map"] = Pitched.empty(M, F, np.float32), Pitched.empty(1, M * F // 8, np.uint8)
        coded("qact", M, F), coded("qactt", F, M), coded("qg", M, K), coded("qgt", K, M), coded("qd", M, F), coded("qdt", F, M)
        new("out", M, K, np.float32), new("dy", M, K, np.float32), new("dyw", M, K, wide)
        new("dw1", F, K, np.float32), new("dw2", K, F, np.float32), new("dx", M, K, wide), new("dw", 1, K, np.float32)
        self.work = capi.DeviceBuffer(capi.rmsnorm_backward_workspace(M, K))

    def q(self, src, dst, dst_t, rows, cols, kind, block_rows=1, fmt=capi.E4M3):
        d = self.d
        p = lambda n: (d[n].ptr, d[n].ld) if n else (None, 0)  # noqa: E731
        capi.f8_quantize(*p(src), kind, rows, cols, block_rows, fmt, self.scale, *p(dst), *p("s_" + dst if dst else None), *p(dst_t),
                         *p("s_" + dst_t if dst_t else None), blocking=False)

    def mm(self, a, fa, b, fb, b_rows, dst, M, N, K, kind, add=None):
        d = self.d
        capi.f8gemm(d[a].ptr, d[a].ld, fa, d["s_" + a].ptr, d["s_" + a].ld, d[b].ptr, d[b].ld, fb, d["s_" + b].ptr, d["s_" + b].ld, b_rows, self.scale,
                    d[dst].ptr, d[dst].ld, kind, M, N, K, d[add].ptr if add else None, d[add].ld if add else 0, blocking=False)

    def run(self):
        """One training step's work on the library's stream, without waiting."""
        M, K, F, d, L = self.M, self.K, self.F, self.d, capi.lib()
        e4, e5, f32 = capi.E4M3, capi.E5M2, capi.F32
        self.q("w1", "qw1", "qw1t", F, K, f32, 128)
        self.q("w2", "qw2", "qw2t", K, F, f32, 128)
        capi.rmsnorm_f8(d["x"].ptr, d["x"].ld, d["r"].ptr, d["r"].ld, d["w"].ptr, EPS, self.kind, M, K, d["h"].ptr, d["h"].ld, d["rstd"].ptr,
                        d["y"].ptr, d["y"].ld, d["qy"].ptr, d["qy"].ld, d["s_qy"].ptr, d["s_qy"].ld, e4, self.scale, blocking=False)
        self.mm("qy", e4, "qw1", e4, 128, "a", M, F, K, f32)
        capi.check(L.decx_hip_relu_f32_async(d["a"].ptr, d["act"].ptr, M * F))
        self.q("act", "qact", "qactt", M, F, f32)
        self.mm("qact", e4, "qw2", e4, 128, "out", M, K, F, f32)
        # backward
        self.q("g", "qg", "qgt", M, K, f32, fmt=e5)
        self.mm("qg", e5, "qw2t", e4, 128, "da", M, F, K, f32)
        self.mm("qgt", e5, "qactt", e4, 1, "dw2", K, F, M, f32)

    def run_rest(self):
        M, K, F, d = self.M, self.K, self.F, self.d
        e4, e5, f32 = capi.E4M3, capi.E5M2, capi.F32
        self.q("dpre", "qd", "qdt", M, F, f32, fmt=e5)
        self.q("y", None, "qyt", M, K, self.kind)
        self.mm("qd", e5, "qw1t", e4, 128, "dyw", M, K, F, self.kind)
        self.mm("qdt", e5, "qyt", e4, 1, "dw1", F, K, M, f32)
        capi.rmsnorm_backward(d["h"].ptr, d["h"].ld, d["w"].ptr, d["rstd"].ptr, d["dyw"].ptr, d["dyw"].ld, None, 0, self.kind, M, K, d["dx"].ptr,
                              d["dx"].ld, d["dw"].ptr, self.work.ptr, self.work.nbytes, blocking=False)

    def relu_backward(self):
        """da where a's sign bit is clear, by the recording form of the activation (blocking entry points)."""
        L, d, n = capi.lib(), self.d, self.M * self.F
        capi.check(L.decx_hip_relu_f32_rec(d["a"].ptr, d["act"].ptr, d["map"].ptr, n))
        capi.check(L.decx_hip_relu_f32_backward(d["da"].ptr, d["dpre"].ptr, d["map"].ptr, n))

    def get(self, name):
        a = self.d[name].result()
        return ref.from_type(a, self.kind) if a.dtype == np.uint16 or self.d[name].dtype == np.float16 else a.astype(np.float64)

    def deq(self, name, fmt, block_rows):
        return ref.dequantize(self.d[name].result(), fmt, self.d["s_" + name].result(), block_rows)


def near(got, want, size, K, kind=capi.F32):
    lost = 7 * 2.0 ** -13 * size if kind != capi.F32 else 0.0     # the 8-bit instructions' alignment, at most (test_gpu_f8gemm.py)
    blocks = -(-K // 128)
    assert np.all(np.abs(got - want) <= size * (128 + 3 * blocks + 2) * 2.0 ** -23 + lost + np.abs(want) * ref.HALF_STEP[kind] * 1.001 + 1e-30)


@pytest.mark.parametrize("M,K,F,kind,scale", [(40, 256, 384, capi.F32, capi.SCALE_F32), (200, 320, 576, capi.BF16, capi.SCALE_E8M0), (8, 136, 264, capi.F16, capi.SCALE_F32)])
def test_training_step(gpu, M, K, F, kind, scale):
    """Each product against 64 bits on the very codes that the step before made, and the step as a whole against the same layer
    in 64 bits without any 8-bit rounding: within what four such roundings cost."""
    s = Layer(M, K, F, kind, scale)
    s.run()
    capi.sync()
    s.relu_backward()
    s.run_rest()
    capi.sync()
    e4, e5 = capi.E4M3, capi.E5M2

    def product(dst, a, fa, b, fb, b_rows, inner, out_kind=capi.F32):
        x, w = s.deq(a, fa, 1), s.deq(b, fb, b_rows)
        near(s.get(dst), x @ w.T, np.abs(x) @ np.abs(w).T, inner, out_kind)

    product("a", "qy", e4, "qw1", e4, 128, K)
    product("out", "qact", e4, "qw2", e4, 128, F)
    product("da", "qg", e5, "qw2t", e4, 128, K)
    product("dw2", "qgt", e5, "qactt", e4, 1, M)
    product("dyw", "qd", e5, "qw1t", e4, 128, F, kind)
    product("dw1", "qdt", e5, "qyt", e4, 1, M)
    # the layer without 8-bit numbers
    h = ref.from_type(s.x, kind) + ref.from_type(s.r, kind)
    rstd = 1 / np.sqrt((h * h).mean(1, keepdims=True) + EPS)
    w = ref.from_type(s.w, kind)
    y = h * rstd * w
    a = y @ s.w1.astype(np.float64).T
    act = np.maximum(a, 0)
    out = act @ s.w2.astype(np.float64).T
    g = s.g.astype(np.float64)
    da = (g @ s.w2.astype(np.float64)) * (a > 0)
    dy = da @ s.w1.astype(np.float64)
    gn = dy * w
    dx = rstd * (gn - h * rstd * (gn * h * rstd).mean(1, keepdims=True))
    for name, want in (("out", out), ("dw2", g.T @ act), ("dw1", da.T @ y), ("dx", dx), ("dw", (dy * h * rstd).sum(0)[None])):
        off = np.linalg.norm(s.get(name) - want) / np.linalg.norm(want)
        # an e4m3 rounding is at most 2^-4 of a value, an e5m2 one 2^-3; independent, a result's norm is off by at most the sum of those on
        # its way (and by what masks flip near zero): 4 * 2^-4 + 2 * 2^-3
        assert off < 0.5, (name, off)


def test_captured_step(gpu):
    """The step captured into a graph and replayed, with other inputs and eager work in between: the eager bits each time."""
    hip = capi.lib()                                             # the runtime's symbols, through the library that links it
    shape = (72, 256, 320, capi.BF16, capi.SCALE_F32)
    s, eager = Layer(*shape, seed=30), Layer(*shape, seed=30)
    names = ("out", "da", "dw2", "dw1", "dyw", "dx", "dw", "h", "qy", "s_qy")

    def step(layer):
        layer.run()
        layer.run_rest()                                         # on the gradient that dpre holds

    for layer in (s, eager):                                     # first calls set kernels up; dpre gets its value
        layer.run(), capi.sync(), layer.relu_backward(), layer.run_rest(), capi.sync()
    stream, graph, exe = ctypes.c_void_p(capi.stream()), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 1) == 0             # 1: calls of other threads stay allowed
    step(s)
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    try:
        for turn in range(4):
            x = ref.to_type(workloads.normal((s.M, s.K), 60 + turn).astype(np.float32), s.kind)
            for layer in (s, eager):                             # in place: the graph holds the addresses
                layer.d["x"].store[:x.size] = x.reshape(-1)
                layer.d["x"].buf.upload(layer.d["x"].store)
            step(eager)
            assert hip.hipGraphLaunch(exe, stream) == 0
            capi.sync()
            for name in names:
                assert np.array_equal(s.d[name].result().view(np.uint8), eager.d[name].result().view(np.uint8)), (turn, name)
    finally:
        assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0


@pytest.mark.parametrize("aligned", [True, False])
def test_operands_beyond_32_bits(gpu, aligned):
    """600 rows a pitch of 8 MiB apart (5 GB): codes written and read, results written, each at its 64-bit place."""
    M, N, K = 600, 520, 272
    pitch = (1 << 23) + (0 if aligned else 1)
    x = workloads.normal((M, K), 91).astype(np.float32)
    b, sb = ref.quantize(workloads.normal((N, K), 92).astype(np.float32), capi.E4M3, capi.SCALE_F32, 128)
    codes, scales = ref.quantize(x, capi.E4M3, capi.SCALE_F32, 1)
    big = capi.DeviceBuffer(pitch * M)                           # the codes' rows; reused for the result's
    dx, dS, dB, dSB, dD = Pitched(x), Pitched.empty(3, M, np.float32), Pitched(b), Pitched(sb), Pitched.empty(M, N, np.float32)

    def rows(count, width):
        out = np.empty((count, width), np.uint8)
        capi.check(capi.lib().decx_hip_memcpy2d(out.ctypes.data, width, big.ptr, pitch, width, count, capi.D2H))
        return out

    capi.f8_quantize(dx.ptr, K, capi.F32, M, K, 1, capi.E4M3, capi.SCALE_F32, big.ptr, pitch, dS.ptr, M)
    assert np.array_equal(rows(M, K), codes) and np.array_equal(dS.result(), scales)
    want = ref.dequantize(codes, capi.E4M3, scales, 1) @ ref.dequantize(b, capi.E4M3, sb, 128).T
    size = np.abs(ref.dequantize(codes, capi.E4M3, scales, 1)) @ np.abs(ref.dequantize(b, capi.E4M3, sb, 128)).T
    try:
        for variant in (0, 1, 3, 5):
            capi.lib().decx_hip_set_f8gemm_variant(variant)
            capi.f8gemm(big.ptr, pitch, 0, dS.ptr, M, dB.ptr, K, 0, dSB.ptr, dSB.ld, 128, 0, dD.ptr, N, capi.F32, M, N, K)
            near(dD.result().astype(np.float64), want, size, K)
    finally:
        capi.lib().decx_hip_set_f8gemm_variant(0)
    if aligned:                                                  # the result far apart: pitch / 2 elements of 2 bytes
        dA = Pitched(codes)
        try:
            for variant in (0, 1, 4, 5, 6):
                capi.lib().decx_hip_set_f8gemm_variant(variant)
                capi.f8gemm(dA.ptr, K, 0, dS.ptr, M, dB.ptr, K, 0, dSB.ptr, dSB.ld, 128, 0, big.ptr, pitch // 2, capi.BF16, M, N, K)
                near(ref.from_type(rows(M, 2 * N).view(np.uint16), capi.BF16), want, size, K, capi.BF16)
        finally:
            capi.lib().decx_hip_set_f8gemm_variant(0)
        h = ref.to_type(x, capi.F16)
        dh, one = Pitched(h), Pitched(np.ones((1, K), np.float16))
        capi.rmsnorm_f8(dh.ptr, K, None, 0, one.ptr, EPS, capi.F16, M, K, big.ptr, pitch // 2,
                        None, None, 0, None, 0, None, 0)
        assert np.array_equal(rows(M, 2 * K).view(np.float16), h)


def test_sizes_beyond_a_launch_are_refused(gpu):
    L, d = capi.lib(), capi.DeviceBuffer(64)
    most = 1 << 29
    assert L.decx_hip_f8_quantize(d.ptr, 16, 0, most + 1, 16, 1, 0, 0, d.ptr, 16, d.ptr, most + 1, None, 0, None, 0) == 0x0d
    assert L.decx_hip_f8_quantize(d.ptr, 128, 0, most, 128, 1, 0, 0, d.ptr, 128, d.ptr, most, None, 0, None, 0) == 0x0d
    assert L.decx_hip_f8gemm(d.ptr, 16, 0, d.ptr, most + 1, d.ptr, 16, 0, d.ptr, 1, 128, 0, None, 0, d.ptr, 16, 0, most + 1, 1, 16) == 0x0d
    assert L.decx_hip_f8gemm(d.ptr, 16, 0, d.ptr, most, d.ptr, 16, 0, d.ptr, most, 128, 0, None, 0, d.ptr, most, 0, most, most, 16) == 0x0d
    assert L.decx_hip_rmsnorm_f8(d.ptr, 4096, None, 0, d.ptr, 1e-5, 0, most, 4096, d.ptr, 4096, None, None, 0, None, 0, None, 0, 0, 0) == 0x0d
    assert L.decx_hip_rmsnorm_backward(d.ptr, 64, d.ptr, d.ptr, d.ptr, 64, None, 0, 0, most + 1, 64, d.ptr, 64, None, None, 0) == 0x0d


@pytest.mark.parametrize("M,K,F,kind,scale", [(40, 256, 384, capi.F32, capi.SCALE_F32), (200, 320, 576, capi.BF16, capi.SCALE_E8M0), (8, 136, 264, capi.F16, capi.SCALE_F32)])
def test_training_step_operator_by_operator(gpu, M, K, F, kind, scale):
    """What test_training_step bounds as a whole only by what 8-bit rounding costs: here each operator between the products, on what
    the step before it made -- codes, scales and the activation bit for bit, the norm and its gradient within their own bounds."""
    from test_gpu_rmsnorm import check, check_backward
    s = Layer(M, K, F, kind, scale)
    s.run()
    capi.sync()
    s.relu_backward()
    s.run_rest()
    capi.sync()
    got = lambda n: s.d[n].result()  # noqa: E731
    e4, e5, f32 = capi.E4M3, capi.E5M2, capi.F32
    act, dpre = got("act"), got("dpre")
    a = got("a")
    assert np.array_equal(act, np.where(np.signbit(a), a * 0, a)) and np.array_equal(dpre, np.where(np.signbit(a), got("da") * 0, got("da")))
    for name, of, of_kind, fmt, block_rows in (("qw1", s.w1, f32, e4, 128), ("qw2", s.w2, f32, e4, 128), ("qact", act, f32, e4, 1), ("qg", s.g, f32, e5, 1),
                                               ("qd", dpre, f32, e5, 1), ("qy", got("y"), kind, e4, 1)):
        v = ref.from_type(of, of_kind).astype(np.float32)
        for n, m in ((name, v), (name + "t", v.T)):
            if n == "qy":
                continue                                         # of y before its rounding: with the norm below
            codes, scales = ref.quantize(m, fmt, scale, block_rows)
            values = lambda c: ref.TABLE[fmt][c]  # noqa: E731
            assert np.array_equal(values(got(n)), values(codes)) and np.array_equal(got("s_" + n), scales), n
    check(s.x, s.r, s.w, kind, {"H": got("h"), "rstd": got("rstd"), "Y": got("y"), "Q": got("qy"), "S": got("s_qy")}, e4, scale)
    check_backward(got("h"), s.w, got("rstd")[0], got("dyw"), None, kind, (got("dx"), got("dw")[0]), M)
