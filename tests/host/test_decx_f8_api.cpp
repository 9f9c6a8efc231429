// Exercises the 8-bit operators of the DECX-named C++ API (Quantize_f8, GEMM_f8, RMSNorm_f8 and its backward, DECX.h) over
// device-resident containers, against plain double arithmetic.  Usage: test_decx_f8_api cpu | gpu
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <string>
#include <vector>

#include "../../backup_1_amd/host/DECX.h"

static int g_fail = 0;
#define CHECK(cond)                                                                                          \
    do {                                                                                                     \
        if (!(cond)) { std::printf("  CHECK FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); ++g_fail; }     \
    } while (0)

static std::mt19937 rng(2024);
static float small_int() { return (float)((int)(rng() % 17) - 8); }
static float normal() { return std::normal_distribution<float>()(rng); }

// host copies with the values a container holds
template <class T> struct Host {
    de::Matrix<T>* m;
    uint w, h;
    Host(uint w_, uint h_) : m(&de::CreateMatrixRef<T>(w_, h_, 0)), w(w_), h(h_) {}
    T& at(uint i, uint j) { return m->index((int)i, (int)j); }
};
static de::GPU_Matrix<float>& upload(Host<float>& x) {
    de::GPU_Matrix<float>& d = de::CreateGPUMatrixRef<float>(x.w, x.h);
    d.Load_from_host(*x.m);
    return d;
}
static de::GPU_Matrix<de::Half>& upload_half(Host<float>& x) {       // values that binary16 holds
    Host<de::Half> y(x.w, x.h);
    for (uint i = 0; i < x.h; ++i)
        for (uint j = 0; j < x.w; ++j) y.at(i, j) = de::Float2Half(x.at(i, j));
    de::GPU_Matrix<de::Half>& d = de::CreateGPUMatrixRef<de::Half>(x.w, x.h);
    d.Load_from_host(*y.m);
    return d;
}
static Host<float> download(de::GPU_Matrix<float>& d) {
    Host<float> x(d.Width(), d.Height());
    d.Load_to_host(*x.m);
    return x;
}
static Host<float> download(de::GPU_Matrix<de::Half>& d) {
    Host<de::Half> y(d.Width(), d.Height());
    d.Load_to_host(*y.m);
    Host<float> x(d.Width(), d.Height());
    for (uint i = 0; i < x.h; ++i)
        for (uint j = 0; j < x.w; ++j) x.at(i, j) = de::Half2Float(y.at(i, j));
    return x;
}
static bool good(const de::DH& h) {
    if (h.error_type != decx::DECX_SUCCESS) std::printf("  status %d: %s\n", h.error_type, h.error_string);
    return h.error_type == decx::DECX_SUCCESS;
}

// Whole numbers of magnitude <= 8 have three significant bits more than none: power-of-two scales lose nothing, so the
// product of the quantised matrices is the matrices' own.
template <class Out>
static void product_of_whole_numbers(int block_rows, bool half_source) {
    const uint M = 45, N = 150, K = 300;
    Host<float> a(K, M), b(K, N);
    for (uint k = 0; k < K; ++k) {
        for (uint i = 0; i < M; ++i) a.at(i, k) = small_int();
        for (uint j = 0; j < N; ++j) b.at(j, k) = small_int();
    }
    de::GPU_Matrix<uchar>&qa = de::CreateGPUMatrixRef<uchar>(), &qb = de::CreateGPUMatrixRef<uchar>(), &sa = de::CreateGPUMatrixRef<uchar>(),
                         &sb = de::CreateGPUMatrixRef<uchar>();
    de::GPU_Matrix<Out>& d = de::CreateGPUMatrixRef<Out>();
    if (half_source) {
        CHECK(good(de::cuda::Quantize_f8(upload_half(a), qa, sa, 1, decx::de_f8_e4m3)));
        CHECK(good(de::cuda::Quantize_f8(upload_half(b), qb, sb, block_rows, decx::de_f8_e4m3)));
    } else {
        CHECK(good(de::cuda::Quantize_f8(upload(a), qa, sa, 1, decx::de_f8_e4m3)));
        CHECK(good(de::cuda::Quantize_f8(upload(b), qb, sb, block_rows, decx::de_f8_e4m3)));
    }
    CHECK(qa.Width() == K && qa.Height() == M && sa.Width() == M && sa.Height() == 3 && sb.Width() == (block_rows == 1 ? N : 2));
    CHECK(good(de::cuda::GEMM_f8(qa, sa, decx::de_f8_e4m3, qb, sb, decx::de_f8_e4m3, d)));
    Host<float> got = download(d);
    int bad = 0;
    for (uint i = 0; i < M; ++i)
        for (uint j = 0; j < N; ++j) {
            float want = 0;
            for (uint k = 0; k < K; ++k) want += a.at(i, k) * b.at(j, k);
            if (sizeof(Out) == 2) want = de::Half2Float(de::Float2Half(want));
            bad += got.at(i, j) != want;
        }
    CHECK(bad == 0);
    // the transposes' product of the same matrix: A^T and B's rows must agree in length, so A with itself
    de::GPU_Matrix<uchar>&qt = de::CreateGPUMatrixRef<uchar>(), &st = de::CreateGPUMatrixRef<uchar>();
    CHECK(good(de::cuda::Quantize_f8_T(upload(a), qt, st, 1, decx::de_f8_e4m3)));
    CHECK(qt.Width() == M && qt.Height() == K && st.Width() == K && st.Height() == 1);
    de::GPU_Matrix<float>& gram = de::CreateGPUMatrixRef<float>();
    CHECK(good(de::cuda::GEMM_f8(qt, st, decx::de_f8_e4m3, qt, st, decx::de_f8_e4m3, gram)));
    Host<float> g = download(gram);
    bad = 0;
    for (uint i = 0; i < K; ++i)
        for (uint j = 0; j < K; ++j) {
            float want = 0;
            for (uint m = 0; m < M; ++m) want += a.at(m, i) * a.at(m, j);
            bad += g.at(i, j) != want;
        }
    CHECK(bad == 0);
    // sizes that do not fit each other
    de::GPU_Matrix<uchar>& other = de::CreateGPUMatrixRef<uchar>(K + 1, N);
    CHECK(de::cuda::GEMM_f8(qa, sa, 0, other, sb, 0, d).error_type == decx::DECX_FAIL_DimsNotMatching);
    CHECK(de::cuda::GEMM_f8(qa, sb, 0, qb, sb, 0, d).error_type == decx::DECX_FAIL_DimsNotMatching);
    CHECK(de::cuda::GEMM_f8(qa, sa, 7, qb, sb, 0, d).error_type == decx::DECX_FAIL_ErrorFlag);
    CHECK(de::cuda::Quantize_f8(upload(a), qa, sa, 64, 0).error_type == decx::DECX_FAIL_ErrorParams);
    CHECK(de::cuda::Quantize_f8(upload(a), qa, qa, 1, 0).error_type == decx::DECX_FAIL_ErrorParams);
}

// norm -> codes -> product with a quantised weight: every result within the formats' half steps of double arithmetic
template <class T>
static void norm_product_and_gradient(bool half) {
    const uint M = 37, N = 65, K = 260;
    const double eps = 1e-5, half_step = half ? 1.0 / 2048 : 1.0 / (1 << 24);
    Host<float> x(K, M), r(K, M), w(K, 1), dy(K, M), f(K, N);
    auto q = [&](float v) { return half ? de::Half2Float(de::Float2Half(v)) : v; };
    for (uint k = 0; k < K; ++k) {
        w.at(0, k) = q(1 + 0.1f * normal());
        for (uint i = 0; i < M; ++i) x.at(i, k) = q(normal()), r.at(i, k) = q(normal()), dy.at(i, k) = q(0.1f * normal());
        for (uint j = 0; j < N; ++j) f.at(j, k) = q(0.1f * normal());
    }
    auto up = [&](Host<float>& v) -> de::GPU_Matrix<T>& {
        if constexpr (sizeof(T) == 2) return upload_half(v);
        else return upload(v);
    };
    de::GPU_Matrix<T>&dx = up(x), &dr = up(r), &dw = up(w), &ddy = up(dy), &df = up(f);
    de::GPU_Matrix<T>&sum = de::CreateGPUMatrixRef<T>(), &out = de::CreateGPUMatrixRef<T>(), &dst = de::CreateGPUMatrixRef<T>();
    de::GPU_Matrix<float>&rstd = de::CreateGPUMatrixRef<float>(), &s = de::CreateGPUMatrixRef<float>(), &sf = de::CreateGPUMatrixRef<float>(),
                         &gw = de::CreateGPUMatrixRef<float>();
    de::GPU_Matrix<uchar>&c = de::CreateGPUMatrixRef<uchar>(), &cf = de::CreateGPUMatrixRef<uchar>();
    CHECK(good(de::nn::RMSNorm_f8(dx, dr, dw, (float)eps, sum, rstd, c, s, decx::de_f8_e4m3)));
    CHECK(good(de::cuda::Quantize_f8(df, cf, sf, 128, decx::de_f8_e4m3)));
    CHECK(good(de::cuda::GEMM_f8(c, s, decx::de_f8_e4m3, cf, sf, decx::de_f8_e4m3, out)));
    CHECK(good(de::nn::RMSNorm_f8_Backward(sum, dw, rstd, ddy, dst, gw)));
    Host<float> h = download(sum), o = download(out), g = download(dst), rs = download(rstd), gws = download(gw);
    int bad = 0;
    std::vector<double> want_gw(K, 0.0), size_gw(K, 0.0);
    for (uint i = 0; i < M; ++i) {
        double ss = 0, dot = 0;
        for (uint k = 0; k < K; ++k) {
            bad += h.at(i, k) != q(x.at(i, k) + r.at(i, k));
            ss += (double)h.at(i, k) * h.at(i, k);
        }
        const double rstd_i = 1 / std::sqrt(ss / K + eps);
        bad += !(std::fabs(rs.at(0, i) - rstd_i) <= 1e-6 * rstd_i);
        std::vector<double> y(K), n(K);
        for (uint k = 0; k < K; ++k) {
            n[k] = h.at(i, k) * rstd_i;
            y[k] = n[k] * w.at(0, k);
            dot += (double)dy.at(i, k) * w.at(0, k) * n[k] / K;
            want_gw[k] += dy.at(i, k) * n[k];
            size_gw[k] += std::fabs(dy.at(i, k) * n[k]);
        }
        for (uint j = 0; j < N; ++j) {
            double want = 0, size = 0;
            for (uint k = 0; k < K; ++k) want += y[k] * f.at(j, k), size += std::fabs(y[k] * f.at(j, k));
            // each factor within half a step (2^-4) of its value, smallest ones within the blocks' tiny steps: in all under 2^-3 + 2^-8
            // of the magnitudes' sum and the tiny steps' share
            double tiny = 0;
            for (uint k = 0; k < K; ++k) tiny += (std::fabs(y[k]) + std::fabs(f.at(j, k))) * 1e-4;
            bad += !(std::fabs(o.at(i, j) - want) <= size * (0.125 + 0.00391) + tiny + std::fabs(want) * half_step);
        }
        for (uint k = 0; k < K; ++k) {
            const double gk = (double)dy.at(i, k) * w.at(0, k), want = rstd_i * (gk - n[k] * dot);
            const double size = rstd_i * (std::fabs(gk) + std::fabs(n[k] * dot));
            bad += !(std::fabs(g.at(i, k) - want) <= 1e-5 * size + std::fabs(want) * half_step * 1.001 + (half ? 3e-8 : 0));
        }
    }
    for (uint k = 0; k < K; ++k) bad += !(std::fabs(gws.at(0, k) - want_gw[k]) <= 1e-5 * size_gw[k]);
    CHECK(bad == 0);
    // in place over the gradient: the same
    CHECK(good(de::nn::RMSNorm_f8_Backward(sum, dw, rstd, ddy, ddy, gw)));
    Host<float> again = download(ddy);
    bad = 0;
    for (uint i = 0; i < M; ++i)
        for (uint k = 0; k < K; ++k) bad += again.at(i, k) != g.at(i, k);
    CHECK(bad == 0);
    de::GPU_Matrix<T>& wrong = de::CreateGPUMatrixRef<T>(K, M + 1);
    CHECK(de::nn::RMSNorm_f8(dx, wrong, dw, (float)eps, sum, rstd, c, s, 0).error_type == decx::DECX_FAIL_DimsNotMatching);
    CHECK(de::nn::RMSNorm_f8_Backward(sum, dw, rstd, wrong, dst, gw).error_type == decx::DECX_FAIL_DimsNotMatching);
    CHECK(de::nn::RMSNorm_f8_Backward(sum, dw, rstd, ddy, dst, rstd).error_type == decx::DECX_FAIL_ErrorParams);
}

static void refuses_before_init() {
    de::GPU_Matrix<float>& x = de::CreateGPUMatrixRef<float>();
    de::GPU_Matrix<uchar>& c = de::CreateGPUMatrixRef<uchar>();
    de::GPU_Matrix<float>& s = de::CreateGPUMatrixRef<float>();
    CHECK(de::cuda::Quantize_f8(x, c, s, 1, 0).error_type == decx::DECX_FAIL_not_init);
    CHECK(de::cuda::GEMM_f8(c, s, 0, c, s, 0, x).error_type == decx::DECX_FAIL_not_init);
    CHECK(de::nn::RMSNorm_f8(x, x, x, 1e-5f, x, s, c, x, 0).error_type == decx::DECX_FAIL_not_init);
}

int main(int argc, char** argv) {
    const std::string mode = argc > 1 ? argv[1] : "cpu";
    if (mode == "cpu") {
        refuses_before_init();
    } else {
        de::InitCuda();
        for (int block_rows : {1, 128}) {
            product_of_whole_numbers<float>(block_rows, false);
            product_of_whole_numbers<float>(block_rows, true);
            product_of_whole_numbers<de::Half>(block_rows, true);
        }
        norm_product_and_gradient<float>(false);
        norm_product_and_gradient<de::Half>(true);
    }
    std::printf("%s: %d failure(s)\n", mode.c_str(), g_fail);
    return g_fail ? 1 : 0;
}
