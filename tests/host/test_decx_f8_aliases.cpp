// Calls of the DECX-named 8-bit operators (DECX.h) whose results name a container that the same call reads, is another result,
// or shares its block with one (operator=): each gives what the same call gives with containers of its own, or is refused.
// Usage: test_decx_f8_aliases [part] over the fake device (FAKE_DEVICE), test_decx_f8_aliases_gpu [part] over the library's.
#ifdef FAKE_DEVICE
#include "fake_device.hpp"
#endif
#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <type_traits>
#include <vector>

#include "../../backup_1_amd/host/DECX.h"

static int g_fail = 0;
#define CHECK(cond)                                                                                          \
    do {                                                                                                     \
        if (!(cond)) { std::printf("  CHECK FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); ++g_fail; }     \
    } while (0)

template <class T> static T from_float(float v) {
    if constexpr (std::is_same_v<T, de::Half>) return de::Float2Half(v);
    else return (T)v;
}
// a container of small whole numbers, 1 to 3
template <class T> static de::GPU_Matrix<T>& filled(uint w, uint h, int seed) {
    de::Matrix<T>& m = de::CreateMatrixRef<T>(w, h, 0);
    for (uint i = 0; i < h; ++i)
        for (uint j = 0; j < w; ++j) m.index((int)i, (int)j) = from_float<T>((float)(1 + (i * 5 + j * 7 + (uint)seed) % 3));
    de::GPU_Matrix<T>& d = de::CreateGPUMatrixRef<T>(w, h);
    d.Load_from_host(m);
    return d;
}
template <class T> static de::GPU_Matrix<T>& empty() { return de::CreateGPUMatrixRef<T>(); }
template <class T> static de::GPU_Matrix<T>& shared(de::GPU_Matrix<T>& of) {
    de::GPU_Matrix<T>& d = de::CreateGPUMatrixRef<T>();
    d = of;
    return d;
}
template <class T> static std::vector<T> values(de::GPU_Matrix<T>& d) {
    de::Matrix<T>& m = de::CreateMatrixRef<T>(d.Width(), d.Height(), 0);
    d.Load_to_host(m);
    std::vector<T> v;
    for (uint i = 0; i < d.Height(); ++i)
        for (uint j = 0; j < d.Width(); ++j) v.push_back(m.index((int)i, (int)j));
    return v;
}
template <class T> static bool same(de::GPU_Matrix<T>& a, de::GPU_Matrix<T>& b) {
    if (a.Width() != b.Width() || a.Height() != b.Height()) return false;
    const std::vector<T> x = values(a), y = values(b);
    return std::memcmp(x.data(), y.data(), x.size() * sizeof(T)) == 0;
}
static bool good(const de::DH& h) { return h.error_type == decx::DECX_SUCCESS; }
static bool refused(const de::DH& h) { return h.error_type == decx::DECX_FAIL_ErrorParams; }

static void quantize() {
    for (bool turn : {false, true})
        for (uint w : {300u, 1u}) {
            auto call = [&](auto& src, auto& codes, auto& scales) {
                return turn ? de::cuda::Quantize_f8_T(src, codes, scales, 1, 0) : de::cuda::Quantize_f8(src, codes, scales, 1, 0);
            };
            de::GPU_Matrix<float>&src = filled<float>(w, w == 1 ? 1 : 5, 1), &scales = empty<float>();
            de::GPU_Matrix<uchar>& codes = empty<uchar>();
            CHECK(good(call(src, codes, scales)));
            for (bool handle : {false, true}) {
                de::GPU_Matrix<float>& x = filled<float>(w, w == 1 ? 1 : 5, 1);
                de::GPU_Matrix<float>& s = handle ? shared(x) : x;
                de::GPU_Matrix<uchar>& c = empty<uchar>();
                CHECK(good(call(x, c, s)) && same(c, codes) && same(s, scales));
                CHECK(!handle || same(x, src));
            }
            // results on one block: 1 x 1 is the size for which neither is made anew
            de::GPU_Matrix<uchar>&c = filled<uchar>(1, 1, 0), &s = shared(c), &want_c = empty<uchar>(), &want_s = empty<uchar>();
            CHECK(good(call(src, want_c, want_s)) && good(call(src, c, s)) && same(c, want_c) && same(s, want_s));
            CHECK(refused(call(src, c, c)));
        }
}

// dst over either operand's scales; M = 1 and N = 1 leave a scales' container its size for some K
static void gemm() {
    for (uint M : {1u, 3u})
        for (uint N : {1u, 40u})
            for (uint K : {100u, 300u}) {
                const uint kb = (K + 127) / 128;
                de::GPU_Matrix<uchar>&a = filled<uchar>(K, M, 1), &b = filled<uchar>(K, N, 2);
                de::GPU_Matrix<float>&sa = filled<float>(M, kb, 3), &sb = filled<float>(N, kb, 4), &want = empty<float>();
                CHECK(good(de::cuda::GEMM_f8(a, sa, 0, b, sb, 0, want)) && want.Width() == N && want.Height() == M);
                for (int which : {0, 1, 2, 3}) {
                    de::GPU_Matrix<float>&pa = filled<float>(M, kb, 3), &pb = filled<float>(N, kb, 4);
                    de::GPU_Matrix<float>& over = which & 1 ? pb : pa;
                    de::GPU_Matrix<float>& dst = which & 2 ? shared(over) : over;
                    CHECK(good(de::cuda::GEMM_f8(a, pa, 0, b, pb, 0, dst)) && same(dst, want));
                    CHECK(which != 2 || (same(pa, sa) && same(pb, sb)));
                    CHECK(which != 3 || (same(pa, sa) && same(pb, sb)));
                }
                de::GPU_Matrix<float>& s1 = filled<float>(M, kb, 3);
                de::GPU_Matrix<uchar>& b1 = filled<uchar>(K, M, 2);              // one container scales both operands and takes the result
                CHECK(good(de::cuda::GEMM_f8(a, s1, 0, b1, s1, 0, s1)) && s1.Width() == M && s1.Height() == M);
            }
}

template <class T> struct NormCase {
    de::GPU_Matrix<T>&src, &residual, &weight, *sum;
    de::GPU_Matrix<float>*rstd, *scales;
    de::GPU_Matrix<uchar>& codes;
    NormCase(uint M, uint K)
        : src(filled<T>(K, M, 1)), residual(filled<T>(K, M, 2)), weight(filled<T>(K, 1, 3)), sum(&empty<T>()), rstd(&empty<float>()),
          scales(&empty<float>()), codes(empty<uchar>()) {}
    de::DH run() { return de::nn::RMSNorm_f8(src, residual, weight, 0.5f, *sum, *rstd, codes, *scales, 0); }
    bool as(NormCase& o) { return same(*sum, *o.sum) && same(*rstd, *o.rstd) && same(codes, o.codes) && same(*scales, *o.scales); }
};
template <class T> static void norm() {
    for (uint M : {1u, 4u})
        for (uint K : {1u, 4u, 300u}) {
            NormCase<T> plain(M, K);
            CHECK(good(plain.run()));
            for (bool handle : {false, true}) {
                for (int which : {0, 1, 2}) {                                  // the sum over src, residual (in place), weight
                    NormCase<T> c(M, K);
                    de::GPU_Matrix<T>& over = which == 0 ? c.src : which == 1 ? c.residual : c.weight;
                    c.sum = handle ? &shared(over) : &over;
                    CHECK(good(c.run()) && c.as(plain));
                    CHECK(which != 2 || !handle || same(c.weight, plain.weight));
                }
                if constexpr (std::is_same_v<T, float>)
                    for (int result : {0, 1})                                  // rstd, the scales over each of the matrices
                        for (int which : {0, 1, 2}) {
                            NormCase<T> c(M, K);
                            de::GPU_Matrix<T>& over = which == 0 ? c.src : which == 1 ? c.residual : c.weight;
                            (result ? c.scales : c.rstd) = handle ? &shared(over) : &over;
                            CHECK(good(c.run()) && c.as(plain));
                            CHECK(!handle || same(over, which == 0 ? plain.src : which == 1 ? plain.residual : plain.weight));
                        }
            }
            if constexpr (std::is_same_v<T, float>) {
                for (int which : {0, 1}) {                                     // two results of one container, or on one block
                    NormCase<T> c(M, K), d(M, K);
                    (which ? c.scales : c.rstd) = c.sum;
                    CHECK(refused(c.run()));
                    d.sum = &filled<float>(K, M, 5);
                    (which ? d.scales : d.rstd) = &shared(*d.sum);
                    CHECK(good(d.run()) && d.as(plain));
                }
            }
            NormCase<T> c(M, K), d(M, K);
            c.scales = c.rstd;
            CHECK(refused(c.run()));
            d.rstd = &filled<float>(M, 1, 5);
            d.scales = &shared(*d.rstd);
            CHECK(good(d.run()) && d.as(plain));
        }
}

template <class T> struct BackwardCase {
    de::GPU_Matrix<T>&sum, &weight, &grad, *dst;
    de::GPU_Matrix<float>&rstd, *grad_weight;
    BackwardCase(uint M, uint K)
        : sum(filled<T>(K, M, 1)), weight(filled<T>(K, 1, 2)), grad(filled<T>(K, M, 3)), dst(&empty<T>()), rstd(filled<float>(M, 1, 4)),
          grad_weight(&empty<float>()) {}
    de::DH run() { return de::nn::RMSNorm_f8_Backward(sum, weight, rstd, grad, *dst, *grad_weight); }
    // dst bit for bit; dW's parts may be added in another order where dst lies over an input: whole numbers, so the same but for rstd's
    bool as(BackwardCase& o) {
        const std::vector<float> x = values(*grad_weight), y = values(*o.grad_weight);
        bool near = x.size() == y.size();
        for (size_t i = 0; near && i < x.size(); ++i) near = std::fabs(x[i] - y[i]) <= 1e-6f * std::fabs(y[i]);
        return same(*dst, *o.dst) && near;
    }
};
template <class T> static void backward() {
    for (uint M : {1u, 4u})
        for (uint K : {1u, 4u, 300u}) {
            BackwardCase<T> plain(M, K);
            CHECK(good(plain.run()));
            for (bool handle : {false, true}) {
                for (int which : {0, 1, 2}) {                                  // dst over grad, sum (in place), weight
                    BackwardCase<T> c(M, K);
                    de::GPU_Matrix<T>& over = which == 0 ? c.grad : which == 1 ? c.sum : c.weight;
                    c.dst = handle ? &shared(over) : &over;
                    CHECK(good(c.run()) && c.as(plain));
                    CHECK(which != 2 || !handle || same(c.weight, plain.weight));
                }
                BackwardCase<T> r(M, K);
                r.grad_weight = handle ? &shared(r.rstd) : &r.rstd;
                CHECK(refused(r.run()));
                if constexpr (std::is_same_v<T, float>) {
                    BackwardCase<T> d(M, K);
                    d.dst = handle ? &shared(d.rstd) : &d.rstd;
                    CHECK(good(d.run()) && d.as(plain));
                    for (int which : {0, 1, 2}) {                              // the weight's gradient over each of the matrices
                        BackwardCase<T> c(M, K);
                        de::GPU_Matrix<T>& over = which == 0 ? c.grad : which == 1 ? c.sum : c.weight;
                        c.grad_weight = handle ? &shared(over) : &over;
                        CHECK(good(c.run()) && c.as(plain));
                        CHECK(!handle || same(over, which == 0 ? plain.grad : which == 1 ? plain.sum : plain.weight));
                    }
                }
            }
            if constexpr (std::is_same_v<T, float>) {
                BackwardCase<T> c(M, K), d(M, K);
                c.grad_weight = c.dst;
                CHECK(refused(c.run()));
                d.dst = &filled<float>(K, M, 5);
                d.grad_weight = &shared(*d.dst);
                CHECK(good(d.run()) && d.as(plain));
            }
        }
}

int main(int argc, char** argv) {
    const std::string only = argc > 1 ? argv[1] : "";
    de::InitCuda();
    struct { const char* name; void (*run)(); } parts[] = {{"quantize", quantize}, {"gemm", gemm}, {"norm", [] { norm<float>(); norm<de::Half>(); }},
                                                           {"backward", [] { backward<float>(); backward<de::Half>(); }}};
    for (auto& part : parts) {
        if (!only.empty() && only != part.name) continue;
        const int before = g_fail;
        part.run();
#ifdef FAKE_DEVICE
        CHECK(fake::faults == 0 && fake::calls > 0);
        fake::faults = fake::calls = 0;
#endif
        std::printf("%s: %d failure(s)\n", part.name, g_fail - before);
        std::fflush(stdout);
    }
    return g_fail ? 1 : 0;
}
