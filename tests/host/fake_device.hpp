// A stand-in for the device behind the C ABI, for tests of the DECX-named layer on the CPU: defined in the test program,
// these functions take the place of libdecx_hip.so's.  Device memory is host memory, and the 8-bit operators are plain
// arithmetic with the entry points' arguments (codes are whole numbers, not 8-bit floats).  What a call reads and writes has
// to lie in blocks that are allocated, and its results off its inputs but where decx_hip.h lets them lie over one; what does
// not is counted in fake::faults and not touched.
#pragma once
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <map>
#include <vector>

#include "../../backup_1_amd/host/DECX.h"
#include "../../include/decx_hip.h"

namespace fake {
static std::map<const char*, size_t> blocks;
static int faults = 0, calls = 0;

struct Region {
    const void* p;
    size_t rows, cols, ld, size;       // elements, bytes an element
    const char* begin() const { return static_cast<const char*>(p); }
    const char* end() const { return begin() + ((rows - 1) * ld + cols) * size; }
};
static bool allocated(const Region& r) {
    auto it = blocks.upper_bound(r.begin());
    if (!r.p || it == blocks.begin()) return false;
    --it;
    return r.end() <= it->first + it->second;
}
static bool meet(const Region& a, const Region& b) { return a.begin() < b.end() && b.begin() < a.end(); }
static bool check(const char* call, std::vector<Region> results, std::vector<Region> inputs, std::function<bool(size_t, size_t)> in_place) {
    int bad = 0;
    ++calls;
    for (const auto& r : results) bad += !allocated(r);
    for (const auto& r : inputs) bad += !allocated(r);
    for (size_t i = 0; i < results.size(); ++i) {
        for (size_t j = 0; j < inputs.size(); ++j)
            bad += meet(results[i], inputs[j]) && !(in_place(i, j) && results[i].p == inputs[j].p && results[i].ld == inputs[j].ld);
        for (size_t j = i + 1; j < results.size(); ++j) bad += meet(results[i], results[j]);
    }
    if (bad) std::printf("  %s: memory it may not use\n", call);
    faults += bad;
    return bad == 0;
}
static size_t size_of(int type) { return type == DECX_HIP_F32 ? 4 : 2; }
static float get(const void* p, size_t at, int type) {
    if (type == DECX_HIP_F32) return static_cast<const float*>(p)[at];
    return de::Half2Float(static_cast<const de::Half*>(p)[at]);
}
static void put(void* p, size_t at, int type, float v) {
    if (type == DECX_HIP_F32) static_cast<float*>(p)[at] = v;
    else static_cast<de::Half*>(p)[at] = de::Float2Half(v);
}
static int blocks_of(int n) { return (n + 127) / 128; }
}  // namespace fake

extern "C" {
int decx_hip_init(int*) { return 0; }
int decx_hip_is_init(void) { return 1; }
const char* decx_hip_last_error(void) { return "fake device\n"; }
int decx_hip_malloc(void** p, size_t bytes) {
    *p = std::calloc(1, bytes);
    fake::blocks[static_cast<char*>(*p)] = bytes;
    return 0;
}
int decx_hip_free(void* p) {
    fake::faults += fake::blocks.erase(static_cast<char*>(p)) != 1;
    std::free(p);
    return 0;
}
int decx_hip_memset(void* p, int v, size_t bytes) { return std::memset(p, v, bytes), 0; }
int decx_hip_memcpy2d(void* d, size_t dp, const void* s, size_t sp, size_t width, size_t height, int) {
    for (size_t i = 0; i < height; ++i) std::memcpy(static_cast<char*>(d) + i * dp, static_cast<const char*>(s) + i * sp, width);
    return 0;
}
int decx_hip_tmp_malloc(void** p, size_t bytes) { return decx_hip_malloc(p, bytes); }
int decx_hip_tmp_free(void* p) { return decx_hip_free(p); }

int decx_hip_f8_quantize(const void* X, int ldx, int type, int M, int K, int block_rows, int, int scale_type, uint8_t* Q, int ldq, void* S,
                         int lds, uint8_t* Qt, int ldqt, void* St, int ldst) {
    using namespace fake;
    const bool turn = Qt != nullptr;
    const int rows = turn ? K : M, cols = turn ? M : K, row_scales = block_rows == 1 ? rows : blocks_of(rows), ld = turn ? ldst : lds;
    uint8_t* codes = turn ? Qt : Q;
    void* scales = turn ? St : S;
    const size_t one = scale_type == DECX_HIP_SCALE_F32 ? 4 : 1;
    if (!check("quantize", {{codes, (size_t)rows, (size_t)cols, (size_t)(turn ? ldqt : ldq), 1}, {scales, (size_t)blocks_of(cols), (size_t)row_scales, (size_t)ld, one}},
               {{X, (size_t)M, (size_t)K, (size_t)ldx, size_of(type)}}, [](size_t, size_t) { return false; }))
        return 0;
    for (int i = 0; i < rows; ++i)
        for (int j = 0; j < cols; ++j) {
            const float v = get(X, turn ? (size_t)j * ldx + i : (size_t)i * ldx + j, type);
            codes[(size_t)i * (turn ? ldqt : ldq) + j] = (uint8_t)v;
            const size_t at = (size_t)(j / 128) * ld + i / block_rows;
            if (one == 4) static_cast<float*>(scales)[at] = std::fmax(static_cast<float*>(scales)[at], v);
            else static_cast<uint8_t*>(scales)[at] = 127;
        }
    return 0;
}
int decx_hip_f8gemm(const uint8_t* A, int lda, int, const void* SA, int ldsa, const uint8_t* B, int ldb, int, const void* SB, int ldsb,
                    int b_block_rows, int scale_type, const void*, int, void* D, int ldd, int type, int M, int N, int K) {
    using namespace fake;
    const size_t one = scale_type == DECX_HIP_SCALE_F32 ? 4 : 1, kb = (size_t)blocks_of(K);
    if (!check("f8gemm", {{D, (size_t)M, (size_t)N, (size_t)ldd, size_of(type)}},
               {{A, (size_t)M, (size_t)K, (size_t)lda, 1}, {B, (size_t)N, (size_t)K, (size_t)ldb, 1}, {SA, kb, (size_t)M, (size_t)ldsa, one},
                {SB, kb, (size_t)(b_block_rows == 1 ? N : blocks_of(N)), (size_t)ldsb, one}}, [](size_t, size_t) { return false; }))
        return 0;
    auto scale = [&](const void* s, size_t at) { return one == 4 ? static_cast<const float*>(s)[at] : (float)static_cast<const uint8_t*>(s)[at]; };
    for (int m = 0; m < M; ++m)
        for (int n = 0; n < N; ++n) {
            float v = 0;
            for (int k = 0; k < K; ++k)
                v += (float)A[(size_t)m * lda + k] * B[(size_t)n * ldb + k] * scale(SA, (size_t)(k / 128) * ldsa + m) *
                     scale(SB, (size_t)(k / 128) * ldsb + n / b_block_rows);
            put(D, (size_t)m * ldd + n, type, v);
        }
    return 0;
}
int decx_hip_rmsnorm_f8(const void* X, int ldx, const void* R, int ldr, const void* W, float eps, int type, int M, int K, void* H, int ldh,
                        float* rstd, void*, int, uint8_t* Q, int ldq, void* S, int lds, int, int) {
    using namespace fake;
    const size_t m_ = (size_t)M, k_ = (size_t)K, w = size_of(type);
    if (!check("rmsnorm_f8", {{H, m_, k_, (size_t)ldh, w}, {rstd, 1, m_, m_, 4}, {Q, m_, k_, (size_t)ldq, 1}, {S, (size_t)blocks_of(K), m_, (size_t)lds, 4}},
               {{X, m_, k_, (size_t)ldx, w}, {R, m_, k_, (size_t)ldr, w}, {W, 1, k_, k_, w}}, [](size_t i, size_t j) { return i == 0 && j < 2; }))
        return 0;
    for (int m = 0; m < M; ++m) {
        float sum = 0;
        for (int k = 0; k < K; ++k) {
            const float h = get(X, (size_t)m * ldx + k, type) + get(R, (size_t)m * ldr + k, type);
            put(H, (size_t)m * ldh + k, type, h);
            sum += h * h;
        }
        rstd[m] = 1 / std::sqrt(sum / K + eps);
        for (int k = 0; k < K; ++k) {
            const float y = get(H, (size_t)m * ldh + k, type) * get(W, (size_t)k, type);
            Q[(size_t)m * ldq + k] = (uint8_t)y;
            float& s = static_cast<float*>(S)[(size_t)(k / 128) * lds + m];
            s = k % 128 ? std::fmax(s, y) : y;
        }
    }
    return 0;
}
size_t decx_hip_rmsnorm_backward_workspace(int, int K) { return (size_t)K * 4; }
int decx_hip_rmsnorm_backward(const void* H, int ldh, const void* W, const float* rstd, const void* dY, int lddy, const void*, int, int type,
                              int M, int K, void* dX, int lddx, float* dW, void* work, size_t bytes) {
    using namespace fake;
    const size_t m_ = (size_t)M, k_ = (size_t)K, w = size_of(type);
    if (!check("rmsnorm_backward", {{dX, m_, k_, (size_t)lddx, w}, {dW, 1, k_, k_, 4}, {work, 1, bytes, bytes, 1}},
               {{H, m_, k_, (size_t)ldh, w}, {dY, m_, k_, (size_t)lddy, w}, {W, 1, k_, k_, w}, {rstd, 1, m_, m_, 4}},
               [](size_t i, size_t j) { return i == 0 && j < 2; }))
        return 0;
    for (int k = 0; k < K; ++k) dW[k] = 0;
    for (int m = 0; m < M; ++m)
        for (int k = 0; k < K; ++k) {
            const float dy = get(dY, (size_t)m * lddy + k, type), h = get(H, (size_t)m * ldh + k, type);
            dW[k] += dy * h * rstd[m];
            put(dX, (size_t)m * lddx + k, type, rstd[m] * dy * get(W, (size_t)k, type) + h);
        }
    return 0;
}
}
