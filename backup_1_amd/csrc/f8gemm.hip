// Scaled 8-bit products: argument checks, kernel choice and launch.
#include "f8gemm_stream.hpp"

namespace decx_hip {

typedef F8StreamShape<1, 1, 8, 4> F8Token;         // a token to 16 rows
typedef F8StreamShape<4, 2, 8, 1> F8Rows;

template <class S, class F>
static int launch_f8gemm_stream(F8GemmArgs g) {
    auto kern = f8gemm_stream_kernel<S, F>;
    g.tiles_m = cdiv(g.M, S::BM), g.tiles_n = cdiv(g.N, S::BN);
    const long total = (long)g.tiles_m * g.tiles_n;
    if (total > 0x7fffffffL) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "problem too large for one launch\n");
    g.group_m = g.tiles_m < g_rt.group_m ? g.tiles_m : g_rt.group_m;
    hipLaunchKernelGGL(kern, dim3((unsigned)total), dim3(S::NT), S::LDS_BYTES, g_rt.stream, g);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <class F>
static int launch_f8gemm(const F8GemmArgs& g) {
    if (g.M <= 16) return launch_f8gemm_stream<F8Token, F>(g);
    return launch_f8gemm_stream<F8Rows, F>(g);
}
template <int FA, int FB>
static int launch_f8gemm_kind(const F8GemmArgs& g, bool e8m0) {
    if (g.type != DECX_HIP_F32) {
        if (e8m0) return launch_f8gemm<F8Kind<FA, FB, true, false, false>>(g);
        return g.b_shift ? launch_f8gemm<F8Kind<FA, FB, false, false, false>>(g) : launch_f8gemm<F8Kind<FA, FB, false, true, false>>(g);
    }
    if (e8m0) return g.b_shift ? launch_f8gemm<F8Kind<FA, FB, true, false, true>>(g) : launch_f8gemm<F8Kind<FA, FB, true, true, true>>(g);
    return g.b_shift ? launch_f8gemm<F8Kind<FA, FB, false, false, true>>(g) : launch_f8gemm<F8Kind<FA, FB, false, true, true>>(g);
}

int f8gemm_enqueue(const uint8_t* A, int lda, int format_a, const void* SA, int ldsa, const uint8_t* B, int ldb, int format_b,
                   const void* SB, int ldsb, int b_block_rows, int scale_type, const void* Cin, int ldc, void* D, int ldd, int type, int M,
                   int N, int K) {
    if (int rc = need_library_device()) return rc;
    if (!A || !B || !SA || !SB || !D) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "null matrix pointer\n");
    if (M <= 0 || N <= 0 || K <= 0) return fail(DECX_HIP_FAIL_DIMS, "Matrix Dims don't match each other");
    if (int rc = check_f8_codes(type, format_a, scale_type)) return rc;
    if (int rc = check_f8_codes(type, format_b, scale_type)) return rc;
    if (b_block_rows != 1 && b_block_rows != kScaleBlock) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "a block has 1 or 128 rows\n");
    if (lda < K || ldb < K || ldd < N || (Cin && ldc < N) || ldsa < M || ldsb < (b_block_rows == 1 ? N : cdiv(N, kScaleBlock)))
        return fail(DECX_HIP_FAIL_ERROR_PARAMS, "leading dimension smaller than the row length\n");
    if (int rc = check_element_alignment(D, type)) return rc;
    if (int rc = check_element_alignment(Cin, type)) return rc;
    if (scale_type == DECX_HIP_SCALE_F32 && ((reinterpret_cast<uintptr_t>(SA) | reinterpret_cast<uintptr_t>(SB)) & 3u))
        return fail(DECX_HIP_FAIL_ERROR_PARAMS, "scales off the grid of their type\n");
    F8GemmArgs g = {};
    g.A = A, g.B = B, g.SA = SA, g.SB = SB, g.C = Cin, g.D = D;
    g.lda = (size_t)lda, g.ldb = (size_t)ldb, g.ldsa = (size_t)ldsa, g.ldsb = (size_t)ldsb, g.ldc = (size_t)ldc, g.ldd = (size_t)ldd;
    g.b_shift = b_block_rows == 1 ? 0 : 7;
    g.type = type, g.M = M, g.N = N, g.K = K;
    const bool e8m0 = scale_type == DECX_HIP_SCALE_E8M0;
    if (format_a == DECX_HIP_E4M3)
        return format_b == DECX_HIP_E4M3 ? launch_f8gemm_kind<0, 0>(g, e8m0) : launch_f8gemm_kind<0, 1>(g, e8m0);
    return format_b == DECX_HIP_E4M3 ? launch_f8gemm_kind<1, 0>(g, e8m0) : launch_f8gemm_kind<1, 1>(g, e8m0);
}

}  // namespace decx_hip
