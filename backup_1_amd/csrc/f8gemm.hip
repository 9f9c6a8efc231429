// Scaled 8-bit products: argument checks, the kernel choice, and the pairing of formats.
#include "f8gemm_common.hpp"

namespace decx_hip {

// The kernel for a product, as the number decx_hip_set_f8gemm_variant would force it with:
//   1: 16 x 16 results a workgroup straight from memory (f8gemm_stream.hpp), 2: 64 x 32
//   3: 128 x 128 LDS-DMA tiles (f8gemm_tile.hpp), 4: 256 x 256; both need `aligned` operands, the latter not the exact sums
//      of fp32 results nor an fp32 scale for each row of B
static int plan_f8gemm(int M, int N, bool aligned, bool large) {
    const int forced = g_rt.f8gemm_variant;
    if (forced == 1 || forced == 2 || (forced == 3 && aligned) || (forced == 4 && aligned && large)) return forced;
    if (aligned && M > 64 && (long)cdiv(M, 128) * cdiv(N, 128) >= 64) return large && (long)cdiv(M, 256) * cdiv(N, 256) >= 128 ? 4 : 3;
    return M <= 16 ? 1 : 2;
}
static bool f8gemm_pitches_fit(long lda, long ldb) { return lda % 16 == 0 && ldb % 16 == 0 && lda < (1L << 24) && ldb < (1L << 24); }
static bool f8gemm_large_fits(int type, int scale_type, int b_block_rows) {
    return type != DECX_HIP_F32 && (scale_type == DECX_HIP_SCALE_E8M0 || b_block_rows != 1);
}
int f8gemm_plan(int M, int N, int type, int scale_type, int b_block_rows, long lda, long ldb, bool aligned) {
    return plan_f8gemm(M, N, aligned && f8gemm_pitches_fit(lda, ldb), f8gemm_large_fits(type, scale_type, b_block_rows));
}

// one translation unit each
int f8gemm_launch_e4m3_e4m3(const F8GemmArgs& g, bool e8m0);
int f8gemm_launch_e4m3_e5m2(const F8GemmArgs& g, bool e8m0);
int f8gemm_launch_e5m2_e4m3(const F8GemmArgs& g, bool e8m0);
int f8gemm_launch_e5m2_e5m2(const F8GemmArgs& g, bool e8m0);

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
    g.variant = plan_f8gemm(M, N, aligned16(A) && aligned16(B) && f8gemm_pitches_fit(lda, ldb), f8gemm_large_fits(type, scale_type, b_block_rows));
    const bool e8m0 = scale_type == DECX_HIP_SCALE_E8M0;
    if (format_a == DECX_HIP_E4M3)
        return format_b == DECX_HIP_E4M3 ? f8gemm_launch_e4m3_e4m3(g, e8m0) : f8gemm_launch_e4m3_e5m2(g, e8m0);
    return format_b == DECX_HIP_E4M3 ? f8gemm_launch_e5m2_e4m3(g, e8m0) : f8gemm_launch_e5m2_e5m2(g, e8m0);
}

}  // namespace decx_hip
