// Scaled 8-bit products: argument checks, the kernel choice, and the pairing of formats.
#include "f8gemm_common.hpp"

#include <cmath>

namespace decx_hip {

// The kernel for a product, as the number decx_hip_set_f8gemm_variant would force it with:
//   1 - 4: 16 x 16, 32 x 16, 64 x 32, 64 x 64 results a workgroup straight from memory (f8gemm_stream.hpp); 4 not for exact
//          sums, whose fragments leave it no registers (3 instead)
//   5: 128 x 128 LDS-DMA tiles (f8gemm_tile.hpp), 6: 256 x 256; both need `aligned` operands, the latter not the exact sums
//      of fp32 results nor an fp32 scale for each row of B
// The cheapest by a model of what was measured on an MI355X, in us:
//   1 - 4: a CU takes in 81 KB a us, a workgroup's share of A and B, once 1.5 us have passed, and again (at most 1.5 us) for
//          each of the workgroups that a CU has after each other (exact sums a third more, an fp32 scale for each row of B half more in 4); and B passes
//          through at 6.5 MB a us at most
//   5: 0.64 a block of K while a CU has one tile, 1 for two; exact sums 1.15 and 2.2
//   6: 1.05 a block of K on a nearly empty chip to 1.47 on a full one
//   plus 2.4 (1 - 4), 3 and half of the store (5) and 7 to 11 (6) for the launch, the first loads and the store.
// On 74 shapes from 1 x 4096 x 4096 to 4096^3, bf16 and fp32 results: within 5 % of the best kernel on all but three, 9 to 14 %
// on those (profiles/f8gemm_choice_sweep.txt has every kernel's time).
static int plan_f8gemm(int M, int N, int K, int type, int scale_type, int b_block_rows, bool aligned, bool large) {
    const int forced = g_rt.f8gemm_variant;
    if ((forced >= 1 && forced <= 4) || (forced == 5 && aligned) || (forced == 6 && aligned && large)) return forced;
    const double cus = g_rt.compute_units > 0 ? g_rt.compute_units : 256;
    const double blocks = cdiv(K, kScaleBlock);
    const bool exact = type == DECX_HIP_F32, row_scales = !exact && scale_type == DECX_HIP_SCALE_F32 && b_block_rows == 1;
    static const int MI[4] = {1, 2, 4, 4}, NI[4] = {1, 1, 2, 4};
    int best = 1;
    double least = 0;
    for (int v = 1; v <= (exact ? 3 : 4); ++v) {
        const int mi = MI[v - 1], ni = NI[v - 1];
        const double rounds = std::ceil((double)cdiv(M, 16 * mi) * cdiv(N, 16 * ni) / cus), slower = exact ? 1.35 : row_scales && v == 4 ? 1.5 : 1.0;
        const double share = (mi + ni) * 16.0 * K * slower / 81e3, passed = (double)N * K / 6.5e6;
        const double taken = 1.5 + rounds * share + (rounds - 1) * (share < 1.5 ? share : 1.5);
        const double cost = 2.4 + (taken > passed ? taken : passed);
        if (v == 1 || cost < least) best = v, least = cost;
    }
    if (!aligned) return best;
    const double small = (double)cdiv(M, 128) * cdiv(N, 128), big = (double)cdiv(M, 256) * cdiv(N, 256);
    const double store = 0.5 * (double)M * N * (exact ? 4 : 2) / 5e6;
    const double cost5 = 3.0 + store + blocks * (small <= cus ? (exact ? 1.15 : 0.64) : std::ceil(small / (2 * cus)) * (exact ? 2.2 : 1.0));
    if (cost5 < least) best = 5, least = cost5;
    const double fill = big < cus ? big / cus : 1.0;
    const double cost6 = 7.0 + 4.0 * fill + blocks * std::ceil(big / cus) * (1.05 + 0.42 * fill);
    if (large && cost6 < least) best = 6;
    return best;
}
static bool f8gemm_pitches_fit(long lda, long ldb) { return lda % 16 == 0 && ldb % 16 == 0 && lda < (1L << 24) && ldb < (1L << 24); }
static bool f8gemm_large_fits(int type, int scale_type, int b_block_rows) {
    return type != DECX_HIP_F32 && (scale_type == DECX_HIP_SCALE_E8M0 || b_block_rows != 1);
}
int f8gemm_plan(int M, int N, int K, int type, int scale_type, int b_block_rows, long lda, long ldb, bool aligned) {
    return plan_f8gemm(M, N, K, type, scale_type, b_block_rows, aligned && f8gemm_pitches_fit(lda, ldb), f8gemm_large_fits(type, scale_type, b_block_rows));
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
    if (M > kMostExtent || N > kMostExtent || K > kMostExtent) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "problem too large for one launch\n");
    if (int rc = check_f8_codes(type, format_a, scale_type)) return rc;
    if (int rc = check_f8_codes(type, format_b, scale_type)) return rc;
    if (b_block_rows != 1 && b_block_rows != kScaleBlock) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "a block has 1 or 128 rows\n");
    if (lda < K || ldb < K || ldd < N || (Cin && ldc < N) || ldsa < M || ldsb < (b_block_rows == 1 ? N : cdiv(N, kScaleBlock)))
        return fail(DECX_HIP_FAIL_ERROR_PARAMS, "leading dimension smaller than the row length\n");
    if (int rc = check_element_alignment(D, type)) return rc;
    if (int rc = check_element_alignment(Cin, type)) return rc;
    if (scale_type == DECX_HIP_SCALE_F32 && ((reinterpret_cast<uintptr_t>(SA) | reinterpret_cast<uintptr_t>(SB)) & 3u))
        return fail(DECX_HIP_FAIL_ERROR_PARAMS, "scales off the grid of their type\n");
    const size_t m = (size_t)M, n = (size_t)N, k = (size_t)K, wide = element_size(type), one = scale_size(scale_type), blocks = cdiv(K, kScaleBlock);
    if (int rc = check_results({{operand(D, m, n, ldd, wide), 1u}},
                               {operand(Cin, m, n, ldc, wide), operand(A, m, k, lda, 1), operand(B, n, k, ldb, 1), operand(SA, blocks, m, ldsa, one),
                                operand(SB, blocks, b_block_rows == 1 ? N : cdiv(N, kScaleBlock), ldsb, one)}))
        return rc;
    F8GemmArgs g = {};
    g.A = A, g.B = B, g.SA = SA, g.SB = SB, g.C = Cin, g.D = D;
    g.lda = (size_t)lda, g.ldb = (size_t)ldb, g.ldsa = (size_t)ldsa, g.ldsb = (size_t)ldsb, g.ldc = (size_t)ldc, g.ldd = (size_t)ldd;
    g.b_shift = b_block_rows == 1 ? 0 : 7;
    g.type = type, g.M = M, g.N = N, g.K = K;
    g.variant = plan_f8gemm(M, N, K, type, scale_type, b_block_rows, aligned16(A) && aligned16(B) && f8gemm_pitches_fit(lda, ldb), f8gemm_large_fits(type, scale_type, b_block_rows));
    const bool e8m0 = scale_type == DECX_HIP_SCALE_E8M0;
    if (format_a == DECX_HIP_E4M3)
        return format_b == DECX_HIP_E4M3 ? f8gemm_launch_e4m3_e4m3(g, e8m0) : f8gemm_launch_e4m3_e5m2(g, e8m0);
    return format_b == DECX_HIP_E4M3 ? f8gemm_launch_e5m2_e4m3(g, e8m0) : f8gemm_launch_e5m2_e5m2(g, e8m0);
}

}  // namespace decx_hip
