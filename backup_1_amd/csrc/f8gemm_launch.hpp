// Launch of the scaled 8-bit products' kernels for one pairing of formats: each pairing's kernels are compiled in a
// translation unit of their own (f8gemm_e4m3_e4m3.hip and its three siblings).
#pragma once
#include "f8gemm_stream.hpp"
#include "f8gemm_tile.hpp"

namespace decx_hip {

typedef F8StreamShape<1, 1, 8, 2> F8Stream16x16;
typedef F8StreamShape<2, 1, 8, 2> F8Stream32x16;
typedef F8StreamShape<4, 2, 8, 1> F8Stream64x32;
typedef F8StreamShape<4, 4, 8, 1> F8Stream64x64;
typedef F8TileShape<128, 128, 2, 2> F8TileSmall;   // 4 waves of 64 x 64, two workgroups a CU
typedef F8TileShape<256, 256, 2, 4> F8TileLarge;   // 8 waves of 128 x 64, two a SIMD

template <class S, class F>
static int launch_f8gemm_tile(F8GemmArgs g) {
    auto kern = f8gemm_tile_kernel<S, F>;
    static bool attr_done = false;
    if (!attr_done) {
        HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)S::LDS_BYTES));
        attr_done = true;
    }
    g.tiles_m = cdiv(g.M, S::BM), g.tiles_n = cdiv(g.N, S::BN);
    const long total = (long)g.tiles_m * g.tiles_n;
    if (total * S::NT > kMostThreads) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "problem too large for one launch\n");
    // raster groups 6 tile rows tall: an XCD's 32 tiles then share the fewest panels.  8192 x 8192 x 2048 119.8 us (8 rows 128.0, 4
    // 120.5, 12 121.7); 8192^3 388 to 391 (389 to 394, 384 to 387, 389 to 393); on seven sizes from 1024 x 4096 x 4096 to 8192 x 2048
    // x 4096, all types, the four are within 2 %, and groups of 2 up to 5 % slower.
    const int group_m = g_rt.group_m_or(6);
    g.group_m = g.tiles_m < group_m ? g.tiles_m : group_m;
    hipLaunchKernelGGL(kern, dim3((unsigned)total), dim3(S::NT), S::LDS_BYTES, g_rt.stream, g);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <class S, class F>
static int launch_f8gemm_stream(F8GemmArgs g) {
    auto kern = f8gemm_stream_kernel<S, F>;
    static bool attr_done = false;
    if (!attr_done) {
        HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)S::LDS_BYTES));
        attr_done = true;
    }
    g.tiles_m = cdiv(g.M, S::BM), g.tiles_n = cdiv(g.N, S::BN);
    const long total = (long)g.tiles_m * g.tiles_n;
    if (total * S::NT > kMostThreads) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "problem too large for one launch\n");
    g.group_m = g.tiles_m < g_rt.group_m ? g.tiles_m : g_rt.group_m;
    hipLaunchKernelGGL(kern, dim3((unsigned)total), dim3(S::NT), S::LDS_BYTES, g_rt.stream, g);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <class F>
static int launch_f8gemm(const F8GemmArgs& g) {
    switch (g.variant) {
        case 1: return launch_f8gemm_stream<F8Stream16x16, F>(g);
        case 2: return launch_f8gemm_stream<F8Stream32x16, F>(g);
        case 3: return launch_f8gemm_stream<F8Stream64x32, F>(g);
        case 4:
            if constexpr (!F::EXACT) return launch_f8gemm_stream<F8Stream64x64, F>(g);
            return launch_f8gemm_stream<F8Stream64x32, F>(g);
        case 5: return launch_f8gemm_tile<F8TileSmall, F>(g);
        default:
            if constexpr (!F::EXACT && !F::B_PER_ROW) return launch_f8gemm_tile<F8TileLarge, F>(g);
            return launch_f8gemm_tile<F8TileSmall, F>(g);
    }
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

}  // namespace decx_hip
