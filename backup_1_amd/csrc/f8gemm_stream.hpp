// Scaled 8-bit product for few rows (a token, a batch of requests) and for operands that the LDS-DMA tiles cannot take.
//
// Bound: reading B.  A workgroup owns 16 MI x 16 NI results; its waves take the blocks of K in turn (wave w the blocks w,
// w + WAVES, ...), each straight from global memory into registers -- nothing is shared between waves until the end, so there
// is no barrier in the walk and every wave keeps DEPTH blocks of loads in flight.  Then the waves' sums meet in LDS and are
// added in wave order: the same bits on every run, without a workspace and in one launch.
#pragma once
#include "f8gemm_common.hpp"

namespace decx_hip {

template <int MI_, int NI_, int WAVES_, int DEPTH_>
struct F8StreamShape {
    static constexpr int MI = MI_, NI = NI_, WAVES = WAVES_, DEPTH = DEPTH_, NT = WAVES * kWave;
    static constexpr int BM = 16 * MI, BN = 16 * NI;
    static constexpr size_t LDS_BYTES = (size_t)WAVES * MI * NI * kWave * 16;
};

template <class S, class F>
__global__ __launch_bounds__(S::NT) void f8gemm_stream_kernel(const F8GemmArgs g) {
    constexpr int MI = S::MI, NI = S::NI, WAVES = S::WAVES, DEPTH = S::DEPTH;
    constexpr bool IN_INSTRUCTION = F::IN_INSTRUCTION, B_PER_ROW = F::B_PER_ROW;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const int lg = lane >> 4, li = lane & 15;
    const TileCoord tc = xcd_grouped_tile(blockIdx.x, g.tiles_m, g.tiles_n, g.group_m);
    const int bm0 = tc.tm * S::BM, bn0 = tc.tn * S::BN;

    // rows and columns past the end repeat the last one and are never stored
    const uint8_t* a_row[MI];
    const uint8_t* b_row[NI];
    int sa_at[MI], sb_at[NI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        const int m = bm0 + 16 * mi + li, mc = m < g.M ? m : g.M - 1;
        a_row[mi] = g.A + (size_t)mc * g.lda + 16 * lg;
        sa_at[mi] = mc;
    }
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
        const int n = bn0 + 16 * ni + li, nc = n < g.N ? n : g.N - 1;
        b_row[ni] = g.B + (size_t)nc * g.ldb + 16 * lg;
        sb_at[ni] = IN_INSTRUCTION ? nc >> g.b_shift : (bn0 + 16 * ni < g.N ? bn0 + 16 * ni : g.N - 1) >> g.b_shift;
    }

    f32x4 acc[MI][NI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Block {
        i32x8 a[MI], b[NI];
        float fa[MI], fb[NI][B_PER_ROW ? 4 : 1];
        int ea[MI], eb[NI];
    };
    auto scale = [&](const void* scales, size_t at) -> float {
        if constexpr (F::E8M0) return e8m0_value(static_cast<const uint8_t*>(scales)[at]);
        else return static_cast<const float*>(scales)[at];
    };
    auto load_scales = [&](Block& x, int kb) {
        const size_t at_a = (size_t)kb * g.ldsa, at_b = (size_t)kb * g.ldsb;
        if constexpr (IN_INSTRUCTION) {
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) x.ea[mi] = static_cast<const uint8_t*>(g.SA)[at_a + sa_at[mi]];
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) x.eb[ni] = static_cast<const uint8_t*>(g.SB)[at_b + sb_at[ni]];
        } else {
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) x.fa[mi] = scale(g.SA, at_a + sa_at[mi]);
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                if constexpr (B_PER_ROW) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int n = bn0 + 16 * ni + 4 * lg + e;
                        x.fb[ni][e] = scale(g.SB, at_b + (n < g.N ? n : g.N - 1));
                    }
                } else {
                    x.fb[ni][0] = scale(g.SB, at_b + sb_at[ni]);
                }
            }
        }
    };
    auto load_whole = [&](Block& x, int kb) {
        const size_t at = (size_t)kb * kScaleBlock;
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
            x.b[ni] = f8_fragment(*reinterpret_cast<const u32x4_any*>(b_row[ni] + at), *reinterpret_cast<const u32x4_any*>(b_row[ni] + at + 64));
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
            x.a[mi] = f8_fragment(*reinterpret_cast<const u32x4_any*>(a_row[mi] + at), *reinterpret_cast<const u32x4_any*>(a_row[mi] + at + 64));
        load_scales(x, kb);
    };
    auto multiply = [&](const Block& x) {
        if constexpr (IN_INSTRUCTION) {
#pragma unroll
            for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                for (int ni = 0; ni < NI; ++ni)
                    acc[mi][ni] = f8_mfma_scaled<F::FA, F::FB>(x.b[ni], x.a[mi], acc[mi][ni], x.eb[ni], x.ea[mi]);
        } else {
            F16Fragment wide_b[NI];
            if constexpr (F::EXACT) {
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) wide_b[ni] = f8_widen<F::FB>(x.b[ni]);
            }
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) {
                F16Fragment wide_a;
                if constexpr (F::EXACT) wide_a = f8_widen<F::FA>(x.a[mi]);
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) {
                    f32x4 p;
                    if constexpr (F::EXACT) p = f8_mfma_exact(wide_b[ni], wide_a);
                    else p = f8_mfma<F::FA, F::FB>(x.b[ni], x.a[mi], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[mi][ni][e] = __builtin_fmaf(p[e], x.fa[mi] * x.fb[ni][B_PER_ROW ? e : 0], acc[mi][ni][e]);
                }
            }
        }
    };

    const int whole = g.K / kScaleBlock;
    int kb = wave;
    for (; kb + (DEPTH - 1) * WAVES < whole; kb += DEPTH * WAVES) {
        Block x[DEPTH];
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) load_whole(x[d], kb + d * WAVES);
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) multiply(x[d]);
    }
    for (; kb < whole; kb += WAVES) {
        Block x;
        load_whole(x, kb);
        multiply(x);
    }
    if (whole * kScaleBlock < g.K && kb == whole) {             // the wave whose turn it is takes the ragged last block
        Block x;
        const size_t at = (size_t)whole * kScaleBlock;
        const int n = g.K - whole * kScaleBlock - 16 * lg;
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) x.b[ni] = f8_fragment(f8_unit_part(b_row[ni] + at, n), f8_unit_part(b_row[ni] + at + 64, n - 64));
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) x.a[mi] = f8_fragment(f8_unit_part(a_row[mi] + at, n), f8_unit_part(a_row[mi] + at + 64, n - 64));
        load_scales(x, whole);
        multiply(x);
    }

    // ---- the waves' sums meet, in wave order
    f32x4* sums = reinterpret_cast<f32x4*>(lds_raw);            // [wave][block of 16 x 16][lane]
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) sums[(wave * MI * NI + mi * NI + ni) * kWave + lane] = acc[mi][ni];
    __syncthreads();
    for (int blk = wave; blk < MI * NI; blk += WAVES) {
        f32x4 v = sums[blk * kWave + lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v += sums[(w * MI * NI + blk) * kWave + lane];
        f8_store_result(g, bm0 + 16 * (blk / NI) + li, bn0 + 16 * (blk % NI) + 4 * lg, v);
    }
}

}  // namespace decx_hip
