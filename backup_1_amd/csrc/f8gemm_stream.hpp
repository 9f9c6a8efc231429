// Scaled 8-bit product for few rows (a token, a batch of requests), for results of too few tiles to fill the chip, and for
// operands that the LDS-DMA tiles cannot take (any alignment, any pitch).
//
// Bound: reading B, and what a CU can take in.  A workgroup owns 16 MI x 16 NI results; its waves take the blocks of K in
// turn (wave w the blocks w, w + WAVES, ...), from global memory into registers -- nothing is shared between waves until the
// end, so there is no barrier in the walk and every wave keeps DEPTH blocks of loads in flight.  Then the waves' sums meet in
// LDS and are added in wave order: the same bits on every run, without a workspace and in one launch.
//
// A load takes whole lines: 8 rows x 128 bytes, lane -> (row lane / 8, unit lane % 8).  In the matrix instruction's own order
// (row lane % 16, 16 lines touched by each load) a CU took in 14 bytes a clock, whatever the depth, half or less of this:
// 48 x 8192 x 4096 12.1 us against 8.1, 1 x 1024 x 8192 6.8 against 4.4.  The fragments get into that order through 2 KB of
// LDS that only the wave itself touches: LDS operations of a wave are carried out in order, so it needs no barrier.
#pragma once
#include "f8gemm_common.hpp"

namespace decx_hip {

template <int MI_, int NI_, int WAVES_, int DEPTH_>
struct F8StreamShape {
    static constexpr int MI = MI_, NI = NI_, WAVES = WAVES_, DEPTH = DEPTH_, NT = WAVES * kWave;
    static constexpr int BM = 16 * MI, BN = 16 * NI;
    static constexpr size_t TURN_BYTES = 16 * kScaleBlock, SUM_BYTES = (size_t)MI * NI * kWave * 16;     // of a wave, one after the other
    static constexpr size_t LDS_BYTES = WAVES * (TURN_BYTES > SUM_BYTES ? TURN_BYTES : SUM_BYTES);
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
    const int line = lane >> 3, unit = lane & 7;                // of a load
    const uint8_t* a_at[MI][2];
    const uint8_t* b_at[NI][2];
    int sa_at[MI], sb_at[NI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int m = bm0 + 16 * mi + 8 * h + line;
            a_at[mi][h] = g.A + (size_t)(m < g.M ? m : g.M - 1) * g.lda + 16 * unit;
        }
        sa_at[mi] = bm0 + 16 * mi + li < g.M ? bm0 + 16 * mi + li : g.M - 1;
    }
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int n = bn0 + 16 * ni + 8 * h + line;
            b_at[ni][h] = g.B + (size_t)(n < g.N ? n : g.N - 1) * g.ldb + 16 * unit;
        }
        const int n = bn0 + 16 * ni + (IN_INSTRUCTION ? li : 0);
        sb_at[ni] = (n < g.N ? n : g.N - 1) >> g.b_shift;
    }

    f32x4 acc[MI][NI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Block {
        u32x4 a[MI][2], b[NI][2];                               // as loaded: lines
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
    auto load_block = [&](Block& x, int kb, auto ragged_tag) {
        const size_t at = (size_t)kb * kScaleBlock;
        const int left = g.K - kb * kScaleBlock - 16 * unit;    // codes of this lane's unit and after it
        auto load = [&](const uint8_t* p) -> u32x4 {
            if constexpr (decltype(ragged_tag)::value) return f8_unit_part(p, left, g.K - left);
            else return *reinterpret_cast<const u32x4_any*>(p);
        };
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
#pragma unroll
            for (int h = 0; h < 2; ++h) x.b[ni][h] = load(b_at[ni][h] + at);
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int h = 0; h < 2; ++h) x.a[mi][h] = load(a_at[mi][h] + at);
        load_scales(x, kb);
    };
    // 16 lines into a fragment: unit q of row r lies in slot q ^ (r % 8), which keeps the writes and the reads free of conflicts
    unsigned char* const turn = lds_raw + (size_t)wave * S::TURN_BYTES;
    unsigned char* const turn_in = turn + line * kScaleBlock + ((unit ^ line) << 4);
    const unsigned char* const turn_out = turn + li * kScaleBlock + ((lg ^ (li & 7)) << 4);
    const unsigned char* const turn_out4 = turn + li * kScaleBlock + (((lg + 4) ^ (li & 7)) << 4);
    auto fragment = [&](const u32x4 (&lines)[2]) -> i32x8 {
        asm volatile("" ::: "memory");                          // in this order: the lanes exchange what they hold
        *reinterpret_cast<u32x4*>(turn_in) = lines[0];
        *reinterpret_cast<u32x4*>(turn_in + 8 * kScaleBlock) = lines[1];
        asm volatile("" ::: "memory");
        const u32x4 lo = *reinterpret_cast<const u32x4*>(turn_out), hi = *reinterpret_cast<const u32x4*>(turn_out4);
        asm volatile("" ::: "memory");
        return f8_fragment(lo, hi);
    };
    auto multiply = [&](const Block& x) {
        i32x8 b[NI];
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) b[ni] = fragment(x.b[ni]);
        F16Fragment wide_b[NI];
        if constexpr (F::EXACT) {
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) wide_b[ni] = f8_widen<F::FB>(b[ni]);
        }
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
            const i32x8 a = fragment(x.a[mi]);
            F16Fragment wide_a;
            if constexpr (F::EXACT) wide_a = f8_widen<F::FA>(a);
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                if constexpr (IN_INSTRUCTION) {
                    acc[mi][ni] = f8_mfma_scaled<F::FA, F::FB>(b[ni], a, acc[mi][ni], x.eb[ni], x.ea[mi]);
                } else {
                    f32x4 p;
                    if constexpr (F::EXACT) p = f8_mfma_exact(wide_b[ni], wide_a);
                    else p = f8_mfma<F::FA, F::FB>(b[ni], a, f32x4{0.f, 0.f, 0.f, 0.f});
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
        for (int d = 0; d < DEPTH; ++d) load_block(x[d], kb + d * WAVES, std::false_type{});
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) multiply(x[d]);
    }
    for (; kb < whole; kb += WAVES) {
        Block x;
        load_block(x, kb, std::false_type{});
        multiply(x);
    }
    if (whole * kScaleBlock < g.K && kb == whole) {             // the wave whose turn it is takes the ragged last block
        Block x;
        load_block(x, whole, std::true_type{});
        multiply(x);
    }

    // ---- the waves' sums meet, in wave order; no wave turns fragments any more
    __syncthreads();
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
