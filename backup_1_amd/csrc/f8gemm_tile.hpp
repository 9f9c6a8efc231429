// Scaled 8-bit product on LDS-DMA tiles: what runs when the result is large enough to fill the chip with tiles.
//
// Bound: the matrix pipe.  A K step is one scale block of 128 codes = 128 contiguous bytes of every row of A and of B, so
// both operands have the same LDS layout: rows of eight 16-byte units, unit q of row r in slot q ^ (r % 8), filled by
// global_load_lds_dwordx4 with the swizzle on the global side.  A fragment is two ds_read_b128 (units lg and lg + 4 of a
// row), free of bank conflicts.  The scales of a step's rows and columns travel the same way, 4 bytes of LDS each
// (global_load_lds_dword, or _ubyte for e8m0), one load a wave, so that the walk waits for nothing but its own stage.
//
// Two stages; the walk is unrolled over them, every LDS address is a lane's base plus a constant.  A step is cut into units
// of two row blocks; a unit's A fragments are read during the unit before it (two sets in turn).  B fragments stay for the
// whole step.  In the last unit everything of the current stage is in registers: after its first column a barrier (which
// also says that the next stage has landed), then its refill goes out and the next step's fragments come in, each column of
// B as soon as its last product is issued.
//
// fp32 scales: an instruction's four sums are multiplied into the accumulators two instructions later (`pending`), so that
// the vector unit never waits for the matrix pipe.
//
// Needs 16-byte aligned A and B with pitches in 16s and below 2^24 (32-bit offsets within a tile).  Of a row's last 16-byte
// unit the bytes past K are read too, and dropped: they lie in the same aligned 16 bytes as one of the row's codes.
#pragma once
#include "f8gemm_common.hpp"

namespace decx_hip {

template <int BM_, int BN_, int WAVES_M_, int WAVES_N_>
struct F8TileShape {
    static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_, STAGES = 2;
    static constexpr int NWAVES = WAVES_M * WAVES_N, NT = NWAVES * kWave;
    static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, MI = WM / 16, NI = WN / 16;
    static constexpr int UM = 2, UNITS = MI / UM;
    static constexpr int A_BYTES = BM * kScaleBlock, B_BYTES = BN * kScaleBlock, S_BYTES = (BM + BN) * 4;
    static constexpr int B_AT = STAGES * A_BYTES, S_AT = B_AT + STAGES * B_BYTES;
    static constexpr size_t LDS_BYTES = (size_t)S_AT + STAGES * S_BYTES;
    static constexpr int A_LOADS = BM / 8 / NWAVES, B_LOADS = BN / 8 / NWAVES, LOADS = A_LOADS + B_LOADS + 1;
    static_assert(UNITS % 2 == 0, "sets of A fragments alternate by unit");
    static_assert(BM % (8 * NWAVES) == 0 && BN % (8 * NWAVES) == 0, "8 rows a load");
    static_assert(BM + BN == NT && BM % kWave == 0, "one scale a thread, a wave's all of one operand");
    static_assert(WN == 64 && 128 % WN == 0, "a wave's columns lie in one 128-row block of B");
    static_assert(A_BYTES + (MI - 1) * 2048 < 65536 && B_BYTES + (NI - 1) * 2048 < 65536, "16-bit offsets from a lane's base");
    static_assert(LDS_BYTES <= 160 * 1024, "LDS of a CU");
};

// 4 bytes (a byte, zero-extended) a lane from global memory to LDS at lds_base + 4 * lane
template <int TAG, bool BYTE>
__device__ __forceinline__ void dma_scale(const void* sbase, uint32_t lane_off, uint32_t lds_base) {
    if constexpr (BYTE)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_ubyte %0, %1 ; load %3"
                     : : "v"(lane_off), "s"(sbase), "s"(lds_base), "n"(TAG) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1 ; load %3"
                     : : "v"(lane_off), "s"(sbase), "s"(lds_base), "n"(TAG) : "memory", "m0");
}

template <class S, class F>
__global__ __launch_bounds__(S::NT, 2) void f8gemm_tile_kernel(const F8GemmArgs g) {
    constexpr int MI = S::MI, NI = S::NI, UM = S::UM, UNITS = S::UNITS, BLK = UM * NI;
    constexpr bool IN_INSTRUCTION = F::IN_INSTRUCTION, B_PER_ROW = F::B_PER_ROW, EXACT = F::EXACT;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
    const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) unsigned char*)lds_raw;
    const TileCoord tc = xcd_grouped_tile(blockIdx.x, g.tiles_m, g.tiles_n, g.group_m);
    const int bm0 = tc.tm * S::BM, bn0 = tc.tn * S::BN;
    const int tid = threadIdx.x, lane = tid % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int wm0 = (wave / S::WAVES_N) * S::WM, wn0 = (wave % S::WAVES_N) * S::WN;
    const int lg = lane >> 4, li = lane & 15;

    // ---- DMA sources.  Rows past the end repeat the last one and are never stored.
    const uint8_t* a_base = g.A + (size_t)bm0 * g.lda;
    const uint8_t* b_base = g.B + (size_t)bn0 * g.ldb;
    uint32_t a_off[S::A_LOADS], b_off[S::B_LOADS];
    const int unit = (lane & 7) ^ (lane >> 3);                  // the unit whose slot of row lane / 8 is lane % 8
#pragma unroll
    for (int j = 0; j < S::A_LOADS; ++j) {
        const int r = (wave * S::A_LOADS + j) * 8 + (lane >> 3), last = g.M - 1 - bm0;
        a_off[j] = (uint32_t)(r < last ? r : last) * (uint32_t)g.lda + 16u * unit;
    }
#pragma unroll
    for (int j = 0; j < S::B_LOADS; ++j) {
        const int r = (wave * S::B_LOADS + j) * 8 + (lane >> 3), last = g.N - 1 - bn0;
        b_off[j] = (uint32_t)(r < last ? r : last) * (uint32_t)g.ldb + 16u * unit;
    }
    constexpr uint32_t SCALE_SIZE = F::E8M0 ? 1 : 4;
    const bool scales_of_a = wave < S::BM / kWave;
    const uint8_t* s_base = static_cast<const uint8_t*>(scales_of_a ? g.SA : g.SB);
    const size_t s_step = (scales_of_a ? g.ldsa : g.ldsb) * SCALE_SIZE;
    uint32_t s_off;
    {
        const int m = bm0 + tid, n = bn0 + tid - S::BM;
        s_off = (uint32_t)(scales_of_a ? (m < g.M ? m : g.M - 1) : (n < g.N ? n : g.N - 1) >> g.b_shift) * SCALE_SIZE;
    }

    // The walk begins with the last block of K, the only one that may be ragged, and goes on with blocks 0, 1, ...  Its loads
    // fetch the 16-byte units that hold at least one code of the row (the lanes of the other units fetch the block's first
    // unit again), and its codes past K are zeroed in registers.
    const int others = (g.K - 1) / kScaleBlock, codes_first = g.K - others * kScaleBlock;
    const uint32_t unit_back = 16 * unit >= codes_first ? 16u * unit : 0u;
#pragma unroll
    for (int j = 0; j < S::A_LOADS; ++j) a_off[j] -= unit_back;
#pragma unroll
    for (int j = 0; j < S::B_LOADS; ++j) b_off[j] -= unit_back;
    a_base += (size_t)others * kScaleBlock, b_base += (size_t)others * kScaleBlock, s_base += (size_t)others * s_step;
    int fetches_left = others;
    // load J of the next step to fetch; the last step's loads are repeated for as long as the walk goes on
    auto issue_one = [&](auto stage_tag, auto j_tag) {
        constexpr int STG = decltype(stage_tag)::value, J = decltype(j_tag)::value;
        if constexpr (J < S::A_LOADS) {
            dma_load16_tagged<STG * 64 + J>(a_base, a_off[J], lds_base + (uint32_t)(STG * S::A_BYTES) + (uint32_t)(wave * S::A_LOADS + J) * 1024u);
        } else if constexpr (J < S::A_LOADS + S::B_LOADS) {
            constexpr int JB = J - S::A_LOADS;
            dma_load16_tagged<STG * 64 + J>(b_base, b_off[JB], lds_base + (uint32_t)(S::B_AT + STG * S::B_BYTES) + (uint32_t)(wave * S::B_LOADS + JB) * 1024u);
        } else {
            dma_scale<STG * 64 + J, F::E8M0>(s_base, s_off, lds_base + (uint32_t)(S::S_AT + STG * S::S_BYTES) + (uint32_t)wave * 256u);
            const bool more = --fetches_left > 0;
            a_base += more ? kScaleBlock : 0;
            b_base += more ? kScaleBlock : 0;
            s_base += more ? s_step : (size_t)0;
        }
    };

    f32x4 acc[MI][NI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = f32x4{0.f, 0.f, 0.f, 0.f};

    // ---- fragments of the current and the next unit, and of B
    struct Half {
        u32x4 lo, hi;
    };
    Half af[2][UM], bf[NI];
    uint32_t sa_raw[2][UM], sb_raw[NI];                         // a scale as it lies in LDS, by lane (row li)
    f32x4 sb_row[NI];                                           // B_PER_ROW: those of columns 4 lg .. 4 lg + 3
    // Every read is one of six lane bases plus a constant of the instruction.  The bases are hidden from the compiler, which
    // would otherwise fold parts of them into constants beyond the instruction's 16 bits, a register for each.
    uint32_t a_rd = (uint32_t)((wm0 + li) * kScaleBlock + ((lg ^ (li & 7)) << 4));
    uint32_t b_rd = (uint32_t)(S::B_AT + (wn0 + li) * kScaleBlock + ((lg ^ (li & 7)) << 4));
    uint32_t a_rd4 = a_rd ^ 64u, b_rd4 = b_rd ^ 64u;            // unit lg + 4 instead of lg
    uint32_t sa_rd = (uint32_t)(S::S_AT + (wm0 + li) * 4);
    uint32_t sb_rd = (uint32_t)(S::S_AT + (S::BM + wn0 + (IN_INSTRUCTION ? li : B_PER_ROW ? 4 * lg : 0)) * 4);
    asm volatile("" : "+v"(a_rd), "+v"(a_rd4), "+v"(b_rd), "+v"(b_rd4), "+v"(sa_rd), "+v"(sb_rd));
    auto read_a = [&](auto set_tag, auto stage_tag, auto rb_tag, auto part_tag) {       // part 0, 1: codes, 2: the scale
        constexpr int SET = decltype(set_tag)::value, STG = decltype(stage_tag)::value, RB = decltype(rb_tag)::value, P = decltype(part_tag)::value;
        constexpr int OFF = STG * S::A_BYTES + RB * 2048;
        if constexpr (P == 0) af[SET][RB % UM].lo = *reinterpret_cast<const u32x4*>(lds_raw + a_rd + OFF);
        else if constexpr (P == 1) af[SET][RB % UM].hi = *reinterpret_cast<const u32x4*>(lds_raw + a_rd4 + OFF);
        else sa_raw[SET][RB % UM] = *reinterpret_cast<const uint32_t*>(lds_raw + sa_rd + STG * S::S_BYTES + RB * 64);
    };
    auto read_b = [&](auto stage_tag, auto ni_tag) {
        constexpr int STG = decltype(stage_tag)::value, NIX = decltype(ni_tag)::value, OFF = STG * S::B_BYTES + NIX * 2048;
        bf[NIX].lo = *reinterpret_cast<const u32x4*>(lds_raw + b_rd + OFF);
        bf[NIX].hi = *reinterpret_cast<const u32x4*>(lds_raw + b_rd4 + OFF);
        constexpr int S_OFF = STG * S::S_BYTES + NIX * 64;
        if constexpr (IN_INSTRUCTION) sb_raw[NIX] = *reinterpret_cast<const uint32_t*>(lds_raw + sb_rd + S_OFF);
        else if constexpr (B_PER_ROW) sb_row[NIX] = *reinterpret_cast<const f32x4*>(lds_raw + sb_rd + S_OFF);
        else if constexpr (NIX == 0) sb_raw[0] = *reinterpret_cast<const uint32_t*>(lds_raw + sb_rd + STG * S::S_BYTES);
    };
    auto scale_value = [&](uint32_t raw) -> float {
        if constexpr (F::E8M0) return e8m0_value(raw);
        else return __uint_as_float(raw);
    };

    // ---- fp32 scales: sums of the last instructions that are not in the accumulators yet
    constexpr int DELAY = 2, RING = 4;
    static_assert((UNITS * BLK) % RING == 0, "a step starts at the ring's beginning");
    struct Pending {
        f32x4 sum;
        float s[B_PER_ROW ? 4 : 1];
    } pending[RING];
    if constexpr (!IN_INSTRUCTION) {
#pragma unroll
        for (int i = 0; i < RING; ++i) {
            pending[i].sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < (B_PER_ROW ? 4 : 1); ++e) pending[i].s[e] = 0.f;
        }
    }
    // MFMA I of unit U works on row block U * UM + row, column ni: column by column, the row order turned on every other
    // column, so that one operand changes between any two
    auto settle = [&](auto n_tag) {                             // the sums of instruction N (modulo a step) join the accumulators
        constexpr int N = (decltype(n_tag)::value + UNITS * BLK) % (UNITS * BLK), U = N / BLK, I = N % BLK;
        constexpr int R = U * UM + ((I & 1) ^ ((I >> 1) & 1)), C = I >> 1;
        const Pending& p = pending[N % RING];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[R][C][e] = __builtin_fmaf(p.sum[e], p.s[B_PER_ROW ? e : 0], acc[R][C][e]);
    };
    F16Fragment wide_b[NI], wide_a[UM];
    float row_scale[UM], col_scale = 0.f;
    // EXACT: B is converted as it comes in, columns 0 and 1 of a step during the last unit of the step before (theirs are done
    // by then), the others before their first product: 128 conversions a step among 64 matrix instructions, evenly
    auto widen_b = [&](auto ni_tag) {
        constexpr int NIX = decltype(ni_tag)::value;
        wide_b[NIX] = f8_widen<F::FB>(f8_fragment(bf[NIX].lo, bf[NIX].hi));
    };
    auto mfma_one = [&](auto u_tag, auto i_tag) {
        constexpr int U = decltype(u_tag)::value, I = decltype(i_tag)::value, NIX = I >> 1, ROW = (I & 1) ^ (NIX & 1), SET = U & 1;
        constexpr int N = U * BLK + I;
        if constexpr (IN_INSTRUCTION) {
            acc[U * UM + ROW][NIX] = f8_mfma_scaled<F::FA, F::FB>(f8_fragment(bf[NIX].lo, bf[NIX].hi), f8_fragment(af[SET][ROW].lo, af[SET][ROW].hi),
                                                                 acc[U * UM + ROW][NIX], (int)sb_raw[NIX], (int)sa_raw[SET][ROW]);
        } else {
            if constexpr (I == 0) {
                if constexpr (U == 0 && !B_PER_ROW) col_scale = scale_value(sb_raw[0]);
#pragma unroll
                for (int r = 0; r < UM; ++r) {
                    row_scale[r] = scale_value(sa_raw[SET][r]) * (B_PER_ROW ? 1.f : col_scale);
                    if constexpr (EXACT) wide_a[r] = f8_widen<F::FA>(f8_fragment(af[SET][r].lo, af[SET][r].hi));
                }
            }
            if constexpr (EXACT && U == 0 && (I & 1) == 0 && NIX >= 2) widen_b(std::integral_constant<int, NIX>{});
            Pending& p = pending[N % RING];
            if constexpr (EXACT) p.sum = f8_mfma_exact(wide_b[NIX], wide_a[ROW]);
            else p.sum = f8_mfma<F::FA, F::FB>(f8_fragment(bf[NIX].lo, bf[NIX].hi), f8_fragment(af[SET][ROW].lo, af[SET][ROW].hi), f32x4{0.f, 0.f, 0.f, 0.f});
            if constexpr (B_PER_ROW) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float s = sb_row[NIX][e];
                    if constexpr (F::E8M0) s = e8m0_value(__float_as_uint(s));
                    p.s[e] = row_scale[ROW] * s;
                }
            } else {
                p.s[0] = row_scale[ROW];
            }
            settle(std::integral_constant<int, N - DELAY>{});
        }
    };
#define DECX_PIN() __builtin_amdgcn_sched_barrier(0)
    typedef std::integral_constant<int, 0> I0;
    typedef std::integral_constant<int, UNITS - 1> Last;
    // zeros past K in a lane's fragments: its units start at codes 16 lg and 16 lg + 64 of the block
    auto unit_mask = [&](int first) {
        u32x4 m;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int n = codes_first - first - 4 * w;                // codes of this word that exist
            m[w] = n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
        }
        return m;
    };
    // units 0 .. UNITS - 2 of a step: products, and the reads of the next unit's A fragments
    auto inner_units = [&](auto stage_tag, auto ragged_tag, u32x4 keep_lo, u32x4 keep_hi) {
        static_for<0, UNITS - 1>([&](auto u_tag) {
            constexpr int U = decltype(u_tag)::value, SET = (U + 1) & 1;
            static_for<0, BLK>([&](auto i_tag) {
                constexpr int I = decltype(i_tag)::value;
                static_assert(BLK >= 3 * UM, "a read a slot");
                if constexpr (I < 3 * UM)
                    read_a(std::integral_constant<int, SET>{}, stage_tag, std::integral_constant<int, (U + 1) * UM + I / 3>{}, std::integral_constant<int, I % 3>{});
                mfma_one(u_tag, i_tag);
                DECX_PIN();
            });
            if constexpr (decltype(ragged_tag)::value) {
#pragma unroll
                for (int r = 0; r < UM; ++r) af[SET][r].lo &= keep_lo, af[SET][r].hi &= keep_hi;
            }
        });
    };
    auto k_step = [&](auto stage_tag, auto ragged_tag) {
        constexpr int STG = decltype(stage_tag)::value;
        typedef std::integral_constant<int, 1 - STG> Next;
        u32x4 keep_lo = {}, keep_hi = {};
        if constexpr (decltype(ragged_tag)::value) {
            keep_lo = unit_mask(16 * lg), keep_hi = unit_mask(16 * lg + 64);
#pragma unroll
            for (int r = 0; r < UM; ++r) af[0][r].lo &= keep_lo, af[0][r].hi &= keep_hi;
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) bf[ni].lo &= keep_lo, bf[ni].hi &= keep_hi;
            if constexpr (EXACT) widen_b(I0{}), widen_b(std::integral_constant<int, 1>{});
        }
        inner_units(stage_tag, ragged_tag, keep_lo, keep_hi);
        mfma_one(Last{}, I0{});
        DECX_PIN();
        mfma_one(Last{}, std::integral_constant<int, 1>{});
        DECX_PIN();
        wait_dma_then_barrier<0>();
        DECX_PIN();
        constexpr int SLOTS = BLK - 2;
        static_for<0, SLOTS>([&](auto s_tag) {
            constexpr int I = decltype(s_tag)::value;
            // the next step's first products need column 0 of B and the first row blocks of A: those first
            if constexpr (I % 2 == 0) read_b(Next{}, std::integral_constant<int, I / 2>{});
            static_assert(SLOTS >= UM * 3 / 2, "the first unit's A fragments come in at two reads a slot");
            if constexpr (I < (3 * UM + 1) / 2) {
                static_for<2 * I, (2 * I + 2 < 3 * UM ? 2 * I + 2 : 3 * UM)>([&](auto r_tag) {
                    constexpr int R = decltype(r_tag)::value;
                    read_a(I0{}, Next{}, std::integral_constant<int, R / 3>{}, std::integral_constant<int, R % 3>{});
                });
            }
            static_for<(I * S::LOADS) / SLOTS, ((I + 1) * S::LOADS) / SLOTS>([&](auto j_tag) { issue_one(stage_tag, j_tag); });
            mfma_one(Last{}, std::integral_constant<int, I + 2>{});
            if constexpr (EXACT && (I == 3 || I == 5)) widen_b(std::integral_constant<int, (I - 3) / 2>{});
            DECX_PIN();
        });
        read_b(Next{}, std::integral_constant<int, NI - 1>{});
        DECX_PIN();
    };
    auto read_first = [&](auto stage_tag) {
        static_for<0, 3 * UM>([&](auto r) {
            constexpr int R = decltype(r)::value;
            read_a(I0{}, stage_tag, std::integral_constant<int, R / 3>{}, std::integral_constant<int, R % 3>{});
        });
        static_for<0, NI>([&](auto ni) { read_b(stage_tag, ni); });
    };

    typedef std::integral_constant<int, 1> I1;
    static_for<0, S::LOADS>([&](auto j) { issue_one(I1{}, j); });
    if (others > 0) {
        a_base = g.A + (size_t)bm0 * g.lda, b_base = g.B + (size_t)bn0 * g.ldb;
        s_base = static_cast<const uint8_t*>(scales_of_a ? g.SA : g.SB);
        fetches_left = others;
#pragma unroll
        for (int j = 0; j < S::A_LOADS; ++j) a_off[j] += unit_back;
#pragma unroll
        for (int j = 0; j < S::B_LOADS; ++j) b_off[j] += unit_back;
    }
    static_for<0, S::LOADS>([&](auto j) { issue_one(I0{}, j); });
    wait_dma_then_barrier<S::LOADS>();
    read_first(I1{});
    DECX_PIN();
    k_step(I1{}, std::true_type{});
    for (int t = others >> 1; t > 0; --t) {
        k_step(I0{}, std::false_type{});
        k_step(I1{}, std::false_type{});
    }
    if (others & 1) k_step(I0{}, std::false_type{});
    wait_dma_then_barrier<0>();                                 // the redundant loads have landed before the workgroup gives up its LDS
    if constexpr (!IN_INSTRUCTION)
        static_for<0, DELAY>([&](auto d) { settle(std::integral_constant<int, UNITS * BLK - DELAY + decltype(d)::value>{}); });

    // ---- epilogue.  fp32 results leave as they lie in the accumulators, 16 bytes a lane (through LDS in 256-byte rows: 2 %
    // slower at 8192^3).  16-bit ones, 8 bytes a lane there, go through LDS (the operands' stages are free) in rows of 16-byte
    // pieces XOR-swizzled by the row, and leave as whole 128-byte lines (8192^3: 431 -> 400 us).  The wave reads back what it
    // wrote itself, in order: no barrier.
    const int m_wave = bm0 + wm0, n_wave = bn0 + wn0;
    if constexpr (EXACT) {                                      // fp32 results, and only those
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) f8_store_result(g, m_wave + 16 * mi + li, n_wave + 16 * ni + 4 * lg, acc[mi][ni]);
    } else {
        constexpr int ROW_BYTES = S::WN * 2, PIECES = ROW_BYTES / 16, ROWS_PER_PASS = kWave / PIECES;
        static_assert(PIECES == 8 && (size_t)S::NWAVES * S::WM * ROW_BYTES <= (size_t)S::S_AT, "every wave's piece fits the stages");
        unsigned char* park = lds_raw + (size_t)wave * (S::WM * ROW_BYTES);
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                const int row = 16 * mi + li, col = 16 * ni + 4 * lg;
                f32x4 v = acc[mi][ni];
                u32x2 r;
                if (g.type == DECX_HIP_F16) {
                    if (g.C) v = f8_add_c<_Float16>(g, m_wave + row, n_wave + col, v);
                    r = f8_round4<_Float16>(v);
                } else {
                    if (g.C) v = f8_add_c<__bf16>(g, m_wave + row, n_wave + col, v);
                    r = f8_round4<__bf16>(v);
                }
                *reinterpret_cast<u32x2*>(park + row * ROW_BYTES + (((col >> 3) ^ (row & 7)) << 4) + ((lg & 1) << 3)) = r;
            }
        asm volatile("" ::: "memory");                          // in this order: the lanes exchange what they hold
        uint16_t* const d = static_cast<uint16_t*>(g.D);
        const bool whole = bm0 + S::BM <= g.M && bn0 + S::BN <= g.N && ((reinterpret_cast<uintptr_t>(d) | (g.ldd * 2)) & 15) == 0;
#pragma unroll 4
        for (int pass = 0; pass < S::WM / ROWS_PER_PASS; ++pass) {
            const int row = pass * ROWS_PER_PASS + lane / PIECES, piece = lane % PIECES;
            const u32x4 v = *reinterpret_cast<const u32x4*>(park + row * ROW_BYTES + ((piece ^ (row & 7)) << 4));
            const int m = m_wave + row, n = n_wave + piece * 8;
            uint16_t* to = d + (size_t)m * g.ldd + n;
            if (whole) {
                __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(to));       // not read by this launch
            } else if (m < g.M && n < g.N) {
                if (n + 8 <= g.N) {
                    *reinterpret_cast<u32x4_any*>(to) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (n + e < g.N) to[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
                }
            }
        }
    }
#undef DECX_PIN
}

}  // namespace decx_hip
