// Root-mean-square norm with the residual's addition, its result as 8-bit codes with a scale for each block of 128 (the
// left operand of f8gemm.hip) and / or in its own type, and the norm's gradient.
//
//   h = round(x + r)      rstd = 1 / sqrt(mean(h^2) + eps)      y = h * rstd * w
//   n = h * rstd          g = dy * w      dx = rstd * (g - n * mean(g n)) + dr      dw = sum over rows of dy * n
//
// Bound: memory, every element read and written once.  A workgroup owns a row at a time and keeps it in registers between
// the sum over the row and what needs that sum; thread t holds the 8-element chunks t, t + NT, ..., so that 16 consecutive
// lanes hold a scale block.  Sums are in fp32 (of rows whose squares leave its range in 64 bits): at most 32 products in a
// thread, then a tree over lanes and waves in a fixed order, which gives the same bits on every run.
#include "runtime.hpp"
#include "f8_common.hpp"

namespace decx_hip {

// Sum over the workgroup, in every thread.  `part` is used by one call at a time: the callers separate calls by a barrier.
template <int NT, class T>
__device__ __forceinline__ T workgroup_sum(T v, T* part) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) v += __shfl_xor(v, d);
    if constexpr (NT > kWave) {
        if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int w = 1; w < NT / kWave; ++w) v += part[w];
    }
    return v;
}

// Consecutive workgroups run on different XCDs; give each XCD a contiguous run of rows, so that the scales of neighbouring
// rows (4 or 1 bytes each, neighbours in memory) meet in one L2 before they leave it.
__device__ __forceinline__ int xcd_row(int pid, int rows) {
    const int xcd = pid % kXcds, local = pid / kXcds, base = rows / kXcds, rem = rows % kXcds;
    return xcd * base + (xcd < rem ? xcd : rem) + local;
}

// Squares of elements beyond 2^64 overflow fp32, those of elements below 2^-63 lose bits.  Where the mean of a row is infinite, or
// so small that lost bits could matter (each square at most 2^-150, half of fp32's smallest step), its squares are added again in
// 64 bits from the registers.
constexpr float kLeastMean = 0x1p-120f;

struct RmsNormArgs {
    const void *X, *R, *W;
    void *H, *Y;
    float* rstd;
    uint8_t* Q;
    void* S;
    size_t ldx, ldr, ldh, ldy, ldq, lds;
    float eps;
    int M, K, e5m2, e8m0, stream;
};

template <int TYPE, int NT, int CH, int ROWS>
__global__ __launch_bounds__(NT) void rmsnorm_f8_kernel(const RmsNormArgs g) {
    typedef typename Wide<TYPE>::T T;
    __shared__ float part[NT / kWave];
    __shared__ double part64[NT / kWave];
    const int K = g.K, m = xcd_row((int)blockIdx.x, g.M);
    const T* x = static_cast<const T*>(g.X) + (size_t)m * g.ldx;
    Eight h[CH];
    RawEight<TYPE> raw_x[CH], raw_r[CH];
    auto load_row = [&](auto stream_tag) {
        constexpr bool STREAM = decltype(stream_tag)::value;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int k = 8 * ((int)threadIdx.x + i * NT), at = k < K ? k : 0;
            raw_x[i] = fetch8_part<TYPE, ROWS, STREAM>(x + at, K - k);
            if (g.R) raw_r[i] = fetch8_part<TYPE, ROWS, STREAM>(static_cast<const T*>(g.R) + (size_t)m * g.ldr + at, K - k);
        }
    };
    if (TYPE != 0 && g.stream) load_row(std::true_type{});
    else load_row(std::false_type{});
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int k = 8 * ((int)threadIdx.x + i * NT);
        settle8_part<TYPE, ROWS>(raw_x[i], K - k);
        h[i] = widen8<TYPE>(raw_x[i]);
        if (g.R) {
            settle8_part<TYPE, ROWS>(raw_r[i], K - k);
            const Eight r = widen8<TYPE>(raw_r[i]);
            // the sum is what the stream carries on, so it is rounded to its type here and the norm is taken of that
#pragma unroll
            for (int e = 0; e < 8; ++e) h[i].v[e] = (float)(T)(h[i].v[e] + r.v[e]);
        }
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(h[i].v[e], h[i].v[e], sum);
    if (g.H) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int k = 8 * ((int)threadIdx.x + i * NT);
            store8_part<TYPE>(static_cast<T*>(g.H) + (size_t)m * g.ldh + (k < K ? k : 0), h[i], K - k);
        }
    }
    const float mean = __fdiv_rn(workgroup_sum<NT>(sum, part), (float)K) + g.eps;
    float rstd;
    if (mean >= kLeastMean && mean < __builtin_inff()) {        // the same for the whole workgroup
        rstd = __fdiv_rn(1.f, __fsqrt_rn(mean));
    } else {
        double squares = 0.0;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) squares += (double)h[i].v[e] * h[i].v[e];
        rstd = (float)(1.0 / sqrt(workgroup_sum<NT>(squares, part64) / K + (double)g.eps));
    }
    if (g.rstd && threadIdx.x == 0) g.rstd[m] = rstd;
    if (!g.Q && !g.Y) return;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int k = 8 * ((int)threadIdx.x + i * NT), at = k < K ? k : 0;
        const Eight w = load8_part<TYPE, ROWS>(static_cast<const T*>(g.W) + at, K - k);
        Eight y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y.v[e] = h[i].v[e] * rstd * w.v[e];     // in this order: |h * rstd| <= sqrt(K), h * w may overflow
        if (g.Y) store8_part<TYPE>(static_cast<T*>(g.Y) + (size_t)m * g.ldy + at, y, K - k);
        if (g.Q) {
            // the codes are rounded from fp32, not from y's own type; elements past K are zeros
            if (k + 8 > K) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (k + e >= K) y.v[e] = 0.f;               // also where rstd is NaN or infinite
            }
            const BlockScale s = block_scale(group16_max(eight_magnitude(y)), g.e5m2, g.e8m0);
            if (k < K) {
                store_codes(g.Q + (size_t)m * g.ldq + k, pack8_f8(y, s.factor, g.e5m2), K - k);
                if ((threadIdx.x & 15) == 0) store_scale(g.S, (size_t)(k / kScaleBlock) * g.lds + m, s, g.e8m0);
            }
        }
    }
}

struct RmsNormBackwardArgs {
    const void *H, *W, *dY, *dR;
    const float* rstd;
    void* dX;
    float* partial;           // [workgroups][K], nullptr: dW not wanted, or made by the column workgroups
    float* dW;                // of the column workgroups
    int row_groups;           // workgroups of rows; those behind them take columns of dW
    size_t ldh, lddy, lddr, lddx;
    int M, K, rows_each;
    int stream;               // the inputs are more than the caches keep
};

// dw of some columns straight from H and dY, in workgroups of their own beside those of the rows: both are read twice, but
// there is one launch and no workspace.  For few rows of inputs that the caches hold (rmsnorm_backward_enqueue).  64 rows a
// pass and four passes in flight; columns for that many lanes.
constexpr int dw_columns(int nt) { return nt / 8 < 64 ? nt / 8 : 64; }
template <int TYPE, int NT, int ROWS>
__device__ __forceinline__ void rmsnorm_dw_columns(const RmsNormBackwardArgs& g, int group) {
    typedef typename Wide<TYPE>::T T;
    constexpr int COLS = dw_columns(NT), LANES = COLS / 8, GROUPS = NT / LANES, AHEAD = 4;
    __shared__ float part[GROUPS][COLS + 1];
    const int k0 = group * COLS, c = threadIdx.x % LANES, r = threadIdx.x / LANES, k = k0 + 8 * c, at = k < g.K ? k : 0;
    float sum[8] = {};
    for (int m0 = r; m0 < g.M; m0 += GROUPS * AHEAD) {
        RawEight<TYPE> h[AHEAD], dy[AHEAD];
        float rstd[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int m = m0 + GROUPS * j, row = m < g.M ? m : 0;
            rstd[j] = m < g.M ? g.rstd[row] : 0.f;
            h[j] = fetch8_part<TYPE, ROWS>(static_cast<const T*>(g.H) + (size_t)row * g.ldh + at, m < g.M ? g.K - k : 0);
            dy[j] = fetch8_part<TYPE, ROWS>(static_cast<const T*>(g.dY) + (size_t)row * g.lddy + at, m < g.M ? g.K - k : 0);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            settle8_part<TYPE, ROWS>(h[j], g.K - k);            // rows past the last are zeros either way
            settle8_part<TYPE, ROWS>(dy[j], g.K - k);
            const Eight hv = widen8<TYPE>(h[j]), yv = widen8<TYPE>(dy[j]);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] = __builtin_fmaf(yv.v[e], hv.v[e] * rstd[j], sum[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) part[r][8 * c + e] = sum[e];
    __syncthreads();
    // 8 threads a column add a share of the rows of lanes each, then meet
    constexpr int SHARE = GROUPS / 8;
    static_assert(COLS * 8 <= NT && GROUPS % 8 == 0, "8 threads a column");
    const int col = threadIdx.x / 8, share = threadIdx.x % 8;
    if (col < COLS) {
        float v = part[share * SHARE][col];
#pragma unroll
        for (int i = 1; i < SHARE; ++i) v += part[share * SHARE + i][col];
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) v += __shfl_xor(v, d);
        if (share == 0 && k0 + col < g.K) g.dW[k0 + col] = v;
    }
}

// Workgroup b owns rows b * rows_each ...: their dx, and their part of dw in a row of `partial`, which the second kernel
// adds up in row order (no atomics: the same bits on every run).
template <int TYPE, int NT, int CH, int ROWS>
__global__ __launch_bounds__(NT, NT >= 512 ? NT / 256 : 2) void rmsnorm_backward_kernel(const RmsNormBackwardArgs g) {
    typedef typename Wide<TYPE>::T T;
    __shared__ float part[2][NT / kWave];
    // The thread's columns of dw: in registers, or, where a thread has 128 of them and 4 chunks, in LDS, in whole vectors of the
    // workgroup one after the other
    constexpr bool DW_IN_LDS = NT >= 1024 && CH == 4;
    if constexpr (!DW_IN_LDS) {                                 // (LDS has no room for the columns' sums beside that)
        if ((int)blockIdx.x >= g.row_groups) {
            rmsnorm_dw_columns<TYPE, NT, ROWS>(g, (int)blockIdx.x - g.row_groups);
            return;
        }
    }
    const int K = g.K, first = (int)blockIdx.x * g.rows_each;
    const int last = first + g.rows_each < g.M ? first + g.rows_each : g.M;
    __shared__ f32x4 dw_lds[DW_IN_LDS ? 2 * CH * NT : 1];
    Eight dw[DW_IN_LDS ? 1 : CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if (DW_IN_LDS) {
            dw_lds[2 * i * NT + threadIdx.x] = f32x4{0.f, 0.f, 0.f, 0.f};
            dw_lds[(2 * i + 1) * NT + threadIdx.x] = f32x4{0.f, 0.f, 0.f, 0.f};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) dw[i].v[e] = 0.f;
        }
    }
    // The next row's loads are in flight while a row waits for its sum.  Not where a workgroup fills the CU and a thread has 128
    // registers (LONG): there a row stays as it was loaded, n and g are made twice, and dr is fetched when it is added.  With all
    // of that in registers, and so in scratch memory, 2048 x 32768 bf16 took 448 us; so, and with dw in LDS, 119.  n and g are
    // also made twice (TWICE) where the moving of row ends would cost the last registers (2048 x 12001 bf16 62.3 -> 58.5 us).
    constexpr bool LONG = NT >= 1024, TWICE = LONG || (TYPE != 0 && CH == 4 && ROWS == kRowsRagged);
    struct Row {
        RawEight<TYPE> h[CH], dy[CH], dr[LONG ? 1 : CH];
        float rstd;
    };
    auto load_row_as = [&](Row& r, int m, auto stream_tag) {
        constexpr bool STREAM = decltype(stream_tag)::value;
        r.rstd = g.rstd[m];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int k = 8 * ((int)threadIdx.x + i * NT), at = k < K ? k : 0;
            r.h[i] = fetch8_part<TYPE, ROWS, STREAM>(static_cast<const T*>(g.H) + (size_t)m * g.ldh + at, K - k);
            r.dy[i] = fetch8_part<TYPE, ROWS, STREAM>(static_cast<const T*>(g.dY) + (size_t)m * g.lddy + at, K - k);
            if (g.dR && !LONG) r.dr[i] = fetch8_part<TYPE, ROWS, STREAM>(static_cast<const T*>(g.dR) + (size_t)m * g.lddr + at, K - k);
        }
    };
    auto load_row = [&](Row& r, int m) {
        if (TYPE != 0 && g.stream) load_row_as(r, m, std::true_type{});
        else load_row_as(r, m, std::false_type{});
    };
    Row next;
    if (!LONG) load_row(next, first);
    for (int m = first; m < last; ++m) {
        if (LONG) load_row(next, m);
        Row row = next;
        if (!LONG && m + 1 < last) load_row(next, m + 1);
        const float rstd = row.rstd;
        Eight n[TWICE ? 1 : CH], dn[TWICE ? 1 : CH];            // n and g; TWICE: of a chunk at a time
        auto weigh = [&](int i, Eight& ni, Eight& gi, bool first_time) {
            const int k = 8 * ((int)threadIdx.x + i * NT), at = k < K ? k : 0;
            const Eight w = load8_part<TYPE, ROWS>(static_cast<const T*>(g.W) + at, K - k);
            ni = widen8<TYPE>(row.h[i]);
            gi = widen8<TYPE>(row.dy[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) ni.v[e] *= rstd;
            if (first_time && DW_IN_LDS) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    f32x4 sums = dw_lds[(2 * i + half) * NT + threadIdx.x];
#pragma unroll
                    for (int e = 0; e < 4; ++e) sums[e] = __builtin_fmaf(gi.v[4 * half + e], ni.v[4 * half + e], sums[e]);
                    dw_lds[(2 * i + half) * NT + threadIdx.x] = sums;
                }
            } else if (first_time) {
#pragma unroll
                for (int e = 0; e < 8; ++e) dw[i].v[e] = __builtin_fmaf(gi.v[e], ni.v[e], dw[i].v[e]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) gi.v[e] *= w.v[e];
        };
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int k = 8 * ((int)threadIdx.x + i * NT);
            settle8_part<TYPE, ROWS>(row.h[i], K - k);
            settle8_part<TYPE, ROWS>(row.dy[i], K - k);
            Eight &ni = n[TWICE ? 0 : i], &gi = dn[TWICE ? 0 : i];
            weigh(i, ni, gi, true);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(gi.v[e], ni.v[e], sum);
        }
        // two sets of partial sums in turn: a wave may be a row ahead of another, never two (it meets it in between)
        const float mean = __fdiv_rn(workgroup_sum<NT>(sum, part[m & 1]), (float)K);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int k = 8 * ((int)threadIdx.x + i * NT), at = k < K ? k : 0;
            Eight &ni = n[TWICE ? 0 : i], &gi = dn[TWICE ? 0 : i];
            if (TWICE) {
                if (LONG && g.dR) row.dr[0] = fetch8_part<TYPE, ROWS>(static_cast<const T*>(g.dR) + (size_t)m * g.lddr + at, K - k);
                weigh(i, ni, gi, false);
            }
            Eight dx;
#pragma unroll
            for (int e = 0; e < 8; ++e) dx.v[e] = rstd * __builtin_fmaf(-ni.v[e], mean, gi.v[e]);
            if (g.dR) {
                RawEight<TYPE>& raw = row.dr[LONG ? 0 : i];
                settle8_part<TYPE, ROWS>(raw, K - k);
                const Eight dr = widen8<TYPE>(raw);
#pragma unroll
                for (int e = 0; e < 8; ++e) dx.v[e] += dr.v[e];
            }
            store8_part<TYPE>(static_cast<T*>(g.dX) + (size_t)m * g.lddx + at, dx, K - k);
        }
    }
    if (!g.partial) return;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int k = 8 * ((int)threadIdx.x + i * NT);
        Eight sums = dw[DW_IN_LDS ? 0 : i];
        if (DW_IN_LDS) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sums.v[e] = dw_lds[(2 * i + e / 4) * NT + threadIdx.x][e % 4];
        }
        store8_part<0>(g.partial + (size_t)blockIdx.x * K + (k < K ? k : 0), sums, K - k);
    }
}

// dw[k] = sum of `rows` rows of partial.  A workgroup takes COLS columns: COLS / 4 lanes with 4 each, 1024 / COLS rows of
// lanes that add every (1024 / COLS)th row, eight loads in flight each, and meet in LDS in their order.
template <int COLS>
__global__ __launch_bounds__(256) void rmsnorm_dw_kernel(const float* __restrict__ partial, int rows, int K, float* __restrict__ dW) {
    constexpr int LANES = COLS / 4, GROUPS = 256 / LANES, AHEAD = 8;
    __shared__ float part[GROUPS][COLS + 1];
    const int c = threadIdx.x % LANES, r = threadIdx.x / LANES;
    const int k = (int)blockIdx.x * COLS + 4 * c;
    const float* p = partial + (k < K ? k : 0);
    const bool whole = k + 4 <= K;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int m0 = r; m0 < rows; m0 += GROUPS * AHEAD) {
        f32x4 v[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int m = m0 + GROUPS * j;
            v[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (m < rows) {
                if (whole) {
                    v[j] = *reinterpret_cast<const f32x4_any*>(p + (size_t)m * K);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (k + e < K) v[j][e] = p[(size_t)m * K + e];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) sum += v[j];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[r][4 * c + e] = sum[e];
    __syncthreads();
    // 8 threads a column add GROUPS / 8 rows of lanes each, then one of them the 8
    constexpr int SHARE = GROUPS / 8;
    static_assert(COLS * 8 <= 256 && GROUPS % 8 == 0, "8 threads a column");
    const int col = threadIdx.x / 8, share = threadIdx.x % 8;
    if (col < COLS) {
        float v = part[share * SHARE][col];
#pragma unroll
        for (int i = 1; i < SHARE; ++i) v += part[share * SHARE + i][col];
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) v += __shfl_xor(v, d);
        const int at = (int)blockIdx.x * COLS + col;
        if (share == 0 && at < K) dW[at] = v;
    }
}

constexpr int kRmsNormMaxK = 32768;       // 1024 threads with 4 chunks each hold a row

// The smallest workgroup that holds a row of K elements with at most MOST chunks a thread, one wave for short rows.  The
// gradient holds three inputs twice, a row's and the next one's: 4 chunks in fp32 would leave registers for one workgroup a CU.
#define DECX_RMSNORM_SHAPES(K, MOST, LAUNCH)               \
    do {                                                   \
        if ((K) <= 512) LAUNCH(64, 1);                     \
        else if ((K) <= 1024) LAUNCH(128, 1);              \
        else if ((K) <= 2048) LAUNCH(256, 1);              \
        else if ((K) <= 4096) LAUNCH(256, 2);              \
        else if ((K) <= 8192) LAUNCH(1024 / (MOST), MOST); \
        else if ((K) <= 16384) LAUNCH(2048 / (MOST), MOST); \
        else LAUNCH(1024, 4);                              \
    } while (0)

template <int TYPE>
static int rmsnorm_f8_launch(const RmsNormArgs& g) {
    // a workgroup a row
    if ((long)g.M * (g.K <= 512 ? 64 : g.K <= 1024 ? 128 : g.K <= 8192 ? 256 : g.K <= 16384 ? 512 : 1024) > kMostThreads)
        return fail(DECX_HIP_FAIL_ERROR_PARAMS, "problem too large for one launch\n");
    const int rows = rows_kind(g.K);
    // Long rows (8 to 32 KB) from memory: 4 workgroups a CU instead of 8, by LDS that nothing uses.  8 have twice the loads in
    // flight that memory needs, from twice the places: 8192 x 8192 bf16 132 us against 119, 4096 x 8192 fp32 134 against 126.
    // Where the caches hold the inputs, 8 are better (1262 x 8192 bf16 16.5 against 17.7), and with shorter rows.
    const size_t row_bytes = (size_t)g.K * sizeof(typename Wide<TYPE>::T), inputs = (size_t)g.M * row_bytes * (g.R ? 2 : 1);
    const size_t unused = row_bytes > 8192 && g.K <= 8192 && inputs >= (size_t)64 << 20 ? 40000 : 0;
#define DECX_LAUNCH(NT, CH)                                                                                                          \
    hipLaunchKernelGGL((rows == kRowsWhole ? rmsnorm_f8_kernel<TYPE, NT, CH, kRowsWhole> : rmsnorm_f8_kernel<TYPE, NT, CH, kRowsRagged>), \
                       dim3((unsigned)g.M), dim3(NT), unused, g_rt.stream, g)
    if (rows == kRowsShort) hipLaunchKernelGGL((rmsnorm_f8_kernel<TYPE, kWave, 1, kRowsShort>), dim3((unsigned)g.M), dim3(kWave), 0, g_rt.stream, g);
    else DECX_RMSNORM_SHAPES(g.K, 4, DECX_LAUNCH);
#undef DECX_LAUNCH
    HIP_TRY(hipGetLastError());
    return 0;
}
template <int TYPE>
static int rmsnorm_backward_launch(const RmsNormBackwardArgs& g) {
    const int rows = rows_kind(g.K);
#define DECX_GRID(NT) dim3((unsigned)(g.row_groups + (g.dW ? cdiv(g.K, dw_columns(NT)) : 0)))
#define DECX_LAUNCH(NT, CH)                                                                                                                  \
    hipLaunchKernelGGL((rows == kRowsWhole ? rmsnorm_backward_kernel<TYPE, NT, CH, kRowsWhole> : rmsnorm_backward_kernel<TYPE, NT, CH, kRowsRagged>), \
                       DECX_GRID(NT), dim3(NT), 0, g_rt.stream, g)
    constexpr int MOST = TYPE == 0 ? 2 : 4;
    if (rows == kRowsShort) hipLaunchKernelGGL((rmsnorm_backward_kernel<TYPE, kWave, 1, kRowsShort>), DECX_GRID(kWave), dim3(kWave), 0, g_rt.stream, g);
    else DECX_RMSNORM_SHAPES(g.K, MOST, DECX_LAUNCH);
#undef DECX_LAUNCH
#undef DECX_GRID
    HIP_TRY(hipGetLastError());
    return 0;
}

int rmsnorm_f8_enqueue(const void* X, int ldx, const void* R, int ldr, const void* W, float eps, int type, int M, int K, void* H, int ldh,
                       float* rstd, void* Y, int ldy, uint8_t* Q, int ldq, void* S, int lds, int format, int scale_type) {
    if (int rc = need_library_device()) return rc;
    if (!X || !W) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "null matrix pointer\n");
    if (!H && !Y && !Q && !rstd) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "no result wanted\n");
    if (Q && !S) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "codes without their scales\n");
    if (M <= 0 || K <= 0) return fail(DECX_HIP_FAIL_DIMS, "Matrix Dims don't match each other");
    if (M > kMostExtent) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "problem too large for one launch\n");
    if (K > kRmsNormMaxK) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "the norm takes rows of at most %d elements\n", kRmsNormMaxK);
    if (int rc = check_f8_codes(type, format, scale_type)) return rc;
    if (!(eps >= 0.f)) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "eps is negative or no number\n");
    if (ldx < K || (R && ldr < K) || (H && ldh < K) || (Y && ldy < K) || (Q && (ldq < K || lds < M)))
        return fail(DECX_HIP_FAIL_ERROR_PARAMS, "leading dimension smaller than the row length\n");
    for (const void* p : {X, R, W, static_cast<const void*>(H), static_cast<const void*>(Y)})
        if (int rc = check_element_alignment(p, type)) return rc;
    if (int rc = check_element_alignment(rstd, DECX_HIP_F32)) return rc;
    if (Q && scale_type == DECX_HIP_SCALE_F32 && (reinterpret_cast<uintptr_t>(S) & 3u))
        return fail(DECX_HIP_FAIL_ERROR_PARAMS, "scales off the grid of their type\n");
    // a thread reads its elements of a row before it writes them, so H or Y may lie over X or R
    const size_t m = (size_t)M, k = (size_t)K, wide = element_size(type);
    if (int rc = check_results({{operand(H, m, k, ldh, wide), 3u}, {operand(Y, m, k, ldy, wide), 3u}, {operand(rstd, 1, m, m, 4)}, {operand(Q, m, k, ldq, 1)},
                                {operand(Q ? S : nullptr, cdiv(K, kScaleBlock), m, lds, scale_size(scale_type))}},
                               {operand(X, m, k, ldx, wide), operand(R, m, k, ldr, wide), operand(W, 1, k, k, wide)}))
        return rc;
    RmsNormArgs g = {};
    g.X = X, g.R = R, g.W = W, g.H = H, g.Y = Y, g.rstd = rstd, g.Q = Q, g.S = S;
    g.ldx = (size_t)ldx, g.ldr = (size_t)ldr, g.ldh = (size_t)ldh, g.ldy = (size_t)ldy, g.ldq = (size_t)ldq, g.lds = (size_t)lds;
    // 16-bit inputs of 96 to 256 MiB are read past the caches, whose 256 MiB the results then have for themselves: 4096 x 8192,
    // 134 MB, 64 us against 68 (59 against 65 where little else is used in between); 4096 x 4096, 67 MB, 29 against 24, and
    // 8192 x 8192, 268 MB, 125 against 119
    const size_t inputs = (size_t)M * K * (R ? 4 : 2);
    g.stream = inputs > ((size_t)96 << 20) && inputs < ((size_t)256 << 20);
    g.eps = eps, g.M = M, g.K = K, g.e5m2 = format == DECX_HIP_E5M2, g.e8m0 = scale_type == DECX_HIP_SCALE_E8M0;
    if (type == DECX_HIP_F32) return rmsnorm_f8_launch<0>(g);
    if (type == DECX_HIP_F16) return rmsnorm_f8_launch<1>(g);
    return rmsnorm_f8_launch<2>(g);
}

// Workgroups of the gradient.  More of them hide more of the wait for a row's sum, but each writes a row of `partial`, so there
// are fewer the longer the rows are, and not many for few rows: 4 rows each from 512 workgroups on.  2048 x 2048 bf16 takes
// 22.4 us with a row each and 13.5 with 4; of 8192 rows, 256 elements 14 us with 2048 workgroups and 18 with 512, 2048
// elements 36 and 29; 2048 x 8192 fp32 62 us with 256 and 66 with 512.  The workspace is sized for the 2-byte types.
static int rmsnorm_backward_groups(int M, int K, int size) {
    const long bytes = (long)K * size;
    const int each = bytes <= 1024 ? 8 : bytes <= 2048 ? 4 : bytes <= 4096 ? 3 : bytes <= 16384 ? 2 : 1;
    const int cus = g_rt.compute_units > 0 ? g_rt.compute_units : 256;
    const int by_rows = cdiv(M, 4) > 2 * cus ? cdiv(M, 4) : 2 * cus, most = each * cus < by_rows ? each * cus : by_rows;
    const int groups = M < most ? M : most;
    return cdiv(M, cdiv(M, groups));
}

size_t rmsnorm_backward_workspace(int M, int K) { return (size_t)rmsnorm_backward_groups(M, K, 2) * K * sizeof(float); }

int rmsnorm_backward_enqueue(const void* H, int ldh, const void* W, const float* rstd, const void* dY, int lddy, const void* dR, int lddr,
                             int type, int M, int K, void* dX, int lddx, float* dW, void* work, size_t work_bytes) {
    if (int rc = need_library_device()) return rc;
    if (!H || !W || !rstd || !dY || !dX) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "null matrix pointer\n");
    if (M <= 0 || K <= 0) return fail(DECX_HIP_FAIL_DIMS, "Matrix Dims don't match each other");
    if (M > kMostExtent) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "problem too large for one launch\n");
    if (K > kRmsNormMaxK) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "the norm takes rows of at most %d elements\n", kRmsNormMaxK);
    if (int rc = check_f8_codes(type, DECX_HIP_E4M3, DECX_HIP_SCALE_F32)) return rc;
    if (ldh < K || lddy < K || (dR && lddr < K) || lddx < K)
        return fail(DECX_HIP_FAIL_ERROR_PARAMS, "leading dimension smaller than the row length\n");
    for (const void* p : {H, W, dY, dR, static_cast<const void*>(dX)})
        if (int rc = check_element_alignment(p, type)) return rc;
    for (const void* p : {static_cast<const void*>(rstd), static_cast<const void*>(dW)})
        if (int rc = check_element_alignment(p, DECX_HIP_F32)) return rc;
    if (dW && (!work || (reinterpret_cast<uintptr_t>(work) & 3u) || work_bytes < rmsnorm_backward_workspace(M, K)))
        return fail(DECX_HIP_FAIL_ERROR_PARAMS, "the weight's gradient needs a workspace of %zu bytes (decx_hip_rmsnorm_backward_workspace)\n",
                    rmsnorm_backward_workspace(M, K));
    const size_t m = (size_t)M, k = (size_t)K, wide = element_size(type), need = rmsnorm_backward_workspace(M, K);
    if (int rc = check_results({{operand(dX, m, k, lddx, wide), 7u}, {operand(dW, 1, k, k, 4)}, {operand(dW ? work : nullptr, 1, need, need, 1)}},
                               {operand(H, m, k, ldh, wide), operand(dY, m, k, lddy, wide), operand(dR, m, k, lddr, wide), operand(W, 1, k, k, wide),
                                operand(rstd, 1, m, m, 4)}))
        return rc;
    const int groups = rmsnorm_backward_groups(M, K, type == DECX_HIP_F32 ? 4 : 2);
    RmsNormBackwardArgs g = {};
    g.H = H, g.W = W, g.dY = dY, g.dR = dR, g.rstd = rstd, g.dX = dX, g.row_groups = groups;
    // Few rows of inputs that the caches hold: the column workgroups (one launch: 200 x 1500 8.4 -> 5.6 us, 512 x 4096 10.7 ->
    // 7.4, 512 x 8192 15.9 -> 13; 2048 x 512 would go 12.5 -> 29.8), unless dX overwrites what they read
    const bool in_place = dX == H || dX == dY;
    const bool columns = dW && !in_place && M <= 512 && (size_t)M * K <= (size_t)1 << 22 && K <= kRmsNormMaxK / 2;      // DW_IN_LDS beyond
    if (columns) g.dW = dW;
    else if (dW) g.partial = static_cast<float*>(work);
    g.ldh = (size_t)ldh, g.lddy = (size_t)lddy, g.lddr = (size_t)lddr, g.lddx = (size_t)lddx;
    g.M = M, g.K = K, g.rows_each = cdiv(M, groups);
    // 16-bit inputs of more than 128 MiB are read past the caches: 8192 x 8192, 402 MB, 99 us against 112, 4096 x 8192, 201 MB, 55
    // against 61; 2048 x 8192, 101 MB, 32 against 29 (and in fp32, whose lanes read a line in two pieces, always slower)
    g.stream = (size_t)M * K * (dR ? 6 : 4) > ((size_t)128 << 20);
    int rc = type == DECX_HIP_F32 ? rmsnorm_backward_launch<0>(g) : type == DECX_HIP_F16 ? rmsnorm_backward_launch<1>(g) : rmsnorm_backward_launch<2>(g);
    if (rc || !g.partial) return rc;
    if (K <= 2048)          // narrow pieces where wide ones would leave most of the chip idle
        hipLaunchKernelGGL(rmsnorm_dw_kernel<8>, dim3((unsigned)cdiv(K, 8)), dim3(256), 0, g_rt.stream, g.partial, groups, K, dW);
    else
        hipLaunchKernelGGL(rmsnorm_dw_kernel<32>, dim3((unsigned)cdiv(K, 32)), dim3(256), 0, g_rt.stream, g.partial, groups, K, dW);
    HIP_TRY(hipGetLastError());
    return 0;
}

}  // namespace decx_hip
