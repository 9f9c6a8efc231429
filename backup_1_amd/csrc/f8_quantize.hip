// Quantisation of a wide matrix to 8-bit codes with a scale for each block of 128 (rows) or 128 x 128 (squares), and of
// its transpose in the same pass: what the operands of f8gemm.hip are made with.
//
// Bound: memory.  A row-major pass reads 2 or 4 bytes an element and writes 1 (2 with the transpose); everything else is
// register work between the load and the store.
#include "runtime.hpp"
#include "f8_common.hpp"

namespace decx_hip {

// Rows only.  16 lanes hold the 128 elements of a block, 8 each: one 16- or 32-byte load, a maximum over the lanes, one
// 8-byte store.  A workgroup takes 16 rows x kQuantCols blocks, so that the scales of a block column leave as 64
// consecutive bytes (one scale for a row and block lies `lds` elements from the row's next one).
constexpr int kQuantCols = 4;
template <int TYPE, int ROWS>
__global__ __launch_bounds__(256) void f8_quantize_rows_kernel(const typename Wide<TYPE>::T* __restrict__ X, size_t ldx, int M, int K,
                                                               int e5m2, int e8m0, uint8_t* __restrict__ Q, size_t ldq,
                                                               void* __restrict__ S, size_t lds, int col_groups) {
    const int group = threadIdx.x >> 4, li = threadIdx.x & 15;
    const int m = (int)(blockIdx.x / (unsigned)col_groups) * 16 + group;
    const int kb0 = (int)(blockIdx.x % (unsigned)col_groups) * kQuantCols;
    const int rows = M;
    const size_t row = (size_t)(m < rows ? m : rows - 1);
    RawEight<TYPE> raw[kQuantCols];
    Eight x[kQuantCols];
#pragma unroll
    for (int j = 0; j < kQuantCols; ++j) {
        const int k = (kb0 + j) * kScaleBlock + 8 * li;
        raw[j] = fetch8_part<TYPE, ROWS>(X + row * ldx + (k < K ? k : 0), K - k);
    }
#pragma unroll
    for (int j = 0; j < kQuantCols; ++j) {
        const int k = (kb0 + j) * kScaleBlock + 8 * li;
        settle8_part<TYPE, ROWS>(raw[j], K - k);
        x[j] = widen8<TYPE>(raw[j]);
    }
    const int blocks = (K + kScaleBlock - 1) / kScaleBlock;
#pragma unroll
    for (int j = 0; j < kQuantCols; ++j) {
        const int kb = kb0 + j, k = kb * kScaleBlock + 8 * li;
        const BlockScale s = block_scale(group16_max(eight_magnitude(x[j])), e5m2, e8m0);
        if (m < rows && kb < blocks) {
            store_codes(Q + row * ldq + k, pack8_f8(x[j], s.factor, e5m2), K - k);
            if (li == 0) store_scale(S, (size_t)kb * lds + m, s, e8m0);
        }
    }
}

// Maxima of N values each over the lanes that differ in bits BIT, 2 BIT, ... of their number, spread over them: with every
// step a lane keeps half of the values, those whose lowest bit is its own bit `id & 1`, then `id >> 1 & 1`, ...  Ends with LEFT
// values: value j is number id % (N / LEFT) + j * (N / LEFT).
template <int N, int BIT, int LEFT = 1>
__device__ __forceinline__ void scatter_max(uint32_t (&v)[8], int id) {
    if constexpr (N > LEFT) {
        const bool odd = id & 1;
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            const uint32_t keep = odd ? v[2 * j + 1] : v[2 * j], give = odd ? v[2 * j] : v[2 * j + 1];
            const uint32_t o = (uint32_t)__shfl_xor((int)give, BIT);
            v[j] = keep > o ? keep : o;
        }
        scatter_max<N / 2, 2 * BIT, LEFT>(v, id >> 1);
    }
}

// A 128 x 128 tile of X for a workgroup: squares, the transpose, or both orders.  Thread (rg, c) of 16 x 16 holds rows
// 8 rg .. 8 rg + 7 of columns 8 c .. 8 c + 7, so that the codes of a column's 8 rows are 8 bytes of the transpose.  Those
// go through LDS ([column][row], 8-byte units XOR-swizzled by the column group, which spreads the 16 units that 16 lanes
// write over all banks) and leave as 128 contiguous bytes a row.
//   rows   : the scale of a row is a maximum over the 16 lanes of its group; lane c ends with that of row c % 8;
//   columns: over the 8 rows of a thread, the 4 groups of a wave and, through LDS, the 4 waves; thread t makes column t's;
//   square : one maximum over the tile, the same codes in both orders.
// So every scale, two divisions in fp32, is made by one or two threads and handed to the others: with all of a row's and
// column's threads making it, 8192 x 8192 bf16 in both orders took 62.6 us instead of 57.1, 2048 x 2048 9.7 instead of 6.9.
template <int TYPE, bool SQUARE, int ROWS>
__global__ __launch_bounds__(256) void f8_quantize_tile_kernel(const typename Wide<TYPE>::T* __restrict__ X, size_t ldx, int M, int K,
                                                               int e5m2, int e8m0, uint8_t* __restrict__ Q, size_t ldq,
                                                               void* __restrict__ S, size_t lds, uint8_t* __restrict__ Qt, size_t ldqt,
                                                               void* __restrict__ St, size_t ldst, int col_blocks) {
    __shared__ uint32_t part[4][kScaleBlock];
    __shared__ __attribute__((aligned(16))) float col_factor[kScaleBlock];
    __shared__ __attribute__((aligned(16))) uint8_t turned[kScaleBlock * kScaleBlock];
    const int tid = threadIdx.x, rg = tid >> 4, c = tid & 15, wave = tid >> 6;
    const int mb = (int)(blockIdx.x / (unsigned)col_blocks), kb = (int)(blockIdx.x % (unsigned)col_blocks);
    const int m0 = mb * kScaleBlock + 8 * rg, k0 = kb * kScaleBlock + 8 * c;
    RawEight<TYPE> raw[8];
    Eight x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool live = m0 + i < M;
        raw[i] = fetch8_part<TYPE, ROWS>(X + (size_t)(live ? m0 + i : 0) * ldx + (k0 < K ? k0 : 0), live ? K - k0 : 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        settle8_part<TYPE, ROWS>(raw[i], K - k0);          // rows past the last are zeros either way
        x[i] = widen8<TYPE>(raw[i]);
    }
    BlockScale square;
    if (SQUARE) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t o = eight_magnitude(x[i]);
            m = m > o ? m : o;
        }
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const uint32_t o = (uint32_t)__shfl_xor((int)m, d);
            m = m > o ? m : o;
        }
        if ((tid & (kWave - 1)) == 0) part[wave][0] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) m = m > part[w][0] ? m : part[w][0];
        square = block_scale(m, e5m2, e8m0);
        if (tid == 0) {
            if (Q) store_scale(S, (size_t)kb * lds + mb, square, e8m0);
            if (Qt) store_scale(St, (size_t)mb * ldst + kb, square, e8m0);
        }
    }
    if (Q) {
        BlockScale mine = square;
        if (!SQUARE) {
            uint32_t m[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) m[i] = eight_magnitude(x[i]);
            scatter_max<8, 1>(m, c);
            const uint32_t o = (uint32_t)__shfl_xor((int)m[0], 8);
            mine = block_scale(m[0] > o ? m[0] : o, e5m2, e8m0);
            if (c < 8 && m0 + c < M) store_scale(S, (size_t)kb * lds + m0 + c, mine, e8m0);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float factor = SQUARE ? square.factor : __shfl(mine.factor, (tid & 48) | i);
            if (m0 + i < M) store_codes(Q + (size_t)(m0 + i) * ldq + k0, pack8_f8(x[i], factor, e5m2), K - k0);
        }
    }
    if (!Qt) return;
    // ---- the transpose
    Eight factors;
    if (!SQUARE) {
        uint32_t m[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            m[e] = magnitude_bits(x[0].v[e]);
#pragma unroll
            for (int i = 1; i < 8; ++i) {
                const uint32_t o = magnitude_bits(x[i].v[e]);
                m[e] = m[e] > o ? m[e] : o;
            }
        }
        scatter_max<8, 16, 2>(m, rg);                           // columns rg % 4 and rg % 4 + 4 of the eight
        part[wave][8 * c + (rg & 3)] = m[0], part[wave][8 * c + (rg & 3) + 4] = m[1];
        __syncthreads();
        if (tid < kScaleBlock) {
            uint32_t most = part[0][tid];
#pragma unroll
            for (int w = 1; w < 4; ++w) most = most > part[w][tid] ? most : part[w][tid];
            const BlockScale s = block_scale(most, e5m2, e8m0);
            if (kb * kScaleBlock + tid < K) store_scale(St, (size_t)mb * ldst + kb * kScaleBlock + tid, s, e8m0);
            col_factor[tid] = s.factor;
        }
        __syncthreads();
        const f32x4 lo = *reinterpret_cast<const f32x4*>(col_factor + 8 * c), hi = *reinterpret_cast<const f32x4*>(col_factor + 8 * c + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) factors.v[e] = e < 4 ? lo[e & 3] : hi[e & 3];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        Eight col;
#pragma unroll
        for (int i = 0; i < 8; ++i) col.v[i] = x[i].v[e];
        *reinterpret_cast<u32x2*>(turned + (8 * c + e) * kScaleBlock + 8 * (rg ^ c)) = pack8_f8(col, SQUARE ? square.factor : factors.v[e], e5m2);
    }
    __syncthreads();
    // row j of the transposed tile: 8 lanes take 16 bytes each = units 2p and 2p + 1, which the swizzle keeps in one
    // 16-byte piece, in either order
#pragma unroll
    for (int pass = 0; pass < 4; ++pass) {
        const int j = pass * 32 + (tid >> 3), p = tid & 7, cg = j >> 3;
        const u32x4 v = *reinterpret_cast<const u32x4*>(turned + j * kScaleBlock + 16 * (p ^ (cg >> 1)));
        const u32x4 w = (cg & 1) ? u32x4{v[2], v[3], v[0], v[1]} : v;
        const int k = kb * kScaleBlock + j, m = mb * kScaleBlock + 16 * p;
        if (k < K && m < M) {
            uint8_t* to = Qt + (size_t)k * ldqt + m;
            if (m + 16 <= M) {
                *reinterpret_cast<u32x4_any*>(to) = w;
            } else {
                store_codes(to, u32x2{w[0], w[1]}, M - m);
                store_codes(to + 8, u32x2{w[2], w[3]}, M - m - 8);
            }
        }
    }
}

template <int TYPE>
static int f8_quantize_launch(const void* X, int ldx, int M, int K, int block_rows, int e5m2, int e8m0, uint8_t* Q, int ldq, void* S,
                              int lds, uint8_t* Qt, int ldqt, void* St, int ldst) {
    typedef typename Wide<TYPE>::T T;
    const T* x = static_cast<const T*>(X);
    const int rows = rows_kind(K);
    const int row_blocks = cdiv(M, kScaleBlock), col_blocks = cdiv(K, kScaleBlock);
    if (block_rows == 1 && !Qt) {
        const int col_groups = cdiv(col_blocks, kQuantCols);
        const long groups = (long)cdiv(M, 16) * col_groups;
        if (groups * 256 > kMostThreads) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "problem too large for one launch\n");
        auto kern = rows == kRowsWhole    ? f8_quantize_rows_kernel<TYPE, kRowsWhole>
                    : rows == kRowsRagged ? f8_quantize_rows_kernel<TYPE, kRowsRagged>
                                          : f8_quantize_rows_kernel<TYPE, kRowsShort>;
        hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(256), 0, g_rt.stream, x, (size_t)ldx, M, K, e5m2, e8m0, Q, (size_t)ldq, S, (size_t)lds,
                           col_groups);
    } else {
        const long tiles = (long)row_blocks * col_blocks;
        if (tiles * 256 > kMostThreads) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "problem too large for one launch\n");
        auto square = rows == kRowsWhole    ? f8_quantize_tile_kernel<TYPE, true, kRowsWhole>
                      : rows == kRowsRagged ? f8_quantize_tile_kernel<TYPE, true, kRowsRagged>
                                            : f8_quantize_tile_kernel<TYPE, true, kRowsShort>;
        auto by_rows = rows == kRowsWhole    ? f8_quantize_tile_kernel<TYPE, false, kRowsWhole>
                       : rows == kRowsRagged ? f8_quantize_tile_kernel<TYPE, false, kRowsRagged>
                                             : f8_quantize_tile_kernel<TYPE, false, kRowsShort>;
        auto kern = block_rows == 1 ? by_rows : square;
        // Large fp32 matrices: 3 workgroups a CU instead of 8, by LDS that nothing uses; their loads are enough and come from fewer
        // places at a time (8192 x 8192 in both orders 85.2 -> 80.8 us; 4096 x 4096, which the caches hold, would go 24.0 -> 25.3)
        const size_t unused = TYPE == 0 && (size_t)M * K * sizeof(T) > (size_t)96 << 20 ? 34000 : 0;
        hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(256), unused, g_rt.stream, x, (size_t)ldx, M, K, e5m2, e8m0, Q, (size_t)ldq, S,
                           (size_t)lds, Qt, (size_t)ldqt, St, (size_t)ldst, col_blocks);
    }
    HIP_TRY(hipGetLastError());
    return 0;
}

int f8_quantize_enqueue(const void* X, int ldx, int type, int M, int K, int block_rows, int format, int scale_type, uint8_t* Q, int ldq,
                        void* S, int lds, uint8_t* Qt, int ldqt, void* St, int ldst) {
    if (int rc = need_library_device()) return rc;
    if (!X || (!Q && !Qt)) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "null matrix pointer\n");
    if ((Q && !S) || (Qt && !St)) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "codes without their scales\n");
    if (M <= 0 || K <= 0) return fail(DECX_HIP_FAIL_DIMS, "Matrix Dims don't match each other");
    if (M > kMostExtent || K > kMostExtent) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "problem too large for one launch\n");
    if (int rc = check_f8_codes(type, format, scale_type)) return rc;
    if (block_rows != 1 && block_rows != kScaleBlock) return fail(DECX_HIP_FAIL_ERROR_PARAMS, "a block has 1 or 128 rows\n");
    const int row_scales = block_rows == 1 ? M : cdiv(M, kScaleBlock), col_scales = block_rows == 1 ? K : cdiv(K, kScaleBlock);
    if (ldx < K || (Q && (ldq < K || lds < row_scales)) || (Qt && (ldqt < M || ldst < col_scales)))
        return fail(DECX_HIP_FAIL_ERROR_PARAMS, "leading dimension smaller than the row length\n");
    if (int rc = check_element_alignment(X, type)) return rc;
    if (scale_type == DECX_HIP_SCALE_F32 && ((reinterpret_cast<uintptr_t>(Q ? S : nullptr) | reinterpret_cast<uintptr_t>(Qt ? St : nullptr)) & 3u))
        return fail(DECX_HIP_FAIL_ERROR_PARAMS, "scales off the grid of their type\n");
    const size_t m = (size_t)M, k = (size_t)K, one = scale_size(scale_type);
    if (int rc = check_results({{operand(Q, m, k, ldq, 1)}, {operand(Q ? S : nullptr, cdiv(K, kScaleBlock), row_scales, lds, one)},
                                {operand(Qt, k, m, ldqt, 1)}, {operand(Qt ? St : nullptr, cdiv(M, kScaleBlock), col_scales, ldst, one)}},
                               {operand(X, m, k, ldx, element_size(type))}))
        return rc;
    const int e5m2 = format == DECX_HIP_E5M2, e8m0 = scale_type == DECX_HIP_SCALE_E8M0;
    if (type == DECX_HIP_F32) return f8_quantize_launch<0>(X, ldx, M, K, block_rows, e5m2, e8m0, Q, ldq, S, lds, Qt, ldqt, St, ldst);
    if (type == DECX_HIP_F16) return f8_quantize_launch<1>(X, ldx, M, K, block_rows, e5m2, e8m0, Q, ldq, S, lds, Qt, ldqt, St, ldst);
    return f8_quantize_launch<2>(X, ldx, M, K, block_rows, e5m2, e8m0, Q, ldq, S, lds, Qt, ldqt, St, ldst);
}

}  // namespace decx_hip
