// Pieces of the scaled 8-bit products' kernels (f8gemm_tile.hpp, f8gemm_stream.hpp): the arguments, the matrix instruction
// with either kind of scale, fragments at the ragged end of K, and the store of a result.
//
//   D[m][n] = C[m][n] + sum over blocks kb of 128 k:  SA[kb][m] * SB[kb][n / b_rows] * sum_{k in kb} A[m][k] * B[n][k]
//
// v_mfma_f32_16x16x128_f8f6f4 multiplies 16 rows of A by 16 rows of B over exactly one scale block and takes both 8-bit
// formats in any pairing.  A lane (lg = lane / 16, li = lane % 16) holds 32 of the 128 codes of row li of each operand; the
// sum does not depend on which 32, as long as both operands agree: here the 16-byte units lg and lg + 4 of the block.
// B is the first operand, so that a lane's four results are columns 4 lg .. 4 lg + 3 of row li.
//
// Scales:
//   e8m0: operands of the instruction's scaled form, one biased exponent for the 32 codes that a lane holds; the same for
//         all four lanes of a row.  The scaling costs nothing.
//   fp32: the instruction starts from zero and its 4 sums are multiplied into the accumulator, 4 fused multiply-adds a lane
//         (8 instructions where every column has a scale of its own).
//
// What the 8-bit instructions lose.  They align the products of 8 consecutive codes to the largest of them and drop what
// lies below 2^-13 of it (measured: 2^16 + 2^3 within 8 codes is exact, 2^16 + 2^2 gives 2^16; between groups of 8 and to
// the accumulator nothing is dropped; v_mfma_f32_16x16x32_fp8_fp8 does the same).  A result is off by at most 7 * 2^-13 of
// the largest product of each group of 8, added over the groups.  That is no bound relative to the result, whose sum may
// cancel; measured as a norm, on activations with outlier channels, it is 1e-5 to 9e-5 of the result's: a fifth of what
// rounding to binary16 costs, and less for bfloat16, but it would be the whole error of an fp32 result.  16-bit results take
// it for twice the rate.  Results in fp32 are computed EXACTly: the codes, which binary16 holds exactly in both formats, are
// converted in registers and multiplied by v_mfma_f32_16x16x32_f16, whose products are exact and whose sums are fp32 ones
// (7e-8), at half the rate.
// Accumulation is in fp32 throughout; a result is rounded to its type once.
#pragma once
#include "runtime.hpp"
#include "f8_common.hpp"

namespace decx_hip {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// How a kernel multiplies: the operands' formats (DECX_HIP_E4M3 = 0, DECX_HIP_E5M2 = 1, the instruction's own codes), the
// kind of scale, whether B has one for each row (0: one for each 128 rows), and whether sums are exact.  The scaled
// instruction takes its scales by lane, whatever rows share them.
template <int FA_, int FB_, bool E8M0_, bool B_PER_ROW_, bool EXACT_>
struct F8Kind {
    static constexpr int FA = FA_, FB = FB_;
    static constexpr bool E8M0 = E8M0_, EXACT = EXACT_, B_PER_ROW = B_PER_ROW_;
    static constexpr bool IN_INSTRUCTION = E8M0 && !EXACT;      // the scales are the matrix instruction's operands
    static_assert(!(IN_INSTRUCTION && B_PER_ROW), "one kernel serves both");
};

struct F8GemmArgs {
    const uint8_t* A;
    const uint8_t* B;
    const void* SA;
    const void* SB;
    const void* C;          // nullable, of the result's type
    void* D;
    size_t lda, ldb, ldsa, ldsb, ldc, ldd;
    int b_shift;            // 7: a scale for each 128 rows of B, 0: for each row
    int type;               // of C and D
    int M, N, K;
    int variant;            // the kernel to launch (plan_f8gemm, f8gemm.hip)
    int tiles_m, tiles_n, group_m;
};

template <int FA, int FB>
__device__ __forceinline__ f32x4 f8_mfma(i32x8 b, i32x8 a, f32x4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, FB, FA, 0, 0, 0, 0);
}
template <int FA, int FB>
__device__ __forceinline__ f32x4 f8_mfma_scaled(i32x8 b, i32x8 a, f32x4 c, int sb, int sa) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, FB, FA, 0, sb, 0, sa);
}
// the 32 codes of a fragment as binary16, 8 to each of 4 matrix instructions
struct F16Fragment {
    f16x8 q[4];
};
template <int FORMAT>
__device__ __forceinline__ F16Fragment f8_widen(i32x8 codes) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    F16Fragment r;
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            f16x2 lo, hi;
            if constexpr (FORMAT == DECX_HIP_E4M3) {
                lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[2 * q + w], 1.f, false);
                hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[2 * q + w], 1.f, true);
            } else {
                lo = __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(codes[2 * q + w], 1.f, false);
                hi = __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(codes[2 * q + w], 1.f, true);
            }
            r.q[q][4 * w] = lo[0], r.q[q][4 * w + 1] = lo[1], r.q[q][4 * w + 2] = hi[0], r.q[q][4 * w + 3] = hi[1];
        }
    return r;
}
__device__ __forceinline__ f32x4 f8_mfma_exact(const F16Fragment& b, const F16Fragment& a) {
    f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; ++q) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(b.q[q], a.q[q], p, 0, 0, 0);
    return p;
}
// a biased exponent in 8 bits as its power of two (0: 2^-127, 255: NaN)
__device__ __forceinline__ float e8m0_value(uint32_t e) {
    return __uint_as_float(e == 255u ? 0x7fc00000u : e == 0u ? 0x00400000u : e << 23);
}

__device__ __forceinline__ i32x8 f8_fragment(u32x4 lo, u32x4 hi) {
    return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
// a 16-byte unit of which only the first n codes exist (n may be <= 0 or >= 16), `at` of the row's codes before it: the others
// are zeros, whose products add nothing whatever the block's scale (but infinity); nothing beyond the n is read
__device__ __forceinline__ u32x4 f8_unit_part(const uint8_t* p, int n, int at) {
    if (n >= 16) return *reinterpret_cast<const u32x4_any*>(p);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (n <= 0) return v;
    if (at >= 16) return bytes_down(*reinterpret_cast<const u32x4_any*>(p + (n - 16)), 16 - n);
#pragma unroll
    for (int e = 0; e < 16; ++e)
        if (e < n) v[e >> 2] |= (uint32_t)p[e] << (8 * (e & 3));
    return v;
}

template <class T>
__device__ __forceinline__ void f8_store4(T* d, const T* c, f32x4 v, int n) {
    typedef T Four __attribute__((ext_vector_type(4)));
    typedef T FourAny __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (n >= 4) {
        if (c) {
            const Four o = *reinterpret_cast<const FourAny*>(c);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += (float)o[e];
        }
        Four r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (T)v[e];
        *reinterpret_cast<FourAny*>(d) = r;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < n) d[e] = (T)(v[e] + (c ? (float)c[e] : 0.f));
}
// columns n .. n + 3 of row m of the result, as far as they exist
__device__ __forceinline__ void f8_store_result(const F8GemmArgs& g, int m, int n, f32x4 v) {
    if (m >= g.M || n >= g.N) return;
    const size_t d = (size_t)m * g.ldd + n, c = (size_t)m * g.ldc + n;
    const int left = g.N - n;
    if (g.type == DECX_HIP_F32)
        f8_store4(static_cast<float*>(g.D) + d, g.C ? static_cast<const float*>(g.C) + c : nullptr, v, left);
    else if (g.type == DECX_HIP_F16)
        f8_store4(static_cast<_Float16*>(g.D) + d, g.C ? static_cast<const _Float16*>(g.C) + c : nullptr, v, left);
    else
        f8_store4(static_cast<__bf16*>(g.D) + d, g.C ? static_cast<const __bf16*>(g.C) + c : nullptr, v, left);
}

// columns n .. n + 3 of row m of C, as far as they exist, on top of v (16-bit results)
template <class T>
__device__ __forceinline__ f32x4 f8_add_c(const F8GemmArgs& g, int m, int n, f32x4 v) {
    if (m >= g.M || n >= g.N) return v;
    const T* c = static_cast<const T*>(g.C) + (size_t)m * g.ldc + n;
    if (n + 4 <= g.N) {
        typedef T Four __attribute__((ext_vector_type(4)));
        typedef T FourAny __attribute__((ext_vector_type(4), aligned(sizeof(T))));
        const Four o = *reinterpret_cast<const FourAny*>(c);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += (float)o[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < g.N) v[e] += (float)c[e];
    }
    return v;
}
template <class T>
__device__ __forceinline__ u32x2 f8_round4(f32x4 v) {
    typedef T Four __attribute__((ext_vector_type(4)));
    const Four r = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    return __builtin_bit_cast(u32x2, r);
}

}  // namespace decx_hip
