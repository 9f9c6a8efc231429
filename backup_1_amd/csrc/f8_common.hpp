// What the 8-bit operators share (f8_quantize.hip, f8gemm.hip, rmsnorm.hip): the wide element types and their rounding,
// the 8-bit codes, the scales of blocks of 128, and loads and stores of 8 consecutive elements at any alignment.
#pragma once
#include "tile_common.hpp"

namespace decx_hip {

constexpr int kScaleBlock = 128;      // elements along the contraction that share a scale
constexpr int kMostExtent = 1 << 29;  // rows or columns of an operand: sums of sizes and 4-byte offsets of scales fit 32 bits
constexpr long kMostThreads = 0xffffffffL;     // of a launch: the hardware counts them in 32 bits

// Wide and vector types that may lie at any address: global memory takes such accesses on gfx950 as one instruction, so
// rows whose pitch is no multiple of 16 bytes need no slower loader of their own.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(1)));

// ---- wide element types, by the codes of the C ABI (DECX_HIP_F32 / F16 / BF16)
template <int TYPE> struct Wide;
template <> struct Wide<0> { typedef float T; };
template <> struct Wide<1> { typedef _Float16 T; };
template <> struct Wide<2> { typedef __bf16 T; };

// 8 consecutive elements in fp32 (exact for every type)
struct Eight {
    float v[8];
};
// ... and as they lie in memory: 16 bytes, or 32 in fp32
template <int TYPE>
struct RawEight {
    u32x4 w[TYPE == 0 ? 2 : 1];
};
// STREAM: non-temporal, for inputs that no cache can hold.  Stores of 16-bit types are non-temporal always: norm of 8192 x
// 8192 5 % faster than with plain ones.  Where the next call reads the result at once (bf16 norms in a row, each on the last
// one's h; us, non-temporal / plain): 16 x 4096 4.4 / 4.4, 256 x 4096 4.2 / 4.3, 1024 x 4096 7.4 / 7.2, 2048 x 4096 12.9 / 13.1,
// 4096 x 4096 23.3 / 20.9, 8192 x 4096 43.1 / 41.0; gradients in a row 4.3 / 4.3, 3.7 / 3.65, 5.8 / 5.9, 10.8 / 10.9, 21.5 / 19.2,
// 39.0 / 37.7.  Those of fp32, a lane's 32 bytes in two, leave half lines that way (8192 x 4096 100 -> 119).
template <int TYPE, bool STREAM = false>
__device__ __forceinline__ RawEight<TYPE> load_raw8(const typename Wide<TYPE>::T* p) {
    RawEight<TYPE> r;
    if constexpr (STREAM) {
        r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
        if constexpr (TYPE == 0) r.w[1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p + 4));
    } else {
        r.w[0] = *reinterpret_cast<const u32x4_any*>(p);
        if constexpr (TYPE == 0) r.w[1] = *reinterpret_cast<const u32x4_any*>(p + 4);
    }
    return r;
}
// 16 bytes moved down by n of them (0 < n < 16), zeros from above
__device__ __forceinline__ u32x4 bytes_down(u32x4 v, int n) {
    uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
    if (n >= 8) lo = hi, hi = 0, n -= 8;
    if (n > 0) lo = lo >> (8 * n) | hi << (64 - 8 * n), hi >>= 8 * n;
    return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}
// The first `n` of 8 elements of a row (n may be <= 0 or > 8), the others 0, in two parts.  Reads nothing beyond the n: what
// is left of a row is fetched as the row's last 8 elements, one load instead of n.  fetch8_part issues the load, settle8_part
// moves the elements down, so that loads may stay in flight in between (moved at once, a wave with a row's end waited before
// its next load: norm's gradient of 4096 x 4095 bf16 took 49 us, now 41).  ROWS says what the kernel's rows are like: shorter
// than 8 elements, of any greater length, or of a multiple of 8 (nothing to move, fewer registers); short rows have kernels of
// their own because their loads one by one, never taken, still cost the others (gradient of 4096 x 8190 bf16 82 -> 77 us).
enum { kRowsShort = 0, kRowsRagged = 1, kRowsWhole = 2 };
inline int rows_kind(int K) { return K % 8 == 0 ? kRowsWhole : K > 8 ? kRowsRagged : kRowsShort; }
template <int TYPE, int ROWS, bool STREAM = false>
__device__ __forceinline__ RawEight<TYPE> fetch8_part(const typename Wide<TYPE>::T* p, int n) {
    RawEight<TYPE> r = {};
    if (n <= 0) return r;
    if constexpr (ROWS != kRowsShort) return load_raw8<TYPE, STREAM>(ROWS == kRowsWhole || n >= 8 ? p : p + (n - 8));
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) {
            if constexpr (TYPE == 0) r.w[e >> 2][e & 3] = reinterpret_cast<const uint32_t*>(p)[e];
            else r.w[0][e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e & 1));
        }
    return r;
}
template <int TYPE, int ROWS>
__device__ __forceinline__ void settle8_part(RawEight<TYPE>& r, int n) {
    if (ROWS != kRowsRagged || n >= 8 || n <= 0) return;
    if constexpr (TYPE == 0) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = r.w[e >> 2][e & 3];
#pragma unroll
        for (int s = 4; s > 0; s >>= 1)
            if ((8 - n) & s) {
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = e + s < 8 ? w[e + s < 8 ? e + s : 0] : 0u;
            }
#pragma unroll
        for (int e = 0; e < 8; ++e) r.w[e >> 2][e & 3] = w[e];
    } else {
        r.w[0] = bytes_down(r.w[0], 2 * (8 - n));
    }
}
template <int TYPE>
__device__ __forceinline__ Eight widen8(const RawEight<TYPE>& raw) {
    Eight r;
    if constexpr (TYPE == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) r.v[e] = __uint_as_float(raw.w[e >> 2][e & 3]);
    } else {
        typedef typename Wide<TYPE>::T Vec __attribute__((ext_vector_type(8)));
        const Vec h = __builtin_bit_cast(Vec, raw.w[0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) r.v[e] = (float)h[e];
    }
    return r;
}
template <int TYPE, int ROWS>
__device__ __forceinline__ Eight load8_part(const typename Wide<TYPE>::T* p, int n) {
    RawEight<TYPE> r = fetch8_part<TYPE, ROWS>(p, n);
    settle8_part<TYPE, ROWS>(r, n);
    return widen8<TYPE>(r);
}
// rounds to nearest even, once
template <int TYPE>
__device__ __forceinline__ void store8_part(typename Wide<TYPE>::T* p, const Eight& x, int n) {
    typedef typename Wide<TYPE>::T T;
    if (n >= 8) {
        if constexpr (TYPE == 0) {
            const u32x4 lo = {__float_as_uint(x.v[0]), __float_as_uint(x.v[1]), __float_as_uint(x.v[2]), __float_as_uint(x.v[3])};
            const u32x4 hi = {__float_as_uint(x.v[4]), __float_as_uint(x.v[5]), __float_as_uint(x.v[6]), __float_as_uint(x.v[7])};
            *reinterpret_cast<u32x4_any*>(p) = lo;
            *reinterpret_cast<u32x4_any*>(p + 4) = hi;
        } else {
            typedef T Vec __attribute__((ext_vector_type(8)));
            Vec h;
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = (T)x.v[e];
            __builtin_nontemporal_store(__builtin_bit_cast(u32x4, h), reinterpret_cast<u32x4_any*>(p));
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) p[e] = (T)x.v[e];
}

// ---- 8-bit codes (DECX_HIP_E4M3 / E5M2: the OCP formats, which gfx950 converts to with one rounding to nearest even).
// The callers' values are within the largest finite one up to the last bit of fp32, which rounds down to it, so no value
// needs a clamp; a NaN stays a NaN.
__device__ __forceinline__ uint32_t pack4_f8(float a, float b, float c, float d, int e5m2) {
    int r = 0;
    if (e5m2) {
        r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, r, false);
        r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
    } else {
        r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    }
    return (uint32_t)r;
}
__device__ __forceinline__ u32x2 pack8_f8(const Eight& x, float factor, int e5m2) {
    return u32x2{pack4_f8(x.v[0] * factor, x.v[1] * factor, x.v[2] * factor, x.v[3] * factor, e5m2),
                 pack4_f8(x.v[4] * factor, x.v[5] * factor, x.v[6] * factor, x.v[7] * factor, e5m2)};
}
__device__ __forceinline__ void store_codes(uint8_t* p, u32x2 codes, int n) {
    if (n >= 8) {
        *reinterpret_cast<u32x2_any*>(p) = codes;
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) p[e] = (uint8_t)(codes[e >> 2] >> (8 * (e & 3)));
}

// ---- the scale of a block, from the bits of its largest magnitude.  The maximum is taken over the bit patterns of the
// magnitudes, which order as the values do with NaN above infinity: a NaN in a block is not lost.
struct BlockScale {
    float scale;       // the fp32 scale (the power of two itself for e8m0)
    float factor;      // what the values are multiplied by before they are rounded to 8 bits
    uint32_t e8m0;     // its biased exponent
};
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t eight_magnitude(const Eight& x) {
    uint32_t m = magnitude_bits(x.v[0]);
#pragma unroll
    for (int e = 1; e < 8; ++e) {
        const uint32_t o = magnitude_bits(x.v[e]);
        m = m > o ? m : o;
    }
    return m;
}
constexpr uint32_t kLeastMagnitude = 0x0d800000u;      // 2^-100: blocks of zeros and of smaller values take its scale
// e4m3's largest value is 1.75 * 2^8, e5m2's 1.75 * 2^15.
//   fp32: scale = amax / largest, factor = 1 / scale, both correctly rounded: amax * factor is within 2^-22 of the largest.
//   e8m0: the least 2^e with largest * 2^e >= amax: amax's exponent, one more where its mantissa is beyond 1.75, less 8
//         (15).  The factor 2^-e is exact, and so is every product with it.  Infinity and NaN give the NaN of e8m0, 255.
__device__ __forceinline__ BlockScale block_scale(uint32_t amax_bits, int e5m2, int e8m0) {
    if (amax_bits < kLeastMagnitude) amax_bits = kLeastMagnitude;
    BlockScale s;
    if (e8m0) {
        const uint32_t e = ((amax_bits + 0x1fffffu) >> 23) - (e5m2 ? 15u : 8u);
        const bool finite = amax_bits < 0x7f800000u;
        s.e8m0 = finite ? e : 255u;
        s.scale = finite ? __uint_as_float(e << 23) : __uint_as_float(0x7fc00000u);
        s.factor = finite ? __uint_as_float((254u - e) << 23) : __uint_as_float(0x7fc00000u);
    } else {
        s.scale = __fdiv_rn(__uint_as_float(amax_bits), e5m2 ? 57344.f : 448.f);
        s.factor = __fdiv_rn(1.f, s.scale);
        s.e8m0 = 0u;
    }
    return s;
}
__device__ __forceinline__ void store_scale(void* scales, size_t at, const BlockScale& s, int e8m0) {
    if (e8m0) static_cast<uint8_t*>(scales)[at] = (uint8_t)s.e8m0;
    else static_cast<float*>(scales)[at] = s.scale;
}

// maximum over the 16 lanes of a group (lanes 16g .. 16g + 15), in every lane of it
__device__ __forceinline__ uint32_t group16_max(uint32_t v) {
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)v, d);
        v = v > o ? v : o;
    }
    return v;
}

}  // namespace decx_hip
