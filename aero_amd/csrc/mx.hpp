// Microscaled rows: blocks of 32 values of a row share a power of two, a byte s that
// stands for 2^(s-127) (255: the block holds NaN or an infinity and is NaN). Two
// formats: AERO_MX_INT8, a signed byte c worth c/64 of the scale, and AERO_MX_FP4,
// four bits (sign, two of exponent, one of mantissa) worth 0 .5 1 1.5 2 3 4 6 of it,
// two codes a byte, the low nibble first.
//
// The scale is the smallest power of two under which the block's largest magnitude
// does not pass the format's largest (127/64, 6): nothing is cut off, and no value is
// off by more than half a step (in 8 bits, past 2^127 * 127/64, where no scale is left, the
// largest code stands in). 8-bit rows keep s >= 4, so that the product can give the low half
// of a code a scale byte of its own, down to s - 4.
#pragma once
#include "common.hpp"
#include "aero_hip.h"

namespace aero {

template <int FMT>
constexpr int kMxLow = FMT == AERO_MX_INT8 ? 4 : 0;

// Largest of v over the 8 lanes that hold a block, four values each.
__device__ __forceinline__ uint32_t mx_max8(uint32_t v) {
    auto step = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    v = step(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));   // lane ^ 1
    v = step(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));   // lane ^ 2
    v = step(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));  // lane ^ 7
    return v;
}

__device__ __forceinline__ uint32_t mx_abs_bits(float v) {
    return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu;
}

// Scale byte of a block from the bits of its largest magnitude (as integers NaN and
// infinities are above every number).
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale(uint32_t amax) {
    const int k = (int)(amax >> 23);
    const int m = (int)(amax & 0x7FFFFFu);
    int s;
    if constexpr (FMT == AERO_MX_INT8)
        s = k + (m > 0x7E0000 ? 1 : 0);        // 127/64 = 2^0 * 1.984375
    else
        s = k - 2 + (m > 0x400000 ? 1 : 0);    // 6 = 2^2 * 1.5
    s = s < kMxLow<FMT> ? kMxLow<FMT> : (s > 254 ? 254 : s);
    return k == 255 ? 255u : (uint32_t)s;
}

// Four codes of one lane: a dword of bytes, or four nibbles in the low 16 bits.
// 8 bits: c = rint(h 2^(133-s)); the sum with 1.5 * 2^23 rounds halves to even and
// leaves c in the low byte. (Past 2^127 * 127/64 the largest code stands in.)
// 4 bits: the hardware's conversion, which divides by the scale's exponent exactly and
// rounds halves to even.
template <int FMT>
__device__ __forceinline__ uint32_t mx_codes(float4 h, uint32_t s) {
    if (s == 255u) return 0u;
    if constexpr (FMT == AERO_MX_INT8) {
        const int e = 133 - (int)s;
        auto code = [e](float v) {
            const float q = __builtin_amdgcn_fmed3f(__builtin_amdgcn_ldexpf(v, e), -127.f, 127.f);
            return __builtin_bit_cast(uint32_t, q + 12582912.f);
        };
        const uint32_t lo = __builtin_amdgcn_perm(code(h.y), code(h.x), 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(code(h.w), code(h.z), 0x04000c0cu);
        return lo | hi;
    } else {
        const float sc = __builtin_bit_cast(float, s << 23);
        uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, h.x, h.y, sc, 0);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, h.z, h.w, sc, 1);
    }
}

// One lane's four values of a block held by 8 lanes: codes to codes[quad], the scale
// (by the first lane) to scales[quad / 8].
__device__ __forceinline__ uint32_t mx_amax(float4 h) {
    const uint32_t ax = mx_abs_bits(h.x), ay = mx_abs_bits(h.y);
    const uint32_t az = mx_abs_bits(h.z), aw = mx_abs_bits(h.w);
    return mx_max8(max(max(ax, ay), max(az, aw)));
}

template <int FMT>
__device__ __forceinline__ void mx_store(float4 h, int64_t quad, uint8_t* codes, uint8_t* scales) {
    const uint32_t s = mx_scale<FMT>(mx_amax(h));
    const uint32_t c = mx_codes<FMT>(h, s);
    if constexpr (FMT == AERO_MX_INT8)
        reinterpret_cast<uint32_t*>(codes)[quad] = c;
    else
        reinterpret_cast<uint16_t*>(codes)[quad] = (uint16_t)c;
    if ((quad & 7) == 0) scales[quad >> 3] = (uint8_t)s;
}

// Whether four values that are only known to a relative d, and the block's largest of which
// mx_max8 gives amax, have the codes they seem to: no border between two codes, nor one of
// the scale, lies within d of any of them. (d counts the rounding to fp32, too.)
template <int FMT>
__device__ __forceinline__ bool mx_sure(float4 h, uint32_t amax, float d) {
    if (amax == 0u) return true;          // (what 32 bits lose below 2^-149 has code 0)
    const float top = __builtin_bit_cast(float, amax);
    const uint32_t s = mx_scale<FMT>(amax);
    // (a block near the subnormals, where errors are not relative, is not sure)
    bool sure = s != 255u && top > 0x1p-100f && mx_scale<FMT>(mx_abs_bits(top * (1.f - d))) == mx_scale<FMT>(mx_abs_bits(top * (1.f + d)));
    if constexpr (FMT == AERO_MX_INT8) {
        const int e = 133 - (int)s;
        float far = 0.f;     // the largest |distance to the code| + |code| d, half a code at a border
        auto one = [&](float v) {
            const float q = __builtin_amdgcn_ldexpf(v, e);
            const float f = q - __builtin_rintf(q);
            far = fmaxf(far, __builtin_fmaf(fabsf(q), d, fabsf(f)));
        };
        one(h.x); one(h.y); one(h.z); one(h.w);
        return sure && far < 0.5f;
    } else {
        const float lo = 1.f - d, hi = 1.f + d;
        return sure && mx_codes<FMT>(make_float4(h.x * lo, h.y * lo, h.z * lo, h.w * lo), s) ==
                           mx_codes<FMT>(make_float4(h.x * hi, h.y * hi, h.z * hi, h.w * hi), s);
    }
}

// Lanes of one launch: HIP takes fewer than 2^32, and the kernels here count quads of a launch in
// 32 bits. Larger calls are several launches.
constexpr int64_t kMxLanes = (int64_t)1 << 31;

inline int64_t mx_row_bytes(int fmt, int64_t cols) { return fmt == AERO_MX_FP4 ? cols / 2 : cols; }

// What every call over rows checks first.
bool mx_rows_ok(const char* what, int fmt, const void* codes, const void* scales, int64_t rows,
                int64_t cols);

}  // namespace aero
