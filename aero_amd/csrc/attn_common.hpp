// Operand helpers of the attention kernels (attention.hip, attn_rows.hip): cache
// elements as fp32, integer codes as fp16 matrix operands, two-part splits.
#pragma once

#include "common.hpp"

namespace aero {
namespace {

template <int DT>
constexpr int kv_bits() { return DT == 0 ? 32 : (DT == 1 ? 8 : 4); }

// N bytes (4-byte multiple, or 2) at p into words.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
    if constexpr (N % 16 == 0) {
#pragma unroll
        for (int i = 0; i < N / 16; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(p + 16 * i);
            w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
        }
    } else if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            const uint2 x = *reinterpret_cast<const uint2*>(p + 8 * i);
            w[2 * i] = x.x; w[2 * i + 1] = x.y;
        }
    } else if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
        static_assert(N == 2, "slice size");
        w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
}

// element e of a slice held as words: fp32 bits, int8 or int4 (low nibble first)
template <int DT>
__device__ __forceinline__ float slice_elem(const uint32_t* w, int e) {
    if constexpr (DT == 0) {
        return __uint_as_float(w[e]);
    } else if constexpr (DT == 1) {
        return (float)((int32_t)(w[e >> 2] << (24 - 8 * (e & 3))) >> 24);
    } else {
        return (float)((int32_t)(w[e >> 3] << (28 - 4 * (e & 7))) >> 28);
    }
}

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef unsigned int v2u __attribute__((ext_vector_type(2)));

__device__ __forceinline__ h2 u32_h2(uint32_t u) { return __builtin_bit_cast(h2, u); }
__device__ __forceinline__ uint32_t h2_u32(h2 h) { return __builtin_bit_cast(uint32_t, h); }

// A reduction over each row of 16 lanes (or 8), and over the lanes c, 16 + c, 32 + c
// and 48 + c (or 32 apart): every lane has the result, the same bits in all of them. By
// lane moves of the vector unit: a shuffle through LDS takes some 100 cycles.
template <int CTRL>
__device__ __forceinline__ uint32_t lane_moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
template <int CTRL, typename T, typename Op>
__device__ __forceinline__ T with_moved(T v, Op op) {
    return op(v, __builtin_bit_cast(T, lane_moved<CTRL>(__builtin_bit_cast(uint32_t, v))));
}
template <typename T, typename Op>
__device__ __forceinline__ T over_eight(T v, Op op) {
    v = with_moved<0xb1>(v, op);           // lane ^ 1
    v = with_moved<0x4e>(v, op);           // lane ^ 2
    return with_moved<0x141>(v, op);       // 7 - lane: the other four
}
template <typename T, typename Op>
__device__ __forceinline__ T over_row(T v, Op op) {
    return with_moved<0x140>(over_eight(v, op), op);   // 15 - lane: the other eight
}
template <typename T, typename Op>
__device__ __forceinline__ T over_halves(T v, Op op) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const v2u r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r.x, b = r.y;     // (not cast as they are: that takes x twice)
    return op(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
}
template <typename T, typename Op>
__device__ __forceinline__ T over_rows(T v, Op op) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const v2u r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a = r.x, b = r.y;
    return over_halves(op(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b)), op);
}
struct Add {
    template <typename T>
    __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
    __device__ __forceinline__ int32_t operator()(int32_t a, int32_t b) const { return max(a, b); }
};
struct Min {
    __device__ __forceinline__ float operator()(float a, float b) const { return fminf(a, b); }
    __device__ __forceinline__ int32_t operator()(int32_t a, int32_t b) const { return min(a, b); }
};

// the 8 codes of key-slice step s as fp16 (bits 0x6400 or u are 1024 + u), in the
// order of key_order
template <int DT>
__device__ __forceinline__ h8 key_codes(const uint32_t* k, int s) {
    constexpr uint32_t E = 0x64646464u;
    if constexpr (DT == 1) {
        const h2 off = h2{(_Float16)-1152.f, (_Float16)-1152.f};
        const uint32_t u0 = k[2 * s] ^ 0x80808080u, u1 = k[2 * s + 1] ^ 0x80808080u;
        const h2 a0 = u32_h2(__builtin_amdgcn_perm(E, u0, 0x04010400u)) + off;
        const h2 a1 = u32_h2(__builtin_amdgcn_perm(E, u0, 0x04030402u)) + off;
        const h2 a2 = u32_h2(__builtin_amdgcn_perm(E, u1, 0x04010400u)) + off;
        const h2 a3 = u32_h2(__builtin_amdgcn_perm(E, u1, 0x04030402u)) + off;
        return __builtin_bit_cast(h8, make_uint4(h2_u32(a0), h2_u32(a1), h2_u32(a2), h2_u32(a3)));
    } else {
        const h2 off = h2{(_Float16)-1032.f, (_Float16)-1032.f};
        const uint32_t u = k[s] ^ 0x88888888u;
        const uint32_t lo = u & 0x0F0F0F0Fu, hi = (u >> 4) & 0x0F0F0F0Fu;
        const h2 a0 = u32_h2(__builtin_amdgcn_perm(E, lo, 0x04020400u)) + off;  // 0, 4
        const h2 a1 = u32_h2(__builtin_amdgcn_perm(E, lo, 0x04030401u)) + off;  // 2, 6
        const h2 a2 = u32_h2(__builtin_amdgcn_perm(E, hi, 0x04020400u)) + off;  // 1, 5
        const h2 a3 = u32_h2(__builtin_amdgcn_perm(E, hi, 0x04030401u)) + off;  // 3, 7
        return __builtin_bit_cast(h8, make_uint4(h2_u32(a0), h2_u32(a1), h2_u32(a2), h2_u32(a3)));
    }
}

// element i of a key-slice operand is slice element 8s + key_order(i)
template <int DT>
__device__ __forceinline__ constexpr int key_order(int i) {
    return DT == 1 ? i : ((i & 1) ? 4 : 0) + ((i >> 1) & 1) * 2 + (i >> 2);
}

// codes of element t of two value rows (words a, b of those rows) as fp16
// (code_a, code_b)
template <int DT>
__device__ __forceinline__ uint32_t value_pair(const uint32_t* a, const uint32_t* b, int t) {
    if constexpr (DT == 1) {
        const uint32_t byte = (uint32_t)(t & 3);
        const uint32_t sel = 0x0C000C00u | ((4u + byte) << 16) | byte;
        const uint32_t x = __builtin_amdgcn_perm(b[t >> 2], a[t >> 2], sel) ^ 0x64806480u;
        return h2_u32(u32_h2(x) + h2{(_Float16)-1152.f, (_Float16)-1152.f});
    } else {
        const uint32_t byte = (uint32_t)((t >> 1) & 3);
        const uint32_t sel = 0x0C000C00u | ((4u + byte) << 16) | byte;
        uint32_t x = __builtin_amdgcn_perm(b[t >> 3], a[t >> 3], sel);
        x = ((t & 1) ? (x >> 4) : x) & 0x000F000Fu;
        return h2_u32(u32_h2(x ^ 0x64086408u) + h2{(_Float16)-1032.f, (_Float16)-1032.f});
    }
}

// v = 2^scale-shifted value split into fp16 hi and lo
__device__ __forceinline__ void split2(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// 2^e as a float, e in [-126, 127]
__device__ __forceinline__ float pow2i(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

}  // namespace
}  // namespace aero
