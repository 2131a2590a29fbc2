// Microscaled rows (mx.hpp) from fp32: plain quantisation, RMSNorm with the residual's
// addition, act(gate) * up, each in one pass that reads its inputs once and writes codes
// and scales; and the way back.
//
// Norms and activations are evaluated in 64 bits and rounded to fp32 once before they are
// quantised. A code is a decision, and next to the border of two an error of the last bit
// of 32 turns it: in 64 bits the codes are those of the formula and do not depend on the
// order of a sum. The arithmetic hides behind the memory: 16384 x 8192 with a residual moves
// 13 bytes a value, for which the card has about 30 instructions a lane.
#include "act_ops.hpp"
#include "mx.hpp"

#pragma clang fp contract(off)

namespace aero {
namespace {

constexpr int64_t kMaxRows = 0x7fffffff;

__device__ __forceinline__ float4 ld4(const float* p, bool vec) {
    if (vec) return ld_stream(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}

// ------------------------------------------------------------- activations
// act(v) in 64 bits; gelu with the erf polynomial of act_ops.hpp, in a form that does not
// cancel on the negative side; gelu_tanh by 1 + tanh(z) = 2 / (1 + exp(-2z)).
template <int KIND>
__device__ __forceinline__ double act64(double v) {
    if constexpr (KIND == AERO_ACT_SILU) {
        return v / (1.0 + exp(-v));
    } else if constexpr (KIND == AERO_ACT_SIGMOID) {
        return 1.0 / (1.0 + exp(-v));
    } else if constexpr (KIND == AERO_ACT_GELU_TANH) {
        return v / (1.0 + exp(-2.0 * 0.7978845608028654 * (v + 0.044715 * v * v * v)));
    } else if constexpr (KIND == AERO_ACT_GELU) {
        const double a = fabs(v * 0.7071067811865476);
        const double t = 1.0 / (1.0 + 0.3275911 * a);
        const double p = ((((1.061405429 * t - 1.453152027) * t + 1.421413741) * t
                           - 0.284496736) * t + 0.254829592) * t * exp(-a * a);
        return 0.5 * v * (v < 0.0 ? p : 2.0 - p);
    } else {
        return v;
    }
}

// exp2(hi + lo), lo small, to 2^-22 (the hardware's exp2 is within 2^-23).
__device__ __forceinline__ float exp2_split(float hi, float lo) {
    const float e = __builtin_amdgcn_exp2f(hi);
    return __builtin_fmaf(e, lo * 0.693147182f, e);
}

// act(v) in 32 bits, to a relative kActOff<KIND>, the later product with `up` and the rounding
// included; ok becomes false where it may be further off (far in the negative tail). The
// arguments of exp are kept in two parts: as one fp32 number their rounding alone would be |v|
// 2^-24 of the result. Hardware exp2 and reciprocal: 2^-23 each.
//   silu, sigmoid: 2^-22 (exp) + 2^-24 (1 + e) + 2^-23 (reciprocal) + 2^-23 (two products)
//   gelu_tanh: the same, its argument from 64 bits
//   gelu: the polynomial's terms are up to 4.5 times its value and it follows t 3.5 times
//   relatively: 14 2^-23 with t's own 2^-22, on the negative side in full
template <int KIND>
constexpr float kActOff = KIND == AERO_ACT_GELU ? 0x1p-18f : 0x1p-20f;

template <int KIND>
__device__ __forceinline__ float act32(float v, bool& ok) {
    constexpr float L = 1.44269502f, LO = 1.92596303e-8f;       // log2(e)
    if constexpr (KIND == AERO_ACT_SILU || KIND == AERO_ACT_SIGMOID) {
        const float hi = -v * L;
        const float e = exp2_split(hi, __builtin_fmaf(-v, L, -hi) - v * LO);
        ok = ok && hi < 90.f;
        const float s = __builtin_amdgcn_rcpf(1.f + e);
        return KIND == AERO_ACT_SILU ? v * s : s;
    } else if constexpr (KIND == AERO_ACT_GELU_TANH) {
        const double x = (double)v;
        const double t = x * __builtin_fma(x * x, -2.0 * 0.7978845608028654 * 1.4426950408889634 * 0.044715,
                                           -2.0 * 0.7978845608028654 * 1.4426950408889634);
        const float hi = (float)t;
        ok = ok && hi < 90.f;
        return v * __builtin_amdgcn_rcpf(1.f + exp2_split(hi, (float)(t - (double)hi)));
    } else {
        const float a = fabsf(v) * 0.707106769f;
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, a, 1.f));
        float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
        p = __builtin_fmaf(p, t, 1.421413741f);
        p = __builtin_fmaf(p, t, -0.284496736f);
        p = __builtin_fmaf(p, t, 0.254829592f);
        // exp(-v^2 / 2)
        const float s = v * v, s2 = __builtin_fmaf(v, v, -s), hi = s * (-0.5f * L);
        const float lo = __builtin_fmaf(s, -0.5f * L, -hi) - 0.5f * (s * LO + s2 * L);
        ok = ok && (v > 0.f || hi > -90.f);
        p = p * t * exp2_split(hi, lo);
        return 0.5f * v * (v < 0.f ? p : 2.f - p);
    }
}

constexpr int kNone = -1;  // no activation, no second input: plain quantisation

// Quad i of rows of nq quads, input rows ld floats apart; 8 consecutive lanes hold a block.
template <int FMT, int KIND, bool UP>
__global__ __launch_bounds__(256)
void mx_rows_kernel(const float* g, const float* u, uint8_t* codes, uint8_t* scales, uint32_t n,
                    uint32_t nq, int64_t ld, bool vec) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= n) return;
    const uint32_t row = i / nq;
    const int64_t at = row * ld + 4 * (int64_t)(i - row * nq);
    float4 h = ld4(g + at, vec);
    if constexpr (KIND == AERO_ACT_IDENTITY) {
        const float4 b = ld4(u + at, vec);      // (a product's fp32 rounding is its only one)
        h = make_float4(h.x * b.x, h.y * b.y, h.z * b.z, h.w * b.w);
    } else if constexpr (KIND != kNone) {
        const float4 x = h, b = UP ? ld4(u + at, vec) : make_float4(1.f, 1.f, 1.f, 1.f);
        // In 32 bits first: where no border of codes is near any value of the wave, they are the
        // formula's. In 64 bits for all, 512 x 14336 took 17.4 us (silu), 512 x 14336 x 9 bytes
        // without the activation 12.0.
        bool ok = true;
        auto fast = [&](float v, float w) {
            const float a = act32<KIND>(v, ok);
            // (a subnormal act(v) has lost bits that a large w would show)
            if (UP && KIND != AERO_ACT_SIGMOID) ok = ok && (fabsf(v) > 0x1p-100f || v == 0.f);
            return UP ? a * w : a;
        };
        h = make_float4(fast(x.x, b.x), fast(x.y, b.y), fast(x.z, b.z), fast(x.w, b.w));
        ok = mx_sure<FMT>(h, mx_amax(h), kActOff<KIND>) && ok;
        if (__any(!ok)) {
            auto one = [](float v, float w) {
                const double a = act64<KIND>((double)v);
                return (float)(UP ? a * (double)w : a);
            };
            h = make_float4(one(x.x, b.x), one(x.y, b.y), one(x.z, b.z), one(x.w, b.w));
        }
    }
    mx_store<FMT>(h, i, codes, scales);
}

template <int FMT, int KIND, bool UP>
bool run_rows(const char* name, const float* g, const float* u, uint8_t* codes, uint8_t* scales,
              int64_t rows, int64_t cols, int64_t ld, hipStream_t s) {
    const bool vec = aligned16(g) && (!UP || aligned16(u)) && ld % 4 == 0;
    const int64_t nq = cols / 4;
    const int64_t step = kMxLanes / nq;
    for (int64_t r = 0; r < rows; r += step) {
        const int64_t n = (rows - r < step ? rows - r : step) * nq;
        if (!launch(name, mx_rows_kernel<FMT, KIND, UP>, dim3((unsigned)((n + 255) / 256)),
                    dim3(256), 0, s, g + r * ld, UP ? u + r * ld : u,
                    codes + r * mx_row_bytes(FMT, cols), scales + r * (cols / 32), (uint32_t)n,
                    (uint32_t)nq, ld, vec))
            return false;
    }
    return true;
}

template <int FMT>
bool run_act(int kind, const float* g, const float* u, uint8_t* codes, uint8_t* scales,
             int64_t rows, int64_t cols, int64_t ld, hipStream_t s) {
#define AERO_MX_ACT(K)                                                                       \
    case K:                                                                                  \
        return u ? run_rows<FMT, K, true>("mx_act_kernel", g, u, codes, scales, rows, cols, ld, s) \
                 : run_rows<FMT, K, false>("mx_act_kernel", g, u, codes, scales, rows, cols, ld, s)
    switch (kind) {
    AERO_MX_ACT(AERO_ACT_SILU);
    AERO_MX_ACT(AERO_ACT_GELU);
    AERO_MX_ACT(AERO_ACT_GELU_TANH);
    AERO_MX_ACT(AERO_ACT_SIGMOID);
    AERO_MX_ACT(AERO_ACT_IDENTITY);
    default:
        set_error("act_mul_mx: unknown kind %d", kind);
        return false;
    }
#undef AERO_MX_ACT
}

// ------------------------------------------------------------------- norm
struct MxNorm {
    const float* x;
    const float* d;      // residual input, or null
    float* xo;           // x + d
    const float* w;      // or null (ones)
    uint8_t* codes;
    uint8_t* scales;
    int64_t cols;
    float eps;
    int flags;
    bool vec;
};

template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xf, 0xf, true);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Sum over a workgroup of BS lanes, the same bits in every lane.
template <int BS>
__device__ __forceinline__ double mx_sum(double v) {
    v = dpp_add<0xB1>(v);       // lane ^ 1, ^ 2, then mirrored in 8 and in 16
    v = dpp_add<0x4E>(v);
    v = dpp_add<0x141>(v);
    v = dpp_add<0x140>(v);
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    if constexpr (BS > 64) {
        __shared__ double part[BS / 64];
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int k = 1; k < BS / 64; ++k) v += part[k];
    }
    return v;
}

__device__ __forceinline__ double sq4(float4 v) {
    return (double)v.x * v.x + (double)v.y * v.y + ((double)v.z * v.z + (double)v.w * v.w);
}

__device__ __forceinline__ float4 add4(float4 a, float4 b) {
    return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

__device__ __forceinline__ float4 scaled4(float4 v, double inv, float4 w, double one) {
    return make_float4((float)(v.x * inv * (w.x + one)), (float)(v.y * inv * (w.y + one)),
                       (float)(v.z * inv * (w.z + one)), (float)(v.w * inv * (w.w + one)));
}

__device__ __forceinline__ double norm_inv(double ss, const MxNorm& p) {
    return 1.0 / sqrt(ss / (double)p.cols + (double)p.eps);
}

// A row a workgroup, V quads of it in each lane's registers. Loads are unconditional, from
// clamped places (a branch around a load waits for those before it). With a residual and up to
// four quads the weights are loaded with the row, otherwise beside each store: as in the fp32
// norm, whose stores the loads behind them would wait for (512 x 4096 with a residual 7.0 us
// without, 6.4 with; 64 x 28672, eight quads, 13.0 and 23.2).
template <int FMT, int BS, int V, bool ADD>
__global__ __launch_bounds__(BS)
void mx_norm_kernel(MxNorm p) {
    constexpr bool EARLY = ADD && V <= 4;
    const int64_t row = blockIdx.x, base = row * p.cols;
    const int nq = (int)(p.cols / 4), t = threadIdx.x;
    const double one = p.w != nullptr && (p.flags & AERO_NORM_UNIT_OFFSET) ? 1.0 : 0.0;
    float4 v[V], d[V], w[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = min(t + i * BS, nq - 1);
        v[i] = ld_stream(p.x + base + 4 * c);
        if constexpr (ADD) d[i] = ld_stream(p.d + base + 4 * c);
    }
    auto weights = [&](int c) {
        return p.w != nullptr ? reinterpret_cast<const float4*>(p.w)[c] : make_float4(1.f, 1.f, 1.f, 1.f);
    };
    if constexpr (EARLY) {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = weights(min(t + i * BS, nq - 1));
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const bool in = t + i * BS < nq;
        if constexpr (ADD) {
            v[i] = add4(v[i], d[i]);
            if (in) {
                const v4f q = {v[i].x, v[i].y, v[i].z, v[i].w};
                __builtin_nontemporal_store(q, reinterpret_cast<v4f*>(p.xo + base) + t + i * BS);
            }
        }
        ss += in ? sq4(v[i]) : 0.0;
    }
    const double inv = norm_inv(mx_sum<BS>(ss), p);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = t + i * BS;
        if (c < nq)
            mx_store<FMT>(scaled4(v[i], inv, EARLY ? w[i] : weights(c), one), row * nq + c, p.codes, p.scales);
    }
}

// Rows of any length and at any address, read twice.
template <int FMT>
__global__ __launch_bounds__(256)
void mx_norm_any_kernel(MxNorm p) {
    const int64_t row = blockIdx.x, nq = p.cols / 4, base = row * p.cols;
    const double one = p.w != nullptr && (p.flags & AERO_NORM_UNIT_OFFSET) ? 1.0 : 0.0;
    double ss = 0.0;
    for (int64_t c = threadIdx.x; c < nq; c += 256) {
        float4 v = ld4(p.x + base + 4 * c, false);
        if (p.d != nullptr) {
            v = add4(v, ld4(p.d + base + 4 * c, false));
            float* o = p.xo + base + 4 * c;
            o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
        }
        ss += sq4(v);
    }
    const double inv = norm_inv(mx_sum<256>(ss), p);
    // (the sum comes from where this lane wrote it: xo may be x or d)
    const float* from = p.d != nullptr ? p.xo : p.x;
    for (int64_t c = threadIdx.x; c < nq; c += 256) {
        const float4 w = p.w != nullptr ? ld4(p.w + 4 * c, false) : make_float4(1.f, 1.f, 1.f, 1.f);
        const float* q = from + base + 4 * c;
        mx_store<FMT>(scaled4(make_float4(q[0], q[1], q[2], q[3]), inv, w, one), row * nq + c, p.codes, p.scales);
    }
}

// A workgroup of bs lanes a row.
template <int FMT>
bool launch_rows(const char* name, void (*kernel)(MxNorm), int bs, const MxNorm& p, int64_t rows, hipStream_t s) {
    const int64_t step = kMxLanes / bs;
    for (int64_t r = 0; r < rows; r += step) {
        MxNorm q = p;
        q.x += r * p.cols;
        if (p.d != nullptr) {
            q.d += r * p.cols;
            q.xo += r * p.cols;
        }
        q.codes += r * mx_row_bytes(FMT, p.cols);
        q.scales += r * (p.cols / 32);
        if (!launch(name, kernel, dim3((unsigned)(rows - r < step ? rows - r : step)), dim3((unsigned)bs), 0, s, q))
            return false;
    }
    return true;
}

template <int FMT, int BS, int V>
bool launch_norm(const MxNorm& p, int64_t rows, hipStream_t s) {
    return launch_rows<FMT>("mx_norm_kernel",
                            p.d != nullptr ? mx_norm_kernel<FMT, BS, V, true> : mx_norm_kernel<FMT, BS, V, false>,
                            BS, p, rows, s);
}

template <int FMT>
bool run_norm(const MxNorm& p, int64_t rows, hipStream_t s) {
    const int64_t nq = p.cols / 4;
    if (!p.vec || nq > 8192)
        return launch_rows<FMT>("mx_norm_any_kernel", mx_norm_any_kernel<FMT>, 256, p, rows, s);
    if (nq <= 64) return launch_norm<FMT, 64, 1>(p, rows, s);
    if (nq <= 128) return launch_norm<FMT, 64, 2>(p, rows, s);
    if (nq <= 256) return launch_norm<FMT, 256, 1>(p, rows, s);
    if (nq <= 512) return launch_norm<FMT, 256, 2>(p, rows, s);
    if (nq <= 1024) return launch_norm<FMT, 256, 4>(p, rows, s);
    if (nq <= 2048) return launch_norm<FMT, 512, 4>(p, rows, s);
    if (nq <= 4096) return launch_norm<FMT, 1024, 4>(p, rows, s);
    return launch_norm<FMT, 1024, 8>(p, rows, s);
}

// --------------------------------------------------------------- the way back
template <int FMT>
__global__ __launch_bounds__(256)
void mx_dequant_kernel(const uint8_t* codes, const uint8_t* scales, float* out, int64_t n, bool vec) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int s = scales[i >> 3];
    float v[4];
    if constexpr (FMT == AERO_MX_INT8) {
        const uint32_t c = reinterpret_cast<const uint32_t*>(codes)[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = __builtin_amdgcn_ldexpf((float)(int8_t)(c >> (8 * k)), s - 133);
    } else {
        const uint32_t c = reinterpret_cast<const uint16_t*>(codes)[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            // twice the magnitude: 0 1 2 3 4 6 8 12, a byte each
            const uint32_t m = __builtin_amdgcn_perm(0x0c080604u, 0x03020100u, (c >> (4 * k)) & 7u) & 255u;
            const float a = __builtin_amdgcn_ldexpf((float)m, s - 128);
            v[k] = (c >> (4 * k)) & 8u ? -a : a;
        }
    }
    if (s == 255) v[0] = v[1] = v[2] = v[3] = __builtin_nanf("");
    if (vec) {
        const v4f q = {v[0], v[1], v[2], v[3]};
        __builtin_nontemporal_store(q, reinterpret_cast<v4f*>(out + 4 * i));
    } else {
        for (int k = 0; k < 4; ++k) out[4 * i + k] = v[k];
    }
}

template <int FMT>
bool run_dequant(const uint8_t* codes, const uint8_t* scales, float* out, int64_t n, hipStream_t s) {
    for (int64_t i = 0; i < n; i += kMxLanes) {
        const int64_t m = n - i < kMxLanes ? n - i : kMxLanes;
        if (!launch("mx_dequant_kernel", mx_dequant_kernel<FMT>, dim3((unsigned)((m + 255) / 256)), dim3(256), 0, s,
                    codes + mx_row_bytes(FMT, 4 * i), scales + i / 8, out + 4 * i, m, aligned16(out)))
            return false;
    }
    return true;
}

}  // namespace

bool mx_rows_ok(const char* what, int fmt, const void* codes, const void* scales, int64_t rows,
                int64_t cols) {
    if (fmt != AERO_MX_INT8 && fmt != AERO_MX_FP4) {
        set_error("%s: unknown format %d", what, fmt);
        return false;
    }
    if (codes == nullptr || scales == nullptr || rows < 0 || rows > kMaxRows) {
        set_error("%s: bad arguments", what);
        return false;
    }
    if (cols <= 0 || cols % 32 != 0 || cols > ((int64_t)1 << 31)) {
        set_error("%s: %lld columns: rows are whole blocks of 32 values", what, (long long)cols);
        return false;
    }
    if ((reinterpret_cast<uintptr_t>(codes) & 3u) != 0) {
        set_error("%s: codes at a multiple of 4 bytes are needed", what);
        return false;
    }
    return true;
}

static bool rows_in_ok(const char* what, const float* a, const float* b, int64_t cols, int64_t ld) {
    if (a == nullptr || ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 3u) != 0) {
        set_error("%s: bad input pointer", what);
        return false;
    }
    if (ld < cols) {
        set_error("%s: rows %lld values apart hold no %lld columns", what, (long long)ld,
                  (long long)cols);
        return false;
    }
    return true;
}

}  // namespace aero

extern "C" {

int aero_hip_mx_quantize(int fmt, const float* x, int64_t ld, uint8_t* codes, uint8_t* scales,
                         int64_t rows, int64_t cols, void* stream) {
    using namespace aero;
    if (!mx_rows_ok("mx_quantize", fmt, codes, scales, rows, cols) ||
        !rows_in_ok("mx_quantize", x, nullptr, cols, ld))
        return 0;
    if (rows == 0) return 1;
    const hipStream_t s = (hipStream_t)stream;
    return (fmt == AERO_MX_INT8
                ? run_rows<AERO_MX_INT8, kNone, false>("mx_quantize_kernel", x, nullptr, codes, scales,
                                                       rows, cols, ld, s)
                : run_rows<AERO_MX_FP4, kNone, false>("mx_quantize_kernel", x, nullptr, codes, scales,
                                                      rows, cols, ld, s))
               ? 1 : 0;
}

int aero_hip_act_mul_mx(int fmt, int kind, const float* gate, const float* up, int64_t ld,
                        uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, void* stream) {
    using namespace aero;
    if (!mx_rows_ok("act_mul_mx", fmt, codes, scales, rows, cols) ||
        !rows_in_ok("act_mul_mx", gate, up, cols, ld))
        return 0;
    if (kind == AERO_ACT_IDENTITY && up == nullptr) {
        set_error("act_mul_mx: identity needs `up`");
        return 0;
    }
    if (rows == 0) return 1;
    const hipStream_t s = (hipStream_t)stream;
    return (fmt == AERO_MX_INT8
                ? run_act<AERO_MX_INT8>(kind, gate, up, codes, scales, rows, cols, ld, s)
                : run_act<AERO_MX_FP4>(kind, gate, up, codes, scales, rows, cols, ld, s))
               ? 1 : 0;
}

int aero_hip_rmsnorm_mx(int fmt, const float* x, const float* d, float* x_out, const float* w,
                        uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, float eps,
                        int flags, void* stream) {
    using namespace aero;
    if (!mx_rows_ok("rmsnorm_mx", fmt, codes, scales, rows, cols) ||
        !rows_in_ok("rmsnorm_mx", x, d, cols, cols) || !rows_in_ok("rmsnorm_mx", x, w, cols, cols))
        return 0;
    if ((d == nullptr) != (x_out == nullptr) || (reinterpret_cast<uintptr_t>(x_out) & 3u) != 0) {
        set_error("rmsnorm_mx: d and x_out go together");
        return 0;
    }
    if (flags & ~AERO_NORM_UNIT_OFFSET) {
        set_error("rmsnorm_mx: unknown flags %d", flags);
        return 0;
    }
    if (rows == 0) return 1;
    MxNorm p{x, d, x_out, w, codes, scales, cols, eps, flags,
             aligned16(x) && aligned16(d) && aligned16(x_out) && aligned16(w)};
    const hipStream_t s = (hipStream_t)stream;
    return (fmt == AERO_MX_INT8 ? run_norm<AERO_MX_INT8>(p, rows, s) : run_norm<AERO_MX_FP4>(p, rows, s))
               ? 1 : 0;
}

int aero_hip_mx_dequant(int fmt, const uint8_t* codes, const uint8_t* scales, float* out, int64_t rows,
                        int64_t cols, void* stream) {
    using namespace aero;
    if (!mx_rows_ok("mx_dequant", fmt, codes, scales, rows, cols) ||
        !rows_in_ok("mx_dequant", out, nullptr, cols, cols))
        return 0;
    if (rows == 0) return 1;
    const int64_t n = rows * (cols / 4);
    const hipStream_t s = (hipStream_t)stream;
    return (fmt == AERO_MX_INT8 ? run_dequant<AERO_MX_INT8>(codes, scales, out, n, s)
                                : run_dequant<AERO_MX_FP4>(codes, scales, out, n, s))
               ? 1 : 0;
}

}  // extern "C"
