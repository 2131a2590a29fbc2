// y = x W^T of microscaled rows (mx.hpp): W in 4 bits, x in 8 or 4, on the scaled matrix
// steps (v_mfma_scale_f32_32x32x64_f8f6f4), which multiply each block of 32 values by
// its two scales themselves.
//
// 8-bit x goes through in two halves. A code c = sign * (16 h + l), h and l in 0 .. 15
// (h up to 8): as 8-bit floats (e4m3) the numbers 0 .. 15 times 2^-9 are the codes 0 .. 15
// themselves, subnormals and first normals, so a half is a mask and a sign. Its products
// with 4-bit weights have 8 bits and one exponent range, so the step's sums lose nothing:
// against 64 bits 1e-7 of the result. The same steps on e4m3 activations keep about 14 bits
// of each sum of eight products, whose exponents differ (5e-5 measured on random codes): that
// is why 8 bits are whole numbers here. l has the scale of h divided by 16, the scale byte
// less 4.
//
// Weights are laid out once, in the order in which the steps take them: 32 rows, then
// blocks of 32 columns, then the 32 rows' 16 bytes of a block; a step's operand is 1 KB in
// one piece. Their scales are a dword (four blocks) a row.
#include <type_traits>

#include "mx.hpp"

#pragma clang fp contract(off)

namespace aero {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kF8 = 0, kF6 = 2, kF4 = 4;  // operand formats of the step

struct MxGemm {
    const uint8_t* x;    // codes [T][K] or [T][K/2]
    const uint8_t* xs;   // scales [T][K/32]
    const uint8_t* w;    // operand codes [N/32][kb][32][16]
    const uint8_t* ws;   // operand scales [N/32][kb/4][32][4]
    float* y;            // [T][N]
    int64_t T, N;
    int KB, KP;          // blocks of 32 columns, and of 128 (rounded up)
    bool vec;            // y rows at 16 bytes
};

// ------------------------------------------------------------- weight layout
// One 16-byte piece (row, block) a lane; rows and blocks past the end are zeros, with the
// smallest scale.
__global__ __launch_bounds__(256)
void mx_pack_kernel(const uint8_t* codes, const uint8_t* scales, uint8_t* w, uint8_t* ws, int64_t rows,
                    int KB, int KP, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int r = (int)(i & 31);
    const int64_t tile = (i >> 5) / (4 * KP);
    const int kb = (int)((i >> 5) - tile * (4 * KP));
    const int64_t row = tile * 32 + r;
    uint4 c = make_uint4(0u, 0u, 0u, 0u);
    uint8_t s = 0;
    if (row < rows && kb < KB) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(codes + (row * KB + kb) * 16);
        c = make_uint4(p[0], p[1], p[2], p[3]);
        s = scales[row * KB + kb];
    }
    reinterpret_cast<uint4*>(w)[i] = c;
    ws[((tile * KP + (kb >> 2)) * 32 + r) * 4 + (kb & 3)] = s;
}

// The halves of four 8-bit codes as e4m3 bytes.
__device__ __forceinline__ void halves(uint32_t c, int& hi, int& lo) {
    const uint32_t s = c & 0x80808080u, t = s >> 7;
    const uint32_t mag = (c ^ ((s - t) | s)) + t;
    hi = (int)(((mag >> 4) & 0x0F0F0F0Fu) | s);
    lo = (int)((mag & 0x0F0F0F0Fu) | s);
}

__device__ __forceinline__ v8i wide(v4i v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// Few tokens: 32 weight rows and up to 32 tokens a workgroup, its four waves each every fourth 128 columns,
// their sums joined in LDS. Lane l of a step holds row (token) l % 32 and, of 64 columns,
// block l / 32 of 4-bit operands; of e4m3 ones the bytes 16 (l / 32) .. of either block.
template <int FMT>
__global__ __launch_bounds__(256)
void mx_gemm_kernel(MxGemm p) {
    __shared__ v4f part[4][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 31, g = lane >> 5;
    const int64_t tile = blockIdx.x, t0 = (int64_t)blockIdx.y * 32;
    const int64_t tok = t0 + r < p.T ? t0 + r : p.T - 1;
    const uint8_t* wt = p.w + (tile * (4 * p.KP) * 32 + r) * 16;
    const uint8_t* wst = p.ws + (tile * p.KP * 32 + r) * 4;
    const uint8_t* xt = p.x + tok * p.KB * (FMT == AERO_MX_INT8 ? 32 : 16);
    const uint8_t* xst = p.xs + tok * p.KB;
    v16f acc;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    const v4i zero = {0, 0, 0, 0};
    for (int k = wave; k < p.KP; k += 4) {
        const uint32_t sw = *reinterpret_cast<const uint32_t*>(wst + (int64_t)k * 128);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int k0 = 4 * k + 2 * j, kb = k0 + g;   // the step's first block; this lane's
            const v4i a = *reinterpret_cast<const v4i*>(wt + (int64_t)kb * 512);
            const int sa = (int)(sw >> (8 * (2 * j + g)));
            int sb = kb < p.KB ? xst[kb] : 0;
            if constexpr (FMT == AERO_MX_INT8) {
                v4i c0 = zero, c1 = zero;
                if (k0 < p.KB) c0 = *reinterpret_cast<const v4i*>(xt + k0 * 32 + 16 * g);
                if (k0 + 1 < p.KB) c1 = *reinterpret_cast<const v4i*>(xt + k0 * 32 + 32 + 16 * g);
                v8i hi, lo;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    int h, l;
                    halves((uint32_t)c0[i], h, l);
                    hi[i] = h; lo[i] = l;
                    halves((uint32_t)c1[i], h, l);
                    hi[4 + i] = h; lo[4 + i] = l;
                }
                sb = sb < 4 ? 4 : sb;
                acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), hi, acc, kF4, kF8, 0, sa,
                                                                      0, sb);
                acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), lo, acc, kF4, kF8, 0, sa,
                                                                      0, sb - 4);
            } else {
                v4i b = zero;
                if (kb < p.KB) b = *reinterpret_cast<const v4i*>(xt + kb * 16);
                acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), wide(b), acc, kF4, kF4, 0,
                                                                      sa, 0, sb);
            }
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const v4f v = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
        part[wave][q][lane] = v;
    }
    __syncthreads();
    v4f v = part[0][wave][lane];
#pragma unroll
    for (int k = 1; k < 4; ++k) v += part[k][wave][lane];
    if constexpr (FMT == AERO_MX_INT8) v *= 128.f;   // h 16 / 64 = (h 2^-9) 2^7
    const int64_t n = tile * 32 + 8 * wave + 4 * g;
    if (t0 + r >= p.T) return;
    float* o = p.y + (t0 + r) * p.N + n;
    if (p.vec && n + 4 <= p.N) {
        *reinterpret_cast<v4f*>(o) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < p.N) o[i] = v[i];
}

// ---------------------------------------------------------- many tokens
// x as operands, once a call: 32 tokens, then steps of 64 columns. 4 bits: as the weights.
// 8 bits: the halves as 6-bit floats (e2m3), whose steps against 4-bit operands take half
// the time of e4m3 ones (35 cycles and 64 measured). There too a number 0 .. 15 is its own
// code (in units of 1/8). A lane's 24 bytes a half lie as 16 and 8, 64 lanes side by side:
// 1024 + 512 for the high halves, the same for the low ones.
template <int FMT>
constexpr int kStepBytes = FMT == AERO_MX_INT8 ? 3072 : 1024;

// 32 codes of 6 bits, the first lowest, from 32 bytes' signs (bit 7) and low halves.
__device__ __forceinline__ void pack6(const uint32_t (&b)[8], uint32_t (&o)[6]) {
    uint64_t q[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const uint32_t v = b[i >> 2] >> (8 * (i & 3));
        const uint64_t c = (v & 15u) | ((v >> 2) & 32u);
        const int at = 6 * i, w = at >> 6, s = at & 63;
        q[w] |= c << s;
        if (s > 58) q[w + 1] |= c >> (64 - s);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        o[2 * i] = (uint32_t)q[i];
        o[2 * i + 1] = (uint32_t)(q[i] >> 32);
    }
}

// One block of one token a lane; tokens and blocks past the end are zeros.
template <int FMT>
__global__ __launch_bounds__(256)
void mx_operand_kernel(const uint8_t* x, const uint8_t* xs, uint8_t* o, uint8_t* os, int64_t T, int KB,
                       int KP, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int lane = (int)(i & 63), r = lane & 31;
    const int64_t step = i >> 6, tile = step / (2 * KP);
    const int kb = 2 * (int)(step - tile * (2 * KP)) + (lane >> 5);
    const int64_t tok = tile * 32 + r;
    const bool in = tok < T && kb < KB;
    const int low = FMT == AERO_MX_INT8 ? 4 : 0;
    int s = in ? xs[tok * KB + kb] : low;
    os[((tile * KP + (kb >> 2)) * 32 + r) * 4 + (kb & 3)] = (uint8_t)(s < low ? low : s);
    uint8_t* to = o + step * kStepBytes<FMT>;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (FMT == AERO_MX_FP4) {
        reinterpret_cast<uint4*>(to)[lane] =
            in ? *reinterpret_cast<const uint4*>(x + (tok * KB + kb) * 16) : zero;
    } else {
        const uint4* p = reinterpret_cast<const uint4*>(x + (tok * KB + kb) * 32);
        const uint4 c0 = in ? p[0] : zero, c1 = in ? p[1] : zero;
        const uint32_t c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        uint32_t hi[8], lo[8], h[6], l[6];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            int a, b;
            halves(c[k], a, b);
            hi[k] = (uint32_t)a;
            lo[k] = (uint32_t)b;
        }
        pack6(hi, h);
        pack6(lo, l);
        reinterpret_cast<uint4*>(to)[lane] = make_uint4(h[0], h[1], h[2], h[3]);
        reinterpret_cast<uint2*>(to + 1024)[lane] = make_uint2(h[4], h[5]);
        reinterpret_cast<uint4*>(to + 1536)[lane] = make_uint4(l[0], l[1], l[2], l[3]);
        reinterpret_cast<uint2*>(to + 2560)[lane] = make_uint2(l[4], l[5]);
    }
}

// A value the compiler knows nothing about. (The host pass has no such registers.)
template <typename T>
__device__ __forceinline__ void opaque(T& v) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" : "+v"(v));
#endif
}

struct MxTiles {
    const uint8_t* w;    // operand codes and scales of both sides
    const uint8_t* ws;
    const uint8_t* x;
    const uint8_t* xs;
    float* y;
    int64_t T, N;
    int KP, steps;       // 128-column groups, 64-column steps
    int nt, tt;          // 32-row and 32-token tiles
    int bn, bt, group;   // workgroups along each; token tiles side by side
};

// A workgroup of GN x GT waves, a wave WA weight tiles by XB token tiles of 32. Steps of 64
// columns go through NB buffers in LDS by direct loads of 1 KB, each wave its share, NB - 1
// steps ahead.
template <int FMT, int WA, int XB, int GN, int GT>
struct MxShape {
    static constexpr int NW = GN * GT, TN = WA * GN, TT = XB * GT;
    static constexpr int XC = kStepBytes<FMT> / 1024;
    static constexpr int SC = (TN + TT + 7) / 8;                 // pieces of 8 tiles' scales
    static constexpr int PIECES = TN + TT * XC + SC;
    static constexpr int LOADS = (PIECES + NW - 1) / NW;
    static constexpr int XOFF = TN * 1024, SOFF = XOFF + TT * XC * 1024;
    static constexpr int BYTES = SOFF + SC * 1024;
};

template <int FMT, int WA, int XB, int GN, int GT, int NB, int WAVES>
__global__ __launch_bounds__(64 * GN * GT, WAVES)
void mx_tiles_kernel(MxTiles p) {
    using S = MxShape<FMT, WA, XB, GN, GT>;
    // (arrays of their own: the compiler tells a load into one from a read of another)
#define AERO_MX_BUF(K) __shared__ __attribute__((aligned(16))) uint8_t b##K[K < NB ? S::BYTES : 16]
    AERO_MX_BUF(0); AERO_MX_BUF(1); AERO_MX_BUF(2); AERO_MX_BUF(3); AERO_MX_BUF(4); AERO_MX_BUF(5);
    AERO_MX_BUF(6); AERO_MX_BUF(7); AERO_MX_BUF(8); AERO_MX_BUF(9); AERO_MX_BUF(10); AERO_MX_BUF(11);
#undef AERO_MX_BUF
    uint8_t* const bufs[12] = {b0, b1, b2, b3, b4, b5, b6, b7, b8, b9, b10, b11};
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, g = lane >> 5;
    // Each XCD (workgroups go round them in turn) takes a run of neighbouring tiles: four
    // token tiles beside one weight tile, then beside the next, so that what runs at a time
    // on an XCD shares both sides through its L2.
    const int per = gridDim.x >> 3;
    const int at = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (at >= p.bn * p.bt) return;
    const int group = at / (p.group * p.bn), rest = at - group * p.group * p.bn;
    const int width = min(p.group, p.bt - group * p.group);
    const int n0 = (rest / width) * S::TN, t0 = (group * p.group + rest % width) * S::TT;

    // This wave's pieces of a step, the scales' first: where they begin, how far a step goes.
    // (A piece past the last is the wave's one before once more, to the same place.)
    static_assert(S::SC <= S::NW, "the scales' pieces are first ones");
    const uint8_t* src[S::LOADS];
    int dst[S::LOADS], stride[S::LOADS];
#pragma unroll
    for (int i = 0; i < S::LOADS; ++i) {
        int c = wave + S::NW * i;
        if (c >= S::PIECES) c -= S::NW;
        c -= S::SC;
        dst[i] = c * 1024;
        if (c < S::TN) {
            src[i] = p.w + (int64_t)min(n0 + max(c, 0), p.nt - 1) * p.KP * 2048;
            stride[i] = 1024;
        } else {
            const int q = c - S::TN;
            src[i] = p.x + (int64_t)min(t0 + q / S::XC, p.tt - 1) * p.KP * (2 * kStepBytes<FMT>) +
                     (q % S::XC) * 1024;
            stride[i] = kStepBytes<FMT>;
        }
    }
    uint32_t lane16 = lane * 16;
    opaque(lane16);
    const uint8_t* first = src[0] + lane16;
    const int half = wave < S::SC ? 1 : 0;
    if (wave < S::SC) {       // eight tiles' scales of 128 columns
        const int k = min(wave * 8 + (lane >> 3), S::TN + S::TT - 1);
        first = (k < S::TN ? p.ws + (int64_t)min(n0 + k, p.nt - 1) * p.KP * 128
                           : p.xs + (int64_t)min(t0 + k - S::TN, p.tt - 1) * p.KP * 128) + (lane & 7) * 16;
        dst[0] = S::SOFF + wave * 1024;
        stride[0] = 128;
    }
    auto fetch = [&](int i, uint8_t* b, int k0, int k1) __attribute__((always_inline)) {
#pragma unroll
        for (int k = k0; k < k1; ++k) {
            const uint8_t* from = k == 0 ? first + (int64_t)(i >> half) * stride[0]
                                         : src[k] + (int64_t)i * stride[k] + lane16;
            uint8_t* to = b + dst[k];
            __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
        }
    };

    const int wn = (wave % GN) * WA, wt = (wave / GN) * XB;
    v16f acc[WA][XB];
#pragma unroll
    for (int a = 0; a < WA; ++a)
#pragma unroll
        for (int b = 0; b < XB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;

    // A lane's places in a buffer. (Opaque, so that each stays one register that the buffers
    // and tiles add constants to.)
    int oa = wn * 1024 + lane * 16, ox = S::XOFF + wt * kStepBytes<FMT> + lane * 16;
    int ox8 = ox - lane * 8, osa = S::SOFF + wn * 128 + r * 4, osx = S::SOFF + (S::TN + wt) * 128 + r * 4;
    opaque(oa);
    opaque(ox);
    opaque(ox8);
    opaque(osa);
    opaque(osx);
    // (the step's operands are read first; the loads of a later step go out between groups of
    // matrix steps, behind which their issue hides)
    auto compute = [&](int i, const uint8_t* buf, uint8_t* nb) __attribute__((always_inline)) {
        constexpr int H = FMT == AERO_MX_INT8 ? 2 : 1, GROUPS = XB * H;
        const int sh = 16 * (i & 1) + 8 * g, next = min(i + NB - 1, p.steps - 1);
        v4i a[WA], q[XB][H];
        v2i e[XB][H];
        int sa[WA], sb[XB];
#pragma unroll
        for (int k = 0; k < WA; ++k) a[k] = *reinterpret_cast<const v4i*>(buf + oa + k * 1024);
#pragma unroll
        for (int k = 0; k < WA; ++k) sa[k] = *reinterpret_cast<const int*>(buf + osa + k * 128);
#pragma unroll
        for (int b = 0; b < XB; ++b) {
            sb[b] = *reinterpret_cast<const int*>(buf + osx + b * 128);
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const int at = b * kStepBytes<FMT> + 1536 * h;
                q[b][h] = *reinterpret_cast<const v4i*>(buf + ox + at);
                if constexpr (H == 2) e[b][h] = *reinterpret_cast<const v2i*>(buf + ox8 + at + 1024);
            }
        }
#pragma unroll
        for (int k = 0; k < WA; ++k) sa[k] = (int)((uint32_t)sa[k] >> sh);
#pragma unroll
        for (int b = 0; b < XB; ++b) sb[b] = (int)((uint32_t)sb[b] >> sh);
#pragma unroll
        for (int b = 0; b < XB; ++b)
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const int n = b * H + h;
                v8i f;
                if constexpr (H == 2) {
                    const v4i e4 = __builtin_shufflevector(e[b][h], e[b][h], 0, 1, -1, -1);
                    f = __builtin_shufflevector(q[b][h], e4, 0, 1, 2, 3, 4, 5, -1, -1);
                } else {
                    f = wide(q[b][h]);
                }
#pragma unroll
                for (int k = 0; k < WA; ++k) {
                    acc[k][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                        f, wide(a[k]), acc[k][b], H == 2 ? kF6 : kF4, kF4, 0, sb[b] - 4 * h, 0, sa[k]);
                    const int at = n * WA + k;
                    __builtin_amdgcn_sched_barrier(0);
                    fetch(next, nb, at * S::LOADS / (GROUPS * WA), (at + 1) * S::LOADS / (GROUPS * WA));
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
    };
    // A step begins when its loads have landed (the next ones' may be on their way) and
    // every wave is done with the step before, whose buffer is then filled again; the last
    // steps load the last one once more, so that every step is alike. (The marks keep the
    // copies of this code apart: merged, the compiler could not tell the buffer that is read
    // from the one that is filled, and would wait for the loads.)
    auto step = [&](auto k, int i) __attribute__((always_inline)) {
        constexpr int K = decltype(k)::value, N = (NB - 2) * S::LOADS;
        __builtin_amdgcn_s_waitcnt((N & 15) | 0x0f70 | ((N >> 4) << 14));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        asm volatile("; buffer %0" ::"n"(K) : "memory");
        compute(i, bufs[K], bufs[(K + NB - 1) % NB]);
        asm volatile("; buffer %0 done" ::"n"(K) : "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
#define AERO_MX_EACH(DO) DO(0) DO(1) DO(2) DO(3) DO(4) DO(5) DO(6) DO(7) DO(8) DO(9) DO(10) DO(11)
#define AERO_MX_FILL(K) if constexpr (K < NB - 1) fetch(min(K, p.steps - 1), bufs[K], 0, S::LOADS);
#define AERO_MX_ROUND(K) if constexpr (K < NB) step(std::integral_constant<int, K>{}, i + K);
#define AERO_MX_REST(K) \
    if constexpr (K < NB - 1) if (i + K < p.steps) step(std::integral_constant<int, K>{}, i + K);
    AERO_MX_EACH(AERO_MX_FILL)
    // (whole rounds, then the rest: with an exit after each step the compiler keeps the sums
    // twice and spills)
    int i = 0;
    for (; i + NB <= p.steps; i += NB) {
        AERO_MX_EACH(AERO_MX_ROUND)
    }
    AERO_MX_EACH(AERO_MX_REST)
#undef AERO_MX_EACH
#undef AERO_MX_FILL
#undef AERO_MX_ROUND
#undef AERO_MX_REST
    __builtin_amdgcn_s_waitcnt(0x0f70);       // (no load is on its way when the wave ends)

    constexpr float UNIT = FMT == AERO_MX_INT8 ? 2.f : 1.f;      // h 16 / 64 = (h / 8) 2
    // lane l holds column l % 32 of 16 tokens: 128 bytes in one piece for each
#pragma unroll
    for (int a = 0; a < WA; ++a) {
        const int64_t n = (int64_t)(n0 + wn + a) * 32 + r;
        if (n >= p.N) continue;
#pragma unroll
        for (int b = 0; b < XB; ++b) {
            const int64_t t1 = (int64_t)(t0 + wt + b) * 32 + 4 * g;
            float* o = p.y + t1 * p.N + n;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int t = 8 * (i >> 2) + (i & 3);
                if (t1 + t < p.T) __builtin_nontemporal_store(acc[a][b][i] * UNIT, o + t * p.N);
            }
        }
    }
}

// The largest calls: 256 weight rows by 256 tokens a workgroup of four waves, each 128 by
// 128 (its 16 tiles of sums take half of a SIMD's registers: one wave each). LDS carries the
// tokens only, stages of 128 columns; a wave loads its weights straight into registers, two
// stages ahead. With both sides in LDS the reads and the direct loads' writes take about as
// many of its cycles as there are matrix steps; so they take half.
// A stage is eight groups of matrix steps (four with x in 4 bits). The operands of a group
// are read while the group before runs, those of a stage's first while the last one of the
// stage before does: the barrier that a stage begins with stands in front of that.
template <int FMT>
struct MxWide {
    static constexpr int H = FMT == AERO_MX_INT8 ? 2 : 1;        // halves
    static constexpr int BT = FMT == AERO_MX_INT8 ? 1 : 2;       // token tiles a group
    static constexpr int GROUPS = 8 / BT;
    static constexpr int XC = 2 * kStepBytes<FMT> / 1024;        // KB of a token tile's stage
    static constexpr int PIECES = 8 * XC + 1, LOADS = (PIECES + 3) / 4;
    static constexpr int SOFF = 8 * XC * 1024, BYTES = SOFF + 1024;
    static constexpr int VMEM = LOADS + 12;                      // and the weights' loads
};

template <int FMT>
__global__ __launch_bounds__(256, 1)
void mx_wide_kernel(MxTiles p) {
    using S = MxWide<FMT>;
    __shared__ __attribute__((aligned(16))) uint8_t b0[S::BYTES];
    __shared__ __attribute__((aligned(16))) uint8_t b1[S::BYTES];
    __shared__ __attribute__((aligned(16))) uint8_t b2[S::BYTES];
    uint8_t* const bufs[3] = {b0, b1, b2};
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, g = lane >> 5;
    const int per = gridDim.x >> 3;
    const int at = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (at >= p.bn * p.bt) return;
    const int group = at / (p.group * p.bn), rest = at - group * p.group * p.bn;
    const int width = min(p.group, p.bt - group * p.group);
    const int n0 = (rest / width) * 8, t0 = (group * p.group + rest % width) * 8;
    const int wn = (wave & 1) * 4, wt = (wave >> 1) * 4;

    // this wave's pieces of a stage's tokens (the first wave's first: their scales), and its
    // weights
    uint32_t lane16 = lane * 16, lane4 = r * 4;
    opaque(lane16);
    opaque(lane4);
    const uint8_t* src[S::LOADS];
    int dst[S::LOADS];
#pragma unroll
    for (int i = 0; i < S::LOADS; ++i) {
        int c = wave + 4 * i;
        if (c >= S::PIECES) c -= 4;
        c = max(c - 1, 0);
        dst[i] = c * 1024;
        src[i] = p.x + (int64_t)min(t0 + c / S::XC, p.tt - 1) * p.KP * (S::XC * 1024) + (c % S::XC) * 1024;
    }
    const uint8_t* first = src[0] + lane16;
    int first_stride = S::XC * 1024;
    if (wave == 0) {
        first = p.xs + (int64_t)min(t0 + (lane >> 3), p.tt - 1) * p.KP * 128 + (lane & 7) * 16;
        first_stride = 128;
        dst[0] = S::SOFF;
    }
    auto piece = [&](int i, uint8_t* b, int k0, int k1) __attribute__((always_inline)) {
#pragma unroll
        for (int k = k0; k < k1; ++k) {
            const uint8_t* from = k == 0 ? first + (int64_t)i * first_stride
                                         : src[k] + (int64_t)i * (S::XC * 1024) + lane16;
            uint8_t* to = b + dst[k];
            __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
        }
    };
    const uint8_t* wp[4];
    const uint8_t* wsp[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        const int64_t tile = min(n0 + wn + a, p.nt - 1);
        wp[a] = p.w + tile * p.KP * 2048;
        wsp[a] = p.ws + tile * p.KP * 128;
    }
    v4i w[3][2][4];
    int sw[3][4];
    auto weights = [&](int i, int set, int n) __attribute__((always_inline)) {   // the n-th of 12 loads
        const int64_t k = i;
        const int a = n / 3;
        if (n % 3 < 2)
            w[set][n % 3][a] = *reinterpret_cast<const v4i*>(wp[a] + k * 2048 + n % 3 * 1024 + lane16);
        else
            sw[set][a] = *reinterpret_cast<const int*>(wsp[a] + k * 128 + lane4);
    };
    auto load = [&](int i, int set, uint8_t* b, int k0, int k1) __attribute__((always_inline)) {
#pragma unroll
        for (int k = k0; k < k1; ++k) {
            if (k < S::LOADS)
                piece(i, b, k, k + 1);
            else
                weights(i, set, k - S::LOADS);
        }
    };

    v16f acc[4][4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;

    struct Frag {
        v4i q[S::BT][S::H];
        v2i e[S::BT][S::H];
        int s[S::BT];
    };
    int ox = wt * (S::XC * 1024) + lane * 16, ox8 = ox - lane * 8, osx = S::SOFF + wt * 128 + r * 4;
    opaque(ox);
    opaque(ox8);
    opaque(osx);
    // group n: columns 64 (n / (4 / BT)) .. of the stage, token tiles BT (n % (4 / BT)) ..
    auto read = [&](Frag& f, const uint8_t* b, int n) __attribute__((always_inline)) {
        const int j = n / (4 / S::BT), b0 = n % (4 / S::BT) * S::BT;
#pragma unroll
        for (int x = 0; x < S::BT; ++x) {
            const int off = (b0 + x) * (S::XC * 1024) + j * kStepBytes<FMT>;
#pragma unroll
            for (int h = 0; h < S::H; ++h) {
                f.q[x][h] = *reinterpret_cast<const v4i*>(b + ox + off + 1536 * h);
                if constexpr (S::H == 2)
                    f.e[x][h] = *reinterpret_cast<const v2i*>(b + ox8 + off + 1536 * h + 1024);
            }
            f.s[x] = *reinterpret_cast<const int*>(b + osx + (b0 + x) * 128);
        }
    };
    const int sh0 = 8 * g, sh1 = 16 + 8 * g;
    Frag f0, f1;
    auto stage = [&](auto kk, int i) __attribute__((always_inline)) {
        constexpr int K = decltype(kk)::value, K1 = (K + 1) % 3, K2 = (K + 2) % 3;
        const int next = min(i + 2, p.KP - 1);
        int sa[2][4];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            sa[0][a] = (int)((uint32_t)sw[K][a] >> sh0);
            sa[1][a] = (int)((uint32_t)sw[K][a] >> sh1);
        }
#pragma unroll
        for (int n = 0; n < S::GROUPS; ++n) {
            Frag& cur = n & 1 ? f1 : f0;
            Frag& nxt = n & 1 ? f0 : f1;
            const int j = n / (4 / S::BT), b0 = n % (4 / S::BT) * S::BT;
            if (n + 1 < S::GROUPS) {
                read(nxt, bufs[K], n + 1);
            } else {
                // every wave has read this stage, and the next one has landed
                __builtin_amdgcn_s_waitcnt((S::VMEM & 15) | 0x0070 | ((S::VMEM >> 4) << 14));
                asm volatile("" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                asm volatile("; buffer %0" ::"n"(K1) : "memory");
                read(nxt, bufs[K1], 0);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < S::BT; ++x)
#pragma unroll
                for (int h = 0; h < S::H; ++h) {
                    v8i f;
                    if constexpr (S::H == 2) {
                        const v4i e4 = __builtin_shufflevector(cur.e[x][h], cur.e[x][h], 0, 1, -1, -1);
                        f = __builtin_shufflevector(cur.q[x][h], e4, 0, 1, 2, 3, 4, 5, -1, -1);
                    } else {
                        f = wide(cur.q[x][h]);
                    }
                    const int sb = (int)((uint32_t)cur.s[x] >> (j ? sh1 : sh0)) - 4 * h;
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        acc[a][b0 + x] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                            f, wide(w[K][j][a]), acc[a][b0 + x], S::H == 2 ? kF6 : kF4, kF4, 0, sb, 0,
                            sa[j][a]);
                        // (one load at a time, each behind a matrix step)
                        constexpr int M = (S::GROUPS - 1) * 8;
                        const int m = n * 8 + (x * S::H + h) * 4 + a;
                        __builtin_amdgcn_sched_barrier(0);
                        if (m < M) load(next, K2, bufs[K2], m * S::VMEM / M, (m + 1) * S::VMEM / M);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
        }
    };
    load(0, 0, b0, 0, S::VMEM);
    load(min(1, p.KP - 1), 1, b1, 0, S::VMEM);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((S::VMEM & 15) | 0x0f70 | ((S::VMEM >> 4) << 14));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(f0, b0, 0);
    using K0 = std::integral_constant<int, 0>;
    using K1 = std::integral_constant<int, 1>;
    using K2 = std::integral_constant<int, 2>;
    int i = 0;
    for (; i + 3 <= p.KP; i += 3) {
        stage(K0{}, i);
        stage(K1{}, i + 1);
        stage(K2{}, i + 2);
    }
    if (i < p.KP) stage(K0{}, i);
    if (i + 1 < p.KP) stage(K1{}, i + 1);
    __builtin_amdgcn_s_waitcnt(0x0f70);       // (no load is on its way when the wave ends)

    constexpr float UNIT = FMT == AERO_MX_INT8 ? 2.f : 1.f;      // h 16 / 64 = (h / 8) 2
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        const int64_t n = (int64_t)(n0 + wn + a) * 32 + r;
        if (n >= p.N) continue;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int64_t t1 = (int64_t)(t0 + wt + b) * 32 + 4 * g;
            float* o = p.y + t1 * p.N + n;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int t = 8 * (i >> 2) + (i & 3);
                if (t1 + t < p.T) __builtin_nontemporal_store(acc[a][b][i] * UNIT, o + t * p.N);
            }
        }
    }
}

int64_t tiles32(int64_t n) { return (n + 31) / 32; }

bool weight_sizes_ok(const char* what, int64_t n_rows, int64_t n_cols) {
    if (n_rows <= 0 || n_rows > ((int64_t)1 << 31) || n_cols <= 0 || n_cols % 32 != 0 ||
        n_cols > ((int64_t)1 << 24)) {
        set_error("%s: %lld rows of %lld columns: rows are whole blocks of 32 values, at most 2^24",
                  what, (long long)n_rows, (long long)n_cols);
        return false;
    }
    return true;
}

int64_t weight_codes_bytes(int64_t n_rows, int64_t n_cols) {
    return tiles32(n_rows) * ((n_cols + 127) / 128) * 2048;
}

// Calls of more tokens go through operands in the workspace.
constexpr int64_t kFewTokens = 32;

template <int FMT>
int64_t operand_bytes(int64_t n_tok, int KP) {
    return tiles32(n_tok) * KP * (2 * kStepBytes<FMT> + 128);
}

template <int FMT, int WA, int XB, int GN, int GT, int NB, int WAVES>
bool launch_tiles(MxTiles p, hipStream_t s) {
    using S = MxShape<FMT, WA, XB, GN, GT>;
    p.bn = (p.nt + S::TN - 1) / S::TN;
    p.bt = (p.tt + S::TT - 1) / S::TT;
    const int64_t grid = ((int64_t)p.bn * p.bt + 7) / 8 * 8;
    if (grid > 0x7fffffff) {
        set_error("mx_matmul: %lld x %lld results are too many", (long long)p.T, (long long)p.N);
        return false;
    }
    return launch("mx_tiles_kernel", mx_tiles_kernel<FMT, WA, XB, GN, GT, NB, WAVES>, dim3((unsigned)grid),
                  dim3(64 * S::NW), 0, s, p);
}

template <int FMT>
bool run_tiles(const MxGemm& g, void* ws, hipStream_t s) {
    const int64_t tt = tiles32(g.T), nt = tiles32(g.N);
    uint8_t* o = (uint8_t*)ws;
    uint8_t* os = o + tt * g.KP * (2 * kStepBytes<FMT>);
    const int64_t n = tt * 32 * 4 * g.KP, blocks = (n + 255) / 256;
    if (blocks > 0x7fffffff || nt > 0x7fffffff || tt > 0x7fffffff) {
        set_error("mx_matmul: %lld tokens are too many", (long long)g.T);
        return false;
    }
    if (!launch("mx_operand_kernel", mx_operand_kernel<FMT>, dim3((unsigned)blocks), dim3(256), 0, s, g.x,
                g.xs, o, os, g.T, g.KB, g.KP, n))
        return false;
    const MxTiles p{g.w, g.ws, o, os, g.y, g.T, g.N, g.KP, (g.KB + 1) / 2, (int)nt, (int)tt, 0, 0, tune("mx_group", 4)};
    const int64_t wide = ((nt + 7) / 8) * ((tt + 7) / 8);
    if (wide >= tune("mx_wide", 200)) {
        MxTiles q = p;
        q.bn = (int)((nt + 7) / 8);
        q.bt = (int)((tt + 7) / 8);
        return launch("mx_wide_kernel", mx_wide_kernel<FMT>, dim3((unsigned)((wide + 7) / 8 * 8)), dim3(256),
                      0, s, q);
    }
    const int64_t big = ((nt + 7) / 8) * ((tt + 3) / 4);
    if (big >= tune("mx_big", 256)) return launch_tiles<FMT, 4, 2, 2, 2, 3, 2>(p, s);
    if (tune("mx_nb", 6) == 3) return launch_tiles<FMT, 2, 1, 2, 2, 3, 2>(p, s);
    if (tune("mx_nb", 6) == 12) return launch_tiles<FMT, 2, 1, 2, 2, 12, 1>(p, s);
    return launch_tiles<FMT, 2, 1, 2, 2, 6, 2>(p, s);
}

}  // namespace
}  // namespace aero

extern "C" {

int64_t aero_hip_mx_weight_bytes(int64_t n_rows, int64_t n_cols) {
    using namespace aero;
    if (!weight_sizes_ok("mx_weight_bytes", n_rows, n_cols)) return -1;
    return tiles32(n_rows) * ((n_cols + 127) / 128) * (2048 + 128);
}

int aero_hip_mx_pack(const uint8_t* codes, const uint8_t* scales, void* w, int64_t w_bytes,
                     int64_t n_rows, int64_t n_cols, void* stream) {
    using namespace aero;
    if (!weight_sizes_ok("mx_pack", n_rows, n_cols) ||
        !mx_rows_ok("mx_pack", AERO_MX_FP4, codes, scales, n_rows, n_cols))
        return 0;
    if (w == nullptr || !aligned16(w) || w_bytes < aero_hip_mx_weight_bytes(n_rows, n_cols)) {
        set_error("mx_pack: w needs %lld bytes at a 16-byte address",
                  (long long)aero_hip_mx_weight_bytes(n_rows, n_cols));
        return 0;
    }
    const int KB = (int)(n_cols / 32), KP = (KB + 3) / 4;
    const int64_t n = tiles32(n_rows) * 32 * 4 * KP, blocks = (n + 255) / 256;
    if (blocks > 0x7fffffff) {
        set_error("mx_pack: %lld rows of %lld columns are too many", (long long)n_rows,
                  (long long)n_cols);
        return 0;
    }
    uint8_t* codes_out = (uint8_t*)w;
    return launch("mx_pack_kernel", mx_pack_kernel, dim3((unsigned)blocks), dim3(256), 0,
                  (hipStream_t)stream, codes, scales, codes_out,
                  codes_out + weight_codes_bytes(n_rows, n_cols), n_rows, KB, KP, n) ? 1 : 0;
}

int64_t aero_hip_mx_matmul_workspace(int fmt, int64_t n_rows, int64_t n_cols, int64_t n_tok) {
    using namespace aero;
    if ((fmt != AERO_MX_INT8 && fmt != AERO_MX_FP4) || n_tok < 0 ||
        !weight_sizes_ok("mx_matmul_workspace", n_rows, n_cols))
        return -1;
    if (n_tok <= kFewTokens) return 0;
    const int KP = (int)((n_cols + 127) / 128);
    return fmt == AERO_MX_INT8 ? operand_bytes<AERO_MX_INT8>(n_tok, KP)
                               : operand_bytes<AERO_MX_FP4>(n_tok, KP);
}

int aero_hip_mx_matmul(int fmt, const uint8_t* codes, const uint8_t* scales, const void* w,
                       int64_t w_bytes, float* y, int64_t n_rows, int64_t n_cols, int64_t n_tok,
                       void* workspace, int64_t ws_bytes, void* stream) {
    using namespace aero;
    if (!weight_sizes_ok("mx_matmul", n_rows, n_cols) ||
        !mx_rows_ok("mx_matmul", fmt, codes, scales, n_tok, n_cols))
        return 0;
    if (w == nullptr || !aligned16(w) || w_bytes < aero_hip_mx_weight_bytes(n_rows, n_cols)) {
        set_error("mx_matmul: weights of %lld x %lld take %lld bytes at a 16-byte address",
                  (long long)n_rows, (long long)n_cols,
                  (long long)aero_hip_mx_weight_bytes(n_rows, n_cols));
        return 0;
    }
    if (!aligned16(codes) || y == nullptr || (reinterpret_cast<uintptr_t>(y) & 3u) != 0) {
        set_error("mx_matmul: codes at a 16-byte address and a y are needed");
        return 0;
    }
    if (n_tok == 0) return 1;
    const int KB = (int)(n_cols / 32), KP = (KB + 3) / 4;
    MxGemm p{codes, scales, (const uint8_t*)w, (const uint8_t*)w + weight_codes_bytes(n_rows, n_cols), y,
             n_tok, n_rows, KB, KP, aligned16(y) && n_rows % 4 == 0};
    const hipStream_t s = (hipStream_t)stream;
    if (n_tok > kFewTokens) {
        const int64_t need = aero_hip_mx_matmul_workspace(fmt, n_rows, n_cols, n_tok);
        if (workspace == nullptr || !aligned16(workspace) || ws_bytes < need) {
            set_error("mx_matmul: the workspace takes %lld bytes at a 16-byte address", (long long)need);
            return 0;
        }
        return (fmt == AERO_MX_INT8 ? run_tiles<AERO_MX_INT8>(p, workspace, s)
                                    : run_tiles<AERO_MX_FP4>(p, workspace, s)) ? 1 : 0;
    }
    const dim3 grid((unsigned)tiles32(n_rows));
    return (fmt == AERO_MX_INT8
                ? launch("mx_gemm_kernel", mx_gemm_kernel<AERO_MX_INT8>, grid, dim3(256), 0, s, p)
                : launch("mx_gemm_kernel", mx_gemm_kernel<AERO_MX_FP4>, grid, dim3(256), 0, s, p))
               ? 1 : 0;
}

}  // extern "C"
