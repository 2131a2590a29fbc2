// y = x W^T of microscaled rows (mx.hpp): W in 4 bits, x in 8 or 4, on the scaled matrix
// steps (v_mfma_scale_f32_32x32x64_f8f6f4), which multiply each block of 32 values by
// its two scales themselves.
//
// 8-bit x goes through in two halves. A code c = sign * (16 h + l), h and l in 0 .. 15
// (h up to 8): as 8-bit floats (e4m3) the numbers 0 .. 15 times 2^-9 are the codes 0 .. 15
// themselves, subnormals and first normals, so a half is a mask and a sign. Its products
// with 4-bit weights have 8 bits and one exponent range, so a step's sums of eight products
// lose nothing; added up in fp32, 1e-7 of the result against 64 bits. The same steps on e4m3
// activations keep about 14 bits of each sum of eight products, whose exponents differ (5e-5
// measured on random codes): that is why 8 bits are whole numbers here.
//
// Sums are in units of y itself. In larger ones (y / 128 would follow from the codes as they
// are) a sum near 2^-126 would be a subnormal number and lose bits that y has. So the halves'
// scale bytes take what their codes leave out: h / 4 of the scale s is the code 2h of e2m3 at s,
// and of e4m3 at s + 6, l / 64 the code l at s - 3 and s + 3.
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
                    int KB, int KP, int64_t first, int64_t n) {
    const int64_t i = first + (int64_t)blockIdx.x * 256 + threadIdx.x;
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

// The halves of four 8-bit codes: bytes of a sign and 2h (0 .. 16), of a sign and l.
__device__ __forceinline__ void halves(uint32_t c, int& hi, int& lo) {
    const uint32_t s = c & 0x80808080u, t = s >> 7;
    const uint32_t mag = (c ^ ((s - t) | s)) + t;
    hi = (int)(((mag >> 3) & 0x1E1E1E1Eu) | s);
    lo = (int)((mag & 0x0F0F0F0Fu) | s);
}

// Bytes of a sign and a number v = 0 .. 15 as e4m3 numbers v / 4: below 8 by table, from
// there 2^1 and three bits.
__device__ __forceinline__ int quarters(int b) {
    const uint32_t v = (uint32_t)b & 0x07070707u, top = (uint32_t)b & 0x08080808u;
    const uint32_t large = (top << 4) | ((top << 4) - (top >> 3));      // 0xFF where v is 8 or more
    const uint32_t small = __builtin_amdgcn_perm(0x3E3C3A38u, 0x34302800u, v);
    return (int)((large & (0x40404040u | v)) | (~large & small) | ((uint32_t)b & 0x80808080u));
}

__device__ __forceinline__ v8i wide(v4i v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// ----------------------------------------------------------- few tokens
// The weights' bytes count: 28672 x 8192 for one token takes 28 us, 4.5 TB/s; small calls are a
// launch and its round trips (9728 x 896: 3.3 us). A workgroup takes 16 WA rows and up to 16 XB tokens; its waves take
// every NW-th 128 columns, D of them on their way at a time, and x as it lies in memory
// (16x16x128 steps: lane l holds row or token l % 16, of 4-bit operands block l / 16 of the 128
// columns, of e4m3 ones the bytes 16 (l / 16) .. of either half of them). The waves' sums are
// joined in LDS, in the order of the waves.
template <int FMT, int WA, int XB, int NW, int D>
__global__ __launch_bounds__(64 * NW)
void mx_stream_kernel(MxGemm p) {
    constexpr bool I8 = FMT == AERO_MX_INT8;
    __shared__ v4f part[NW][XB][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * WA), last = ((p.N + 31) >> 5) * 32 - 16;

    const uint8_t* wt[WA];
    const uint8_t* wst[WA];
#pragma unroll
    for (int a = 0; a < WA; ++a) {
        const int64_t n = min(n0 + 16 * a, last), tile = n >> 5;
        const int row = (int)(n & 31) + r;
        wt[a] = p.w + ((tile * (4 * p.KP) + q) * 32 + row) * 16;
        wst[a] = p.ws + (tile * p.KP * 32 + row) * 4 + q;
    }
    const uint8_t* xt[XB];
    const uint8_t* xst[XB];
#pragma unroll
    for (int b = 0; b < XB; ++b) {
        const int64_t tok = min((int64_t)(16 * b + r), p.T - 1);
        xt[b] = p.x + tok * p.KB * (I8 ? 32 : 16) + 16 * q;
        xst[b] = p.xs + tok * p.KB;
    }

    v4i w[D][WA], x0[D][XB], x1[D][XB];
    int sw[D][WA], sx[D][XB];
    auto load = [&](int d, int kk) __attribute__((always_inline)) {
        const int k = min(kk, p.KP - 1);
#pragma unroll
        for (int a = 0; a < WA; ++a) {
            w[d][a] = *reinterpret_cast<const v4i*>(wt[a] + (int64_t)k * 2048);
            sw[d][a] = wst[a][(int64_t)k * 128];
        }
        // (places past a row's last block: its last one, taken out below)
        const int kb = 4 * k + q, top = p.KB - 1;
#pragma unroll
        for (int b = 0; b < XB; ++b) {
            if constexpr (I8) {
                const int k0 = min(4 * k + (q >> 1), top), k1 = min(4 * k + 2 + (q >> 1), top);
                x0[d][b] = *reinterpret_cast<const v4i*>(xt[b] + 32 * k0 - 32 * (q >> 1));
                x1[d][b] = *reinterpret_cast<const v4i*>(xt[b] + 32 * k1 - 32 * (q >> 1));
            } else {
                x0[d][b] = *reinterpret_cast<const v4i*>(xt[b] + 16 * (min(kb, top) - q));
            }
            sx[d][b] = xst[b][min(kb, top)];
        }
    };
    v4f acc[WA][XB];
#pragma unroll
    for (int a = 0; a < WA; ++a)
#pragma unroll
        for (int b = 0; b < XB; ++b) acc[a][b] = v4f{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](int d, int k) __attribute__((always_inline)) {
        const bool whole = 4 * k + 4 <= p.KB;
        const v4i zero = {0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < XB; ++b) {
            int s = sx[d][b];
            if constexpr (I8) {
                v4i c0 = x0[d][b], c1 = x1[d][b];
                s = s < 4 ? 4 : s;
                if (!whole) {
                    if (4 * k + (q >> 1) >= p.KB) c0 = zero;
                    if (4 * k + 2 + (q >> 1) >= p.KB) c1 = zero;
                    if (4 * k + q >= p.KB) s = 4;
                }
                int sh = s + 6, sl = s + 3;
                const bool far = __any(s > 248);
                v8i hi, lo;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    int h, l;
                    halves((uint32_t)c0[i], h, l);
                    hi[i] = h; lo[i] = l;
                    halves((uint32_t)c1[i], h, l);
                    hi[4 + i] = h; lo[4 + i] = l;
                }
                // No scale byte is left for s + 6 above 2^121 (nor for NaN's 255): there the halves
                // go in as h / 4 and l / 4 of s and s - 4. (Unlikely, and in a loop, for the code
                // that all calls load: unrolled in place 9728 x 896 3.34 us for 3.32, 8 tokens of
                // 14336 x 4096 9.0 for 8.9. A second walk at the end instead: 3.40, 9.2.)
                if (__builtin_expect(far, 0)) {
#pragma unroll 1
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int t = hi[i];
                            hi[i] = lo[i];
                            lo[i] = quarters(n == 0 ? (t & 0x1E1E1E1E) >> 1 | (t & (int)0x80808080) : t);
                        }
                    sh -= 6;
                    sl -= 7;
                }
#pragma unroll
                for (int a = 0; a < WA; ++a)
                    acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        wide(w[d][a]), hi, acc[a][b], kF4, kF8, 0, sw[d][a], 0, sh);
#pragma unroll
                for (int a = 0; a < WA; ++a)
                    acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        wide(w[d][a]), lo, acc[a][b], kF4, kF8, 0, sw[d][a], 0, sl);
            } else {
                v4i c0 = x0[d][b];
                if (!whole && 4 * k + q >= p.KB) {
                    c0 = zero;
                    s = 0;
                }
#pragma unroll
                for (int a = 0; a < WA; ++a)
                    acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        wide(w[d][a]), wide(c0), acc[a][b], kF4, kF4, 0, sw[d][a], 0, s);
            }
        }
    };
#pragma unroll
    for (int d = 0; d < D; ++d) load(d, wave + d * NW);
    for (int k = wave; k < p.KP; k += D * NW) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int kk = k + d * NW;
            if (kk < p.KP) compute(d, kk);
            if (kk + D * NW < p.KP) load(d, kk + D * NW);
        }
    }

#pragma unroll
    for (int a = 0; a < WA; ++a) {
        if (a > 0) __syncthreads();
#pragma unroll
        for (int b = 0; b < XB; ++b) part[wave][b][lane] = acc[a][b];
        __syncthreads();
        const int64_t n = n0 + 16 * a + 4 * q;
        for (int b = wave; b < XB; b += NW) {
            v4f v = part[0][b][lane];
#pragma unroll
            for (int k = 1; k < NW; ++k) v += part[k][b][lane];
            const int64_t tok = 16 * b + r;
            if (tok >= p.T) continue;
            float* o = p.y + tok * p.N + n;
            if (p.vec && n + 4 <= p.N) {
                *reinterpret_cast<v4f*>(o) = v;
                continue;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < p.N) o[i] = v[i];
        }
    }
}

// ---------------------------------------------------------- many tokens
// x as operands, once a call: 32 tokens, then steps of 64 columns. 4 bits: as the weights.
// 8 bits: the halves as 6-bit floats (e2m3), whose steps against 4-bit operands take half
// the time of e4m3 ones (35 cycles and 64 measured). There too a number 0 .. 16 is its own
// code (in units of 1/8). A lane's 24 bytes a half lie as 16 and 8, 64 lanes side by side:
// 1024 + 512 for the high halves, the same for the low ones.
template <int FMT>
constexpr int kStepBytes = FMT == AERO_MX_INT8 ? 2 * (1024 + 512) : 1024;

// 32 codes of 6 bits, the first lowest, from bytes of a sign (bit 7) and a number 0 .. 16.
__device__ __forceinline__ void pack6(const uint32_t (&b)[8], uint32_t (&o)[6]) {
    uint32_t d[8];       // four codes each, 24 bits
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t c = (b[i] & 0x1F1F1F1Fu) | ((b[i] >> 2) & 0x20202020u);
        const uint32_t e = (c & 0x003F003Fu) | ((c >> 2) & 0x0FC00FC0u);
        d[i] = (e & 0xFFFu) | ((e >> 4) & 0xFFF000u);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        o[3 * i] = d[4 * i] | (d[4 * i + 1] << 24);
        o[3 * i + 1] = (d[4 * i + 1] >> 8) | (d[4 * i + 2] << 16);
        o[3 * i + 2] = (d[4 * i + 2] >> 16) | (d[4 * i + 3] << 8);
    }
}

// Two blocks of one token (columns 32 g .. and 64 + 32 g .. of 128) a lane; tokens and blocks
// past the end are zeros.
template <int FMT>
__global__ __launch_bounds__(256)
void mx_operand_kernel(const uint8_t* x, const uint8_t* xs, uint8_t* o, uint8_t* os, int64_t T, int KB,
                       int KP, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    constexpr int LOW = kMxLow<FMT>;
    const int lane = (int)(i & 63), r = lane & 31, g = lane >> 5;
    const uint32_t group = (uint32_t)(i >> 6), tile = group / (uint32_t)KP;
    const int k0 = 4 * (int)(group - tile * KP);
    const int64_t row = (int64_t)tile * 32 + r;
    // (loads from clamped places, all at once, then what is past the end taken out)
    const int64_t at = min(row, T - 1) * KB;
    constexpr int PIECE = FMT == AERO_MX_INT8 ? 2 : 1;      // 16 bytes a block
    uint4 c[2][PIECE];
    uint32_t s[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint4* p = reinterpret_cast<const uint4*>(x) + (at + min(k0 + 2 * j + g, KB - 1)) * PIECE;
#pragma unroll
        for (int h = 0; h < PIECE; ++h) c[j][h] = p[h];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] = xs[at + min(k0 + k, KB - 1)];
    const bool in = row < T;
    uint32_t four = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        four |= (uint32_t)(in && k0 + k < KB && s[k] > (uint32_t)LOW ? s[k] : LOW) << (8 * k);
    if (g == 0) reinterpret_cast<uint32_t*>(os)[(int64_t)group * 32 + r] = four;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < PIECE; ++h)
            if (!(in && k0 + 2 * j + g < KB)) c[j][h] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        uint8_t* to = o + (2 * (int64_t)group + j) * kStepBytes<FMT>;
        if constexpr (FMT == AERO_MX_FP4) {
            reinterpret_cast<uint4*>(to)[lane] = c[j][0];
        } else {
            const uint4 a = c[j][0], b = c[j][PIECE - 1];
            const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            uint32_t hi[8], lo[8], h[6], l[6];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                int e, f;
                halves(v[k], e, f);
                hi[k] = (uint32_t)e;
                lo[k] = (uint32_t)f;
            }
            pack6(hi, h);
            pack6(lo, l);
            reinterpret_cast<uint4*>(to)[lane] = make_uint4(h[0], h[1], h[2], h[3]);
            reinterpret_cast<uint2*>(to + 1024)[lane] = make_uint2(h[4], h[5]);
            reinterpret_cast<uint4*>(to + 1536)[lane] = make_uint4(l[0], l[1], l[2], l[3]);
            reinterpret_cast<uint2*>(to + 2560)[lane] = make_uint2(l[4], l[5]);
        }
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

// A workgroup's place. Each XCD (workgroups go round them in turn) takes a run of neighbouring
// tiles: four token tiles beside one weight tile, then beside the next, so that what runs at a time
// on an XCD shares both sides through its L2 (2048 x 28672 x 4096: 278 us with sixteen, 274 with
// four; 8192 x 4096 x 4096 184 and 172).
__device__ __forceinline__ bool tile_of(const MxTiles& p, int& n, int& t) {
    const int at = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (at >= p.bn * p.bt) return false;
    const int group = at / (p.group * p.bn), rest = at - group * p.group * p.bn;
    const int width = min(p.group, p.bt - group * p.group);
    n = rest / width;
    t = group * p.group + rest % width;
    return true;
}

// A tile of 32 x 32 sums: lane l holds column l % 32 of 16 tokens, 128 bytes of y in one piece for
// each.
__device__ __forceinline__ void store_tile(const MxTiles& p, int nt, int tt, const v16f& v) {
    const int lane = threadIdx.x & 63;
    const int64_t n = (int64_t)nt * 32 + (lane & 31), t1 = (int64_t)tt * 32 + 4 * (lane >> 5);
    if (n >= p.N) return;
    float* o = p.y + t1 * p.N + n;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int t = 8 * (i >> 2) + (i & 3);
        if (t1 + t < p.T) __builtin_nontemporal_store(v[i], o + t * p.N);
    }
}

// Large tiles (256 x 128 and 256 x 64 results). A workgroup of GN x GT waves, a wave WA weight
// tiles by XB token tiles of 32; with GK = 2 two such sets of waves, one for the first 64 of every
// 128 columns, one for the others, whose sums are joined at the end: as many waves on tiles half
// the size. Stages of 64 GK columns go through NB buffers in LDS by direct loads of 1 KB, each wave
// its share, NB - 1 stages ahead. With PIPE a stage's operands are read into registers while the
// one before is multiplied.
//
// 256 x 128 (two workgroups a CU, two waves a SIMD): 2048 x 28672 x 4096 in 243-256 us, 1.9-2.0
// PFLOP/s in twice as many steps as 4-bit x takes (150-156, 3.1). Its steps alone would take 131 at
// the rate they reach from registers (7.3 PFLOP/s, 1.9 GHz). No one thing bounds it: the clock is
// down to 1.75 GHz (a tenth), the fourth round of workgroups is half full (an eighth), and within a
// round the parts overlap only in part: loads alone take 106 us, steps and LDS reads 155, stores 35,
// past the caches (42 through them). Counters: matrix steps busy 52% of the time, LDS reads 24%,
// a wave waits to issue 49% of its time and for data or the others at the barrier 23%. Measured and
// not kept: 256 x 256 tiles with the weights straight into registers (282 us, one wave a SIMD).
template <int FMT, int WA, int XB, int GN, int GT, int GK>
struct MxShape {
    static constexpr int NW = GN * GT * GK, TN = WA * GN, TT = XB * GT;
    static constexpr int XS = kStepBytes<FMT> * GK;              // bytes of a token tile's stage
    static constexpr int XC = XS / 1024;
    static constexpr int SC = (TN + TT + 7) / 8;                 // pieces of 8 tiles' scales
    static constexpr int PIECES = TN * GK + TT * XC + SC;
    static constexpr int LOADS = (PIECES + NW - 1) / NW;
    static constexpr int XOFF = TN * GK * 1024, SOFF = XOFF + TT * XS;
    static constexpr int BYTES = SOFF + SC * 1024;
};

template <int FMT, int WA, int XB, int GN, int GT, int GK, int NB, bool PIPE>
__global__ __launch_bounds__(64 * GN * GT * GK, 2)
void mx_tiles_kernel(MxTiles p) {
    using S = MxShape<FMT, WA, XB, GN, GT, GK>;
    // (arrays of their own: the compiler tells a load into one from a read of another)
#define AERO_MX_BUF(K) __shared__ __attribute__((aligned(16))) uint8_t b##K[K < NB ? S::BYTES : 16]
    AERO_MX_BUF(0); AERO_MX_BUF(1); AERO_MX_BUF(2); AERO_MX_BUF(3);
#undef AERO_MX_BUF
    static_assert(NB == 3 || NB == 4, "");
    uint8_t* const bufs[4] = {b0, b1, b2, b3};
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, g = lane >> 5;
    int n0, t0;
    if (!tile_of(p, n0, t0)) return;
    n0 *= S::TN;
    t0 *= S::TT;

    // This wave's pieces of a step, the scales' first: where they begin, how far a step goes.
    // (A piece past the last is the wave's one before once more, to the same place.)
    static_assert(S::SC <= S::NW && S::PIECES >= S::NW, "each wave has a piece, the scales' are first ones");
    const uint8_t* src[S::LOADS];
    int dst[S::LOADS], stride[S::LOADS];
#pragma unroll
    for (int i = 0; i < S::LOADS; ++i) {
        int c = wave + S::NW * i;
        if (c >= S::PIECES) c -= S::NW;
        c -= S::SC;
        dst[i] = c * 1024;
        if (c < S::TN * GK) {
            const int q = max(c, 0);
            src[i] = p.w + (int64_t)min(n0 + q / GK, p.nt - 1) * p.KP * 2048 + q % GK * 1024;
            stride[i] = 1024 * GK;
        } else {
            const int q = max(c - S::TN * GK, 0);
            src[i] = p.x + (int64_t)min(t0 + q / S::XC, p.tt - 1) * p.KP * (2 * kStepBytes<FMT>) +
                     (q % S::XC) * 1024;
            stride[i] = S::XS;
        }
    }
    uint32_t lane16 = lane * 16;
    opaque(lane16);
    const uint8_t* first = src[0] + lane16;
    const int half = GK == 1 && wave < S::SC ? 1 : 0;
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
            __builtin_amdgcn_sched_barrier(0);     // (in this order: the waits below count them)
            const uint8_t* from = k == 0 ? first + (int64_t)(i >> half) * stride[0]
                                         : src[k] + (int64_t)i * stride[k] + lane16;
            uint8_t* to = b + dst[k];
            __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
        }
    };

    const int kg = GK == 1 ? 0 : wave / (GN * GT);
    const int wn = (wave % GN) * WA, wt = (wave / GN % GT) * XB;
    const int stages = GK == 1 ? p.steps : p.KP;
    v16f acc[WA][XB];
#pragma unroll
    for (int a = 0; a < WA; ++a)
#pragma unroll
        for (int b = 0; b < XB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;

    // A lane's places in a buffer. (Opaque, so that each stays one register that the buffers
    // and tiles add constants to.)
    int oa = (wn * GK + kg) * 1024 + lane * 16;
    int ox = S::XOFF + wt * S::XS + kg * kStepBytes<FMT> + lane * 16;
    int ox8 = ox - lane * 8, osa = S::SOFF + wn * 128 + r * 4, osx = S::SOFF + (S::TN + wt) * 128 + r * 4;
    opaque(oa);
    opaque(ox);
    opaque(ox8);
    opaque(osa);
    opaque(osx);
    constexpr int H = FMT == AERO_MX_INT8 ? 2 : 1, GROUPS = XB * H;
    struct Operands {
        v4i a[WA];
        v8i x[XB][H];        // (4-bit: the first four)
        int sa[WA], sb[XB];  // dwords of four blocks' scales
    };
    auto read = [&](Operands& f, const uint8_t* buf) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < WA; ++k) f.a[k] = *reinterpret_cast<const v4i*>(buf + oa + k * GK * 1024);
#pragma unroll
        for (int k = 0; k < WA; ++k) f.sa[k] = *reinterpret_cast<const int*>(buf + osa + k * 128);
#pragma unroll
        for (int b = 0; b < XB; ++b) {
            f.sb[b] = *reinterpret_cast<const int*>(buf + osx + b * 128);
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const int at = b * S::XS + 1536 * h;
                const v4i q = *reinterpret_cast<const v4i*>(buf + ox + at);
                if constexpr (H == 2) {
                    const v2i e = *reinterpret_cast<const v2i*>(buf + ox8 + at + 1024);
                    const v4i e4 = __builtin_shufflevector(e, e, 0, 1, -1, -1);
                    f.x[b][h] = __builtin_shufflevector(q, e4, 0, 1, 2, 3, 4, 5, -1, -1);
                } else {
                    f.x[b][h] = wide(q);
                }
            }
        }
    };
    // the matrix steps; the loads of a later stage go out behind them, one at a time
    auto multiply = [&](const Operands& f, int i, uint8_t* nb) __attribute__((always_inline)) {
        const int next = min(i + NB - 1, stages - 1);
        const int sh = 16 * (GK == 1 ? i & 1 : kg) + 8 * g;
        int sa[WA];
#pragma unroll
        for (int k = 0; k < WA; ++k) sa[k] = (int)((uint32_t)f.sa[k] >> sh);
#pragma unroll
        for (int b = 0; b < XB; ++b) {
            const int sb = (int)((uint32_t)f.sb[b] >> sh);
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int k = 0; k < WA; ++k) {
                    acc[k][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                        f.x[b][h], wide(f.a[k]), acc[k][b], H == 2 ? kF6 : kF4, kF4, 0, sb - 3 * h, 0, sa[k]);
                    const int at = (b * H + h) * WA + k;
                    __builtin_amdgcn_sched_barrier(0);
                    fetch(next, nb, at * S::LOADS / (GROUPS * WA), (at + 1) * S::LOADS / (GROUPS * WA));
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    };
    Operands even, odd;
    // A step begins when its loads have landed (the next ones' may be on their way) and
    // every wave is done with the step before, whose buffer is then filled again; the last
    // steps load the last one once more, so that every step is alike. (The marks keep the
    // copies of this code apart: merged, the compiler could not tell the buffer that is read
    // from the one that is filled, and would wait for the loads.)
    auto step = [&](auto k, int i) __attribute__((always_inline)) {
        constexpr int K = decltype(k)::value, R = PIPE ? (K + 1) % NB : K;
        constexpr int N = (PIPE ? NB - 3 : NB - 2) * S::LOADS;
        __builtin_amdgcn_s_waitcnt((N & 15) | 0x0f70 | ((N >> 4) << 14));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        asm volatile("; buffer %0" ::"n"(R) : "memory");
        if constexpr (PIPE) {
            if constexpr (K % 2 == 0) {
                read(odd, bufs[R]);
                __builtin_amdgcn_sched_barrier(0);
                multiply(even, i, bufs[(K + NB - 1) % NB]);
            } else {
                read(even, bufs[R]);
                __builtin_amdgcn_sched_barrier(0);
                multiply(odd, i, bufs[(K + NB - 1) % NB]);
            }
        } else {
            read(even, bufs[K]);
            multiply(even, i, bufs[(K + NB - 1) % NB]);
        }
        asm volatile("; buffer %0 done" ::"n"(R) : "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
#define AERO_MX_EACH(DO) DO(0) DO(1) DO(2) DO(3)
#define AERO_MX_FILL(K) if constexpr (K < NB - 1) fetch(min(K, stages - 1), bufs[K], 0, S::LOADS);
#define AERO_MX_ROUND(K) if constexpr (K < NB) step(std::integral_constant<int, K>{}, i + K);
#define AERO_MX_REST(K) \
    if constexpr (K < NB - 1) if (i + K < stages) step(std::integral_constant<int, K>{}, i + K);
    AERO_MX_EACH(AERO_MX_FILL)
    if constexpr (PIPE) {
        static_assert(NB >= 4 && NB % 2 == 0, "two sets of operands in turn, two stages ahead of the loads");
        constexpr int N = (NB - 2) * S::LOADS;
        __builtin_amdgcn_s_waitcnt((N & 15) | 0x0f70 | ((N >> 4) << 14));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        read(even, bufs[0]);
    }
    // (whole rounds, then the rest: with an exit after each step the compiler keeps the sums
    // twice and spills)
    int i = 0;
    for (; i + NB <= stages; i += NB) {
        AERO_MX_EACH(AERO_MX_ROUND)
    }
    AERO_MX_EACH(AERO_MX_REST)
#undef AERO_MX_EACH
#undef AERO_MX_FILL
#undef AERO_MX_ROUND
#undef AERO_MX_REST
    __builtin_amdgcn_s_waitcnt(0x0f70);       // (no load is on its way when the wave ends)

    auto put = [&](int a, int b, const v16f& v) __attribute__((always_inline)) {
        store_tile(p, n0 + wn + a, t0 + wt + b, v);
    };
    if constexpr (GK == 1) {
#pragma unroll
        for (int a = 0; a < WA; ++a)
#pragma unroll
            for (int b = 0; b < XB; ++b) put(a, b, acc[a][b]);
    } else {
        // each set of waves ends with half of the tiles, the other's sums of them passed
        // through LDS
        constexpr int HALF = WA * XB / 2;
        static_assert(WA * XB % 2 == 0, "half of the tiles each");
        // (a tile a wave, in the first three buffers)
        static_assert((S::NW + 2) / 3 * 4096 <= S::BYTES, "room for a tile a wave");
        auto room = [&](int x) {
            return reinterpret_cast<v4f*>(x % 3 == 0 ? b0 : x % 3 == 1 ? b1 : b2) + x / 3 * 256 + lane;
        };
        v4f* mine = room(wave);
        const v4f* other = room(wave ^ (GN * GT));
#pragma unroll
        for (int m = 0; m < HALF; ++m) {
            const v16f &lo = acc[m / XB][m % XB], &up = acc[(m + HALF) / XB][(m + HALF) % XB];
            __syncthreads();
            const v16f give = kg ? lo : up;
            v16f sum = kg ? up : lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const v4f q = {give[4 * i], give[4 * i + 1], give[4 * i + 2], give[4 * i + 3]};
                mine[64 * i] = q;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const v4f q = other[64 * i];
#pragma unroll
                for (int k = 0; k < 4; ++k) sum[4 * i + k] += q[k];
            }
            const int tile = kg ? m + HALF : m;
            put(tile / XB, tile % XB, sum);
        }
    }
}

// Smaller tiles: 32 WA rows by 32 XB tokens, the columns split over the waves. Every NW-th 128
// columns are one wave's, so that each operand is loaded once, straight into the registers of the
// one wave that multiplies it, and LDS holds nothing but the waves' sums at the end. D groups of
// 128 columns are in registers: one is multiplied, and behind each of its steps goes a load or two
// of the group D - 1 ahead (loads in one piece before the steps: 512 x 4096 x 14336 in 43.5 us, so
// in 42.1, 512 x 28672 x 4096 on the same tiles 100 and 88).
//
// What bounds it is the way from the L2 to the CUs: 128 x 64 results take 21 KB for 128 columns, and
// 256 workgroups get 18 TB/s (303 ns a group, 512 x 4096 x 14336), about 30 bytes a cycle each; the
// matrix steps would take half of that. For 64 tokens of 28672 x 8192 HBM is the other bound (3.6
// TB/s on 224 CUs). The same tiles through LDS, with two sets of waves: 512 x 4096 x 14336 50.5 us
// and 42.1, 333 x 2560 x 10240 in 4 bits 18.0 and 14.7, 48 x 4096 x 14336 26.8 and 19.8, 100 x 4096 x
// 4096 13.4 and 11.1, 64 x 28672 x 8192 39.9 and 38.9: there each byte crossed LDS three to four
// times. Eight waves instead of four: 64 x 64 results 56 us for 54 (512 x 4096 x 14336), 64 x 32 65
// for 62. Weights by loads that pass the caches: 64 x 28672 x 8192 41.4, the others a tenth to a
// third slower, as their weights no longer come from the last-level cache.
template <int FMT, int WA, int XB, int NW, int D>
__global__ __launch_bounds__(64 * NW, NW / 4)
void mx_split_kernel(MxTiles p) {
    constexpr int H = FMT == AERO_MX_INT8 ? 2 : 1, TILES = WA * XB;
    __shared__ v4f part[NW][TILES][4][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, g = lane >> 5;
    int n0, t0;
    if (!tile_of(p, n0, t0)) return;
    n0 *= WA;
    t0 *= XB;

    const uint8_t *w[WA], *ws[WA], *x[XB], *xs[XB];
#pragma unroll
    for (int a = 0; a < WA; ++a) {
        const int64_t n = min(n0 + a, p.nt - 1);
        w[a] = p.w + n * p.KP * 2048;
        ws[a] = p.ws + n * p.KP * 128;
    }
#pragma unroll
    for (int b = 0; b < XB; ++b) {
        const int64_t t = min(t0 + b, p.tt - 1);
        x[b] = p.x + t * p.KP * (2 * kStepBytes<FMT>);
        xs[b] = p.xs + t * p.KP * 128;
    }
    struct Group {
        v4i w[2][WA];
        v8i x[2][XB][H];
        int sw[WA], sx[XB];
    };
    Group f[D];
    // load l of a group: the scales, then the operands in the order of the steps
    constexpr int XL = 2 * H - (H == 1), STEP = WA + XB * XL, LOADS = WA + XB + 2 * STEP;
    auto load = [&](Group& f, int k, int l) __attribute__((always_inline)) {
        if (l < WA) {
            f.sw[l] = *reinterpret_cast<const int*>(ws[l] + (int64_t)k * 128 + r * 4);
        } else if (l < WA + XB) {
            f.sx[l - WA] = *reinterpret_cast<const int*>(xs[l - WA] + (int64_t)k * 128 + r * 4);
        } else {
            const int j = (l - WA - XB) / STEP, i = (l - WA - XB) % STEP;
            if (i < WA) {
                f.w[j][i] = *reinterpret_cast<const v4i*>(w[i] + (int64_t)k * 2048 + j * 1024 + lane * 16);
            } else {
                const int b = (i - WA) / XL, h = (i - WA) % XL / (H == 2 ? 2 : 1), e = (i - WA) % XL % 2;
                const uint8_t* q = x[b] + ((int64_t)k * 2 + j) * kStepBytes<FMT> + 1536 * h;
                if (H == 2 && e == 1) {
                    const v2i v = *reinterpret_cast<const v2i*>(q + 1024 + lane * 8);
                    const v8i e8 = __builtin_shufflevector(v, v, 0, 1, -1, -1, -1, -1, -1, -1);
                    f.x[j][b][h] = __builtin_shufflevector(f.x[j][b][h], e8, 0, 1, 2, 3, 8, 9, -1, -1);
                } else {
                    f.x[j][b][h] = wide(*reinterpret_cast<const v4i*>(q + lane * 16));
                }
            }
        }
    };
    v16f acc[WA][XB];
#pragma unroll
    for (int a = 0; a < WA; ++a)
#pragma unroll
        for (int b = 0; b < XB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;
    // the matrix steps of a group; the loads of a later one go out behind them
    auto compute = [&](const Group& f, Group& nf, int k, bool more) __attribute__((always_inline)) {
        constexpr int M = 2 * XB * H * WA;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int sh = 16 * j + 8 * g;
#pragma unroll
            for (int b = 0; b < XB; ++b) {
                const int sb = (int)((uint32_t)f.sx[b] >> sh);
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int a = 0; a < WA; ++a) {
                        acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                            f.x[j][b][h], wide(f.w[j][a]), acc[a][b], H == 2 ? kF6 : kF4, kF4, 0, sb - 3 * h, 0,
                            (int)((uint32_t)f.sw[a] >> sh));
                        const int m = ((j * XB + b) * H + h) * WA + a;
                        if (more) {
                            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                            for (int l = m * LOADS / M; l < (m + 1) * LOADS / M; ++l) load(nf, k, l);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
            }
        }
    };
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            load(f[d], min(wave + d * NW, p.KP - 1), l);
            __builtin_amdgcn_sched_barrier(0);
        }
    int k = wave;
    for (; k + (D - 1) * NW < p.KP; k += D * NW) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            compute(f[d], f[(d + D - 1) % D], min(k + (d + D - 1) * NW, p.KP - 1), true);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
        if (k + d * NW < p.KP) compute(f[d], f[d], 0, false);

    // each tile's sums by one wave, the others' through LDS
#pragma unroll
    for (int m = 0; m < TILES; ++m)
        if (m % NW != wave) {
            const v16f v = acc[m / XB][m % XB];
#pragma unroll
            for (int i = 0; i < 4; ++i) part[wave][m][i][lane] = v4f{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < TILES; ++m)
        if (m % NW == wave) {
            v16f v = acc[m / XB][m % XB];
#pragma unroll
            for (int o = 1; o < NW; ++o)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const v4f q = part[(wave + o) % NW][m][i][lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[4 * i + e] += q[e];
                }
            store_tile(p, n0 + m / XB, t0 + m % XB, v);
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

// Rows that a workgroup of the few-token kernel takes. More of them share x (and, in 8 bits, its
// halves), more workgroups keep more of the chip busy. Measured, us, with 16 (32) rows: 4096 x
// 4096, one token, 4.1 (5.0); 14336 x 4096, 8 tokens, 12.1 (8.7); 28672 x 8192, one token, 31 (27);
// with 17 to 32 tokens, 16 / 32 / 64 rows: 4096 x 4096 7.4 / 8.8 / 11.3, 8192 x 8192 18 / 12.8 /
// 16, 14336 x 4096 22 / 16.7 / 12.1. Short rows (up to 12 groups of 128 columns) leave little for
// eight waves: 9728 x 896, 24 tokens, 5.4 with 16 rows and one group on its way, 7.9 with 32 rows.
int stream_rows(int64_t n_tok, int64_t n_rows, int KP) {
    if (n_tok > 16) return n_rows >= 12288 ? 64 : n_rows >= 6144 && KP > 12 ? 32 : 16;
    return n_rows >= 12288 ? 32 : 16;
}

// Calls that run on the few-token kernel; the others go through operands in the workspace. Up to
// 16 tokens all, from 17 to 32 while rounds of workgroups on the CUs * tokens * columns stay below
// a limit: the tiles take a launch more (6 us in all), and then less for each column. Measured
// for 17 / 24 / 32 tokens, us on the few-token kernel and on tiles:
//   8 bits, 16 rows: 4096 x 14336 16.9, 18.7 / 19.9, 18.8 / 23.3, 19.0; 4096 x 8192 10.8, 13.1 /
//     12.5, 13.4 / 14.3, 13.5; in two rounds 5120 x 2560 7.2, 8.0 / 7.9, 8.2 / 9.1, 8.4 and 5120 x
//     4096 11.0, 9.6 / 13.0, 9.9 / 15.0, 10.0
//   8 bits, 32 rows: 8192 x 4096 8.5, 10.1 / 9.4, 10.4 / 10.2, 10.6; 8192 x 8192 13.2, 13.8 / 15.3,
//     13.9 / 16.8, 14.2; in two rounds 8224 x 2048 8.8, 7.9 / 9.9, 8.2 / 11.0, 8.4
//   8 bits, 64 rows: 16384 x 2048 7.6, 9.3 / 8.1, 9.6 / 8.5, 9.9; 14336 x 4096 11.2, 10.9 / 12.1, 11.2 /
//     12.7, 11.4; in two rounds 16416 x 512 8.6, 7.4 / 9.0, 7.6 / 9.6, 7.9, 20000 x 8192 32.0, 19.7 /
//     35.2, 19.9 / 39.0, 23.1
//   4 bits, 16 rows: 4096 x 14336 11.2, 12.7 / 13.8, 12.8 / 16.4, 13.1; in two rounds 5120 x 2560 4.8, 6.1 /
//     5.4, 6.3 / 6.2, 6.4 and 5120 x 4096 7.3, 7.3 / 9.1, 7.5 / 10.2, 7.6
//   4 bits, 32 rows: 8192 x 8192 9.2, 10.4 / 10.7, 10.5 / 11.9, 10.7; in two rounds 8224 x 2048 5.4,
//     6.1 / 6.2, 6.4 / 6.9, 6.5
//   4 bits, 64 rows: 16384 x 8192 14.2, 15.1 / 14.9, 15.2 / 16.0, 15.4; in two rounds 16416 x 512 7.2,
//     6.3 / 7.4, 6.1 / 7.8, 6.2
bool few_tokens(int fmt, int64_t n_tok, int64_t n_rows, int64_t n_cols) {
    if (n_tok <= 16) return true;
    if (n_tok > 32) return false;
    // thousands: one round, more of them; by rows a workgroup (16, 32, 64)
    static const int kLimit[2][3][2] = {{{290, 130}, {150, 0}, {66, 0}}, {{290, 165}, {200, 100}, {230, 0}}};
    const int rows = stream_rows(n_tok, n_rows, (int)((n_cols + 127) / 128)), cus = cu_count();
    const int64_t rounds = ((n_rows + rows - 1) / rows + cus - 1) / cus;
    return rounds * n_tok * n_cols <= 1000 * (int64_t)kLimit[fmt == AERO_MX_INT8 ? 0 : 1][rows >> 5][rounds > 1];
}

template <int FMT>
int64_t operand_bytes(int64_t n_tok, int KP) {
    return tiles32(n_tok) * KP * (2 * kStepBytes<FMT> + 128);
}

// Workgroups of one launch: fewer than 2^32 lanes.
bool grid_ok(int64_t T, int64_t N, int64_t grid, int lanes) {
    if (grid * lanes <= 0xffffffff) return true;
    set_error("mx_matmul: %lld x %lld results are too many", (long long)T, (long long)N);
    return false;
}

template <int FMT, int WA, int XB, int NW, int D>
bool launch_stream(const MxGemm& p, hipStream_t s) {
    const int64_t grid = (p.N + 16 * WA - 1) / (16 * WA);
    return grid_ok(p.T, p.N, grid, 64 * NW) &&
           launch("mx_stream_kernel", mx_stream_kernel<FMT, WA, XB, NW, D>, dim3((unsigned)grid), dim3(64 * NW), 0, s, p);
}

// (eight waves a workgroup; four on short rows: 9728 x 896, one token, 3.3 us and 3.7)
template <int FMT>
bool run_stream(const MxGemm& p, hipStream_t s) {
    const int rows = stream_rows(p.T, p.N, p.KP);
    if (p.T > 16) {
        if (rows == 64) return launch_stream<FMT, 4, 2, 8, 2>(p, s);
        return rows == 32 ? launch_stream<FMT, 2, 2, 8, 2>(p, s) : launch_stream<FMT, 1, 2, 8, 1>(p, s);
    }
    if (rows == 32) return launch_stream<FMT, 2, 1, 8, 2>(p, s);
    return p.KP <= 12 ? launch_stream<FMT, 1, 1, 4, 2>(p, s) : launch_stream<FMT, 1, 1, 8, 2>(p, s);
}

template <int FMT, int WA, int XB, int GN, int GT, int GK, int NB, bool PIPE>
bool launch_tiles(MxTiles p, hipStream_t s) {
    using S = MxShape<FMT, WA, XB, GN, GT, GK>;
    p.bn = (p.nt + S::TN - 1) / S::TN;
    p.bt = (p.tt + S::TT - 1) / S::TT;
    const int64_t grid = ((int64_t)p.bn * p.bt + 7) / 8 * 8;
    return grid_ok(p.T, p.N, grid, 64 * S::NW) &&
           launch("mx_tiles_kernel", mx_tiles_kernel<FMT, WA, XB, GN, GT, GK, NB, PIPE>, dim3((unsigned)grid),
                  dim3(64 * S::NW), 0, s, p);
}

template <int FMT, int WA, int XB, int NW, int D>
bool launch_split(MxTiles p, hipStream_t s) {
    p.bn = (p.nt + WA - 1) / WA;
    p.bt = (p.tt + XB - 1) / XB;
    const int64_t grid = ((int64_t)p.bn * p.bt + 7) / 8 * 8;
    return grid_ok(p.T, p.N, grid, 64 * NW) &&
           launch("mx_split_kernel", mx_split_kernel<FMT, WA, XB, NW, D>, dim3((unsigned)grid), dim3(64 * NW), 0, s, p);
}

// The tiles by what rounds of them take: the workgroups that run at a time, and microseconds of
// such a round, for each 128 columns and beside them, fitted to measured calls. All six on the same
// call, us: 512 x 28672 x 4096 73 / 88 / 88 / 108 / 104 / 108, 512 x 6144 x 4096 42 / 27 / 29 / 29 / 27 /
// 29, 512 x 4096 x 14336 113 / 58 / 42 / 54 / 49 / 62, 300 x 9728 x 896 17 / 13 / 16 / 16 / 16 / 15, 64 x 4096
// x 4096 38 / 22 / 16 / 12 / 12 / 10; in 4 bits 333 x 2560 x 10240 (the last four) 20 / 15 / 16 / 18,
// 1500 x 5120 x 2048 21 / 23 / 28 / 24 / 26 / 26.
int best_tiles(int fmt, int64_t T, int64_t N, int KP) {
    struct Tiles {
        int n, t, per_cu;
        float each[2], once[2];      // 8 bits, 4 bits
    };
    static const Tiles kTiles[6] = {{8, 4, 2, {1.75f, 1.1f}, {5.f, 1.f}},     {8, 2, 1, {0.57f, 0.39f}, {4.5f, 3.3f}},
                                    {4, 2, 1, {0.31f, 0.15f}, {2.5f, 3.8f}},  {2, 2, 1, {0.21f, 0.1f}, {2.4f, 1.4f}},
                                    {4, 1, 1, {0.2f, 0.12f}, {2.2f, 1.4f}},   {2, 1, 1, {0.118f, 0.075f}, {1.f, 0.5f}}};
    const int F = fmt == AERO_MX_INT8 ? 0 : 1;
    const int64_t tt = tiles32(T), nt = tiles32(N), cus = cu_count();
    // The largest run two to a CU. A last round of one each has a time of its own: 1939 x 3200 x
    // 12512 in 4 bits 71.7 us, 75.8 on the best of the others; 1932 x 3456 x 3488 28.6 and 28.4, 1609 x
    // 2624 x 1344 15.3 and 15.3. (For up to 512 columns it stands above the time of a whole round,
    // which is then set too low, its stores left out; no choice hangs on that, and the lower of the
    // two would be wrong for small calls: 128 x 14336 x 128 in 4 bits 9.4 on these tiles, 8.1 on 64
    // x 32.)
    const float alone = F == 0 ? 1.f * KP + 6.f : 0.65f * KP + 3.f;
    int best = 0;
    float least = 0.f;
    for (int i = 0; i < 6; ++i) {
        const Tiles& c = kTiles[i];
        const int64_t n = ((nt + c.n - 1) / c.n) * ((tt + c.t - 1) / c.t);
        const int64_t slots = c.per_cu * cus, last = n % slots;
        const float round = c.each[F] * KP + c.once[F];
        const float cost = (float)(n / slots) * round +
                           (last == 0 ? 0.f : i == 0 && last <= cus ? alone : round);
        if (i == 0 || cost < least) {
            best = i;
            least = cost;
        }
    }
    return best;
}

template <int FMT>
bool run_tiles(const MxGemm& g, void* ws, hipStream_t s) {
    const int64_t tt = tiles32(g.T), nt = tiles32(g.N);
    uint8_t* o = (uint8_t*)ws;
    uint8_t* os = o + tt * g.KP * (2 * kStepBytes<FMT>);
    const int64_t n = tt * 64 * g.KP, blocks = (n + 255) / 256;
    if (n >> 6 > 0x7fffffff || nt > 0x7fffffff || tt > 0x7fffffff) {
        set_error("mx_matmul: %lld tokens are too many", (long long)g.T);
        return false;
    }
    if (!launch("mx_operand_kernel", mx_operand_kernel<FMT>, dim3((unsigned)blocks), dim3(256), 0, s, g.x,
                g.xs, o, os, g.T, g.KB, g.KP, n))
        return false;
    const MxTiles p{g.w, g.ws, o, os, g.y, g.T, g.N, g.KP, (g.KB + 1) / 2, (int)nt, (int)tt, 0, 0, 4};
    switch (tune("mx_tiles", best_tiles(FMT, g.T, g.N, g.KP))) {
    case 0: return launch_tiles<FMT, 4, 2, 2, 2, 1, 3, false>(p, s);
    case 1: return launch_tiles<FMT, 4, 1, 2, 2, 2, 4, true>(p, s);
    case 2: return launch_split<FMT, 4, 2, 4, 2>(p, s);
    case 3: return launch_split<FMT, 2, 2, 4, 3>(p, s);
    case 4: return launch_split<FMT, 4, 1, 4, 3>(p, s);
    default: return launch_split<FMT, 2, 1, 4, 3>(p, s);
    }
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
    const int64_t n = tiles32(n_rows) * 32 * 4 * KP;
    uint8_t* codes_out = (uint8_t*)w;
    for (int64_t i = 0; i < n; i += kMxLanes) {
        const int64_t m = n - i < kMxLanes ? n - i : kMxLanes;
        if (!launch("mx_pack_kernel", mx_pack_kernel, dim3((unsigned)((m + 255) / 256)), dim3(256), 0,
                    (hipStream_t)stream, codes, scales, codes_out,
                    codes_out + weight_codes_bytes(n_rows, n_cols), n_rows, KB, KP, i, n))
            return 0;
    }
    return 1;
}

int64_t aero_hip_mx_matmul_workspace(int fmt, int64_t n_rows, int64_t n_cols, int64_t n_tok) {
    using namespace aero;
    if ((fmt != AERO_MX_INT8 && fmt != AERO_MX_FP4) || n_tok < 0 || n_tok > 0x7fffffff) {
        set_error("mx_matmul_workspace: format %d, %lld tokens", fmt, (long long)n_tok);
        return -1;
    }
    if (!weight_sizes_ok("mx_matmul_workspace", n_rows, n_cols)) return -1;
    if (few_tokens(fmt, n_tok, n_rows, n_cols)) return 0;
    const int KP = (int)((n_cols + 127) / 128);
    return fmt == AERO_MX_INT8 ? operand_bytes<AERO_MX_INT8>(n_tok, KP)
                               : operand_bytes<AERO_MX_FP4>(n_tok, KP);
}

int aero_hip_mx_matmul_tiles(int fmt, int64_t n_rows, int64_t n_cols, int64_t n_tok) {
    using namespace aero;
    if (aero_hip_mx_matmul_workspace(fmt, n_rows, n_cols, n_tok) < 0) return -1;
    if (few_tokens(fmt, n_tok, n_rows, n_cols)) return 6;
    return best_tiles(fmt, n_tok, n_rows, (int)((n_cols + 127) / 128));
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
    const int64_t need = aero_hip_mx_matmul_workspace(fmt, n_rows, n_cols, n_tok);
    const bool room = workspace != nullptr && aligned16(workspace) && ws_bytes >= need;
    // (without a workspace the few-token kernel takes all that it can)
    if (!few_tokens(fmt, n_tok, n_rows, n_cols) && (room || n_tok > 32)) {
        if (!room) {
            set_error("mx_matmul: the workspace takes %lld bytes at a 16-byte address", (long long)need);
            return 0;
        }
        return (fmt == AERO_MX_INT8 ? run_tiles<AERO_MX_INT8>(p, workspace, s)
                                    : run_tiles<AERO_MX_FP4>(p, workspace, s)) ? 1 : 0;
    }
    return (fmt == AERO_MX_INT8 ? run_stream<AERO_MX_INT8>(p, s) : run_stream<AERO_MX_FP4>(p, s)) ? 1 : 0;
}

}  // extern "C"
