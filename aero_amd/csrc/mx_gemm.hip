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
#include "mx.hpp"

#pragma clang fp contract(off)

namespace aero {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kF8 = 0, kF4 = 4;  // operand formats of the step

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

// 32 weight rows and 32 tokens a workgroup, its four waves each every fourth 128 columns,
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
    return 0;
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
    const int64_t tt = tiles32(n_tok);
    if (tt > 65535) {
        set_error("mx_matmul: %lld tokens are too many", (long long)n_tok);
        return 0;
    }
    const int KB = (int)(n_cols / 32), KP = (KB + 3) / 4;
    MxGemm p{codes, scales, (const uint8_t*)w, (const uint8_t*)w + weight_codes_bytes(n_rows, n_cols), y,
             n_tok, n_rows, KB, KP, aligned16(y) && n_rows % 4 == 0};
    const dim3 grid((unsigned)tiles32(n_rows), (unsigned)tt);
    const hipStream_t s = (hipStream_t)stream;
    return (fmt == AERO_MX_INT8
                ? launch("mx_gemm_kernel", mx_gemm_kernel<AERO_MX_INT8>, grid, dim3(256), 0, s, p)
                : launch("mx_gemm_kernel", mx_gemm_kernel<AERO_MX_FP4>, grid, dim3(256), 0, s, p))
               ? 1 : 0;
}

}  // extern "C"
