// A paged KV cache's rows and pages: new keys and values into their pages
// (quantised as include/aero/kv.hpp:62-92), rows back as fp32 (src/kv.cpp:30-46),
// pages copied for forks and compaction, table entries written in stream order.
//
// A vector (token, kv head) of position pos of sequence s lies in page
// table[s][pos / page], row pos % page of the head's [page, dim] block.
#include "paged.hpp"

#include <climits>
#include <cmath>
#include <memory>
#include <new>

namespace aero {

bool pool_ok(const aero_kv_pool_t& p, const char* what) {
    if (p.kv_dt < 0 || p.kv_dt > 2 || p.page < 16 || p.page > 256 || (p.page & (p.page - 1)) ||
        p.n_layers <= 0 || p.n_pages <= 0 || p.n_head_kv <= 0 || p.head_dim <= 0 ||
        p.value_dim <= 0 || p.head_dim > 256 || p.value_dim > 256 || p.n_pages > INT_MAX ||
        p.n_layers > (1 << 20) || p.n_head_kv > 65535 ||
        (p.kv_dt == 0 && (p.head_dim % 4 || p.value_dim % 4)) ||
        (p.kv_dt == 2 && (p.head_dim % 2 || p.value_dim % 2))) {
        set_error("%s: bad pool (kv_dt=%d page=%lld layers=%lld pages=%lld heads=%lld "
                  "head_dim=%lld value_dim=%lld; pages of 16-256 tokens, a power of two; dims up "
                  "to 256, a multiple of 4 in fp32, of 2 in int4)", what, p.kv_dt,
                  (long long)p.page, (long long)p.n_layers, (long long)p.n_pages,
                  (long long)p.n_head_kv, (long long)p.head_dim, (long long)p.value_dim);
        return false;
    }
    if (p.k == nullptr || p.v == nullptr || !aligned16(p.k) || !aligned16(p.v) ||
        (p.kv_dt != 0 && (p.k_scale == nullptr || p.v_scale == nullptr ||
                          !aligned16(p.k_scale) || !aligned16(p.v_scale)))) {
        set_error("%s: the pool's K, V and scales must be there and 16-byte aligned", what);
        return false;
    }
    return true;
}

namespace {

struct RowsIo {
    float* rows[2];        // k, v: [n_seq, n_q, heads, dim]
    uint8_t* pages[2];
    float* scales[2];
    const int32_t* table;
    const int32_t* lens;
    int32_t* bad;
    int32_t dim[2];
    int32_t n_q, heads, n_pages, max_pages, shift;
    int64_t n_rows;        // n_seq * n_q * heads
};

// The vector of the pool that row r is; -1: no token, or no page
// (rows are fewer than 2^26)
__device__ __forceinline__ int64_t pool_vector(const RowsIo& p, uint32_t r) {
    const uint32_t tok = r / (uint32_t)p.heads, h = r - tok * p.heads;
    const uint32_t s = tok / (uint32_t)p.n_q;
    const int64_t pos = (int64_t)p.lens[s] - p.n_q + (tok - s * p.n_q);
    if (pos < 0) return -1;
    const int64_t col = pos >> p.shift;
    const int32_t page = col < p.max_pages ? p.table[(int64_t)s * p.max_pages + col] : -1;
    if (page < 0 || page >= p.n_pages) {
        if (p.bad != nullptr) *p.bad = 1;
        return -1;
    }
    return (((int64_t)page * p.heads + h) << p.shift) + (pos & ((1 << p.shift) - 1));
}

// A row (a vector of K or V) is L lanes' work, four elements each at a time: a
// workgroup takes 256 / L rows of K (blockIdx.y 0) or V (1). The rows come and go
// in fp32 as 16-byte pieces and in the pages as whole words. L is the lanes a row
// of dim / 4 pieces fills: 16, 32 or 64. Bound by the copy: 1,999 tokens of 8 heads of
// 128 in fp32, 32.8 MB, 7.0 us (4.7 TB/s; element by element, a wave a row, 11.4); of
// a serving step by the launch and three round trips (length, page id, row): 4 tokens
// of 64 sequences, int8, written and read back, two launches, 10 us.
struct Codes {
    float top, scale;
    __device__ __forceinline__ int operator()(float v) const {
        return (int)fminf(fmaxf(roundf(v / scale), -top), top);
    }
};

template <int DT, int L>
__global__ __launch_bounds__(256) void paged_write_kernel(RowsIo p) {
    const int w = blockIdx.y, dim = p.dim[w], li = threadIdx.x % L;
    const int64_t r = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (r >= p.n_rows) return;
    const float* x = p.rows[w] + r * dim;
    // (the row is on its way while its place is looked up; dim <= 256: a lane of
    // 64 has one piece, and no row two)
    const bool in = 4 * li < dim;
    const float4 f = in ? *reinterpret_cast<const float4*>(x + 4 * li)
                        : make_float4(0.f, 0.f, 0.f, 0.f);
    const int64_t vec = pool_vector(p, (uint32_t)r);
    if (vec < 0) return;
    if constexpr (DT == 0) {
        if (in) *reinterpret_cast<float4*>(p.pages[w] + (vec * dim + 4 * li) * 4) = f;
    } else {
        float amax = fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w)));
#pragma unroll
        for (int off = L / 2; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, L));
        constexpr float top = DT == 1 ? 127.0f : 7.0f;
        const float sc = amax > 0.0f ? amax / top : 1.0f;
        if (li == 0) p.scales[w][vec] = sc;
        const Codes code{top, sc};
        const int a = code(f.x), b = code(f.y), c = code(f.z), d = code(f.w);
        if (!in) return;
        if constexpr (DT == 1)
            *reinterpret_cast<uint32_t*>(p.pages[w] + vec * dim + 4 * li) =
                (a & 255) | ((b & 255) << 8) | ((c & 255) << 16) | ((uint32_t)(d & 255) << 24);
        else
            *reinterpret_cast<uint16_t*>(p.pages[w] + vec * (dim / 2) + 2 * li) =
                (uint16_t)((a & 15) | ((b & 15) << 4) | ((c & 15) << 8) | ((d & 15) << 12));
    }
}

template <int DT, int L>
__global__ __launch_bounds__(256) void paged_read_kernel(RowsIo p) {
    const int w = blockIdx.y, dim = p.dim[w], li = threadIdx.x % L;
    const int64_t r = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (r >= p.n_rows || 4 * li >= dim) return;
    const int64_t vec = pool_vector(p, (uint32_t)r);
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (vec >= 0) {
        if constexpr (DT == 0) {
            f = *reinterpret_cast<const float4*>(p.pages[w] + (vec * dim + 4 * li) * 4);
        } else {
            const float sc = p.scales[w][vec];
            int n[4];
            if constexpr (DT == 1) {
                const uint32_t c = *reinterpret_cast<const uint32_t*>(p.pages[w] + vec * dim + 4 * li);
#pragma unroll
                for (int e = 0; e < 4; ++e) n[e] = (int32_t)(c << (24 - 8 * e)) >> 24;
            } else {
                const uint32_t c =
                    *reinterpret_cast<const uint16_t*>(p.pages[w] + vec * (dim / 2) + 2 * li);
#pragma unroll
                for (int e = 0; e < 4; ++e) n[e] = (int32_t)(c << (28 - 4 * e)) >> 28;
            }
            f = make_float4((float)n[0] * sc, (float)n[1] * sc, (float)n[2] * sc, (float)n[3] * sc);
        }
    }
    *reinterpret_cast<float4*>(p.rows[w] + r * dim + 4 * li) = f;
}

// The same for dims that are no multiple of 4, or rows that are not 16-byte
// aligned: a wave a row, element by element.
template <int DT>
__global__ __launch_bounds__(64) void paged_write_any_kernel(RowsIo p) {
    const int w = blockIdx.y, dim = p.dim[w], lane = threadIdx.x;
    const int64_t r = blockIdx.x;
    const int64_t vec = pool_vector(p, (uint32_t)r);
    if (vec < 0) return;
    const float* x = p.rows[w] + r * dim;
    if constexpr (DT == 0) {
        float* o = reinterpret_cast<float*>(p.pages[w]) + vec * dim;
        for (int i = lane; i < dim; i += 64) o[i] = x[i];
    } else {
        float amax = 0.0f;
        for (int i = lane; i < dim; i += 64) amax = fmaxf(amax, fabsf(x[i]));
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 64));
        constexpr float top = DT == 1 ? 127.0f : 7.0f;
        const float sc = amax > 0.0f ? amax / top : 1.0f;
        if (lane == 0) p.scales[w][vec] = sc;
        const Codes code{top, sc};
        if constexpr (DT == 1) {
            int8_t* o = reinterpret_cast<int8_t*>(p.pages[w]) + vec * dim;
            for (int i = lane; i < dim; i += 64) o[i] = (int8_t)code(x[i]);
        } else {
            uint8_t* o = p.pages[w] + vec * (dim / 2);
            for (int i = lane; i < dim / 2; i += 64)
                o[i] = (uint8_t)((code(x[2 * i]) & 15) | ((code(x[2 * i + 1]) & 15) << 4));
        }
    }
}

template <int DT>
__global__ __launch_bounds__(64) void paged_read_any_kernel(RowsIo p) {
    const int w = blockIdx.y, dim = p.dim[w], lane = threadIdx.x;
    const int64_t r = blockIdx.x;
    const int64_t vec = pool_vector(p, (uint32_t)r);
    float* o = p.rows[w] + r * dim;
    const float sc = DT != 0 && vec >= 0 ? p.scales[w][vec] : 0.0f;
    for (int i = lane; i < dim; i += 64) {
        float v = 0.0f;
        if (vec >= 0) {
            if constexpr (DT == 0) {
                v = reinterpret_cast<const float*>(p.pages[w])[vec * dim + i];
            } else if constexpr (DT == 1) {
                v = (float)reinterpret_cast<const int8_t*>(p.pages[w])[vec * dim + i] * sc;
            } else {
                const uint8_t b = p.pages[w][vec * (dim / 2) + i / 2];
                const int n = (i & 1) ? b >> 4 : b & 15;
                v = (float)(n >= 8 ? n - 16 : n) * sc;
            }
        }
        o[i] = v;
    }
}

using RowsIoKernel = void (*)(RowsIo);

// the kernel for rows of dims d0 and d1 and its rows a workgroup
template <int DT>
RowsIoKernel rows_io_kernel(bool write, bool vector, int most, int& rows, int& threads) {
    threads = 256;
    if (vector && most <= 64) {
        rows = 16;
        return write ? paged_write_kernel<DT, 16> : paged_read_kernel<DT, 16>;
    }
    if (vector && most <= 128) {
        rows = 8;
        return write ? paged_write_kernel<DT, 32> : paged_read_kernel<DT, 32>;
    }
    if (vector) {
        rows = 4;
        return write ? paged_write_kernel<DT, 64> : paged_read_kernel<DT, 64>;
    }
    rows = 1;
    threads = 64;
    return write ? paged_write_any_kernel<DT> : paged_read_any_kernel<DT>;
}

bool launch_rows_io(const RowsIo& p, int dt, bool write, hipStream_t s) {
    if (p.n_rows == 0) return true;
    const bool vector = p.dim[0] % 4 == 0 && p.dim[1] % 4 == 0 && aligned16(p.rows[0]) &&
                        aligned16(p.rows[1]);
    const int most = p.dim[0] > p.dim[1] ? p.dim[0] : p.dim[1];
    int rows, threads;
    RowsIoKernel k = dt == 0 ? rows_io_kernel<0>(write, vector, most, rows, threads)
                             : (dt == 1 ? rows_io_kernel<1>(write, vector, most, rows, threads)
                                        : rows_io_kernel<2>(write, vector, most, rows, threads));
    return launch(write ? "paged_write_kernel" : "paged_read_kernel", k,
                  dim3((unsigned)((p.n_rows + rows - 1) / rows), 2), dim3(threads), 0, s, p);
}

bool rows_io(const aero_kv_pool_t& pool, int64_t layer, float* k, float* v, const int32_t* table,
             int64_t max_pages, const int32_t* lens, int64_t n_seq, int64_t n_q, int32_t* bad,
             const char* what, RowsIo& p) {
    if (!pool_ok(pool, what)) return false;
    if (layer < 0 || layer >= pool.n_layers || n_seq < 0 || n_q <= 0 || max_pages <= 0 ||
        max_pages > (int64_t(1) << 30) / pool.page || n_q > (int64_t(1) << 30) ||
        n_seq > ((1 << 26) - 1) / (n_q * pool.n_head_kv)) {   // (a grid row: 2^32 threads)
        set_error("%s: bad sizes (layer=%lld n_seq=%lld n_q=%lld max_pages=%lld)", what,
                  (long long)layer, (long long)n_seq, (long long)n_q, (long long)max_pages);
        return false;
    }
    if (n_seq > 0 && (k == nullptr || v == nullptr || table == nullptr || lens == nullptr)) {
        set_error("%s: null pointer", what);
        return false;
    }
    const PoolLayer at = pool_layer(pool, layer);
    p.rows[0] = k; p.rows[1] = v;
    p.pages[0] = at.k; p.pages[1] = at.v;
    p.scales[0] = at.ks; p.scales[1] = at.vs;
    p.table = table; p.lens = lens; p.bad = bad;
    p.dim[0] = (int32_t)pool.head_dim; p.dim[1] = (int32_t)pool.value_dim;
    p.n_q = (int32_t)n_q; p.heads = (int32_t)pool.n_head_kv;
    p.n_pages = (int32_t)pool.n_pages; p.max_pages = (int32_t)max_pages;
    p.shift = 0;
    while ((1 << p.shift) < pool.page) ++p.shift;
    p.n_rows = n_seq * n_q * pool.n_head_kv;
    return true;
}

// ------------------------------------------------------------------- pages
constexpr int kCopyPairs = 256;   // pairs a launch (by value: 2 KB of arguments)

struct PageCopy {
    uint8_t* base[4];        // K, V, their scales
    int64_t bytes[4];        // of a page in one layer (0: no such plane)
    int64_t layer[4];        // from a layer to the next
    int32_t src[kCopyPairs], dst[kCopyPairs];
};

// Workgroup (x, pair, layer): 16-byte pieces of the page's planes, one after the
// other, a workgroup 4 KB of the largest plane: enough of them for a short list, and
// the pairs are arguments, so nothing is copied to the device first.
// Bound by the copy: 34.6 MB 6.4 us, 1.02 GB 175 us (5.8 TB/s; a copy of one buffer
// 4.65).
__global__ __launch_bounds__(256) void pages_copy_kernel(PageCopy p) {
    const int64_t src = p.src[blockIdx.y], dst = p.dst[blockIdx.y];
    const int64_t step = (int64_t)gridDim.x * 256;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const v4u* a = reinterpret_cast<const v4u*>(p.base[x] + blockIdx.z * p.layer[x] +
                                                    src * p.bytes[x]);
        v4u* b = reinterpret_cast<v4u*>(p.base[x] + blockIdx.z * p.layer[x] + dst * p.bytes[x]);
        for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < p.bytes[x] / 16; i += step)
            b[i] = a[i];
    }
}

constexpr int kEdits = 256;
struct Edits {
    int32_t* base;
    int64_t at[kEdits];
    int32_t value[kEdits];
    int32_t n;
};
__global__ __launch_bounds__(256) void write_i32_kernel(Edits e) {
    const int i = threadIdx.x;
    if (i < e.n) e.base[e.at[i]] = e.value[i];
}

bool pages_copy_dev(const aero_kv_pool_t& pool, const int32_t* src, const int32_t* dst, int64_t n,
                    hipStream_t s) {
    if (!pool_ok(pool, "kv_pages_copy")) return false;
    if (n < 0 || (n > 0 && (src == nullptr || dst == nullptr)) || n > pool.n_pages ||
        pool.n_layers > 65535) {
        set_error("kv_pages_copy: bad list of %lld pairs (a pool of %lld pages, at most 65535 "
                  "layers)", (long long)n, (long long)pool.n_pages);
        return false;
    }
    // every destination once, and none of them a source: the copies then have no
    // order among them
    std::unique_ptr<uint8_t[]> seen(new (std::nothrow) uint8_t[(size_t)pool.n_pages]());
    if (!seen) {
        set_error("kv_pages_copy: out of host memory");
        return false;
    }
    for (int64_t i = 0; i < n; ++i) {
        if (src[i] < 0 || src[i] >= pool.n_pages || dst[i] < 0 || dst[i] >= pool.n_pages) {
            set_error("kv_pages_copy: pair %lld (%d -> %d) is outside the pool's %lld pages",
                      (long long)i, src[i], dst[i], (long long)pool.n_pages);
            return false;
        }
        seen[src[i]] |= 1;
        if (seen[dst[i]] & 2) {
            set_error("kv_pages_copy: page %d is a destination twice", dst[i]);
            return false;
        }
        seen[dst[i]] |= 2;
    }
    for (int64_t i = 0; i < n; ++i)
        if (seen[dst[i]] & 1) {
            set_error("kv_pages_copy: page %d is a source and a destination", dst[i]);
            return false;
        }
    PageCopy p{};
    const PoolLayer l0 = pool_layer(pool, 0);
    const int64_t vecs = pool.n_head_kv * pool.page;
    void* base[4] = {l0.k, l0.v, l0.ks, l0.vs};
    const int64_t bytes[4] = {vecs * kv_vec_bytes(pool.kv_dt, pool.head_dim),
                              vecs * kv_vec_bytes(pool.kv_dt, pool.value_dim),
                              pool.kv_dt ? vecs * 4 : 0, pool.kv_dt ? vecs * 4 : 0};
    int64_t most = 0;
    for (int x = 0; x < 4; ++x) {
        p.base[x] = static_cast<uint8_t*>(base[x]);
        p.bytes[x] = bytes[x];
        p.layer[x] = bytes[x] * pool.n_pages;
        most = bytes[x] > most ? bytes[x] : most;
    }
    const unsigned gx = (unsigned)((most + 4095) / 4096);
    for (int64_t i = 0; i < n; i += kCopyPairs) {
        const int m = (int)(n - i < kCopyPairs ? n - i : kCopyPairs);
        for (int x = 0; x < m; ++x) {
            p.src[x] = src[i + x];
            p.dst[x] = dst[i + x];
        }
        if (!launch("pages_copy_kernel", pages_copy_kernel,
                    dim3(gx, (unsigned)m, (unsigned)pool.n_layers), dim3(256), 0, s, p))
            return false;
    }
    return true;
}

}  // namespace
}  // namespace aero

extern "C" {

int aero_hip_paged_kv_write(const aero_kv_pool_t* pool, int64_t layer, const float* k,
                            const float* v, const int32_t* table, int64_t max_pages,
                            const int32_t* lens, int64_t n_seq, int64_t n_q, int32_t* bad,
                            void* stream) {
    using namespace aero;
    clear_error();
    RowsIo p{};
    if (pool == nullptr) {
        set_error("paged_kv_write: null pool");
        return 0;
    }
    if (!rows_io(*pool, layer, const_cast<float*>(k), const_cast<float*>(v), table, max_pages,
                 lens, n_seq, n_q, bad, "paged_kv_write", p))
        return 0;
    return launch_rows_io(p, pool->kv_dt, true, (hipStream_t)stream) ? 1 : 0;
}

int aero_hip_paged_kv_read(const aero_kv_pool_t* pool, int64_t layer, float* k, float* v,
                           const int32_t* table, int64_t max_pages, const int32_t* lens,
                           int64_t n_seq, int64_t n_q, int32_t* bad, void* stream) {
    using namespace aero;
    clear_error();
    RowsIo p{};
    if (pool == nullptr) {
        set_error("paged_kv_read: null pool");
        return 0;
    }
    if (!rows_io(*pool, layer, k, v, table, max_pages, lens, n_seq, n_q, bad, "paged_kv_read", p))
        return 0;
    return launch_rows_io(p, pool->kv_dt, false, (hipStream_t)stream) ? 1 : 0;
}

int aero_hip_kv_pages_copy(const aero_kv_pool_t* pool, const int32_t* src, const int32_t* dst,
                           int64_t n, void* stream) {
    aero::clear_error();
    if (pool == nullptr) {
        aero::set_error("kv_pages_copy: null pool");
        return 0;
    }
    return aero::pages_copy_dev(*pool, src, dst, n, (hipStream_t)stream) ? 1 : 0;
}

int aero_hip_write_i32(int32_t* base, int64_t n_base, const int64_t* at, const int32_t* value,
                       int64_t n, void* stream) {
    using namespace aero;
    clear_error();
    if (n < 0 || n_base < 0 || (n > 0 && (base == nullptr || at == nullptr || value == nullptr))) {
        set_error("write_i32: bad arguments");
        return 0;
    }
    for (int64_t i = 0; i < n; ++i)
        if (at[i] < 0 || at[i] >= n_base || (i > 0 && at[i] <= at[i - 1])) {
            set_error("write_i32: index %lld outside %lld elements, or not above the one before "
                      "it", (long long)at[i], (long long)n_base);
            return 0;
        }
    Edits e{};
    e.base = base;
    for (int64_t i = 0; i < n; i += kEdits) {
        e.n = (int32_t)(n - i < kEdits ? n - i : kEdits);
        for (int x = 0; x < e.n; ++x) {
            e.at[x] = at[i + x];
            e.value[x] = value[i + x];
        }
        if (!launch("write_i32_kernel", write_i32_kernel, dim3(1), dim3(256), 0,
                    (hipStream_t)stream, e))
            return 0;
    }
    return 1;
}

}  // extern "C"
