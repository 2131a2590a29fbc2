// Attention of few query rows over a paged KV cache, and over a contiguous one
// with a sliding window and sinks: GQA with an online softmax, as
// src/transformer.cpp:120-214, for several sequences.
//
//   out[s, t, h] = sum_j softmax_j(scale q[s, t, h] . k[j, kh]) v[j, kh],
//   kh = h / (H / HK), over the keys j that position p of token t sees:
//   j <= p and (no window, or p - j < window, or j < sinks); none: zeros.
//
// A query vector's running maximum m, sum l = sum e^(s - m) and accumulator
// sum e^(s - m) v are carried over its keys, and parts of them are joined by
// the same rule: m = max m_i, l = sum l_i e^(m_i - m).
//
// Work (paged_sched.hpp): an item is a sequence, a kv head and a tile of query
// vectors (token t, head kh rep + r: every head of the group shares the keys);
// its key tiles are cut into units.
//  * paged: a fixed number of workgroups take equal spans of all items' units,
//    read from the lengths on the device: a batch of ragged lengths is balanced,
//    and a recorded plan stays right as the sequences grow. An item cut by a
//    span's end leaves parts that rows_join_kernel joins.
//  * contiguous: every item's units go to n_chunks workgroups.
// Page ids are checked against the pool: tiles of a bad page are not seen.
#include "attn_common.hpp"
#include "paged_sched.hpp"
#include "paged.hpp"
#include "aero_hip.h"

#include <algorithm>
#include <climits>
#include <cmath>

namespace aero {
namespace {

struct RowsParams {
    const float* q;        // [n_seq, n_q, n_head, head_dim]
    float* out;            // [n_seq, n_q, n_head, value_dim]
    const void* k;         // paged: the layer's pages [n_pages, n_head_kv, page, head_dim]
    const void* v;         // contiguous: [n_kv, n_head_kv, head_dim]
    const float* ks;
    const float* vs;
    const int32_t* table;  // paged: [n_seq, max_pages]
    const int32_t* lens;   // paged: [n_seq]
    const int32_t* qpos;   // contiguous: [n_q] or null (= t)
    const int32_t* kpos;   // contiguous: [n_kv] or null (= j)
    int32_t* bad;          // set to 1 when a bad page was met, or null
    float* part;           // [workers][2][VEC] rows of pitch floats, then (m, l) of each
    int2* spans;           // [items]: first and last worker of the item
    int32_t n_seq, n_q, n_head, n_head_kv, rep, head_dim, value_dim, pitch;
    int32_t n_pages, max_pages, page_shift;
    int32_t n_kv;          // contiguous: keys; paged: the table's room in tokens
    int32_t tiles;         // query tiles a kv head and sequence
    int32_t window, sinks;
    int32_t workers, n_chunks;
    float scale;
};

// One item and the keys of it
struct Item {
    int32_t s, kh, z;   // sequence, kv head, query tile
    int32_t len;        // keys there are
    int32_t pos0;       // paged: position of token 0
    KeyTiles kt;
};

__device__ __forceinline__ int64_t item_index(const RowsParams& p, const Item& it) {
    return ((int64_t)it.s * p.n_head_kv + it.kh) * p.tiles + it.z;
}

__device__ __forceinline__ bool key_seen(int64_t kp, int64_t qp, int window, int sinks) {
    return kp <= qp && (window <= 0 || qp - kp < window || kp < sinks);
}

__device__ __forceinline__ float* part_row(const RowsParams& p, int64_t row) {
    return p.part + row * p.pitch;
}
__device__ __forceinline__ float2* part_ml(const RowsParams& p, int vec, int64_t row) {
    return reinterpret_cast<float2*>(p.part + (int64_t)p.workers * 2 * vec * p.pitch) + row;
}

// The page of table column col of sequence s, or -1 (none, or not of the pool)
__device__ __forceinline__ int32_t page_at(const RowsParams& p, int32_t s, int32_t col) {
    const int32_t page =
        col < p.max_pages ? p.table[(int64_t)s * p.max_pages + col] : -1;
    const bool ok = page >= 0 && page < p.n_pages;
    if (!ok && p.bad != nullptr) *p.bad = 1;
    return ok ? page : -1;
}

// ------------------------------------------------------------ any head width
// 16-lane groups own a key each (a 16-key tile a step of the workgroup), lane
// li of a group elements E li .. of the head; dot products by lane shuffles,
// four query vectors a workgroup.
template <int DT, int E>
__device__ __forceinline__ void load_slice(const void* base, const float* scales, int64_t vec,
                                           int dim, int e0, float (&o)[E]) {
    if constexpr (DT == 0) {
        const float* p = static_cast<const float*>(base) + vec * dim + e0;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            if (e0 + e < dim) {   // (dim % 4 == 0)
                const float4 f = *reinterpret_cast<const float4*>(p + e);
                o[e] = f.x; o[e + 1] = f.y; o[e + 2] = f.z; o[e + 3] = f.w;
            } else {
                o[e] = o[e + 1] = o[e + 2] = o[e + 3] = 0.0f;
            }
        }
    } else if constexpr (DT == 1) {
        const int8_t* p = static_cast<const int8_t*>(base) + vec * dim + e0;
        const float s = scales[vec];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = (e0 + e < dim) ? (float)p[e] * s : 0.0f;
    } else {
        const uint8_t* p = static_cast<const uint8_t*>(base) + vec * (dim / 2) + e0 / 2;
        const float s = scales[vec];
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const uint32_t b = (e0 + e < dim) ? p[e / 2] : 0u;
            const int lo = (int)(b & 15u), hi = (int)(b >> 4);
            o[e] = (float)(lo >= 8 ? lo - 16 : lo) * s;
            o[e + 1] = (float)(hi >= 8 ? hi - 16 : hi) * s;
        }
    }
}

template <int DT, int E, bool PAGED>
struct VecCore {
    static constexpr int VEC = 4;            // query vectors an item
    static constexpr int UNIT = 4;           // key tiles a unit
    static constexpr int DVP = 16 * E;
    struct Shared {
        float m[16][VEC], l[16][VEC], acc[16][VEC][DVP];
    };

    const RowsParams& p;
    const Item& it;
    Shared& sh;
    int grp, li, e0;
    int64_t qrow[VEC];
    int64_t qp[VEC];
    bool qok[VEC];
    float q[VEC][E], m[VEC], l[VEC], acc[VEC][E];

    __device__ __forceinline__ VecCore(const RowsParams& p_, const Item& it_, Shared& sh_)
        : p(p_), it(it_), sh(sh_) {
        grp = threadIdx.x >> 4;
        li = threadIdx.x & 15;
        e0 = E * li;
        const int n_vec = p.n_q * p.rep;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int u = it.z * VEC + i;
            qok[i] = u < n_vec;
            const int uc = qok[i] ? u : n_vec - 1;
            const int t = uc / p.rep;
            qrow[i] = ((int64_t)it.s * p.n_q + t) * p.n_head + it.kh * p.rep + uc % p.rep;
            qp[i] = PAGED ? it.pos0 + t : (p.qpos ? p.qpos[t] : t);
            m[i] = -INFINITY;
            l[i] = 0.0f;
            const float* src = p.q + qrow[i] * p.head_dim;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                q[i][e] = e0 + e < p.head_dim ? src[e0 + e] : 0.0f;
                acc[i][e] = 0.0f;
            }
        }
    }

    // positions of the item's rows, least and greatest
    static __device__ __forceinline__ void reach(const RowsParams& p, int z, int64_t& lo,
                                                 int64_t& hi) {
        const int n_vec = p.n_q * p.rep;
        lo = INT64_MAX;
        hi = INT64_MIN;
        for (int i = 0; i < VEC; ++i) {
            const int t = min(z * VEC + i, n_vec - 1) / p.rep;
            const int64_t x = p.qpos ? p.qpos[t] : t;
            lo = min(lo, x);
            hi = max(hi, x);
        }
    }

    // places [x0, x1) of the item's key tiles
    __device__ __forceinline__ void walk(int x0, int x1) {
        for (int x = x0; x < x1; ++x) {
            const int tile = it.kt.at(x);
            const int j = 16 * tile + grp;
            int64_t vec;
            if constexpr (PAGED) {
                const int32_t page = page_at(p, it.s, tile >> (p.page_shift - 4));
                if (page < 0) continue;
                vec = (((int64_t)page * p.n_head_kv + it.kh) << p.page_shift) +
                      (j & ((1 << p.page_shift) - 1));
            } else {
                vec = (int64_t)j * p.n_head_kv + it.kh;
            }
            if (j >= it.len) continue;
            float kv[E], vv[E];
            load_slice<DT, E>(p.k, p.ks, vec, p.head_dim, e0, kv);
            load_slice<DT, E>(p.v, p.vs, vec, p.value_dim, e0, vv);
            const int64_t kp = !PAGED && p.kpos ? p.kpos[j] : j;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float d = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) d = __builtin_fmaf(q[i][e], kv[e], d);
                d = group_sum<16>(d);
                if (key_seen(kp, qp[i], p.window, p.sinks)) {
                    const float s = d * p.scale;
                    const float mn = fmaxf(m[i], s);
                    const float a = m[i] == -INFINITY ? 0.0f : expf(m[i] - mn);
                    const float w = s == -INFINITY ? 0.0f : expf(s - mn);
                    l[i] = l[i] * a + w;
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        acc[i][e] = __builtin_fmaf(w, vv[e], acc[i][e] * a);
                    m[i] = mn;
                }
            }
        }
    }

    // the groups' sums joined; the rows written out (row < 0), or as a part
    __device__ __forceinline__ void finish(int64_t row) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (li == 0) {
                sh.m[grp][i] = m[i];
                sh.l[grp][i] = l[i];
            }
#pragma unroll
            for (int e = 0; e < E; ++e) sh.acc[grp][i][e0 + e] = acc[i][e];
        }
        __syncthreads();
        const int n_vec = p.n_q * p.rep;
        for (int w = threadIdx.x; w < VEC * DVP; w += 256) {
            const int i = w / DVP, d = w % DVP;
            const int u = it.z * VEC + i;
            if (u >= n_vec || d >= p.value_dim) continue;
            float mt = -INFINITY, lt = 0.0f, at = 0.0f;
            for (int g = 0; g < 16; ++g) mt = fmaxf(mt, sh.m[g][i]);
            for (int g = 0; g < 16; ++g) {
                const float c = sh.m[g][i] == -INFINITY ? 0.0f : expf(sh.m[g][i] - mt);
                lt = __builtin_fmaf(sh.l[g][i], c, lt);
                // (0 times what a group without keys holds is 0: its sums are 0)
                at = __builtin_fmaf(sh.acc[g][i][d], c, at);
            }
            if (row < 0) {
                const int64_t r = ((int64_t)it.s * p.n_q + u / p.rep) * p.n_head +
                                  it.kh * p.rep + u % p.rep;
                p.out[r * p.value_dim + d] = at / fmaxf(lt, 1e-30f);
            } else {
                part_row(p, row + i)[d] = at;
                if (d == 0) *part_ml(p, VEC, row + i) = make_float2(mt, lt);
            }
        }
    }
};

// Inclusive sums over the wave's lanes
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t o = __shfl_up(v, off, 64);
        if ((int)(threadIdx.x & 63) >= off) v += o;
    }
    return v;
}
__device__ __forceinline__ int64_t wave_value(int64_t v, int lane) {
    return __shfl(v, lane, 64);
}
__device__ __forceinline__ int64_t uniform64(int64_t v) {
    return (int64_t)(((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32)) << 32) |
                     __builtin_amdgcn_readfirstlane((uint32_t)v));
}

__device__ __forceinline__ int32_t seq_len(const RowsParams& p, int32_t s) {
    return min(max(p.lens[s], 0), p.n_kv);
}
__device__ __forceinline__ KeyTiles seq_tiles(const RowsParams& p, int32_t len) {
    return key_tiles((int64_t)len - p.n_q, (int64_t)len - 1, len, p.window, p.sinks);
}

// Paged: worker blockIdx.x's span of units, item by item. Every wave works out
// the span from the lengths by itself: a sum over the lanes, a scan over the 64
// sequences around the span's begin.
template <typename Core>
__global__ __launch_bounds__(256) void rows_paged_kernel(RowsParams p) {
    __shared__ typename Core::Shared sh;
    const int lane = threadIdx.x & 63;
    const int32_t per_seq = p.n_head_kv * p.tiles;
    int64_t total = 0;
    for (int s = lane; s < p.n_seq; s += 64)
        total += (int64_t)item_units(seq_tiles(p, seq_len(p, s)).n, Core::UNIT) * per_seq;
    total = uniform64(wave_value(wave_scan(total), 63));
    const int64_t g = total < p.workers ? total : p.workers;
    const int w = blockIdx.x;
    if (w >= g) return;
    int64_t u = span_begin(w, total, g);
    const int64_t u_end = span_begin(w + 1, total, g);
    // the sequence of unit u, and the units before it
    int64_t base = 0;
    int s = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += 64) {
        const int x = s0 + lane;
        const int64_t n = x < p.n_seq
                              ? (int64_t)item_units(seq_tiles(p, seq_len(p, x)).n, Core::UNIT) *
                                    per_seq
                              : 0;
        const int64_t upto = wave_scan(n);
        const uint64_t past = __ballot(base + upto > u);
        if (past != 0) {
            const int f = __ffsll((unsigned long long)past) - 1;
            s = s0 + f;
            base = uniform64(base + wave_value(upto - n, f));
            break;
        }
        base += uniform64(wave_value(upto, 63));
    }
    s = __builtin_amdgcn_readfirstlane(s);

    while (u < u_end && s < p.n_seq) {
        Item it;
        it.s = s;
        it.len = __builtin_amdgcn_readfirstlane(seq_len(p, s));
        it.pos0 = it.len - p.n_q;
        it.kt = seq_tiles(p, it.len);
        const int units = item_units(it.kt.n, Core::UNIT);
        const int64_t end = base + (int64_t)units * per_seq;
        while (u < u_end && u < end) {
            const int64_t rel = u - base;
            const int64_t item = rel / units;
            const int a = (int)(rel % units);
            const int b = (int)min<int64_t>(units, a + (u_end - u));
            it.kh = (int)(item / p.tiles);
            it.z = (int)(item % p.tiles);
            // (keys past the tile's own last position are not walked)
            const int t_last = min(it.z * Core::VEC + Core::VEC - 1, p.n_q * p.rep - 1) / p.rep;
            const int x1 = min(b * Core::UNIT, it.kt.upto(it.pos0 + t_last));
            Core core(p, it, sh);
            core.walk(a * Core::UNIT, x1);
            const bool whole = a == 0 && b == units;
            core.finish(whole ? -1 : ((int64_t)w * 2 + (a == 0 ? 1 : 0)) * Core::VEC);
            if (a == 0 && threadIdx.x == 0) {
                const int64_t first = base + item * units;
                p.spans[item_index(p, it)] =
                    make_int2(w, (int)span_of(first + units - 1, total, g));
            }
            u += b - a;
        }
        base = end;
        ++s;
    }
}

// Contiguous: chunk blockIdx.x of n_chunks of item (kv head blockIdx.y, query
// tile), the last query tiles (a prompt's longest) first.
template <typename Core>
__global__ __launch_bounds__(256) void rows_linear_kernel(RowsParams p) {
    __shared__ typename Core::Shared sh;
    Item it;
    it.s = 0;
    it.kh = blockIdx.y;
    it.z = gridDim.z - 1 - blockIdx.z;
    it.len = p.n_kv;
    it.pos0 = 0;
    if (p.kpos != nullptr) {
        it.kt = KeyTiles{0, 0, (p.n_kv + 15) / 16};
    } else {
        int64_t lo, hi;
        Core::reach(p, it.z, lo, hi);
        it.kt = key_tiles(uniform64(lo), uniform64(hi), p.n_kv, p.window, p.sinks);
    }
    const int units = item_units(it.kt.n, Core::UNIT);
    const int c = blockIdx.x;
    const int a = (int)((int64_t)c * units / p.n_chunks);
    const int b = (int)((int64_t)(c + 1) * units / p.n_chunks);
    const int64_t item = item_index(p, it);
    Core core(p, it, sh);
    core.walk(a * Core::UNIT, min(b * Core::UNIT, it.kt.n));
    core.finish(p.n_chunks == 1 ? -1
                                : ((item * p.n_chunks + c) * 2 + (c == 0 ? 1 : 0)) * Core::VEC);
    if (c == 0 && threadIdx.x == 0 && p.n_chunks > 1)
        p.spans[item] = make_int2((int)(item * p.n_chunks), (int)((item + 1) * p.n_chunks - 1));
}

// The parts of one row (row blockIdx.x % VEC of item blockIdx.x / VEC) joined: a
// group of pitch / 4 lanes takes every G-th part, then the groups meet in LDS.
// The first worker's part is its slot 1 (it begins the item), the others' 0.
template <int VEC>
__global__ __launch_bounds__(512) void rows_join_kernel(RowsParams p) {
    __shared__ float sm[512], sl[512];
    __shared__ float4 sa[512];
    const int64_t item = blockIdx.x / VEC;
    const int i = blockIdx.x % VEC;
    const int z = (int)(item % p.tiles);
    const int u = z * VEC + i;
    if (u >= p.n_q * p.rep) return;
    const int2 span = p.spans[item];
    const int n = span.y - span.x + 1;
    if (n <= 1) return;
    const int tid = threadIdx.x;
    const int lpr = p.pitch / 4, G = 512 / lpr;
    const int d4 = tid % lpr, grp = tid / lpr;
    float M = -INFINITY, L = 0.0f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int B = 4;
    if (grp < G) {
        for (int c0 = grp; c0 < n; c0 += B * G) {
            float2 ml[B];
            float4 a[B];
#pragma unroll
            for (int x = 0; x < B; ++x) {
                const int c = min(c0 + x * G, n - 1);
                const int64_t row = ((int64_t)(span.x + c) * 2 + (c == 0 ? 1 : 0)) * VEC + i;
                ml[x] = *part_ml(p, VEC, row);
                a[x] = *reinterpret_cast<const float4*>(part_row(p, row) + 4 * d4);
            }
            float mb = M;
#pragma unroll
            for (int x = 0; x < B; ++x)
                if (c0 + x * G < n) mb = fmaxf(mb, ml[x].x);
            const float sc = M == -INFINITY ? 0.0f : expf(M - mb);
            L *= sc;
            A.x *= sc; A.y *= sc; A.z *= sc; A.w *= sc;
#pragma unroll
            for (int x = 0; x < B; ++x) {
                // (a part without keys holds zeros; not so one that is no part)
                if (c0 + x * G >= n || ml[x].x == -INFINITY) continue;
                const float w = expf(ml[x].x - mb);
                L = __builtin_fmaf(ml[x].y, w, L);
                A.x = __builtin_fmaf(a[x].x, w, A.x);
                A.y = __builtin_fmaf(a[x].y, w, A.y);
                A.z = __builtin_fmaf(a[x].z, w, A.z);
                A.w = __builtin_fmaf(a[x].w, w, A.w);
            }
            M = mb;
        }
        if (d4 == 0) sm[grp] = M;
    }
    __syncthreads();
    if (grp < G) {
        float mt = -INFINITY;
        for (int k = 0; k < G; ++k) mt = fmaxf(mt, sm[k]);
        const float w = M == -INFINITY ? 0.0f : expf(M - mt);
        sa[tid] = make_float4(A.x * w, A.y * w, A.z * w, A.w * w);
        if (d4 == 0) sl[grp] = L * w;
    }
    __syncthreads();
    if (tid < lpr) {
        float lt = 0.0f;
        float4 at = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < G; ++k) {
            const float4 a = sa[k * lpr + tid];
            lt += sl[k];
            at.x += a.x; at.y += a.y; at.z += a.z; at.w += a.w;
        }
        const float r = 1.0f / fmaxf(lt, 1e-30f);
        const int64_t s = item / ((int64_t)p.n_head_kv * p.tiles);
        const int kh = (int)(item / p.tiles % p.n_head_kv);
        float* o = p.out + ((s * p.n_q + u / p.rep) * p.n_head + (int64_t)kh * p.rep + u % p.rep) *
                               p.value_dim + 4 * tid;
        const float v[4] = {at.x * r, at.y * r, at.z * r, at.w * r};
        for (int x = 0; x < 4; ++x)
            if (4 * tid + x < p.value_dim) o[x] = v[x];
    }
}

// ------------------------------------------------------------------- host
using RowsKernel = void (*)(RowsParams);

// A variant of the kernels: query vectors an item, key tiles a unit
struct RowsVariant {
    const char* name;
    int vec, unit;
    RowsKernel paged, linear;
};

template <int DT>
RowsVariant vec_variant(int width) {
    if (width <= 64)
        return {"rows_vec_kernel", 4, 4, rows_paged_kernel<VecCore<DT, 4, true>>,
                rows_linear_kernel<VecCore<DT, 4, false>>};
    if (width <= 128)
        return {"rows_vec_kernel", 4, 4, rows_paged_kernel<VecCore<DT, 8, true>>,
                rows_linear_kernel<VecCore<DT, 8, false>>};
    return {"rows_vec_kernel", 4, 4, rows_paged_kernel<VecCore<DT, 16, true>>,
            rows_linear_kernel<VecCore<DT, 16, false>>};
}

RowsVariant pick_variant(int dt, int64_t head_dim, int64_t value_dim) {
    const int width = (int)std::max(head_dim, value_dim);
    return dt == 0 ? vec_variant<0>(width) : (dt == 1 ? vec_variant<1>(width) : vec_variant<2>(width));
}

constexpr int kRowsWorkers = 512;   // workgroups that fill the chip

// Bytes of the parts and spans: parts (16-byte aligned), (m, l), spans
int64_t rows_workspace(const RowsVariant& k, int64_t workers, int64_t items, int64_t pitch) {
    return workers * 2 * k.vec * (pitch + 2) * 4 + items * 8;
}

void place_workspace(RowsParams& p, const RowsVariant& k, void* ws) {
    p.part = static_cast<float*>(ws);
    p.spans = reinterpret_cast<int2*>(p.part + (int64_t)p.workers * 2 * k.vec * (p.pitch + 2));
}

bool join(const RowsVariant& k, int64_t items, const RowsParams& p, hipStream_t s) {
    return launch("rows_join_kernel", k.vec == 4 ? rows_join_kernel<4> : rows_join_kernel<16>,
                  dim3((unsigned)(items * k.vec)), dim3(512), 0, s, p);
}

int log2_of(int64_t x) {
    int n = 0;
    while ((int64_t(1) << n) < x) ++n;
    return n;
}

// The call's variant, workers and items; false with a reason when its sizes are
// not possible. (Pointers are checked apart.)
struct PagedPlan {
    RowsVariant k;
    int64_t tiles, items, workers, bytes;
    bool cut;   // some item may have more than one unit
};

bool paged_plan(const aero_kv_pool_t& pool, int64_t n_seq, int64_t n_q, int64_t n_head,
                int64_t max_pages, PagedPlan& pl) {
    if (!pool_ok(pool, "paged_attention")) return false;
    if (n_seq < 0 || n_q <= 0 || n_head <= 0 || n_head % pool.n_head_kv || max_pages <= 0 ||
        max_pages > (int64_t(1) << 30) / pool.page) {
        set_error("paged_attention: bad sizes (n_seq=%lld n_q=%lld n_head=%lld n_head_kv=%lld "
                  "max_pages=%lld of %lld tokens)", (long long)n_seq, (long long)n_q,
                  (long long)n_head, (long long)pool.n_head_kv, (long long)max_pages,
                  (long long)pool.page);
        return false;
    }
    pl.k = pick_variant(pool.kv_dt, pool.head_dim, pool.value_dim);
    const int64_t n_vec = n_q * (n_head / pool.n_head_kv);
    pl.tiles = (n_vec + pl.k.vec - 1) / pl.k.vec;
    if (n_q > (int64_t(1) << 24) || n_vec > (int64_t(1) << 28) || n_seq > (int64_t(1) << 24) ||
        n_seq * pool.n_head_kv > (int64_t(1) << 30) / (pl.tiles * pl.k.vec)) {
        set_error("paged_attention: %lld sequences of %lld rows are too many for one call",
                  (long long)n_seq, (long long)n_vec);
        return false;
    }
    pl.items = n_seq * pool.n_head_kv * pl.tiles;
    const int64_t units = std::max<int64_t>(1, (max_pages * pool.page / 16 + pl.k.unit - 1) /
                                                   pl.k.unit);
    pl.cut = units > 1;
    pl.workers = std::min<int64_t>(kRowsWorkers, pl.items * units);
    pl.bytes = rows_workspace(pl.k, pl.workers, pl.items, (pool.value_dim + 3) / 4 * 4);
    return true;
}

bool paged_attention_dev(const aero_kv_pool_t& pool, int64_t layer, const float* q, float* out,
                         const int32_t* table, int64_t max_pages, const int32_t* lens,
                         int64_t n_seq, int64_t n_q, int64_t n_head, float scale, int window,
                         int sinks, int32_t* bad, void* ws, int64_t ws_bytes, hipStream_t s) {
    PagedPlan pl;
    if (!paged_plan(pool, n_seq, n_q, n_head, max_pages, pl)) return false;
    if (layer < 0 || layer >= pool.n_layers || window < 0 || sinks < 0) {
        set_error("paged_attention: bad layer %lld, window %d or sinks %d", (long long)layer,
                  window, sinks);
        return false;
    }
    if (n_seq == 0) return true;
    if (q == nullptr || out == nullptr || table == nullptr || lens == nullptr || ws == nullptr ||
        ws_bytes < pl.bytes || !aligned16(ws)) {
        set_error("paged_attention: null pointer, or a workspace of %lld bytes < %lld needed "
                  "(16-byte aligned)", (long long)ws_bytes, (long long)pl.bytes);
        return false;
    }
    const PoolLayer at = pool_layer(pool, layer);
    RowsParams p{};
    p.q = q;
    p.out = out;
    p.k = at.k; p.v = at.v; p.ks = at.ks; p.vs = at.vs;
    p.table = table; p.lens = lens;
    p.bad = bad;
    p.n_seq = (int32_t)n_seq; p.n_q = (int32_t)n_q; p.n_head = (int32_t)n_head;
    p.n_head_kv = (int32_t)pool.n_head_kv; p.rep = (int32_t)(n_head / pool.n_head_kv);
    p.head_dim = (int32_t)pool.head_dim; p.value_dim = (int32_t)pool.value_dim;
    p.pitch = (int32_t)((pool.value_dim + 3) / 4 * 4);
    p.n_pages = (int32_t)pool.n_pages; p.max_pages = (int32_t)max_pages;
    p.page_shift = log2_of(pool.page);
    p.n_kv = (int32_t)(max_pages * pool.page);
    p.tiles = (int32_t)pl.tiles;
    p.window = window; p.sinks = sinks;
    p.workers = (int32_t)pl.workers;
    p.scale = scale;
    place_workspace(p, pl.k, ws);
    if (!launch(pl.k.name, pl.k.paged, dim3((unsigned)pl.workers), dim3(256), 0, s, p))
        return false;
    return !pl.cut || join(pl.k, pl.items, p, s);
}

// -------------------------------------------------- contiguous, with sinks
struct LinearPlan {
    RowsVariant k;
    int64_t tiles, n_chunks, bytes;
};

bool linear_plan(int64_t n_q, int64_t n_head, int64_t n_head_kv, int64_t head_dim,
                 int64_t value_dim, int64_t n_kv, int window, int sinks, int kv_dt,
                 LinearPlan& pl) {
    pl.k = pick_variant(kv_dt, head_dim, value_dim);
    const int64_t rep = n_head / n_head_kv;
    pl.tiles = (n_q * rep + pl.k.vec - 1) / pl.k.vec;
    // about the key tiles of an item, and enough chunks of them to fill the chip
    const int64_t keys = std::min<int64_t>(n_kv, (int64_t)window + sinks + pl.k.vec / rep + 32);
    const int64_t units = (keys + 16 * pl.k.unit - 1) / (16 * pl.k.unit);
    const int64_t base = n_head_kv * pl.tiles;
    pl.n_chunks = std::max<int64_t>(1, std::min<int64_t>(units, kRowsWorkers / base));
    pl.bytes = pl.n_chunks > 1 ? rows_workspace(pl.k, base * pl.n_chunks, base,
                                                (value_dim + 3) / 4 * 4) : 0;
    return true;
}

}  // namespace

int64_t rows_sinks_workspace(int64_t n_q, int64_t n_head, int64_t n_head_kv, int64_t head_dim,
                             int64_t value_dim, int64_t n_kv, int window, int sinks, int kv_dt) {
    LinearPlan pl;
    linear_plan(n_q, n_head, n_head_kv, head_dim, value_dim, n_kv, window, sinks, kv_dt, pl);
    return pl.bytes;
}

// (sizes and pointers checked by the caller)
bool rows_sinks_dev(const float* q, int kv_dt, const void* k, const float* k_scale, const void* v,
                    const float* v_scale, float* out, int64_t n_q, int64_t n_head,
                    int64_t n_head_kv, int64_t head_dim, int64_t value_dim, float scale,
                    const int32_t* qpos, const int32_t* kpos, int64_t n_kv, int window, int sinks,
                    void* ws, int64_t ws_bytes, hipStream_t s) {
    LinearPlan pl;
    linear_plan(n_q, n_head, n_head_kv, head_dim, value_dim, n_kv, window, sinks, kv_dt, pl);
    if (pl.bytes > 0 && (ws == nullptr || ws_bytes < pl.bytes || !aligned16(ws))) {
        set_error("attention_sinks: workspace %lld bytes < %lld needed (16-byte aligned)",
                  (long long)ws_bytes, (long long)pl.bytes);
        return false;
    }
    if (pl.tiles > 65535 || n_head_kv > 65535 || pl.n_chunks * n_head_kv * pl.tiles > INT_MAX) {
        set_error("attention_sinks: grid too large");
        return false;
    }
    RowsParams p{};
    p.q = q;
    p.out = out;
    p.k = k; p.v = v; p.ks = k_scale; p.vs = v_scale;
    p.qpos = qpos; p.kpos = kpos;
    p.n_seq = 1; p.n_q = (int32_t)n_q; p.n_head = (int32_t)n_head;
    p.n_head_kv = (int32_t)n_head_kv; p.rep = (int32_t)(n_head / n_head_kv);
    p.head_dim = (int32_t)head_dim; p.value_dim = (int32_t)value_dim;
    p.pitch = (int32_t)((value_dim + 3) / 4 * 4);
    p.page_shift = 4;
    p.n_kv = (int32_t)n_kv;
    p.tiles = (int32_t)pl.tiles;
    p.window = window; p.sinks = sinks;
    p.n_chunks = (int32_t)pl.n_chunks;
    p.workers = (int32_t)(n_head_kv * pl.tiles * pl.n_chunks);
    p.scale = scale;
    if (pl.n_chunks > 1) place_workspace(p, pl.k, ws);
    if (!launch(pl.k.name, pl.k.linear,
                dim3((unsigned)pl.n_chunks, (unsigned)n_head_kv, (unsigned)pl.tiles), dim3(256), 0,
                s, p))
        return false;
    return pl.n_chunks == 1 || join(pl.k, n_head_kv * pl.tiles, p, s);
}

}  // namespace aero

extern "C" {

int64_t aero_hip_paged_attention_workspace(const aero_kv_pool_t* pool, int64_t n_seq, int64_t n_q,
                                           int64_t n_head, int64_t max_pages) {
    aero::clear_error();
    aero::PagedPlan pl;
    if (pool == nullptr || !aero::paged_plan(*pool, n_seq, n_q, n_head, max_pages, pl)) return -1;
    return pl.bytes;
}

int aero_hip_paged_attention(const aero_kv_pool_t* pool, int64_t layer, const float* q, float* out,
                             const int32_t* table, int64_t max_pages, const int32_t* lens,
                             int64_t n_seq, int64_t n_q, int64_t n_head, float scale, int window,
                             int sinks, int32_t* bad, void* ws, int64_t ws_bytes, void* stream) {
    aero::clear_error();
    if (pool == nullptr) {
        aero::set_error("paged_attention: null pool");
        return 0;
    }
    return aero::paged_attention_dev(*pool, layer, q, out, table, max_pages, lens, n_seq, n_q,
                                     n_head, scale, window, sinks, bad, ws, ws_bytes,
                                     (hipStream_t)stream) ? 1 : 0;
}

}  // extern "C"
