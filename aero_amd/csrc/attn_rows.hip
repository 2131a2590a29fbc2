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
// its key tiles are cut into chunks, one a workgroup.
//  * paged: workgroups find their chunk from the lengths on the device: items are
//    cut so that all chunks are about as long, and the grid has room for as many
//    as there can be, so a batch of ragged lengths is balanced and a recorded plan
//    stays right as the sequences grow.
//  * contiguous: every item has n_chunks.
// The parts of an item of several chunks are joined by rows_join_kernel.
// Page ids are checked against the pool: tiles of a bad page are not seen.
//
// What bounds it (MI355X; 8 kv heads of 128, 4 query heads each): reading the cache.
// 4 fp32 sequences of up to 50,001 tokens, 887 MB: 159 us, 5.6 TB/s (a large copy reaches
// 4.65, reads alone 6.25). 48 int8 ones of up to 8,192, 282 MB: 70 us, the walk 58 of it
// at 4.9 TB/s (5 us until the first loads are in, as long again at the end), the join 6.
// Few keys: memory round trips one after another (length, page ids, keys), about 1 us
// each, and 1 us for the four waves' sums to meet: 333 tokens 7.5 us, one launch.
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
    float* part;           // [parts][VEC] rows of pitch floats, then (m, l) of each
    int2* spans;           // [items]: the item's first part, and how many
    int32_t n_seq, n_q, n_head, n_head_kv, rep, head_dim, value_dim, pitch;
    int32_t n_pages, max_pages, page_shift;
    int32_t n_kv;          // contiguous: keys; paged: the table's room in tokens
    int32_t tiles;         // query tiles a kv head and sequence
    int32_t window, sinks;
    int32_t parts;         // room for
    int32_t target;        // paged: chunks that fill the chip (0: an item is one chunk)
    int32_t item_tokens;   // paged: tokens that an item has, at most
    int32_t n_chunks;      // contiguous
    float scale;
};

// One item and the keys of it
struct Item {
    int32_t s, kh, z;   // sequence, kv head, query tile
    int32_t len;        // keys there are
    int32_t pos0;       // paged: position of token 0
    bool early;         // paged: id is the page of the table's column threadIdx.x
    int32_t id;
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
    return reinterpret_cast<float2*>(p.part + (int64_t)p.parts * vec * p.pitch) + row;
}

// A table entry, or -1 where it is no page of the pool
__device__ __forceinline__ int32_t checked_page(const RowsParams& p, int32_t page) {
    const bool ok = page >= 0 && page < p.n_pages;
    if (!ok && p.bad != nullptr) *p.bad = 1;
    return ok ? page : -1;
}
// The page of table column col of sequence s, or -1 (none, or not of the pool)
__device__ __forceinline__ int32_t page_at(const RowsParams& p, int32_t s, int32_t col) {
    return checked_page(p, col < p.max_pages ? p.table[(int64_t)s * p.max_pages + col] : -1);
}

// ------------------------------------------------------------ any head width
// 16-lane groups own a key each (a 16-key tile a step of the workgroup), lane
// li of a group elements E li .. of the head; dot products by lane moves, four
// query vectors a workgroup. For widths and addresses that the matrix operands do not
// take: bound by its vector steps and element-wise loads. 8 sequences of up to 20,000
// tokens, 8 kv heads of 80: fp32 138 us here, 66 on the matrix cores, int8 224 / 32.
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
    static constexpr int EU = 1;
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
    __device__ __forceinline__ void reach(int64_t& lo, int64_t& hi) const {
        lo = hi = qp[0];
#pragma unroll
        for (int i = 1; i < VEC; ++i) {
            lo = min(lo, qp[i]);
            hi = max(hi, qp[i]);
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
                d = over_row(d, Add{});
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

// ---------------------------------------------------------------- matrix cores
// A 16-vector query tile on the matrix cores, as attention.hip lays it out: lane
// (g, c) = (l / 16, l % 16) holds of a 16-key tile D/4 elements of key c (the
// scores' operand) and D/16 elements of the values of keys 4g .. 4g + 3, so the
// scores a lane receives are the value sum's operand as they come. Each of the
// four waves takes every fourth step of the item's list; their sums meet in LDS.
enum Source { kPaged, kLinear, kLinearPos };
constexpr int kIds = 1024;   // page ids a workgroup holds at a time

// One kv head's tiles in memory, through buffer descriptors: lane offsets within
// a tile are fixed, the tile's place is wave-uniform, and what lies past the
// cache's end, or on a bad page, reads as zeros.
//
// PAD: vectors of fewer than D elements, K's and V's of any two widths in whole
// pieces (integers: of 8 bytes at most). Pieces past a vector's end read as zeros.
template <int DT, int D, Source SRC, bool PAD>
struct Tiles {
    static constexpr int KVEC = D * kv_bits<DT>() / 8;   // bytes of a vector (PAD: at most)
    static constexpr int KS = D / 4, VS = D / 16;        // elements a lane holds
    static constexpr int KB = KVEC / 4, VB = KVEC / 16;
    static constexpr int MOST = PAD && DT != 0 ? 8 : 16; // bytes of a piece
    static constexpr int KLB = KB < MOST ? KB : MOST, KNI = KB / KLB, KLE = KLB * 8 / kv_bits<DT>();
    static constexpr int VLB = VB < MOST ? VB : MOST, VNI = VB / VLB, VLE = VLB * 8 / kv_bits<DT>();
    static constexpr uint32_t kPast = 0x7ffffff0u;       // an offset past every end
    // head dimension of element j of lane group g's key slice, value dimension
    // of element t of lane c's value slice: pieces of the lanes interleave, so a
    // load instruction reads whole runs of a vector
    static __device__ __forceinline__ int kdim(int g, int j) {
        return (j / KLE) * (4 * KLE) + g * KLE + j % KLE;
    }
    static __device__ __forceinline__ int vdim(int c, int t) {
        return (t / VLE) * (16 * VLE) + c * VLE + t % VLE;
    }
    // a tile's place in memory (wave-uniform)
    struct Place {
        int64_t vec;     // its first vector
        int32_t kb;      // its first key
        int32_t left;    // keys there are from it on (0: no such tile, or no page)
    };
    struct K {
        uint32_t k[(KB + 3) / 4];
        float s[DT ? 4 : 1];                      // scales of keys 4g .. 4g + 3
    };
    struct V {
        int32_t kp[SRC == kLinearPos ? 4 : 1];    // positions of keys 4g .. 4g + 3
        float s[DT ? 4 : 1];
        uint32_t v[4][(VB + 3) / 4];
    };

    const RowsParams& p;
    int kh, g, c;
    uint32_t k_bytes, v_bytes;      // of a vector
    uint32_t k_stride, v_stride;    // from a key to the next
    const int32_t* ids;  // paged: in LDS, the pages of the list from place0 on
    int32_t place0;

    __device__ __forceinline__ Tiles(const RowsParams& p_, const int32_t* ids_, int kh_, int g_,
                                     int c_)
        : p(p_), kh(kh_), g(g_), c(c_), ids(ids_) {
        k_bytes = PAD ? (uint32_t)p.head_dim * kv_bits<DT>() / 8 : KVEC;
        v_bytes = PAD ? (uint32_t)p.value_dim * kv_bits<DT>() / 8 : KVEC;
        k_stride = SRC == kPaged ? k_bytes : p.n_head_kv * k_bytes;
        v_stride = SRC == kPaged ? v_bytes : p.n_head_kv * v_bytes;
    }
    // whether a vector has no piece there
    static __device__ __forceinline__ bool past(uint32_t at, uint32_t bytes) {
        return PAD && at >= bytes;
    }

    // the ids for places x .. x1 - 1 of the list into LDS (no more than
    // id_tiles() places; the workgroup's threads, between barriers)
    __device__ __forceinline__ void pages(const Item& it, int x, int x1, int32_t* to) {
        if constexpr (SRC == kPaged) {
            const int shift = p.page_shift - 4;
            place0 = it.kt.page_place(x, shift);
            const int n = it.kt.page_place(x1 - 1, shift) - place0 + 1;
            for (int i = threadIdx.x; i < n; i += 256) {
                const int32_t col = it.kt.column(place0 + i, shift);
                to[i] = it.early && col == (int32_t)threadIdx.x ? checked_page(p, it.id)
                                                                : page_at(p, it.s, col);
            }
        }
    }
    // (the sinks' and the window's first and last pages may be partly used)
    __device__ __forceinline__ int id_tiles(int all) const {
        return SRC == kPaged ? (kIds - 8) << (p.page_shift - 4) : all;
    }

    template <int N>
    static __device__ __forceinline__ void words(__amdgpu_buffer_rsrc_t r, uint32_t off,
                                                 uint32_t* w) {
        if constexpr (N == 16) {
            const v4u x = __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0);
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
        } else if constexpr (N == 8) {
            const v2u x = __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0);
            w[0] = x.x; w[1] = x.y;
        } else if constexpr (N == 4) {
            w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0);
        } else {
            static_assert(N == 2, "slice size");
            w[0] = __builtin_amdgcn_raw_buffer_load_b16(r, (int)off, 0, 0);
        }
    }
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* base, int64_t off,
                                                                  uint32_t bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(static_cast<const uint8_t*>(base)) + off, 0, (int)bytes,
            kBufferDword3);
    }

    // place x of the list (none at or past x1); x wave-uniform
    __device__ __forceinline__ Place locate(const Item& it, int x, int x1) const {
        const int tile = it.kt.at(x);
        Place l;
        l.kb = 16 * tile;
        if constexpr (SRC == kPaged) {
            const int shift = p.page_shift - 4;
            const int32_t page = x < x1 ? __builtin_amdgcn_readfirstlane(
                                              ids[it.kt.page_place(x, shift) - place0])
                                        : -1;
            l.left = page >= 0 ? 16 : 0;
            l.vec = (((int64_t)max(page, 0) * p.n_head_kv + kh) << p.page_shift) +
                    16 * (tile & ((1 << shift) - 1));
        } else {
            l.left = x < x1 ? min(it.len - l.kb, 16) : 0;
            l.vec = l.left > 0 ? (int64_t)l.kb * p.n_head_kv + kh : 0;
        }
        return l;
    }
    static __device__ __forceinline__ uint32_t reach(const Place& l, uint32_t stride,
                                                     uint32_t bytes) {
        return l.left > 0 ? (uint32_t)(l.left - 1) * stride + bytes : 0u;
    }
    // scales of keys 4g .. 4g + 3 (paged: a head's scales of a page lie together)
    __device__ __forceinline__ void load_scales(float (&o)[4], const float* s,
                                                const Place& l) const {
        if constexpr (SRC == kPaged) {
            uint32_t w[4];
            words<16>(rsrc(s, l.vec * 4, 4 * l.left), 16 * g, w);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = __uint_as_float(w[r]);
        } else {
            const __amdgpu_buffer_rsrc_t b = rsrc(
                s, l.vec * 4, l.left > 0 ? ((uint32_t)(l.left - 1) * p.n_head_kv + 1) * 4 : 0u);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                o[r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                    b, (4 * g + r) * p.n_head_kv * 4, 0, 0));
        }
    }
    __device__ __forceinline__ void load(K& t, const Place& l) const {
        const __amdgpu_buffer_rsrc_t r = rsrc(p.k, l.vec * k_bytes, reach(l, k_stride, k_bytes));
#pragma unroll
        for (int i = 0; i < KNI; ++i) {
            const uint32_t at = (4 * i + g) * KLB;
            words<KLB>(r, past(at, k_bytes) ? kPast : c * k_stride + at, t.k + i * KLB / 4);
        }
        if constexpr (DT != 0) load_scales(t.s, p.ks, l);
    }
    __device__ __forceinline__ void load(V& t, const Place& l) const {
        if constexpr (SRC == kLinearPos) {
            const __amdgpu_buffer_rsrc_t b = rsrc(p.kpos, l.left > 0 ? (int64_t)l.kb * 4 : 0,
                                                  4 * max(l.left, 0));
#pragma unroll
            for (int r = 0; r < 4; ++r)
                t.kp[r] = (int32_t)__builtin_amdgcn_raw_buffer_load_b32(b, (4 * g + r) * 4, 0, 0);
        }
        if constexpr (DT != 0) load_scales(t.s, p.vs, l);
        const __amdgpu_buffer_rsrc_t b = rsrc(p.v, l.vec * v_bytes, reach(l, v_stride, v_bytes));
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < VNI; ++i) {
                const uint32_t at = (16 * i + c) * VLB;
                words<VLB>(b, past(at, v_bytes) ? kPast : (4 * g + r) * v_stride + at,
                           t.v[r] + i * VLB / 4);
            }
    }
};

// the row of q and out of query vector i of an item's tile (a copy of the last
// one past it)
__device__ __forceinline__ int64_t query_row(const RowsParams& p, const Item& it, int i) {
    const int u = min(16 * it.z + i, p.n_q * p.rep - 1);
    return ((int64_t)it.s * p.n_q + u / p.rep) * p.n_head + it.kh * p.rep + u % p.rep;
}

// A tile's query vectors: column c's position and the keys it sees
template <Source SRC>
struct Columns {
    int rows;            // vectors there are
    int32_t qp, klo;     // kept: kp <= qp and (kp >= klo or kp < sinks)
    int32_t qmin, qmax, klo_max;
    bool mixed;          // positions differ

    __device__ __forceinline__ Columns(const RowsParams& p, const Item& it, int c) {
        const int n_vec = p.n_q * p.rep;
        rows = min(n_vec - 16 * it.z, 16);
        // (a column past the last vector is a copy of that one, never written)
        const int u = min(16 * it.z + c, n_vec - 1);
        const int t = u / p.rep;
        qp = SRC == kPaged ? it.pos0 + t : (p.qpos ? p.qpos[t] : t);
        klo = p.window > 0 ? (int32_t)max<int64_t>((int64_t)qp - p.window + 1, INT32_MIN)
                           : INT32_MIN;
        qmin = __builtin_amdgcn_readfirstlane(over_row(qp, Min{}));
        qmax = __builtin_amdgcn_readfirstlane(over_row(qp, Max{}));
        klo_max = p.window > 0 ? (int32_t)max<int64_t>((int64_t)qmax - p.window + 1, INT32_MIN)
                               : INT32_MIN;
        mixed = qmin != qmax;
    }
    // every column keeps every key of the tile at kb (left keys there are)
    __device__ __forceinline__ bool whole(const RowsParams& p, const Item& it, int32_t kb,
                                          int32_t left) const {
        return SRC != kLinearPos && left > 0 && kb + 16 <= it.len && kb + 15 <= qmin &&
               (kb >= klo_max || kb + 16 <= p.sinks);
    }
    // whether column c keeps key 4g + r of it (kp: its position)
    __device__ __forceinline__ bool keeps(const RowsParams& p, const Item& it, int32_t kb,
                                          int32_t left, int g, int r, int32_t kp) const {
        const int32_t kj = kb + 4 * g + r;
        if (SRC != kLinearPos) kp = kj;
        return left > 0 && kj < it.len && kp <= qp && (kp >= klo || kp < p.sinks);
    }
};

template <int D>
struct TileShared {
    float m[4][16], l[4][16], w[4][16], mt[16], lt[16];
    float qscale[16];
    int32_t ids[kIds];
    union {
        float acc[4][16][D + 4];
        // the queries in the order that the lanes' matrix operands have
        v4f q[D / 16][64];        // fp32: elements 4j .. 4j + 3 of lane l's slice
        h8 qh[D / 32][2][64];     // fp16 parts: elements 8j .. 8j + 7
    };
};

// The four waves' (m, l, acc) of a tile joined through LDS; its rows written out
// (row < 0) or as a part. Lane (g, c) holds acc of query 4g + r, dimension
// vdim(c, t), and (m, l) of query c, l a share.
template <typename TL, int D, bool PAD>
__device__ __forceinline__ void finish_tile(const RowsParams& p, const Item& it, int rows, float m,
                                            float ls, const v4f (&acc)[D / 16], int64_t row,
                                            TileShared<D>& sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
    ls = over_rows(ls, Add{});
    __syncthreads();     // (the item before is read)
    if (g == 0) {
        sh.m[wave][c] = m;
        sh.l[wave][c] = ls;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (4 * g + r < rows) {
#pragma unroll
            for (int t = 0; t < D / 16; ++t) sh.acc[wave][4 * g + r][TL::vdim(c, t)] = acc[t][r];
        }
    __syncthreads();
    if (tid < 64) {
        const int x = tid >> 4, i = tid & 15;
        const float mt = fmaxf(fmaxf(sh.m[0][i], sh.m[1][i]), fmaxf(sh.m[2][i], sh.m[3][i]));
        const float w = sh.m[x][i] == -INFINITY ? 0.0f : expf(sh.m[x][i] - mt);
        sh.w[x][i] = w;
        const float lw = over_rows(sh.l[x][i] * w, Add{});
        if (x == 0) {
            sh.mt[i] = mt;
            sh.lt[i] = lw;
        }
    }
    __syncthreads();
    for (int x = tid; x < rows * (D / 4); x += 256) {
        const int i = x / (D / 4), d = 4 * (x % (D / 4));
        if (PAD && d >= p.value_dim) continue;
        v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const v4f a = *reinterpret_cast<const v4f*>(&sh.acc[y][i][d]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(a[e], sh.w[y][i], o[e]);
        }
        if (row < 0) {
            const int u = 16 * it.z + i;
            const int64_t r = ((int64_t)it.s * p.n_q + u / p.rep) * p.n_head + it.kh * p.rep +
                              u % p.rep;
            const float inv = 1.0f / fmaxf(sh.lt[i], 1e-30f);
            *reinterpret_cast<v4f*>(p.out + r * (PAD ? p.value_dim : D) + d) =
                v4f{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        } else {
            *reinterpret_cast<v4f*>(part_row(p, row + i) + d) = o;
            if (d == 0) *part_ml(p, 16, row + i) = make_float2(sh.mt[i], sh.lt[i]);
        }
    }
}

// Integer caches on the fp16 matrix cores (v_mfma_f32_16x16x32_f16): the codes are
// exact in fp16; q, scaled per query to below 2^15, and the weights (probability times
// value scale) go in two fp16 parts (hi, lo = v - hi: 22 bits), so every product is
// exact and added in fp32. 32 keys a step, scores in log2 units.
//
// A query's weights and sums are in units of 2^(e - 6), e the exponent of its own
// largest weight so far: the parts' last bit, 2^-24, is 2^-29 of that one or less, and
// large values of keys that the query does not keep, or that have no weight, cost it
// nothing. The reference m is a whole number and moves up when a maximum passes it by
// 8; e goes down with it (the sums stay as they are) and up where a weight passes
// 2^(e + 9), 2^15 in these units: only then are the sums rescaled. (One exponent a wave
// from the value scales alone: 0-2% faster, and rows of zeros where a neighbour's were
// 2^32 times larger.)
//
// A step is about 340 vector and 32 matrix instructions for 8 KB of codes (dim 128):
// a third of the vector units' time at the memory's rate. So as many waves a SIMD as
// the registers allow without spilling (EU 3; 2 at dim 256), each with the next step's
// codes on their way: 96 KB a CU. 64 sequences in a window of 1,024, 4 kv heads of
// 256, 3 tokens each: 102 MB in 27 us (3.8 TB/s; 22 B/ns a CU, of the 24 of reads
// alone, but for 5 us at the start).
template <int DT, int D, Source SRC, bool PAD = false>
struct F16Core {
    static constexpr int VEC = 16;
    static constexpr int UNIT = 8;
    static constexpr int EU = D == 256 ? 2 : 3;
    using TL = Tiles<DT, D, SRC, PAD>;
    using Shared = TileShared<D>;
    static constexpr int KS = TL::KS, VS = TL::VS, NS = KS / 8;

    const RowsParams& p;
    const Item& it;
    Shared& sh;
    int g, c;
    Columns<SRC> col;
    float m = -INFINITY, ls = 0.0f;    // of query c
    int e_acc = -120;
    v4f acc[VS];
    float qsl;

    __device__ __forceinline__ F16Core(const RowsParams& p_, const Item& it_, Shared& sh_)
        : p(p_), it(it_), sh(sh_), g((threadIdx.x >> 4) & 3), c(threadIdx.x & 15),
          col(p_, it_, threadIdx.x & 15) {
#pragma unroll
        for (int t = 0; t < VS; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void reach(int64_t& lo, int64_t& hi) const {
        lo = col.qmin;
        hi = col.qmax;
    }

    // The queries' parts into LDS: 16 lanes a row, a row's 4 NS operands (step
    // st, lane group) among them, scaled by a power of two per row.
    static constexpr int QI = (4 * NS + 15) / 16;
    __device__ __forceinline__ void load_query(float (&f)[QI][8]) const {
        const int row = threadIdx.x >> 4;
        const int64_t qrow = query_row(p, it, row);
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            const int x = min(16 * i + (int)(threadIdx.x & 15), 4 * NS - 1);
            const int d = TL::kdim(x & 3, 8 * (x >> 2));
            const float* src = p.q + qrow * (PAD ? p.head_dim : D) + d;
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 v = PAD && d + e >= p.head_dim
                                     ? make_float4(0.f, 0.f, 0.f, 0.f)
                                     : *reinterpret_cast<const float4*>(src + e);
                f[i][e] = v.x; f[i][e + 1] = v.y; f[i][e + 2] = v.z; f[i][e + 3] = v.w;
            }
        }
    }
    __device__ __forceinline__ void split_query(const float (&f)[QI][8]) {
        const int row = threadIdx.x >> 4;
        float qmax = 0.0f;
#pragma unroll
        for (int i = 0; i < QI; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) qmax = fmaxf(qmax, fabsf(f[i][e]));
        qmax = over_row(qmax, Max{});
        int eq = 0;
        if (qmax > 0.0f && qmax <= 3.4028235e38f) frexpf(qmax, &eq);
        eq = max(eq, -112);     // (2^(14 - e) is finite; what is smaller keeps its bits)
        const float qsc = ldexpf(1.0f, 14 - eq);
        if ((threadIdx.x & 15) == 0) sh.qscale[row] = ldexpf(p.scale * kLog2e, eq - 14);
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            const int x = 16 * i + (threadIdx.x & 15);
            if (x >= 4 * NS) break;
            h8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                _Float16 a, b;
                split2(f[i][key_order<DT>(e)] * qsc, a, b);
                hi[e] = a;
                lo[e] = b;
            }
            sh.qh[x >> 2][0][16 * (x & 3) + row] = hi;
            sh.qh[x >> 2][1][16 * (x & 3) + row] = lo;
        }
    }

    // scores of keys 4g + r of both tiles, in log2 units
    __device__ __forceinline__ void scores(const typename TL::K& A, const typename TL::K& B,
                                           float (&sc)[8]) const {
        v4f sa = {0.f, 0.f, 0.f, 0.f}, sb = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            const h8 qhi = sh.qh[st][0][threadIdx.x & 63], qlo = sh.qh[st][1][threadIdx.x & 63];
            const h8 ka = key_codes<DT>(A.k, st), kb = key_codes<DT>(B.k, st);
            sa = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qlo, sa, 0, 0, 0);
            sb = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qlo, sb, 0, 0, 0);
            sa = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qhi, sa, 0, 0, 0);
            sb = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb, qhi, sb, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            sc[r] = sa[r] * (qsl * A.s[r]);
            sc[4 + r] = sb[r] * (qsl * B.s[r]);
        }
    }

    // the scores' probabilities times the values (la, lb: the tiles' places)
    __device__ __forceinline__ void values(float (&sc)[8], const typename TL::V& A,
                                           const typename TL::V& B, const typename TL::Place& la,
                                           const typename TL::Place& lb) {
        float vs[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            vs[r] = A.s[r];
            vs[4 + r] = B.s[r];
        }
        const bool full = col.whole(p, it, la.kb, la.left) && col.whole(p, it, lb.kb, lb.left);
        if (!full) {
            // what lies in a key that a query does not keep (a scale that is not
            // finite, say) is nothing to it
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const int r = x & 3, i = SRC == kLinearPos ? r : 0;
                const bool keep = x < 4 ? col.keeps(p, it, la.kb, la.left, g, r, A.kp[i])
                                        : col.keeps(p, it, lb.kb, lb.left, g, r, B.kp[i]);
                sc[x] = keep ? sc[x] : -INFINITY;
                vs[x] = keep ? vs[x] : 0.0f;
            }
        }
        float tm = sc[0];
#pragma unroll
        for (int x = 1; x < 8; ++x) tm = fmaxf(tm, sc[x]);
        tm = over_rows(tm, Max{});
        const bool up = __any(tm > m + 8.0f);
        const float mn = up ? fmaxf(m, ceilf(tm)) : m;
        const float msafe = mn == -INFINITY ? 0.0f : mn;
        float pr[8], psum = 0.0f, wmax = 0.0f;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            pr[x] = __builtin_amdgcn_exp2f(sc[x] - msafe);
            psum += pr[x];
            wmax = fmaxf(wmax, fabsf(pr[x] * vs[x]));
        }
        wmax = over_rows(wmax, Max{});
        // the exponent of the step's largest weight (past fp32: below 2^136)
        int ew = (int)(__builtin_bit_cast(uint32_t, wmax) >> 23) - 126;
        ew = ew > 128 ? 136 : ew;
        // (from -inf on, or past 2^-400, nothing of the sums is left)
        const float rise = mn > m ? mn - m : 0.0f;
        const int e_now = e_acc - (int)fminf(rise, 400.0f);
        const int e_new = min(max(ew > e_now + 9 ? ew : e_now, -120), 128);
        if (up) ls *= __builtin_amdgcn_exp2f(-rise);
        if (__any(e_new != e_now)) {
            const float f = ldexpf(1.0f, e_now - e_new);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float fr = __shfl(f, 4 * g + r);
#pragma unroll
                for (int t = 0; t < VS; ++t) acc[t][r] *= fr;
            }
        }
        m = mn;
        e_acc = e_new;
        // (2^(6 - e) before or after the value scale, so that no product on the way
        // leaves fp32)
        const float psc = pow2i(6 - e_acc);
        const float pa = e_acc > 0 ? psc : 1.0f, pb = e_acc > 0 ? 1.0f : psc;
        h8 phi, plo;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            _Float16 hi, lo;
            split2(pr[x] * pa * vs[x] * pb, hi, lo);
            phi[x] = hi;
            plo[x] = lo;
        }
        ls += psum;
#pragma unroll
        for (int t = 0; t < VS; ++t) {
            const h8 v = __builtin_bit_cast(
                h8, make_uint4(value_pair<DT>(A.v[0], A.v[1], t), value_pair<DT>(A.v[2], A.v[3], t),
                               value_pair<DT>(B.v[0], B.v[1], t), value_pair<DT>(B.v[2], B.v[3], t)));
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(plo, v, acc[t], 0, 0, 0);
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(phi, v, acc[t], 0, 0, 0);
        }
    }

    __device__ __forceinline__ void walk(int x0, int x1) {
        if (x0 >= x1) return;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        TL tl(p, sh.ids, it.kh, g, c);
        float f[QI][8];
        load_query(f);
        const int span = tl.id_tiles(x1 - x0);
        for (int xb = x0; xb < x1; xb += span) {
            const int xe = min(x1, xb + span);
            if (xb != x0) __syncthreads();     // (the ids before are read)
            tl.pages(it, xb, xe, sh.ids);
            if (SRC == kPaged) __syncthreads();
            typename TL::K ka, kb;
            typename TL::V va, vb;
            int x = xb + 2 * wave;
            typename TL::Place la = tl.locate(it, x, xe), lb = tl.locate(it, x + 1, xe);
            // (a wave without a tile loads nothing, but counts as many loads: what the
            // queries wait for is told from the count)
            tl.load(ka, la);
            tl.load(kb, lb);
            tl.load(va, la);
            tl.load(vb, lb);
            // (the queries' parts while the first keys and values are on their way)
            __builtin_amdgcn_sched_barrier(0);
            if (xb == x0) {
                split_query(f);
                __syncthreads();
                qsl = sh.qscale[c];
            }
            // the next step's keys are on their way during this one's softmax and
            // value sum, its values during the next scores
            while (x < xe) {
                const typename TL::Place na = tl.locate(it, x + 8, xe),
                                         nb = tl.locate(it, x + 9, xe);
                float sc[8];
                scores(ka, kb, sc);
                __builtin_amdgcn_sched_barrier(0);
                tl.load(ka, na);
                tl.load(kb, nb);
                __builtin_amdgcn_sched_barrier(0);
                values(sc, va, vb, la, lb);
                __builtin_amdgcn_sched_barrier(0);
                tl.load(va, na);
                tl.load(vb, nb);
                __builtin_amdgcn_sched_barrier(0);
                la = na;
                lb = nb;
                x += 8;
            }
        }
    }

    __device__ __forceinline__ void finish(int64_t row) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int e = __shfl(e_acc, 4 * g + r) - 6;
#pragma unroll
            for (int t = 0; t < VS; ++t) acc[t][r] = ldexpf(acc[t][r], e);
        }
        finish_tile<TL, D, PAD>(p, it, col.rows, m * kLn2, ls, acc, row, sh);
    }
};

// fp32 caches on the fp32 matrix cores (v_mfma_f32_16x16x4_f32): 16 keys a step,
// products and sums in fp32. Keys and values are matrix operands as they are loaded,
// 16 KB a step and wave at dim 128, so two waves a SIMD (one at dim 256, three at 64)
// keep enough on the way: 5.6 TB/s over long caches. One token over 2,052 keys, 4 kv
// heads of 256: 132 workgroups of a step each, 16.8 MB in 11 us and the join's 4.5:
// one round trip to memory at half of the CUs.
template <int D, Source SRC, bool PAD = false>
struct F32Core {
    static constexpr int VEC = 16;
    static constexpr int UNIT = 4;
    static constexpr int EU = D == 256 ? 1 : (D == 128 ? 2 : 3);
    using TL = Tiles<0, D, SRC, PAD>;
    using Shared = TileShared<D>;
    static constexpr int KS = TL::KS, VS = TL::VS;

    const RowsParams& p;
    const Item& it;
    Shared& sh;
    int g, c;
    Columns<SRC> col;
    float m = -INFINITY, ls = 0.0f;    // (log2 units)
    v4f acc[VS];

    __device__ __forceinline__ F32Core(const RowsParams& p_, const Item& it_, Shared& sh_)
        : p(p_), it(it_), sh(sh_), g((threadIdx.x >> 4) & 3), c(threadIdx.x & 15),
          col(p_, it_, threadIdx.x & 15) {
#pragma unroll
        for (int t = 0; t < VS; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void reach(int64_t& lo, int64_t& hi) const {
        lo = col.qmin;
        hi = col.qmax;
    }

    __device__ __forceinline__ void scores(const typename TL::K& t, float (&sc)[4]) const {
        v4f s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KS; j += 4) {
            const v4f q = sh.q[j / 4][threadIdx.x & 63];
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(t.k[j + e]), q[e], s0, 0,
                                                          0, 0);
                s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(t.k[j + e + 1]),
                                                          q[e + 1], s1, 0, 0, 0);
            }
        }
        const float c0 = p.scale * kLog2e;
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[r] = (s0[r] + s1[r]) * c0;
    }

    __device__ __forceinline__ void values(float (&sc)[4], typename TL::V& t,
                                           const typename TL::Place& l) {
        bool leak = false;
        uint64_t kept[4] = {~0ull, ~0ull, ~0ull, ~0ull};
        if (!col.whole(p, it, l.kb, l.left)) {
            // Values of keys that no query keeps become zeros; where some do and
            // some do not and a value is not finite, 0 times it would reach the
            // others: such a tile's value sum is done lane by lane.
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool keep = col.keeps(p, it, l.kb, l.left, g, r,
                                            t.kp[SRC == kLinearPos ? r : 0]);
                sc[r] = keep ? sc[r] : -INFINITY;
                kept[r] = __ballot(keep);
                const uint32_t mine = (uint32_t)(kept[r] >> (16 * g)) & 0xffffu;
#pragma unroll
                for (int e = 0; e < VS; ++e) {
                    t.v[r][e] = mine == 0 ? 0u : t.v[r][e];
                    leak = leak || (mine != 0xffffu &&
                                    !(fabsf(__uint_as_float(t.v[r][e])) <= 3.4028235e38f));
                }
            }
            leak = col.mixed && __any(leak);
        }
        float tm = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        tm = over_rows(tm, Max{});
        // the sums move when a query's maximum passes the reference by 2^8
        if (__any(tm > m + 8.0f)) {
            const float mn = fmaxf(m, tm);
            const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            ls = ls * alpha;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float ar = __shfl(alpha, 4 * g + r);
#pragma unroll
                for (int e = 0; e < VS; ++e) acc[e][r] *= ar;
            }
            m = mn;
        }
        const float msafe = m == -INFINITY ? 0.0f : m;
        float pr[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            pr[r] = __builtin_amdgcn_exp2f(sc[r] - msafe);
            ls += pr[r];
        }
        if (leak) {
            leaky_values(t, pr, kept);
            return;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < VS; ++e)
                acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(pr[r], __uint_as_float(t.v[r][e]),
                                                              acc[e], 0, 0, 0);
    }

    // acc[query 4g + r] += p v over the keys that the query keeps, by shuffles
    // (a value at a time: it is rare, and must not hold registers)
    __device__ __forceinline__ void leaky_values(const typename TL::V& t, const float (&pr)[4],
                                                 const uint64_t (&kept)[4]) {
#pragma unroll 1
        for (int gk = 0; gk < 4; ++gk)
#pragma unroll
            for (int rk = 0; rk < 4; ++rk)
#pragma unroll
                for (int e = 0; e < VS; ++e) {
                    const float v = __shfl(__uint_as_float(t.v[rk][e]), 16 * gk + c);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int q = 4 * g + r;
                        const float w = __shfl(pr[rk], 16 * gk + q);
                        const bool keep = (kept[rk] >> (16 * gk + q)) & 1;
                        acc[e][r] = keep ? __builtin_fmaf(w, v, acc[e][r]) : acc[e][r];
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
    }

    __device__ __forceinline__ void walk(int x0, int x1) {
        if (x0 >= x1) return;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        TL tl(p, sh.ids, it.kh, g, c);
        // the queries into LDS: 16 lanes a row
        constexpr int QI = D / 64;
        const int row = threadIdx.x >> 4;
        const float* src = p.q + query_row(p, it, row) * (PAD ? p.head_dim : D);
        v4f f[QI];
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            const int x = 16 * i + (threadIdx.x & 15);
            const int d = TL::kdim(x & 3, 4 * (x >> 2));
            f[i] = PAD && d >= p.head_dim ? v4f{0.f, 0.f, 0.f, 0.f}
                                          : *reinterpret_cast<const v4f*>(src + d);
        }
        const int span = tl.id_tiles(x1 - x0);
        for (int xb = x0; xb < x1; xb += span) {
            const int xe = min(x1, xb + span);
            if (xb != x0) __syncthreads();     // (the ids before are read)
            tl.pages(it, xb, xe, sh.ids);
            if (SRC == kPaged) __syncthreads();
            typename TL::K k;
            typename TL::V v;
            int x = xb + wave;
            typename TL::Place l = tl.locate(it, x, xe);
            tl.load(k, l);
            tl.load(v, l);
            __builtin_amdgcn_sched_barrier(0);
            if (xb == x0) {
#pragma unroll
                for (int i = 0; i < QI; ++i) {
                    const int x = 16 * i + (threadIdx.x & 15);
                    sh.q[x >> 2][16 * (x & 3) + row] = f[i];
                }
                __syncthreads();
            }
            while (x < xe) {
                const typename TL::Place n = tl.locate(it, x + 4, xe);
                float sc[4];
                scores(k, sc);
                __builtin_amdgcn_sched_barrier(0);
                tl.load(k, n);
                __builtin_amdgcn_sched_barrier(0);
                values(sc, v, l);
                __builtin_amdgcn_sched_barrier(0);
                tl.load(v, n);
                __builtin_amdgcn_sched_barrier(0);
                l = n;
                x += 4;
            }
        }
    }

    __device__ __forceinline__ void finish(int64_t row) {
        finish_tile<TL, D, PAD>(p, it, col.rows, m * kLn2, ls, acc, row, sh);
    }
};

// Inclusive sums over the wave's lanes, by lane moves within rows of 16 and from
// a row's last lane to the next rows
template <int CTRL, int ROWS>
__device__ __forceinline__ int32_t moved(int32_t v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int32_t wave_scan(int32_t v) {
    v += moved<0x111, 0xf>(v);    // from 1, 2, 4, 8 lanes below
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);    // lane 15 to row 1, 47 to row 3
    v += moved<0x143, 0xc>(v);    // lane 31 to rows 2 and 3
    return v;
}
__device__ __forceinline__ int64_t uniform64(int64_t v) {
    return (int64_t)(((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32)) << 32) |
                     __builtin_amdgcn_readfirstlane((uint32_t)v));
}

__device__ __forceinline__ int32_t seq_len(const RowsParams& p, int32_t s) {
    return min(max(p.lens[s], 0), p.n_kv);
}
// the keys of a sequence's last item (none has many more)
__device__ __forceinline__ KeyTiles seq_tiles(const RowsParams& p, int32_t len) {
    return key_tiles((int64_t)len - p.item_tokens, (int64_t)len - 1, len, p.window, p.sinks);
}

__device__ __forceinline__ int32_t chunks_of(const RowsParams& p, int32_t units, int32_t total) {
    return p.target == 0 ? 1 : item_chunks(units, total, p.target);
}

// Chunk b of all: its sequence (-1: there are no so many chunks) and that one's
// length, its place from the sequence's first on, the parts before that one's, and
// all items' units. Every wave finds it by itself: the units summed over the lanes,
// then the chunks of 64 sequences at a time.
struct Chunk {
    int32_t s, len, b, part, total;
};

template <int UNIT>
__device__ __forceinline__ Chunk find_chunk(const RowsParams& p, int32_t b, int32_t per_seq) {
    const int lane = threadIdx.x & 63;
    auto units = [&](int32_t len) __attribute__((always_inline)) {
        return item_units(seq_tiles(p, len).n, UNIT);
    };
    auto len_of = [&](int s) __attribute__((always_inline)) {
        return s < p.n_seq ? seq_len(p, s) : -1;
    };
    Chunk k{-1, 0, b, 0, 0};
    const int32_t len0 = len_of(lane), u0 = units(len0);
    // (the host keeps the units that the table has room for below 2^31)
    if (len0 >= 0) k.total = u0 * per_seq;
    for (int s = lane + 64; s < p.n_seq; s += 64) k.total += units(seq_len(p, s)) * per_seq;
    k.total = __builtin_amdgcn_readlane(wave_scan(k.total), 63);
    for (int s0 = 0; s0 < p.n_seq; s0 += 64) {
        const int32_t len = s0 == 0 ? len0 : len_of(s0 + lane);
        const int32_t n =
            len >= 0 ? chunks_of(p, s0 == 0 ? u0 : units(len), k.total) * per_seq : 0;
        const int32_t m = n > per_seq ? n : 0;   // (an item of one chunk has no parts)
        const int32_t upto = wave_scan(n), parts = wave_scan(m);
        const uint64_t past = __ballot(upto > k.b);
        if (past != 0) {
            const int f = __ffsll((unsigned long long)past) - 1;
            k.s = s0 + f;
            k.len = __builtin_amdgcn_readlane(len, f);
            k.b -= __builtin_amdgcn_readlane(upto - n, f);
            k.part += __builtin_amdgcn_readlane(parts - m, f);
            break;
        }
        k.b -= __builtin_amdgcn_readlane(upto, 63);
        k.part += __builtin_amdgcn_readlane(parts, 63);
    }
    return k;
}

// Paged: workgroup blockIdx.x's chunk. Where items are one chunk each, the first
// columns of its sequence's table are on their way while the length is.
template <typename Core>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Core::EU))) void
rows_paged_kernel(RowsParams p) {
    __shared__ typename Core::Shared sh;
    const int32_t per_seq = p.n_head_kv * p.tiles;
    Item it;
    it.early = p.target == 0;
    Chunk k{(int32_t)blockIdx.x / per_seq, 0, (int32_t)blockIdx.x % per_seq, 0, 0};
    if (p.target == 0) {
        it.id = p.table[(int64_t)k.s * p.max_pages +
                        min((int32_t)threadIdx.x, p.max_pages - 1)];
        k.len = seq_len(p, k.s);
    } else {
        k = find_chunk<Core::UNIT>(p, blockIdx.x, per_seq);
    }
    const int32_t s = k.s, b = k.b, part = k.part, total = k.total;
    if (s < 0) return;
    it.s = __builtin_amdgcn_readfirstlane(s);
    it.len = __builtin_amdgcn_readfirstlane(k.len);
    // (a length past the table's room is cut to it)
    if (p.bad != nullptr && threadIdx.x == 0 && p.lens[it.s] > p.n_kv) *p.bad = 1;
    it.pos0 = it.len - p.n_q;
    const int32_t chunks = chunks_of(p, item_units(seq_tiles(p, it.len).n, Core::UNIT), total);
    const int32_t item = b / chunks, c = b % chunks;
    it.kh = item / p.tiles;
    it.z = item % p.tiles;
    // the keys that the item's own tokens see, in as many chunks (some empty then)
    it.kt = key_tiles(it.pos0 + it.z * Core::VEC / p.rep,
                      it.pos0 + min(it.z * Core::VEC + Core::VEC - 1, p.n_q * p.rep - 1) / p.rep,
                      it.len, p.window, p.sinks);
    const int32_t units = item_units(it.kt.n, Core::UNIT);
    const int x1 = min(chunk_begin(c + 1, chunks, units) * Core::UNIT, it.kt.n);
    Core core(p, it, sh);
    core.walk(chunk_begin(c, chunks, units) * Core::UNIT, x1);
    core.finish(chunks == 1 ? -1 : (int64_t)(part + b) * Core::VEC);
    if (c == 0 && threadIdx.x == 0 && p.target != 0)
        p.spans[item_index(p, it)] = make_int2(part + b, chunks);
}

// Contiguous: chunk blockIdx.x of n_chunks of item (kv head blockIdx.y, query
// tile), the last query tiles (a prompt's longest) first.
template <typename Core>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Core::EU))) void
rows_linear_kernel(RowsParams p) {
    __shared__ typename Core::Shared sh;
    Item it;
    it.s = 0;
    it.kh = blockIdx.y;
    int c = blockIdx.x, z = blockIdx.z;
    if ((int)gridDim.x != p.n_chunks) {    // (more than 65535 tiles)
        z += c / p.n_chunks * (int)gridDim.z;
        c %= p.n_chunks;
    }
    if (z >= p.tiles) return;
    it.z = p.tiles - 1 - z;
    it.len = p.n_kv;
    it.pos0 = 0;
    Core core(p, it, sh);
    if (p.kpos != nullptr) {
        it.kt = KeyTiles{0, 0, (p.n_kv + 15) / 16};
    } else {
        int64_t lo, hi;
        core.reach(lo, hi);
        it.kt = key_tiles(uniform64(lo), uniform64(hi), p.n_kv, p.window, p.sinks);
    }
    const int units = item_units(it.kt.n, Core::UNIT);
    const int a = chunk_begin(c, p.n_chunks, units), b = chunk_begin(c + 1, p.n_chunks, units);
    core.walk(a * Core::UNIT, min(b * Core::UNIT, it.kt.n));
    core.finish(p.n_chunks == 1 ? -1 : (item_index(p, it) * p.n_chunks + c) * Core::VEC);
}

// The parts of an item's rows joined: `groups` groups of pitch / 4 lanes a row
// take every groups-th part, then the groups meet in LDS; 256 threads do as many
// rows as fit. B: parts that a group has in flight. Bound by its launch and one or
// two round trips (the span, the parts): 4.2-6 us from 8 to 33 parts an item. Joining
// in the kernel above instead, by an item's last workgroup, takes a counter that
// starts at zero and a fence a workgroup: faster only where items have few parts.
template <int VEC, int B>
__global__ __launch_bounds__(256) void rows_join_kernel(RowsParams p, int32_t rows, int32_t groups) {
    __shared__ float sm[256], sl[256];
    __shared__ float4 sa[256];
    const int tid = threadIdx.x;
    const int lpr = p.pitch / 4, lanes = lpr * groups, per = 256 / lanes;
    const int sub = (rows + per - 1) / per;      // workgroups an item
    const int64_t item = blockIdx.x / sub;
    // (contiguous: every item has n_chunks)
    const int2 span = p.n_chunks > 0 ? make_int2((int)(item * p.n_chunks), p.n_chunks)
                                     : p.spans[item];
    const int n = span.y;
    if (n <= 1) return;
    const int i = (int)(blockIdx.x % sub) * per + tid / lanes;
    const int d4 = tid % lpr, grp = tid % lanes / lpr;
    const int z = (int)(item % p.tiles);
    const int u = z * VEC + i;
    const bool ok = tid < per * lanes && i < rows && u < p.n_q * p.rep;
    float M = -INFINITY, L = 0.0f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
    if (ok) {
        for (int c0 = grp; c0 < n; c0 += B * groups) {
            float2 ml[B];
            float4 a[B];
#pragma unroll
            for (int x = 0; x < B; ++x) {
                const int c = min(c0 + x * groups, n - 1);
                const int64_t row = (int64_t)(span.x + c) * VEC + i;
                ml[x] = *part_ml(p, VEC, row);
                a[x] = *reinterpret_cast<const float4*>(part_row(p, row) + 4 * d4);
            }
            float mb = M;
#pragma unroll
            for (int x = 0; x < B; ++x)
                if (c0 + x * groups < n) mb = fmaxf(mb, ml[x].x);
            const float sc = M == -INFINITY ? 0.0f : expf(M - mb);
            L *= sc;
            A.x *= sc; A.y *= sc; A.z *= sc; A.w *= sc;
#pragma unroll
            for (int x = 0; x < B; ++x) {
                // (a copy of the last is no part; where all scores are NaN m is -inf too: a
                // part without keys adds zeros, that one its NaN)
                if (c0 + x * groups >= n) continue;
                const float w = ml[x].x == -INFINITY ? 0.0f : expf(ml[x].x - mb);
                L = __builtin_fmaf(ml[x].y, w, L);
                A.x = __builtin_fmaf(a[x].x, w, A.x);
                A.y = __builtin_fmaf(a[x].y, w, A.y);
                A.z = __builtin_fmaf(a[x].z, w, A.z);
                A.w = __builtin_fmaf(a[x].w, w, A.w);
            }
            M = mb;
        }
    }
    sm[tid] = M;
    sl[tid] = L;
    sa[tid] = A;
    __syncthreads();
    if (ok && grp == 0) {
        float mt = M;
        for (int k = 1; k < groups; ++k) mt = fmaxf(mt, sm[tid + k * lpr]);
        float lt = 0.0f;
        float4 at = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < groups; ++k) {
            const int x = tid + k * lpr;
            const float w = sm[x] == -INFINITY ? 0.0f : expf(sm[x] - mt);
            const float4 a = sa[x];
            lt = __builtin_fmaf(sl[x], w, lt);
            at.x = __builtin_fmaf(a.x, w, at.x);
            at.y = __builtin_fmaf(a.y, w, at.y);
            at.z = __builtin_fmaf(a.z, w, at.z);
            at.w = __builtin_fmaf(a.w, w, at.w);
        }
        const float r = 1.0f / fmaxf(lt, 1e-30f);
        const int64_t s = item / ((int64_t)p.n_head_kv * p.tiles);
        const int kh = (int)(item / p.tiles % p.n_head_kv);
        float* o = p.out + ((s * p.n_q + u / p.rep) * p.n_head + (int64_t)kh * p.rep + u % p.rep) *
                               p.value_dim + 4 * d4;
        const float v[4] = {at.x * r, at.y * r, at.z * r, at.w * r};
        for (int x = 0; x < 4; ++x)
            if (4 * d4 + x < p.value_dim) o[x] = v[x];
    }
}

// ------------------------------------------------------------------- host
using RowsKernel = void (*)(RowsParams);

// A variant of the kernels: query vectors an item, key tiles a unit, workgroups
// that fill the chip (two a CU, or one where a wave has a SIMD to itself)
struct RowsVariant {
    const char* name;
    int vec, unit, workers;
    RowsKernel paged, linear, linear_pos;
};

template <int DT, int E>
RowsVariant vec_variant() {
    return {"rows_vec_kernel", 4, 4, 512, rows_paged_kernel<VecCore<DT, E, true>>,
            rows_linear_kernel<VecCore<DT, E, false>>, rows_linear_kernel<VecCore<DT, E, false>>};
}

template <int DT>
RowsVariant vec_variant(int width) {
    return width <= 64 ? vec_variant<DT, 4>()
                       : (width <= 128 ? vec_variant<DT, 8>() : vec_variant<DT, 16>());
}

template <int DT, int D, bool PAD>
RowsVariant f16_variant() {
    return {"rows_f16_kernel", 16, 8, 256 * F16Core<DT, D, kPaged>::EU,
            rows_paged_kernel<F16Core<DT, D, kPaged, PAD>>,
            rows_linear_kernel<F16Core<DT, D, kLinear, PAD>>,
            rows_linear_kernel<F16Core<DT, D, kLinearPos, PAD>>};
}

template <int D, bool PAD>
RowsVariant f32_variant() {
    return {"rows_f32_kernel", 16, 4, 256 * F32Core<D, kPaged>::EU,
            rows_paged_kernel<F32Core<D, kPaged, PAD>>, rows_linear_kernel<F32Core<D, kLinear, PAD>>,
            rows_linear_kernel<F32Core<D, kLinearPos, PAD>>};
}

template <int D, bool PAD>
RowsVariant mfma_variant(int dt) {
    return dt == 0   ? f32_variant<D, PAD>()
           : dt == 1 ? f16_variant<1, D, PAD>()
                     : f16_variant<2, D, PAD>();
}

template <bool PAD>
RowsVariant mfma_variant(int dt, int width) {
    return width <= 64    ? mfma_variant<64, PAD>(dt)
           : width <= 128 ? mfma_variant<128, PAD>(dt)
                          : mfma_variant<256, PAD>(dt);
}

// The matrix cores take 16-byte aligned rows: of 64, 128 and 256 elements as they
// are, others in the next of these widths where both dims are whole 16-byte pieces
// (fp32) or 8-byte ones (int8: a multiple of 8, int4: of 16). The rest, the vector
// kernel.
RowsVariant pick_variant(int dt, int64_t head_dim, int64_t value_dim, bool aligned) {
    const int width = (int)std::max(head_dim, value_dim);
    const int whole = dt == 0 ? 4 : (dt == 1 ? 8 : 16);
    if (aligned && head_dim == value_dim && (width == 64 || width == 128 || width == 256))
        return mfma_variant<false>(dt, width);
    if (aligned && head_dim % whole == 0 && value_dim % whole == 0)
        return mfma_variant<true>(dt, width);
    return dt == 0 ? vec_variant<0>(width) : (dt == 1 ? vec_variant<1>(width) : vec_variant<2>(width));
}

// Items of no more keys than this (whole units) are not cut: a unit more takes a
// workgroup less than the parts and their join do. One sequence of 333 int8 tokens,
// two kv heads of dim 64: cut 11.9 us, whole 8.5. More where the items fill half of
// the chip. 64 sequences, cut / whole, us, int8 and fp32:
//   4 kv heads of 256, 3 tokens, window 1024 36.4 / 26.9, 103 / 83.0; 1984 47.6 / 43.1,
//     147 / 135; 4096 77.0 / 78.3, 246 / 250
//   8 of 128, one token, window 1024 35.5 / 26.4, 86.7 / 80.9; 1984 47.8 / 45.6, 131 /
//     135; 4096 76.9 / 83.5, 223 / 253
//   8 of 128, ragged up to 1024 27.1 / 18.7, 49.4 / 52.2; 2048 36.1 / 30.9, 80.8 / 95.7
//   4 of 256, ragged up to 1024 26.1 / 22.6, 60.3 / 61.5; 2048 32.5 / 37.6, 92.6 / 112
// So it holds for items of a length (a window's) and for most int8 batches; ragged fp32
// ones of up to 2176 tokens lose up to a fifth, the balance that cutting gives.
constexpr int kWholeKeys = 512, kWholeKeysMany = 2176;
// (a launch has fewer than 2^32 threads in a row of its grid, 256 a workgroup)
constexpr int64_t kMostWgs = (1 << 24) - 1;

// Bytes of the parts (16-byte aligned), their (m, l), and the spans
int64_t rows_workspace(const RowsVariant& k, int64_t parts, int64_t items, int64_t pitch) {
    return parts * k.vec * (pitch + 2) * 4 + items * 8;
}

void place_workspace(RowsParams& p, const RowsVariant& k, void* ws) {
    p.part = static_cast<float*>(ws);
    p.spans = reinterpret_cast<int2*>(p.part + (int64_t)p.parts * k.vec * (p.pitch + 2));
}

bool join(const RowsVariant& k, int64_t items, const RowsParams& p, hipStream_t s) {
    // a group of lanes for each part that an item has on the average, as far as a
    // row's groups fit a workgroup
    const int lpr = p.pitch / 4;
    const int rows = std::min(k.vec, p.n_q * p.rep);
    int groups = 1;
    while (groups < p.parts / items && 2 * groups * lpr <= 256) groups *= 2;
    const int per = 256 / (lpr * groups);
    const int64_t grid = items * ((rows + per - 1) / per);    // (at most 16 an item)
    // (2 or 8 parts of a group in flight, us in all: 48 sequences of up to 8,192, 8 parts
    // an item in 8 groups 69.9 / 72.6, at dim 64 21.2 / 21.8, and within 1% at dim 256.
    // One token over a ring of 2,052, dim 256, 33 parts in 4 groups 17.1 / 15.4; over
    // 8,192 keys, int8 dim 256 19.5 / 15.7, fp32 dim 64 13.8 / 11.9)
    const bool many = p.parts / items > 2 * groups;
    return launch("rows_join_kernel",
                  k.vec == 4 ? (many ? rows_join_kernel<4, 8> : rows_join_kernel<4, 2>)
                             : (many ? rows_join_kernel<16, 8> : rows_join_kernel<16, 2>),
                  dim3((unsigned)grid), dim3(256), 0, s, p, rows, groups);
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
    int64_t tiles, items, item_tokens, target, bytes;
    bool cut;   // some item may have more than one chunk
};

bool paged_plan(const aero_kv_pool_t& pool, int64_t n_seq, int64_t n_q, int64_t n_head,
                int64_t max_pages, int window, int sinks, bool aligned, PagedPlan& pl) {
    if (!pool_ok(pool, "paged_attention")) return false;
    if (n_seq < 0 || n_q <= 0 || n_head <= 0 || n_head % pool.n_head_kv || max_pages <= 0 ||
        max_pages > (int64_t(1) << 30) / pool.page) {
        set_error("paged_attention: bad sizes (n_seq=%lld n_q=%lld n_head=%lld n_head_kv=%lld "
                  "max_pages=%lld of %lld tokens)", (long long)n_seq, (long long)n_q,
                  (long long)n_head, (long long)pool.n_head_kv, (long long)max_pages,
                  (long long)pool.page);
        return false;
    }
    pl.k = pick_variant(pool.kv_dt, pool.head_dim, pool.value_dim, aligned);
    const int64_t n_vec = n_q * (n_head / pool.n_head_kv);
    pl.tiles = (n_vec + pl.k.vec - 1) / pl.k.vec;
    if (n_q > (int64_t(1) << 24) || n_vec > (int64_t(1) << 28) || n_seq > (int64_t(1) << 24) ||
        n_seq * pool.n_head_kv > (int64_t(1) << 30) / (pl.tiles * pl.k.vec)) {
        set_error("paged_attention: %lld sequences of %lld rows are too many for one call",
                  (long long)n_seq, (long long)n_vec);
        return false;
    }
    pl.items = std::max<int64_t>(n_seq * pool.n_head_kv * pl.tiles, 1);
    const int64_t units = std::max<int64_t>(1, (max_pages * pool.page / 16 + pl.k.unit - 1) /
                                                   pl.k.unit);
    if (units > INT_MAX / pl.items) {
        set_error("paged_attention: a table of %lld pages for %lld sequences has room for more "
                  "work than one call takes", (long long)max_pages, (long long)n_seq);
        return false;
    }
    const int64_t rep = n_head / pool.n_head_kv;
    pl.item_tokens = std::min<int64_t>(n_q, (pl.k.vec + rep - 1) / rep + 1);
    // (a window's keys, and what is left of the tiles at the runs' ends)
    const int64_t seen = window > 0 ? std::min<int64_t>(max_pages * pool.page,
                                                        (int64_t)window + sinks + pl.item_tokens + 45)
                                    : max_pages * pool.page;
    const int64_t fill = pl.k.workers, most = (seen + 16 * pl.k.unit - 1) / (16 * pl.k.unit);
    pl.cut = most * 16 * pl.k.unit > (2 * pl.items >= fill ? kWholeKeysMany : kWholeKeys);
    // Few items: all chunks run at once; else twice as many as fit, so that those of
    // short sequences make room early. 8 kv heads of 128, all at once / twice, us: 4
    // fp32 sequences of up to 50,001 tokens 158 / 161, 16 of 16,000 134 / 142, 32 of
    // 8,192 163 / 146, 48 322 / 205; int8, 4 of 50,001 54.5 / 58.0, 48 of 8,192 80.5 /
    // 69.7, 256 of 4,000 177 / 166 (four times as many: 172).
    const int64_t target = pl.items <= fill / 4 ? fill - pl.items : 2 * fill;
    pl.target = pl.cut ? std::min<int64_t>(target, pl.items * units) : 0;
    pl.bytes = pl.cut ? rows_workspace(pl.k, 2 * pl.target, pl.items, (pool.value_dim + 3) / 4 * 4)
                      : 0;
    if (pl.target + pl.items > kMostWgs || (pl.cut && pl.items * pl.k.vec > kMostWgs)) {
        set_error("paged_attention: %lld sequences of %lld rows are too many for one call",
                  (long long)n_seq, (long long)n_vec);
        return false;
    }
    return true;
}

bool paged_attention_dev(const aero_kv_pool_t& pool, int64_t layer, const float* q, float* out,
                         const int32_t* table, int64_t max_pages, const int32_t* lens,
                         int64_t n_seq, int64_t n_q, int64_t n_head, float scale, int window,
                         int sinks, int32_t* bad, void* ws, int64_t ws_bytes, hipStream_t s) {
    PagedPlan pl;
    if (!paged_plan(pool, n_seq, n_q, n_head, max_pages, window, sinks,
                    aligned16(q) && aligned16(out), pl))
        return false;
    if (layer < 0 || layer >= pool.n_layers || window < 0 || sinks < 0) {
        set_error("paged_attention: bad layer %lld, window %d or sinks %d", (long long)layer,
                  window, sinks);
        return false;
    }
    if (n_seq == 0) return true;
    if (q == nullptr || out == nullptr || table == nullptr || lens == nullptr ||
        (pl.bytes > 0 && (ws == nullptr || ws_bytes < pl.bytes || !aligned16(ws)))) {
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
    p.target = (int32_t)pl.target;
    p.item_tokens = (int32_t)pl.item_tokens;
    p.parts = (int32_t)(2 * pl.target);
    p.scale = scale;
    if (pl.cut) place_workspace(p, pl.k, ws);
    // (as many workgroups as there can be chunks)
    if (!launch(pl.k.name, pl.k.paged, dim3((unsigned)(pl.target + pl.items)), dim3(256), 0, s, p))
        return false;
    return !pl.cut || join(pl.k, pl.items, p, s);
}

// -------------------------------------------------- contiguous, with sinks
struct LinearPlan {
    RowsVariant k;
    int64_t tiles, n_chunks, bytes;
};

bool linear_plan(int64_t n_q, int64_t n_head, int64_t n_head_kv, int64_t head_dim,
                 int64_t value_dim, int64_t n_kv, int window, int sinks, int kv_dt, bool aligned,
                 LinearPlan& pl) {
    pl.k = pick_variant(kv_dt, head_dim, value_dim, aligned);
    const int64_t rep = n_head / n_head_kv;
    pl.tiles = (n_q * rep + pl.k.vec - 1) / pl.k.vec;
    // about the key tiles of an item, and enough chunks of them to fill the chip
    const int64_t keys = std::min<int64_t>(n_kv, (int64_t)window + sinks + pl.k.vec / rep + 32);
    const int64_t units = (keys + 16 * pl.k.unit - 1) / (16 * pl.k.unit);
    const int64_t base = n_head_kv * pl.tiles;
    pl.n_chunks = units * 16 * pl.k.unit <= kWholeKeys
                      ? 1 : std::max<int64_t>(1, std::min<int64_t>(units, pl.k.workers / base));
    pl.bytes = pl.n_chunks > 1 ? rows_workspace(pl.k, base * pl.n_chunks, base,
                                                (value_dim + 3) / 4 * 4) : 0;
    return true;
}

}  // namespace

int64_t rows_sinks_workspace(int64_t n_q, int64_t n_head, int64_t n_head_kv, int64_t head_dim,
                             int64_t value_dim, int64_t n_kv, int window, int sinks, int kv_dt) {
    LinearPlan a, b;     // (whichever the pointers' alignment will choose)
    linear_plan(n_q, n_head, n_head_kv, head_dim, value_dim, n_kv, window, sinks, kv_dt, true, a);
    linear_plan(n_q, n_head, n_head_kv, head_dim, value_dim, n_kv, window, sinks, kv_dt, false, b);
    return std::max(a.bytes, b.bytes);
}

// (sizes and pointers checked by the caller)
bool rows_sinks_dev(const float* q, int kv_dt, const void* k, const float* k_scale, const void* v,
                    const float* v_scale, float* out, int64_t n_q, int64_t n_head,
                    int64_t n_head_kv, int64_t head_dim, int64_t value_dim, float scale,
                    const int32_t* qpos, const int32_t* kpos, int64_t n_kv, int window, int sinks,
                    void* ws, int64_t ws_bytes, hipStream_t s) {
    LinearPlan pl;
    linear_plan(n_q, n_head, n_head_kv, head_dim, value_dim, n_kv, window, sinks, kv_dt,
                aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), pl);
    if (pl.bytes > 0 && (ws == nullptr || ws_bytes < pl.bytes || !aligned16(ws))) {
        set_error("attention_sinks: workspace %lld bytes < %lld needed (16-byte aligned)",
                  (long long)ws_bytes, (long long)pl.bytes);
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
    p.parts = (int32_t)(n_head_kv * pl.tiles * pl.n_chunks);
    p.scale = scale;
    if (pl.n_chunks > 1) place_workspace(p, pl.k, ws);
    if (!launch(pl.k.name, kpos == nullptr ? pl.k.linear : pl.k.linear_pos,
                dim3((unsigned)(pl.n_chunks * ((pl.tiles + 65534) / 65535)), (unsigned)n_head_kv,
                     (unsigned)std::min<int64_t>(pl.tiles, 65535)), dim3(256), 0, s, p))
        return false;
    return pl.n_chunks == 1 || join(pl.k, n_head_kv * pl.tiles, p, s);
}

}  // namespace aero

extern "C" {

int64_t aero_hip_paged_attention_workspace(const aero_kv_pool_t* pool, int64_t n_seq, int64_t n_q,
                                           int64_t n_head, int64_t max_pages) {
    aero::clear_error();
    aero::PagedPlan a, b;    // (whichever the pointers' alignment will choose)
    if (pool == nullptr ||
        !aero::paged_plan(*pool, n_seq, n_q, n_head, max_pages, 0, 0, true, a) ||
        !aero::paged_plan(*pool, n_seq, n_q, n_head, max_pages, 0, 0, false, b))
        return -1;
    return std::max(a.bytes, b.bytes);
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
