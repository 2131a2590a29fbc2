// Prompt attention with a sliding window and sinks over an fp32 KV cache, on the
// fp16 matrix cores (included by attention.hip after attn_split.hpp, whose
// transposed layout and splitting this shares).
//
// Two launches. prompt_parts_kernel splits the keys and values that the call sees
// into two fp16 parts each (hi = fp16(x), lo = fp16(x - hi)), once, scaled by a
// power of two per 32-key tile (K and V of a kv head), and lays them out as the
// matrix steps' operands, 1 KB a step: a tile's image goes to LDS as it is, by
// direct loads, and is read without bank conflicts. With a window a key meets the
// queries of several workgroups: split in each of them, as attn_split_kernel has
// it, the splitting is as long as the matrix steps.
//
// attn_prompt_kernel: a workgroup owns GQ groups of 32 query vectors of a kv head,
// GK waves a group on every GK-th tile (their sums meet at the end); all tiles of
// a step are in LDS, the next step's on their way.
//   S^T = K Q^T: lane (n, h) = (l % 32, l / 32) holds the scores of query n against
//   keys 8j + 4h + r; O^T += V^T P^T with the probabilities as they come.
// Products are hi hi + hi lo + lo hi, exact, added in fp32 by the matrix cores. The
// reference maximum m is a whole number of log2 units and moves when a query's
// maximum passes it by 1; probabilities are taken in units of 2^(12 + ev - E), ev
// the exponent of the tile's values and E that of the walk's: below 2^13 in fp16.
//
// Measured (2048 tokens, 32 heads of 128 on 8, window 512): 68 us, the splitting 12 of
// it (latency of 512 workgroups: positions, rows, the dimensions' maxima in LDS), the
// walk 2.1 us a tile of 256 query vectors; the queries' 33 MB in 5-9 us and the
// results' 2 us have nothing to overlap with: each CU has one workgroup. What bounds
// the walk is power: over long windows the matrix cores are busy 62% of the cycles and
// the clock is at 1.8 GHz, 1.17 PFLOP/s, a large fp16 product's rate. 1001 tokens, 14
// heads of 64 on 2, window 1024: 28 us, 2.1 a step of four tiles: half the matrix steps
// for the same softmax and LDS reads (41% at 2.1 GHz). So fewer instructions count (all
// three products into one accumulator, 16 sums less a tile: 128 -> 120 us in a window of
// 4096, dim 64), their order does not: the next tile's scores among this one's softmax
// were no faster.
//
// What the parts cannot carry is known before the walk, from each tile's record
// (exponents, the least of a row's, the largest value of each dimension, whether
// all is finite): a workgroup that meets it does its queries on fp32 matrix steps
// (attn_tile_fp32). The limits are attn_split_kernel's: keys and queries whose
// products pass 2^kScoreExp, dimensions of V kSpreadCh apart; and rows of V 2^14
// apart, where a query that keeps the small ones alone has 2^-23 of its result left
// (probabilities keep 2^-25 in units where 1 is 2^12).

struct PromptTile {
    float kf;          // 2^(exponent of K - 14)
    int32_t ek, ev;    // exponents: |x| < 2^e
    int32_t ev_lo;     // of the smallest row of V that is not zeros
    int32_t bad;       // a value is not finite
    int32_t pad[3];
};

struct PromptParams {
    AttnParams a;
    uint8_t* image;         // [head][cap] images of a tile's K, then V: 256 D bytes
    PromptTile* tile;       // [head][cap]
    uint32_t* channel;      // [head][cap][D]: the largest |V| of each dimension (its bits)
    KeyTiles* list;         // the call's tiles (of 32 keys)
    int32_t cap;            // tiles there is room for
};

constexpr int kRowSpread = 14;

// positions of all queries, least and greatest, in every thread of a workgroup
__device__ __forceinline__ void call_reach(const AttnParams& p, int32_t* s, int32_t& lo,
                                           int32_t& hi) {
    lo = INT32_MAX;
    hi = INT32_MIN;
    if (p.qpos == nullptr) {
        lo = 0;
        hi = (int32_t)p.n_q - 1;
        return;
    }
    // (loads of 8 at a time: one memory round trip for most prompts)
    for (int64_t t0 = threadIdx.x; t0 < p.n_q; t0 += 8 * 256) {
        int32_t q[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) q[x] = p.qpos[min(t0 + 256 * x, p.n_q - 1)];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            lo = min(lo, q[x]);
            hi = max(hi, q[x]);
        }
    }
    lo = over_rows(over_row(lo, Min{}), Min{});
    hi = over_rows(over_row(hi, Max{}), Max{});
    if ((threadIdx.x & 63) == 0) {
        s[threadIdx.x >> 6] = lo;
        s[4 + (threadIdx.x >> 6)] = hi;
    }
    __syncthreads();
    lo = min(min(s[0], s[1]), min(s[2], s[3]));
    hi = max(max(s[4], s[5]), max(s[6], s[7]));
}

// Tile blockIdx.x of the call's list, kv head blockIdx.y. Keys that no query can
// keep (by the positions' extremes) become zeros, whatever lies in them.
template <int D, bool KPOS>
__global__ __launch_bounds__(256) void prompt_parts_kernel(PromptParams pp) {
    const AttnParams& p = pp.a;
    constexpr int NS = D / 16, RC = D / 64;     // K steps; 8-element chunks a lane of 8 takes
    __shared__ int32_t s_reach[8];
    __shared__ float s_row[2][32];
    __shared__ uint32_t s_ch[D], s_bad, s_seen;
    const int tid = threadIdx.x, place = blockIdx.x, kh = blockIdx.y;
    if (tid < D) s_ch[tid] = 0;
    if (tid == 0) s_bad = 0;
    int32_t qmin, qmax;
    call_reach(p, s_reach, qmin, qmax);
    const int32_t n_kv = (int32_t)p.n_kv;
    const KeyTiles list = KPOS ? KeyTiles{0, 0, (n_kv + 31) / 32}
                               : key_tiles(qmin, qmax, n_kv, p.window, p.sinks, 32);
    if (place == 0 && kh == 0 && tid == 0) *pp.list = list;
    if (place >= list.n) return;
    const int32_t key0 = 32 * list.at(place);
    const float* kb = static_cast<const float*>(p.k) + (int64_t)kh * D;
    const float* vb = static_cast<const float*>(p.v) + (int64_t)kh * D;
    auto row_of = [&](int x) __attribute__((always_inline)) {
        return (int64_t)min(key0 + x, n_kv - 1) * p.n_head_kv * D;
    };
    // K and V by rows (row tid / 8, chunks tid % 8 + 8 i of 8 dimensions), V by
    // columns too (dimension d, the 8 keys 16 s + 8 b + 4 h + r of an operand)
    const int row = tid >> 3;
    v4f k[RC][2], v[RC][2];
#pragma unroll
    for (int i = 0; i < RC; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int d = 8 * ((tid & 7) + 8 * i) + 4 * x;
            k[i][x] = *reinterpret_cast<const v4f*>(kb + row_of(row) + d);
            v[i][x] = *reinterpret_cast<const v4f*>(vb + row_of(row) + d);
        }
    constexpr int VC = 4 * D / 256;
    float f[VC][8];
#pragma unroll
    for (int i = 0; i < VC; ++i) {
        const int x = tid + 256 * i, d = x % D, s = (x / D) >> 1, h = (x / D) & 1;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] = vb[row_of(16 * s + 8 * (e >> 2) + 4 * h + (e & 3)) + d];
    }
    auto is_seen = [&](int x, int32_t kp) __attribute__((always_inline)) {
        return key0 + x < n_kv && kp <= qmax &&
               (p.window <= 0 || (int64_t)qmin - kp < p.window || kp < p.sinks);
    };
    if (tid < 64) {     // which of the 32 keys are seen
        const int x = tid & 31;
        const uint64_t m = __ballot(is_seen(x, KPOS ? p.kpos[min(key0 + x, n_kv - 1)] : key0 + x));
        if (tid == 0) s_seen = (uint32_t)m;
    }
    __syncthreads();
    const uint32_t seen_rows = s_seen;
    const bool seen = (seen_rows >> row) & 1;
    float ak = 0.0f, av = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < RC; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                k[i][x][e] = seen ? k[i][x][e] : 0.0f;
                const float y = seen ? v[i][x][e] : 0.0f;
                bad = bad || !(fabsf(k[i][x][e]) <= 3.4028235e38f) || !(fabsf(y) <= 3.4028235e38f);
                ak = fmaxf(ak, fabsf(k[i][x][e]));
                av = fmaxf(av, fabsf(y));
            }
    ak = over_eight(ak, Max{});
    av = over_eight(av, Max{});
    if ((tid & 7) == 0) {
        s_row[0][row] = ak;
        s_row[1][row] = av;
    }
    if (bad) s_bad = 1;
    __syncthreads();
    // (32 rows in each half of a wave)
    float kmax = s_row[0][tid & 31], vmax = s_row[1][tid & 31];
    float vmin = vmax > 0.0f ? vmax : INFINITY;
    kmax = over_rows(over_row(kmax, Max{}), Max{});
    vmax = over_rows(over_row(vmax, Max{}), Max{});
    vmin = over_rows(over_row(vmin, Min{}), Min{});
    const int ek = block_exp(kmax), ev = block_exp(vmax);
    const bool finite = s_bad == 0;     // (else the image is not read)
    const float fk = finite ? pow2i(14 - ek) : 0.0f, fv = finite ? pow2i(14 - ev) : 0.0f;

    uint8_t* image = pp.image + ((int64_t)kh * pp.cap + place) * (256 * D);
    h8* ki = reinterpret_cast<h8*>(image);
#pragma unroll
    for (int i = 0; i < RC; ++i) {
        const int c = (tid & 7) + 8 * i, st = c >> 1, h = c & 1;
        h2 hi[4], lo[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
            split_pair(k[i][x >> 1][2 * (x & 1)] * fk, k[i][x >> 1][2 * (x & 1) + 1] * fk, hi[x],
                       lo[x]);
        ki[(2 * st) * 64 + row + 32 * h] = __builtin_bit_cast(
            h8, make_uint4(h2_u32(hi[0]), h2_u32(hi[1]), h2_u32(hi[2]), h2_u32(hi[3])));
        ki[(2 * st + 1) * 64 + row + 32 * h] = __builtin_bit_cast(
            h8, make_uint4(h2_u32(lo[0]), h2_u32(lo[1]), h2_u32(lo[2]), h2_u32(lo[3])));
    }
    h8* vi = ki + 2 * NS * 64;
#pragma unroll
    for (int i = 0; i < VC; ++i) {
        const int x = tid + 256 * i, d = x % D, s = (x / D) >> 1, h = (x / D) & 1;
        float m = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int r = 16 * s + 8 * (e >> 2) + 4 * h + (e & 3);
            f[i][e] = (seen_rows >> r) & 1 ? f[i][e] : 0.0f;
            m = fmaxf(m, fabsf(f[i][e]));
        }
        atomicMax(&s_ch[d], __builtin_bit_cast(uint32_t, m));
        h2 hi[4], lo[4];
#pragma unroll
        for (int y = 0; y < 4; ++y)
            split_pair(f[i][2 * y] * fv, f[i][2 * y + 1] * fv, hi[y], lo[y]);
        const int at = ((2 * (d >> 5) + s) * 2) * 64 + (d & 31) + 32 * h;
        vi[at] = __builtin_bit_cast(
            h8, make_uint4(h2_u32(hi[0]), h2_u32(hi[1]), h2_u32(hi[2]), h2_u32(hi[3])));
        vi[at + 64] = __builtin_bit_cast(
            h8, make_uint4(h2_u32(lo[0]), h2_u32(lo[1]), h2_u32(lo[2]), h2_u32(lo[3])));
    }
    __syncthreads();
    if (tid < D) pp.channel[((int64_t)kh * pp.cap + place) * D + tid] = s_ch[tid];
    if (tid == 0)
        pp.tile[(int64_t)kh * pp.cap + place] =
            PromptTile{pow2i(min(ek, 128) - 14), ek, ev,
                       vmin < INFINITY ? block_exp(vmin) : 1000, finite ? 0 : 1, {0, 0, 0}};
}

// GK waves on the same queries; TS tiles a step of a workgroup (one a wave of a
// group, or two), NB steps in LDS: the one in use and NB - 1 on their way. 32 KB a
// step: four, of the 160 KB of a CU; 64 KB: two.
template <int D, int GK>
struct PromptCfg {
    static constexpr int NW = D == 256 ? 4 : 8;       // waves
    static constexpr int IMG = 256 * D;               // bytes of a tile's image
    static constexpr int TS = D == 64 && GK == 1 ? 2 : GK;
    static constexpr int NB = TS * IMG <= 32768 ? 4 : 2;
    static constexpr int LOADS = TS * IMG / (NW * 1024) + 1;   // a wave's, a step
    // (two of the buffers also hold the sums of an fp32 tile)
    static constexpr int BUF = TS * IMG > (int)sizeof(TileSums<D>) ? TS * IMG
                                                                   : (int)sizeof(TileSums<D>);
};

// A tile's record and its keys' positions, as they are in LDS
struct PromptLds {
    PromptTile tile;
    int32_t kp[32];
};

// GK waves on the same queries, 32 NW / GK query vectors a workgroup
template <int D, int GK, bool KPOS>
__global__ __launch_bounds__((64 * PromptCfg<D, GK>::NW))
__attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2))) void attn_prompt_kernel(PromptParams pp) {
    using C = PromptCfg<D, GK>;
    const AttnParams& p = pp.a;
    constexpr int NT = D / 32, NS = D / 16, GQ = C::NW / GK, QV = 32 * GQ;
    // (objects of their own, so that reads of one need not wait for loads into another)
    __shared__ __attribute__((aligned(16))) uint8_t buf0[C::BUF], buf1[C::BUF],
        buf2[C::NB > 2 ? C::BUF : 16], buf3[C::NB > 2 ? C::BUF : 16];
    __shared__ PromptLds rec0[C::TS], rec1[C::TS], rec2[C::TS], rec3[C::TS];
    __shared__ uint32_t s_ch[D];
    __shared__ int32_t s_lo[C::NW], s_hi[C::NW], s_eq[C::NW];
    __shared__ int s_bad, s_emax, s_lomin, s_ekmax;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int qg = wave % GQ, gk = wave / GQ;
    const int n = lane & 31, h = lane >> 5;
    const int kh = blockIdx.y;
    const uint32_t n_vec = (uint32_t)p.n_q * (uint32_t)p.rep;
    const uint32_t tile = gridDim.z - 1 - blockIdx.z;     // (a prompt's longest first)
    const int n_kv = (int)p.n_kv;

    // the lane's query vector: token tq, head kh * rep + u % rep
    const uint32_t u = tile * QV + qg * 32 + n;
    const bool qok = u < n_vec;
    const uint32_t uc = qok ? u : n_vec - 1;
    const uint32_t tq = uc / (uint32_t)p.rep;
    const uint32_t qrow = tq * (uint32_t)p.n_head + (uint32_t)(kh * p.rep) + uc % (uint32_t)p.rep;
    const int32_t qp = p.qpos ? p.qpos[tq] : (int32_t)tq;
    int32_t qmin = qp, qmax = qp;
    qmin = __builtin_amdgcn_readfirstlane(over_rows(over_row(qmin, Min{}), Min{}));
    qmax = __builtin_amdgcn_readfirstlane(over_rows(over_row(qmax, Max{}), Max{}));

    // the query, on its way; then its parts, times scale * log2(e) (its product with
    // two floats): dimensions 16 st + 8 h .. + 7 of step st, scaled by a power of two
    v4f f[NS][2];
    {
        const float* src = p.q + (int64_t)qrow * D + 8 * h;
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
            for (int x = 0; x < 2; ++x)
                f[st][x] = *reinterpret_cast<const v4f*>(src + 16 * st + 4 * x);
    }
    const KeyTiles call = *pp.list;
    h8 qhi[NS], qlo[NS];
    float qsc;
    auto split_query = [&]() __attribute__((always_inline)) {
        float am = 0.0f;
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // (a NaN counts as an infinity)
                    const float y = fabsf(f[st][x][e]);
                    am = y <= am ? am : (y <= 3.4028235e38f ? y : INFINITY);
                }
        am = over_halves(am, Max{});
        const float c0 = p.scale * kLog2e;
        const float c1 = __builtin_fmaf(p.scale, kLog2e, -c0) + p.scale * kLog2eLo;
        int eq = block_exp(am * fabsf(c0) * 1.0001f);
        const float f0 = pow2i(14 - min(eq, 128));
        qsc = pow2i(min(eq, 128) - 14);
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            h2 hi[4], lo[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float a = f[st][x >> 1][2 * (x & 1)], b = f[st][x >> 1][2 * (x & 1) + 1];
                split_pair(__builtin_fmaf(a, c0, a * c1) * f0, __builtin_fmaf(b, c0, b * c1) * f0,
                           hi[x], lo[x]);
            }
            qhi[st] = __builtin_bit_cast(
                h8, make_uint4(h2_u32(hi[0]), h2_u32(hi[1]), h2_u32(hi[2]), h2_u32(hi[3])));
            qlo[st] = __builtin_bit_cast(
                h8, make_uint4(h2_u32(lo[0]), h2_u32(lo[1]), h2_u32(lo[2]), h2_u32(lo[3])));
        }
        eq = over_rows(over_row(eq, Max{}), Max{});
        if (lane == 0) s_eq[wave] = eq;
    };
    for (int d = threadIdx.x; d < D; d += 64 * C::NW) s_ch[d] = 0;
    if (lane == 0) {
        s_lo[wave] = qmin;
        s_hi[wave] = qmax;
        if (wave == 0) {
            s_bad = 0;
            s_emax = -112;
            s_lomin = 1000;
            s_ekmax = -112;
        }
    }
    __syncthreads();
    int32_t wmin = s_lo[0], wmax = s_hi[0];
#pragma unroll
    for (int x = 1; x < C::NW; ++x) {
        wmin = min(wmin, s_lo[x]);
        wmax = max(wmax, s_hi[x]);
    }
    wmin = __builtin_amdgcn_readfirstlane(wmin);
    wmax = __builtin_amdgcn_readfirstlane(wmax);

    // the workgroup's tiles, and their places among the call's
    const KeyTiles kt = KPOS ? call : key_tiles(wmin, wmax, n_kv, p.window, p.sinks, 32);
    const int64_t head0 = (int64_t)kh * pp.cap;
    const int steps = (kt.n + C::TS - 1) / C::TS;

    // step i of the walk, tiles TS i .. of the list, into b and rec (tiles past the
    // list's end are its last; past the room, noticed below, what is there)
    auto fetch = [&](int i, uint8_t* b, PromptLds* rec) __attribute__((always_inline)) {
        constexpr int W = C::IMG / (C::NW * 1024);      // KB of a tile's image a wave
#pragma unroll
        for (int sub = 0; sub < C::TS; ++sub) {
            const int x = min(C::TS * i + sub, kt.n - 1);
            const int64_t pl = head0 + min(call.place(kt.at(x)), pp.cap - 1);
            const uint8_t* src = pp.image + pl * C::IMG + wave * (W * 1024) + lane * 16;
            uint8_t* dst = b + sub * C::IMG + wave * (W * 1024);
#pragma unroll
            for (int y = 0; y < W; ++y)
                __builtin_amdgcn_global_load_lds(
                    src + y * 1024,
                    (__attribute__((address_space(3))) void*)(dst + y * 1024), 16, 0, 0);
        }
        if (lane < (KPOS ? 40 : 8)) {     // (a record a wave, some twice)
            const int x = min(C::TS * i + wave % C::TS, kt.n - 1), tl = kt.at(x);
            const int64_t pl = head0 + min(call.place(tl), pp.cap - 1);
            const int32_t* src = reinterpret_cast<const int32_t*>(pp.tile + pl) + lane;
            if (KPOS && lane >= 8) src = p.kpos + min(32 * tl + lane - 8, n_kv - 1);
            __builtin_amdgcn_global_load_lds(
                src, (__attribute__((address_space(3))) void*)(rec + wave % C::TS), 4, 0, 0);
        }
    };
    // The tiles' records: the walk's exponents, the largest value of each dimension,
    // and whether the parts carry it. (The first of each thread go out ahead of the
    // walk's loads, which they then need not wait for.)
    constexpr int G = 64 * C::NW / D, CL = 4;
    auto place = [&](int x) __attribute__((always_inline)) {
        return call.place(kt.at(max(min(x, kt.n - 1), 0)));
    };
    const int pl0 = place(threadIdx.x);
    const PromptTile r0 = pp.tile[head0 + min(max(pl0, 0), pp.cap - 1)];
    uint32_t c0[CL];
#pragma unroll
    for (int y = 0; y < CL; ++y)
        c0[y] = pp.channel[(head0 + min(max(place(threadIdx.x / D + G * y), 0), pp.cap - 1)) * D +
                           threadIdx.x % D];
    __builtin_amdgcn_sched_barrier(0);
    if (steps > 0) fetch(0, buf0, rec0);
    if constexpr (C::NB > 2) {
        if (steps > 1) fetch(1, buf1, rec1);
        if (steps > 2) fetch(2, buf2, rec2);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (kt.n > 0) {
        int em = r0.ev, lo = r0.ev_lo, ekm = r0.ek;
        bool bad = r0.bad != 0 || pl0 >= pp.cap;
        for (int x = threadIdx.x + 64 * C::NW; x < kt.n; x += 64 * C::NW) {
            const int pl = place(x);
            const PromptTile r = pp.tile[head0 + min(pl, pp.cap - 1)];
            em = max(em, r.ev);
            lo = min(lo, r.ev_lo);
            ekm = max(ekm, r.ek);
            bad = bad || r.bad != 0 || pl >= pp.cap;
        }
        uint32_t c = max(max(c0[0], c0[1]), max(c0[2], c0[3]));
#pragma unroll 4
        for (int x = threadIdx.x / D + G * CL; x < kt.n; x += G)
            c = max(c, pp.channel[(head0 + min(place(x), pp.cap - 1)) * D + threadIdx.x % D]);
        atomicMax(&s_ch[threadIdx.x % D], c);
        em = over_rows(over_row(em, Max{}), Max{});
        lo = over_rows(over_row(lo, Min{}), Min{});
        ekm = over_rows(over_row(ekm, Max{}), Max{});
        if (lane == 0) {
            atomicMax(&s_emax, em);
            atomicMin(&s_lomin, lo);
            atomicMax(&s_ekmax, ekm);
        }
        if (bad) s_bad = 1;
    }
    split_query();
    __syncthreads();
    const int E = __builtin_amdgcn_readfirstlane(s_emax);
    int wq = s_eq[0];
#pragma unroll
    for (int x = 1; x < C::NW; ++x) wq = max(wq, s_eq[x]);
    bool redo = s_bad != 0 || E > 128 || E - s_lomin > kRowSpread || wq > 128 ||
                s_ekmax + wq > kScoreExp;
    // (a dimension of V far below the others; one of zeros is exact)
#pragma unroll
    for (int d = lane; d < D; d += 64) {
        const uint32_t c = s_ch[d];
        redo = redo || (c != 0 && E - block_exp(__builtin_bit_cast(float, c)) > kSpreadCh);
    }
    redo = __any(redo);
    if (redo) {
        constexpr int PAIR = C::NW / 4;       // four waves a 16-query tile
        TileSums<D>* mine = reinterpret_cast<TileSums<D>*>(wave < 4 ? buf0 : buf1);
        __builtin_amdgcn_s_waitcnt(0x0f70);   // (the buffers are still being filled)
#pragma unroll 1
        for (int x = wave / 4; x < QV / 16; x += PAIR) {
            __syncthreads();
            attn_tile_fp32<D, true>(p, (int64_t)tile * (QV / 16) + x, kh, *mine);
        }
        return;
    }

    // the positions the lane's query keeps: klo .. qp, and those below the sinks
    const int32_t klo = p.window > 0 ? (int32_t)max<int64_t>((int64_t)qp - p.window + 1, INT32_MIN)
                                     : INT32_MIN;
    const int32_t klo_max =
        p.window > 0 ? (int32_t)max<int64_t>((int64_t)qmax - p.window + 1, INT32_MIN) : INT32_MIN;

    const int32_t klo_min =
        p.window > 0 ? (int32_t)max<int64_t>((int64_t)qmin - p.window + 1, INT32_MIN) : INT32_MIN;

    int m = kNoMax;
    float ls = 0.0f;
    v16f acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 16; ++x) acc[t][x] = 0.0f;

    auto compute = [&](int i, const uint8_t* b, const PromptLds* recs) __attribute__((always_inline)) {
#pragma unroll 1
        for (int sub = gk; sub < C::TS; sub += GK) {
            const int x = C::TS * i + sub;
            if (x >= kt.n) break;
            const int kb = 32 * kt.at(x);
            // (nothing of it for the wave's queries)
            if (!KPOS && (kb > qmax || (kb + 31 < klo_min && kb >= p.sinks))) continue;
            const h8* ki = reinterpret_cast<const h8*>(b + sub * C::IMG) + lane;
            const h8* vi = ki + 2 * NS * 64;
            // operands are read two steps ahead
            h8 ah[3], al[3];
            auto key_parts = [&](int st) __attribute__((always_inline)) {
                ah[st % 3] = ki[2 * st * 64];
                al[st % 3] = ki[(2 * st + 1) * 64];
            };
            auto value_parts = [&](int y) __attribute__((always_inline)) {   // y = 2 t + k
                ah[y % 3] = vi[2 * y * 64];
                al[y % 3] = vi[(2 * y + 1) * 64];
            };
            key_parts(0);
            key_parts(1);
            const float kf = recs[sub].tile.kf;
            const int ev = __builtin_amdgcn_readfirstlane(recs[sub].tile.ev);
            v16f s;
#pragma unroll
            for (int y = 0; y < 16; ++y) s[y] = 0.0f;
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                if (st + 2 < NS) key_parts(st + 2);
                __builtin_amdgcn_sched_barrier(0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[st % 3], qhi[st], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[st % 3], qlo[st], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[st % 3], qhi[st], s, 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
            value_parts(0);
            value_parts(1);
            __builtin_amdgcn_sched_barrier(0);
            // (at least the smallest normal: -inf times c stays -inf)
            const float c = fmaxf(kf * qsc, 1.17549435e-38f);
            if (KPOS || kb + 31 > min(qmin, n_kv - 1) ||
                (kb < klo_max && kb + 32 > p.sinks)) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int key = kb + 8 * j + 4 * h + r;
                        const int32_t kp = KPOS ? recs[sub].kp[8 * j + 4 * h + r] : key;
                        const bool keep = key < n_kv && kp <= qp && (kp >= klo || kp < p.sinks);
                        s[4 * j + r] = keep ? s[4 * j + r] : -INFINITY;
                    }
            }
            float tm = max3(s[0], s[1], s[2]);
#pragma unroll
            for (int y = 3; y < 15; y += 2) tm = max3(tm, s[y], s[y + 1]);
            tm = fmaxf(tm, s[15]);
            tm = over_halves(tm, Max{}) * c;
            const int mt = tm > -INFINITY ? (int)ceilf(fminf(fmaxf(tm, -1e8f), 1e8f)) : kNoMax;
            if (__any(mt > m + 1)) {
                const int mn = max(m, mt);
                const float alpha = m - mn < -126 ? 0.0f : pow2i(m - mn);
                ls *= alpha;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int y = 0; y < 16; ++y) acc[t][y] *= alpha;
                m = mn;
            }
            // (a tile of zeros: its keys count in the sum)
            const int fe = max(ev - E, -kRowSpread) + 12;
            const float off = (float)fe - (m == kNoMax ? 0.0f : (float)m);
            h8 phi[2], plo[2];
            float sum[4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                h2 hi[4], lo[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * k + 2 * y], c, off));
                    const float p1 =
                        __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * k + 2 * y + 1], c, off));
                    sum[y] = k == 0 ? p0 + p1 : sum[y] + (p0 + p1);
                    split_pair(p0, p1, hi[y], lo[y]);
                }
                phi[k] = __builtin_bit_cast(h8, make_uint4(h2_u32(hi[0]), h2_u32(hi[1]),
                                                           h2_u32(hi[2]), h2_u32(hi[3])));
                plo[k] = __builtin_bit_cast(h8, make_uint4(h2_u32(lo[0]), h2_u32(lo[1]),
                                                           h2_u32(lo[2]), h2_u32(lo[3])));
            }
            ls += ((sum[0] + sum[1]) + (sum[2] + sum[3])) * pow2i(-fe);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int y = 0; y < 2 * NT; ++y) {
                const int t = y >> 1, k = y & 1;
                if (y + 2 < 2 * NT) value_parts(y + 2);
                __builtin_amdgcn_sched_barrier(0);
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[y % 3], phi[k], acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[y % 3], plo[k], acc[t], 0, 0, 0);
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[y % 3], phi[k], acc[t], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
        }
    };
    // A step begins when its loads have landed (those of the NB - 2 steps after it
    // may be on their way) and every wave is done with the step before, whose
    // buffer is then filled again.
    // (the copies of this code are marked apart: merged, they would read a buffer that
    // the compiler cannot tell from the one being filled, and wait for the loads)
    auto step = [&](auto k, int i, const uint8_t* b, const PromptLds* recs, uint8_t* nb,
                    PromptLds* nrec) __attribute__((always_inline)) {
        constexpr int N = (C::NB - 2) * C::LOADS;
        if (i + C::NB - 2 < steps)
            __builtin_amdgcn_s_waitcnt((N & 15) | 0x0f70 | ((N >> 4) << 14));
        else
            __builtin_amdgcn_s_waitcnt(0x0f70);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (i + C::NB - 1 < steps) fetch(i + C::NB - 1, nb, nrec);
        asm volatile("; buffer %0" ::"n"(decltype(k)::value) : "memory");
        compute(i, b, recs);
        asm volatile("; buffer %0 done" ::"n"(decltype(k)::value) : "memory");
    };
    using K0 = std::integral_constant<int, 0>;
    using K1 = std::integral_constant<int, 1>;
    using K2 = std::integral_constant<int, 2>;
    using K3 = std::integral_constant<int, 3>;
    for (int i = 0; i < steps; i += C::NB) {
        if constexpr (C::NB > 2) {
            step(K0{}, i, buf0, rec0, buf3, rec3);
            if (i + 1 >= steps) break;
            step(K1{}, i + 1, buf1, rec1, buf0, rec0);
            if (i + 2 >= steps) break;
            step(K2{}, i + 2, buf2, rec2, buf1, rec1);
            if (i + 3 >= steps) break;
            step(K3{}, i + 3, buf3, rec3, buf2, rec2);
        } else {
            step(K0{}, i, buf0, rec0, buf1, rec1);
            if (i + 1 >= steps) break;
            step(K1{}, i + 1, buf1, rec1, buf0, rec0);
        }
    }

    // the halves of a column added; the groups' sums joined
    ls = over_halves(ls, Add{});
    if constexpr (GK > 1) {
        constexpr int ROW = 64 * (16 * NT + 2);       // floats of a wave's sums
        constexpr int HALF = sizeof(buf0) / (4 * ROW);
        static_assert((GK - 1) * GQ <= 2 * HALF, "merge buffer");
        __syncthreads();
        auto at = [&](int w) __attribute__((always_inline)) {
            return reinterpret_cast<float*>(w < HALF ? buf0 : buf1) + (w < HALF ? w : w - HALF) * ROW +
                   lane;
        };
        if (gk > 0) {
            float* xs = at((gk - 1) * GQ + qg);
            xs[0] = (float)m;
            xs[64] = ls;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int y = 0; y < 16; ++y) xs[64 * (2 + 16 * t + y)] = acc[t][y];
        }
        __syncthreads();
        if (gk > 0) return;
#pragma unroll 1
        for (int o = 1; o < GK; ++o) {
            const float* xs = at((o - 1) * GQ + qg);
            const float m0 = (float)m, m1 = xs[0];
            const float mt = fmaxf(m0, m1);
            const float w0 = __builtin_amdgcn_exp2f(m0 - mt), w1 = __builtin_amdgcn_exp2f(m1 - mt);
            ls = ls * w0 + xs[64] * w1;
            m = max(m, (int)m1);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int y = 0; y < 16; ++y)
                    acc[t][y] = acc[t][y] * w0 + xs[64 * (2 + 16 * t + y)] * w1;
        }
    }
    if (qok) {
        const float inv = 1.0f / fmaxf(ls, 1e-30f);
        float* o = p.out + (int64_t)qrow * D + 4 * h;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v4f r;
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = ldexpf(acc[t][4 * j + e] * inv, E - 26);
                *reinterpret_cast<v4f*>(o + 32 * t + 8 * j) = r;
            }
    }
}
