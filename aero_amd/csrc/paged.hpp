// A paged KV pool as the translation units see it: checks, and one layer of it.
#pragma once

#include "common.hpp"
#include "aero_hip.h"

namespace aero {

// sizes, pointers and alignment; false with a reason (what: the operator's name)
bool pool_ok(const aero_kv_pool_t& p, const char* what);

// bytes of one (token, head) vector of dim elements
inline int64_t kv_vec_bytes(int dt, int64_t dim) {
    return dt == 0 ? 4 * dim : (dt == 1 ? dim : dim / 2);
}

struct PoolLayer {
    uint8_t* k;
    uint8_t* v;
    float* ks;
    float* vs;
};

inline PoolLayer pool_layer(const aero_kv_pool_t& p, int64_t layer) {
    const int64_t vecs = layer * p.n_pages * p.n_head_kv * p.page;   // (up to 64 bits)
    PoolLayer l;
    l.k = static_cast<uint8_t*>(p.k) + vecs * kv_vec_bytes(p.kv_dt, p.head_dim);
    l.v = static_cast<uint8_t*>(p.v) + vecs * kv_vec_bytes(p.kv_dt, p.value_dim);
    l.ks = p.kv_dt == 0 ? nullptr : p.k_scale + vecs;
    l.vs = p.kv_dt == 0 ? nullptr : p.v_scale + vecs;
    return l;
}

}  // namespace aero
