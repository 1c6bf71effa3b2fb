// What the scored attention kernels share: the rule that forms a score and decides which keys a query sees
// (include/om.h, om_attention_scores), and small vector helpers.
#pragma once

#include "om_internal.hpp"

namespace osc {

typedef float floatx4 __attribute__((ext_vector_type(4)));
constexpr float kLog2e = 1.4426950408889634f;

// The rule with its sizes. Rows of a key head's queries are numbered rr = t * G + g (query t, head g of the group), so
// one row index covers a whole group and a block of rows shares its keys.
struct Rule {
    int B, Hk, G, lq, lk, d, off;  // off = lk - lq: query t stands at position t + off
    int causal, window;            // window 0: none; else below the larger of lq and lk
    float scale, cl2;              // cl2 = scale log2 e
    float icap, capl2;             // cap > 0: icap = scale / cap, capl2 = cap log2 e; else icap = 0
    const float *slopes;
    const int *qd, *kd, *prefix;
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh(u) within 2e-7 of itself: an odd polynomial up to 0.6 (its relative error by least maximum, 2.5e-9, fitted over
// u^2), (1 - t) / (1 + t) with t = 2^(-2 |u| log2 e) above.
__device__ __forceinline__ float tanh_small(float u) {
    const float z = u * u;
    float p = __builtin_fmaf(z, -0x1.7f8718p-8f, 0x1.540706p-6f);
    p = __builtin_fmaf(z, p, -0x1.b87926p-5f);
    p = __builtin_fmaf(z, p, 0x1.110872p-3f);
    p = __builtin_fmaf(z, p, -0x1.555534p-2f);
    return __builtin_fmaf(u * z, p, u);
}
constexpr float kTanhSmall = 0.6f;
__device__ __forceinline__ float tanh_any(float u) {
    const float a = __builtin_fabsf(u), t = exp2_hw(a * -2.8853900817779268f);
    const float big = __builtin_copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t), u);
    return a < kTanhSmall ? tanh_small(u) : big;
}

// A raw product's score in log2 units, before the distance bias; tanh's value for the gradient in *th (1 - th^2 is the
// score's slope in scale * raw; 0 without a cap).
__device__ __forceinline__ float score(const Rule &u, float raw, float &th) {
    if (u.icap == 0.0f) {
        th = 0.0f;
        return raw * u.cl2;
    }
    th = tanh_any(raw * u.icap);
    return th * u.capl2;
}

// Whether the query at position i sees key j (i - j = gap) with prefix keys `pre`, documents aside.
__host__ __device__ __forceinline__ bool in_reach(const Rule &u, int gap, int j, int pre) {
    if (j < pre) return true;
    if (u.causal && gap < 0) return false;
    return u.window == 0 || (gap < u.window && gap > -u.window);
}
// The rule for one query as an interval of keys and a prefix, so that a score's test is two or three integer operations
// without a branch: key j is seen when j - lo < n (unsigned) or j < pre, documents aside. Nothing for a padded query.
struct Reach {
    int lo;
    uint32_t n;
    int pre;
    __host__ __device__ __forceinline__ bool has(int j) const { return ((uint32_t)(j - lo) < n) | (j < pre); }
};
__host__ __device__ __forceinline__ Reach keys_seen(const Rule &u, int pos, int doc, int pre) {
    int lo = 0, hi = u.lk - 1;
    if (u.causal) hi = min(hi, pos);
    if (u.window) {
        lo = max(lo, pos - u.window + 1);
        hi = min(hi, pos + u.window - 1);
    }
    const bool on = doc >= 0;
    return Reach{lo, on && hi >= lo ? (uint32_t)(hi - lo + 1) : 0u, on ? min(pre, u.lk) : 0};
}
// The same for one key: the positions that see it.
__host__ __device__ __forceinline__ Reach rows_seeing(const Rule &u, int j, int doc, int pre) {
    int lo = u.off, hi = u.lk - 1;
    if (j >= pre) {
        if (u.causal) lo = max(lo, j);
        if (u.window) {
            lo = max(lo, j - u.window + 1);
            hi = min(hi, j + u.window - 1);
        }
    }
    return Reach{lo, doc >= 0 && hi >= lo ? (uint32_t)(hi - lo + 1) : 0u, INT32_MIN};
}
// The hull [lo, hi] of the keys that queries at positions i0 .. i1 can see.
__host__ __device__ __forceinline__ void key_range(const Rule &u, int i0, int i1, int pre, int &lo, int &hi) {
    lo = 0;
    hi = u.lk - 1;
    if (u.causal) hi = min(hi, i1);
    if (u.window) {
        lo = max(lo, i0 - u.window + 1);
        if (!u.causal) hi = min(hi, i1 + u.window - 1);
    }
    if (pre > 0) {
        lo = 0;
        hi = max(hi, min(pre, u.lk) - 1);
    }
}
// The hull [lo, hi] of the positions that can see one of the keys j0 .. j1.
__host__ __device__ __forceinline__ void pos_range(const Rule &u, int j0, int j1, int pre, int &lo, int &hi) {
    lo = u.off;
    hi = u.lk - 1;
    if (j0 < pre) return;
    if (u.causal) lo = max(lo, j0);
    if (u.window) {
        hi = min(hi, j1 + u.window - 1);
        if (!u.causal) lo = max(lo, j0 - u.window + 1);
    }
}
// The rows r0 .. r1 - 1 of the group that can see one of the keys j0 .. j1. A window may leave the hull before the first
// query's position, by up to lk: it is cut there before the group's size multiplies it, since lk * G may pass 32 bits.
__host__ __device__ __forceinline__ void row_range(const Rule &u, int j0, int j1, int pre, int &r0, int &r1) {
    int lo, hi;
    pos_range(u, j0, j1, pre, lo, hi);
    r0 = (lo - u.off) * u.G;
    r1 = hi < lo ? r0 : (hi - u.off + 1) * u.G;
}

// Sum over the 16 lanes of a DPP row; every lane gets the same bits (each step adds partners' equal sums).
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float row_sum(float v) {
    v += dpp<0x128>(v);  // row_ror:8
    v += dpp<0x124>(v);
    v += dpp<0x122>(v);
    v += dpp<0x121>(v);
    return v;
}

// Values c .. c + 3 of a row of d; those past d are zero. VEC: d and the rows' alignment are multiples of four floats.
template <bool VEC>
__device__ __forceinline__ floatx4 load4(const float *row, int c, int d) {
    if constexpr (VEC) {
        return c < d ? *reinterpret_cast<const floatx4 *>(row + c) : floatx4{0.f, 0.f, 0.f, 0.f};
    } else {
        floatx4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = c + e < d ? row[c + e] : 0.0f;
        return v;
    }
}

// Workgroups of `threads` that one launch takes: the runtime counts its threads in 32 bits.
constexpr int64_t most_groups(int threads) { return (int64_t)UINT32_MAX / threads; }

// Everything the kernels read and write besides the rule.
struct Ptrs {
    const float *q, *k, *v, *o, *g;
    float *out, *stats;  // forward's o and statistics (stats may be NULL)
    const float *st;     // backward's statistics
    float *dq, *dk, *dv;
    int64_t ldq, ldkv, ldo, ldg, lddq, lddkv;
    int acc;
};

// Row rr of key head hk in batch b: query t, head h.
struct Row {
    int t, h;
};
__device__ __forceinline__ Row row_of(const Rule &u, int hk, int rr) {
    const int t = rr / u.G;
    return Row{t, hk * u.G + rr - t * u.G};
}
__device__ __forceinline__ int64_t stat_at(const Rule &u, int b, const Row &r) {
    return ((int64_t)b * u.Hk * u.G + r.h) * u.lq + r.t;
}

// The forward by the matrix cores (om_attention_scored_fwd.hip), d up to 128; *joins gets the number of key splits left to
// join (1: none) and *part their sums.
om_status fwd_by_matrix(om_ctx *ctx, const Rule &u, const Ptrs &p, int *joins, float **part);
// The backward by the matrix cores (om_attention_scored_bwd.hip), d up to 128.
om_status bwd_by_matrix(om_ctx *ctx, const Rule &u, const Ptrs &p);

}  // namespace osc
