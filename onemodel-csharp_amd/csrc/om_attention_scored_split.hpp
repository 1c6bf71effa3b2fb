// The pass that splits operands for the scored attention's matrix kernels (om_attention_scored_mm.hpp): one workgroup per
// block of 64 rows of a head, four rows x four values a thread. Bound: HBM, 4 bytes read and 4 or 8 written per value (16 heads
// of 128 values over 8192 rows, 4 key heads: 550 MB in 99 to 107 us, 5.1 to 5.6 TB/s), in small calls a workgroup's chain of
// barriers (32 x 12 heads of 128 x 32: 19 us, 2 of them for the columns' largest values).
#pragma once

#include "om_attention_scored_mm.hpp"

namespace osc {

struct SplitOut {
    char *rows, *cols;  // either may be NULL
    Stats *stats;
    float *keys;  // the steps' words (kKeyWords for each 32 keys); K writes the documents too
    bool is_v;
};

// This thread's share of a block: values 64 n + 4 (tid % 16) .. + 3 of rows 4 (tid / 16) + i.
template <int DP>
struct Share {
    static constexpr int NCH = (DP + 63) / 64;
    floatx4 x[4][NCH];
    template <bool VEC>
    __device__ __forceinline__ void load(int i, const float *row, int d) {
#pragma unroll
        for (int n = 0; n < NCH; n++) {
            const int c = 64 * n + 4 * (threadIdx.x & 15);
            x[i][n] = c < DP ? load4<VEC>(row, c, d) : floatx4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // Zeros in place of a row that does not count, whatever it holds: once it is here, so that the loads wait for nothing.
    __device__ __forceinline__ void keep(int i, bool on) {
#pragma unroll
        for (int n = 0; n < NCH; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[i][n][e] = on ? x[i][n][e] : 0.0f;
    }
    // Largest magnitude of row i as bits (infinities and NaN above every finite one), the same in the row's 16 lanes.
    __device__ __forceinline__ uint32_t row_top(int i) const {
        uint32_t t = 0;
#pragma unroll
        for (int n = 0; n < NCH; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) t = max(t, __float_as_uint(x[i][n][e]) & 0x7FFFFFFFu);
        auto step = [&](auto ctrl) {
            t = max(t, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)t, decltype(ctrl)::value, 0xf, 0xf, true));
        };
        step(std::integral_constant<int, 0x128>());
        step(std::integral_constant<int, 0x124>());
        step(std::integral_constant<int, 0x122>());
        step(std::integral_constant<int, 0x121>());
        return t;
    }
    // Sum of row i's squares, the same in the row's 16 lanes.
    __device__ __forceinline__ float row_norm(int i) const {
        float s = 0.0f;
#pragma unroll
        for (int n = 0; n < NCH; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) s = __builtin_fmaf(x[i][n][e], x[i][n][e], s);
        return row_sum(s);
    }
    __device__ __forceinline__ void scale(int i, float w) {
#pragma unroll
        for (int n = 0; n < NCH; n++) x[i][n] *= w;
    }
};

// Largest of a value over the wavefront's four rows of 16 lanes, whose lanes hold the same.
__device__ __forceinline__ uint32_t rows_umax(uint32_t v) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(p[0], p[1]);
    const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(q[0], q[1]);
}
// Sum of a count over the same.
__device__ __forceinline__ uint32_t rows_usum(uint32_t v) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = p[0] + p[1];
    const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return q[0] + q[1];
}
// What a block of 64 rows holds: the largest magnitude (bits), the smallest nonzero row and column maximum, its rows that are
// not zero, and the largest of the threads' `norm`.
struct BlockTop {
    uint32_t top, low, column, rows;
    float norm;
};
// Of a block with these row maxima; every thread gets it. COLUMNS: columns too (else they count as even), from the staging
// buffer `lds` (16 bytes a column). Uses 16 words of `sh`.
template <int DP, bool COLUMNS>
__device__ __forceinline__ BlockTop block_top(const Share<DP> &s, const uint32_t (&row)[4], float norm, uint32_t *sh, char *lds) {
    constexpr int NCH = Share<DP>::NCH;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t t = 0, l = 0xFFFFFFFFu, live = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        t = max(t, row[i]);
        l = row[i] ? min(l, row[i]) : l;
        live += row[i] ? 1 : 0;
    }
    t = rows_umax(t);
    l = ~rows_umax(~l);
    const uint32_t n = rows_umax(__float_as_uint(norm));  // as bits: a NaN is above all
    live = rows_usum(live);
    u32x4 c[NCH];
    if constexpr (COLUMNS) {
#pragma unroll
        for (int k = 0; k < NCH; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(s.x[i][k][e]) & 0x7FFFFFFFu);
                c[k][e] = rows_umax(m);
            }
    }
    __syncthreads();
    if (lane == 0) {
        sh[w] = t;
        sh[4 + w] = l;
        sh[8 + w] = n;
        sh[12 + w] = live;
    }
    uint32_t *columns = reinterpret_cast<uint32_t *>(lds);
    if constexpr (COLUMNS) {
#pragma unroll
        for (int k = 0; k < NCH; k++)
            if (lane < 16 && 64 * k + 4 * lane < DP) *reinterpret_cast<u32x4 *>(columns + w * DP + 64 * k + 4 * lane) = c[k];
    }
    __syncthreads();
    BlockTop r = {sh[0], sh[4], 0xFFFFFFFFu, sh[12], 0.0f};
    uint32_t most = sh[8];
#pragma unroll
    for (int i = 1; i < 4; i++) {
        r.top = max(r.top, sh[i]);
        r.low = min(r.low, sh[4 + i]);
        most = max(most, sh[8 + i]);
        r.rows += sh[12 + i];
    }
    r.norm = __uint_as_float(most);
    if constexpr (COLUMNS) {
#pragma unroll
        for (int k = 0; k < NCH; k++) {
            const int at = min(64 * k + lane, DP - 1);
            const uint32_t m = max(max(columns[at], columns[DP + at]), max(columns[2 * DP + at], columns[3 * DP + at]));
            r.column = min(r.column, m ? m : 0xFFFFFFFFu);
        }
        r.column = wave_umin(r.column);
    }
    return r;
}
// Whether every column that is not zero keeps its bits: its largest value within 2^14 of the block's, so held to 2^-22 of
// itself. In a single row, as a last block may hold, each column is one value, and of a normal's one in 8000 is 2^14 below the
// largest, one in 2 million 2^22: there 2^22 is asked for, or every few calls would have a head that sums plainly for nothing.
__device__ __forceinline__ bool even_columns(const BlockTop &b) {
    return b.top == 0 || (b.top >> 23) - (b.column >> 23) <= (b.rows > 1 ? 14 : 22);
}
__device__ __forceinline__ float larger(float a, float b) {  // of sums of squares; a NaN is the largest
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}

// Writes the block's two planes in rows or columns form: through LDS (DP * 256 bytes), so that memory gets whole lines.
template <int DP, bool COLS>
__device__ __forceinline__ void put_block(const Share<DP> &s, char *out, char *lds) {
    constexpr int NCH = Share<DP>::NCH;
    const int rq = threadIdx.x >> 4;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NCH; n++) {
        const int c = 64 * n + 4 * (threadIdx.x & 15);
        if (c >= DP) continue;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t h0, m0, h1, m1;
            char *to;
            if constexpr (COLS) {  // four rows of value c + i
                split2(s.x[0][n][i], s.x[1][n][i], h0, m0);
                split2(s.x[2][n][i], s.x[3][n][i], h1, m1);
                const int v = c + i;
                to = lds + (((rq >> 2) * (DP / 32) + (v >> 5)) * 2) * 1024 + ((rq & 1) * 32 + (v & 31)) * 16 + ((rq >> 1) & 1) * 8;
            } else {  // four values of row 4 rq + i
                split2(s.x[i][n][0], s.x[i][n][1], h0, m0);
                split2(s.x[i][n][2], s.x[i][n][3], h1, m1);
                const int row = 4 * rq + i;
                to = lds + (((row >> 5) * (DP / 16) + (c >> 4)) * 2) * 1024 + (((c >> 3) & 1) * 32 + (row & 31)) * 16 + ((c >> 2) & 1) * 8;
            }
            *reinterpret_cast<u32x2 *>(to) = u32x2{h0, h1};
            *reinterpret_cast<u32x2 *>(to + 1024) = u32x2{m0, m1};
        }
    }
    __syncthreads();
    for (int f = threadIdx.x; f < DP * 16; f += 256)
        *reinterpret_cast<u32x4 *>(out + 16 * f) = *reinterpret_cast<const u32x4 *>(lds + 16 * f);
}

// Block t of the keys of (b, hk): K or V (src) scaled by one power of two, in the forms asked for. Keys of padding
// documents become zeros, so that nothing they hold reaches a product.
template <int DP, bool VEC>
__device__ __forceinline__ void split_keys(const Rule &u, const float *src, int64_t ld, int b, int hk, int t, int64_t at,
                                           const SplitOut &o, char *lds, uint32_t *sh) {
    Share<DP> s;
    uint32_t top4[4];
    float norm = 0.0f;
    int dlo = INT32_MAX, dhi = -1, doc[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int j = t * kBlock + 4 * (threadIdx.x >> 4) + i;
        const int64_t tok = (int64_t)b * u.lk + min(j, u.lk - 1);
        doc[i] = u.kd ? u.kd[tok] : 0;
        s.template load<VEC>(i, src + tok * ld + (int64_t)hk * u.d, u.d);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const bool there = t * kBlock + 4 * (int)(threadIdx.x >> 4) + i < u.lk;
        s.keep(i, there && doc[i] >= 0);
        top4[i] = s.row_top(i);
        if (!o.is_v) norm = larger(norm, s.row_norm(i));
        dhi = max(dhi, there ? doc[i] : -1);
        dlo = min(dlo, there ? doc[i] : INT32_MAX);
    }
    const BlockTop bt = block_top<DP, true>(s, top4, norm, sh, lds);
    // V's columns are a product's rows or columns either way, K's only in dq: a score bounded by kMostScore loses nothing
    const bool even = even_columns(bt), ok = in_range(bt.top) && even_rows(bt.top, bt.low) && (even || !o.is_v);
    const int e = ok && bt.top ? scale_exp(bt.top) : 0;
    const float w = pow2(-e);
#pragma unroll
    for (int i = 0; i < 4; i++) s.scale(i, w);
    if (o.rows) put_block<DP, false>(s, o.rows + at * plane_bytes(DP, 1), lds);
    if (o.cols) put_block<DP, true>(s, o.cols + at * plane_bytes(DP, 1), lds);
    // the block's document range
    __syncthreads();
    if ((threadIdx.x & 15) == 0) {
        sh[threadIdx.x >> 4] = (uint32_t)dlo;
        sh[16 + (threadIdx.x >> 4)] = (uint32_t)dhi;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 0; i < 16; i++) {
            dlo = min(dlo, (int)sh[i]);
            dhi = max(dhi, (int)sh[16 + i]);
        }
        Stats st = {};
        st.top = ok ? bt.top : 0xFFFFFFFFu;
        st.low = bt.low;
        st.columns = ok && even;
        st.scale = pow2(e);
        st.doc_lo = dlo;
        st.doc_hi = dhi;
        st.norm = bt.norm;
        o.stats[at] = st;
    }
    __syncthreads();
    // the words of the block's two steps
    if (threadIdx.x < 2 * kKeyWords) {
        const int half = threadIdx.x / kKeyWords, n = threadIdx.x % kKeyWords;
        float *to = o.keys + (2 * at + half) * kKeyWords;
        if (o.is_v) {
            if (n == kKeyScaleV) to[n] = pow2(e);
        } else if (n < 32) {
            const int j = t * kBlock + 32 * half + n;
            to[n] = __int_as_float(j >= u.lk ? -1 : u.kd ? u.kd[(int64_t)b * u.lk + j] : 0);
        } else if (n == kKeyScaleK) {
            to[n] = pow2(e);
        } else if (n == kKeyDocLo || n == kKeyDocHi) {
            for (int i = 0; i < 16; i++) {
                dlo = min(dlo, (int)sh[i]);
                dhi = max(dhi, (int)sh[16 + i]);
            }
            to[n] = __int_as_float(n == kKeyDocLo ? dlo : dhi);
        }
    }
}

// What the backward keeps of its rows (queries of one head): a record of 1 KB per 32 rows, a value of all 32 after another.
enum {
    kRowM,      // kLift less the forward's reference exponent; -kNoRow for a row that has nothing to give (its weights become 0)
    kRowDelta,  // g . o times 2^-re, re the exponent of g's row scale
    kRowPos,    // position (int)
    kRowSlope,  // slope of its head, in log2 units
    kRowDoc,    // document (int)
    kRowW,      // 2^re / l: what dq's sums are multiplied with at the end; 0 for a row without gradient
    kRowBlock,  // of the rows' block of 64: its scales of q and q f, its documents' range
    kRowGrad,   // 2^ge, ge the exponent of the row's g / l: what its weights are multiplied with for dk and dv; 0 without gradient
    kRowValues = 8
};
__host__ __device__ __forceinline__ int64_t row_value(int64_t row, int which) { return (row >> 5) * (32 * kRowValues) + which * 32 + (row & 31); }
// A block of 64 rows. Either role needs the rows' values and the rows form; only dk and dv the columns form, where q's rows and
// the columns have to be near each other. g's rows need not: each is scaled by itself there too. (At one scale a block, one row
// in ten peaked and gradients spread as exp of a normal sent most calls to plain sums: 30 ms for both directions of 12 heads of 64
// over 4096 causal rows, where 0.6 are taken now.)
enum { kBadRows = 1, kBadColumns = 2 };
struct RowStats {
    float q, q2;              // scales 2^e of q and of q f
    uint32_t g2_top, q2_top;  // largest magnitudes (bits) of g 2^-ge / l and q f
    uint32_t bad;          // what the split cannot hold of the block: kBadRows, kBadColumns
    int32_t doc_lo, doc_hi;
    float norm;            // largest sum of the squares of a row of q
};
struct RowsOut {
    char *q, *g;    // rows form: q by one scale per block, g by one per row
    char *g2, *q2;  // columns form: g / l (for dv) by one scale per row, q f (for dk) by one per block, f = 2^(re - ge) / l, 1/2 .. 2
    float *v;       // row_value
    RowStats *stats;
};
constexpr uint32_t kWideMost = (127u + 100) << 23, kWideLeast = (127u - 100) << 23, kGradMost = (127u + 60) << 23;
constexpr float kNoRow = 3e38f;
// The exponent e of a row's own scale 2^-e, which brings its largest magnitude to 2^14 .. 2^15.
__device__ __forceinline__ int row_exp(uint32_t top) { return (int)(top >> 23) - 127 - 14; }
constexpr int kLift = 12;  // weights are kept as 2^kLift times themselves, so that their split's second half is normal fp16

// Block t of the rows of (b, hk) for the backward.
template <int DP, bool VEC>
__device__ __forceinline__ void split_rows(const Rule &u, const Ptrs &p, int b, int hk, int t, int64_t at, const RowsOut &o,
                                           char *lds, uint32_t *sh) {
    constexpr int NCH = Share<DP>::NCH;
    const int rows = u.G * u.lq;
    const int64_t all = (int64_t)u.B * u.Hk * rows;
    Share<DP> s, g, ov;
    float rl[4], f[4], gd[4], delta[4], m[4], slope[4];
    uint32_t qt[4], gt[4];
    float norm = 0.0f;
    int dlo = INT32_MAX, dhi = INT32_MIN, doc[4];
    bool bad = false, bad_columns = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const Row row = row_of(u, hk, min(t * kBlock + 4 * (int)(threadIdx.x >> 4) + i, rows - 1));
        const int64_t tok = (int64_t)b * u.lq + row.t, sr = stat_at(u, b, row);
        m[i] = p.st[sr];
        rl[i] = p.st[all + sr];
        doc[i] = u.qd ? u.qd[tok] : 0;
        slope[i] = u.slopes ? u.slopes[row.h] * kLog2e : 0.0f;
        s.template load<VEC>(i, p.q + tok * p.ldq + (int64_t)row.h * u.d, u.d);
        g.template load<VEC>(i, p.g + tok * p.ldg + (int64_t)row.h * u.d, u.d);
        ov.template load<VEC>(i, p.o + tok * p.ldo + (int64_t)row.h * u.d, u.d);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int rr = t * kBlock + 4 * (threadIdx.x >> 4) + i;
        const bool there = rr < rows;
        const Row row = row_of(u, hk, min(rr, rows - 1));
        if (!there) rl[i] = 0.0f;
        const bool on = rl[i] != 0.0f;
        if (there) {
            dlo = min(dlo, doc[i]);
            dhi = max(dhi, doc[i]);
        }
        s.keep(i, on);
        g.keep(i, on);
        ov.keep(i, on);
        float dot = 0.0f;
#pragma unroll
        for (int n = 0; n < NCH; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) dot = __builtin_fmaf(g.x[i][n][e], ov.x[i][n][e], dot);
        dot = row_sum(dot);
        qt[i] = s.row_top(i);
        norm = larger(norm, s.row_norm(i));
        gt[i] = g.row_top(i);
        const bool fine = gt[i] == 0 || (gt[i] >= kWideLeast && gt[i] <= kWideMost);
        const int re = fine && gt[i] ? row_exp(gt[i]) : 0;
        // weights take g / l's size, at most 2^60, so that their products with a row's g . v, below 2^63, stay fp32 numbers
        const uint32_t lt = __float_as_uint(__uint_as_float(gt[i]) * rl[i]);
        const bool gives = gt[i] && fine && lt >= kWideLeast && lt <= kGradMost;
        const int ge = gives ? row_exp(lt) : 0;
        bad_columns = bad_columns || (gt[i] && !gives);
        // a row that gives nothing, and one that the split cannot hold, keep finite stand-ins
        const float w = gt[i] && fine ? rl[i] * pow2(re) : 0.0f;
        f[i] = gives ? rl[i] * pow2(re - ge) : 0.0f;
        gd[i] = gives ? pow2(-ge) : 0.0f;
        delta[i] = fine ? dot * pow2(-re) : 0.0f;
        bad = bad || !fine || (on && !bias_fits(u, slope[i])) || (on && !(__builtin_fabsf(m[i]) < 1e30f && rl[i] > 0.0f && rl[i] < 1e30f && __builtin_fabsf(dot) < 1e38f));
        m[i] = on ? (float)kLift - m[i] : -kNoRow;
        if ((threadIdx.x & 15) == 0) {
            const int64_t r = at * kBlock + 4 * (threadIdx.x >> 4) + i;
            o.v[row_value(r, kRowM)] = m[i];
            o.v[row_value(r, kRowDelta)] = delta[i];
            o.v[row_value(r, kRowPos)] = __int_as_float(row.t + u.off);
            o.v[row_value(r, kRowSlope)] = on ? slope[i] : 0.0f;
            o.v[row_value(r, kRowDoc)] = __int_as_float(doc[i]);
            o.v[row_value(r, kRowW)] = w;
            o.v[row_value(r, kRowGrad)] = gives ? pow2(ge) : 0.0f;
        }
    }
    RowStats st = {};
    // q, one scale
    const BlockTop qb = block_top<DP, false>(s, qt, norm, sh, lds);
    st.norm = qb.norm;
    const bool qok = in_range(qb.top);
    bad = bad || !qok;
    const int eq = qok && qb.top ? scale_exp(qb.top) : 0;
    st.q = pow2(eq);
    Share<DP> x;
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int n = 0; n < NCH; n++) x.x[i][n] = s.x[i][n] * pow2(-eq);
    }
    put_block<DP, false>(x, o.q + at * plane_bytes(DP, 1), lds);
    // g, a scale for each row
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const bool fine = gt[i] >= kWideLeast && gt[i] <= kWideMost;
        const float sc = fine ? pow2(-row_exp(gt[i])) : 0.0f;
#pragma unroll
        for (int n = 0; n < NCH; n++) x.x[i][n] = g.x[i][n] * sc;
    }
    put_block<DP, false>(x, o.g + at * plane_bytes(DP, 1), lds);
    // g / l, a scale for each row: their columns are looked at as they are scaled
    uint32_t t4[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        g.scale(i, rl[i]);
        g.scale(i, gd[i]);
        t4[i] = g.row_top(i);
    }
    const BlockTop gb = block_top<DP, true>(g, t4, 0.0f, sh, lds);
    bad_columns = bad_columns || !even_columns(gb);
    st.g2_top = gb.top;
    put_block<DP, true>(g, o.g2 + at * plane_bytes(DP, 1), lds);
    // q f, one scale
#pragma unroll
    for (int i = 0; i < 4; i++) {
        s.scale(i, f[i]);
        t4[i] = s.row_top(i);
    }
    const BlockTop fb = block_top<DP, true>(s, t4, 0.0f, sh, lds);
    const bool fok = fb.top == 0 || (fb.top >= kWideLeast && fb.top <= kWideMost && even_rows(fb.top, fb.low) && even_columns(fb));
    bad_columns = bad_columns || !fok;
    const int ef = fok && fb.top ? scale_exp(fb.top) : 0;
    st.q2 = pow2(ef);
    st.q2_top = fb.top;
#pragma unroll
    for (int i = 0; i < 4; i++) s.scale(i, pow2(-ef));
    put_block<DP, true>(s, o.q2 + at * plane_bytes(DP, 1), lds);
    __syncthreads();
    const uint32_t wave_bad = (__any(bad) ? kBadRows : 0) | (__any(bad_columns) ? kBadColumns : 0);
    if ((threadIdx.x & 15) == 0) {
        sh[threadIdx.x >> 4] = (uint32_t)dlo;
        sh[16 + (threadIdx.x >> 4)] = (uint32_t)dhi;
        sh[32 + (threadIdx.x >> 4)] = wave_bad;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 0; i < 16; i++) {
            dlo = min(dlo, (int)sh[i]);
            dhi = max(dhi, (int)sh[16 + i]);
            st.bad |= sh[32 + i];
        }
        st.doc_lo = dlo;
        st.doc_hi = dhi;
        o.stats[at] = st;
        for (int half = 0; half < 2; half++) {
            float *to = o.v + row_value(at * kBlock + 32 * half, kRowBlock);
            to[0] = st.q;
            to[1] = st.q2;
            to[2] = __int_as_float(dlo);
            to[3] = __int_as_float(dhi);
        }
    }
}

}  // namespace osc
