// Attention with scored rules over grouped heads (include/om.h, om_attention_fwd_scored / _bwd_scored): the row kernels,
// right for every shape and value, and the entry points.
//
// Forward, per row (a query of one head): m = max x, l = sum 2^(x - m) over the keys it sees, o = sum 2^(x - m) v / l,
// in one pass with the running maximum and sum. Backward: p = 2^(x - m) / l from the saved m and 1 / l,
// ds = p (g . v - delta) (1 - tanh^2), delta = g . o, dq = scale sum ds k, dk = scale sum ds q, dv = sum p g.
//
// A workgroup holds R rows (or R keys) in registers and streams the keys (or rows) past them: 16 lanes share a streamed
// row, four values each per 64, so that 16 streams of rows run side by side in a workgroup and every load is 16 bytes;
// a product is four multiply-adds a lane and a sum over the 16 lanes in four DPP additions. The streams are joined
// through LDS in a fixed order. With few rows the pass over K and V is bound by memory (8 x 4 key heads, three rows each over 4096
// keys of 64 values: 67 MB in 24.5 us with the join, 2.7 TB/s); with many it is bound by the vector unit.
#include <cmath>

#include "om_attention_scored.hpp"

namespace {

using namespace osc;

constexpr int kStreams = 16;  // streams of a workgroup: four per wavefront
constexpr float kInf = __builtin_inff();

// dot of a held row with a streamed one, over this lane's values
template <int NC>
__device__ __forceinline__ float dot(const floatx4 (&a)[NC], const floatx4 (&b)[NC]) {
    float s = 0.0f;
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) s = __builtin_fmaf(a[n][e], b[n][e], s);
    return s;
}
template <int NC, bool VEC>
__device__ __forceinline__ void load_row(floatx4 (&x)[NC], const float *row, int l16, int d) {
#pragma unroll
    for (int n = 0; n < NC; n++) x[n] = load4<VEC>(row, 64 * n + 4 * l16, d);
}
template <int NC>
__device__ __forceinline__ void add_scaled(floatx4 (&a)[NC], float w, const floatx4 (&x)[NC]) {
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) a[n][e] = __builtin_fmaf(w, x[n][e], a[n][e]);
}

// One batch item, key head and split of the keys, rows rr0 .. rr0 + R - 1. part NULL: o and the statistics; else the
// split's unnormalised sums [split][B Hk][G lq][d], then its maxima and sums [split][B Hk][G lq] each.
template <int NC, int R, bool VEC>
__device__ __forceinline__ void fwd_rows(const Rule &u, const Ptrs &p, int b, int hk, int rr0, int split, int nsplit,
                                         int per, float *part) {
    __shared__ __attribute__((aligned(16))) float sa[kStreams][R][NC * 64];
    __shared__ float sm[kStreams][R], sl[kStreams][R];
    constexpr int U = NC * R >= 8 ? 2 : 4;  // streamed rows in flight per stream
    const int lane = threadIdx.x & 63, l16 = lane & 15, st = (threadIdx.x >> 6) * 4 + (lane >> 4);
    const int rows = u.G * u.lq, d = u.d, pre = u.prefix ? u.prefix[b] : 0;
    floatx4 q[R][NC], acc[R][NC];
    float m[R], l[R], slope[R];
    int pos[R], doc[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const Row row = row_of(u, hk, min(rr0 + r, rows - 1));
        load_row<NC, VEC>(q[r], p.q + ((int64_t)b * u.lq + row.t) * p.ldq + (int64_t)row.h * d, l16, d);
        pos[r] = row.t + u.off;
        doc[r] = u.qd ? u.qd[(int64_t)b * u.lq + row.t] : 0;
        if (rr0 + r >= rows) doc[r] = -1;
        slope[r] = u.slopes ? u.slopes[row.h] * kLog2e : 0.0f;
        m[r] = -kInf;
        l[r] = 0.0f;
#pragma unroll
        for (int n = 0; n < NC; n++) acc[r][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    int lo, hi;
    key_range(u, rr0 / u.G + u.off, (min(rr0 + R, rows) - 1) / u.G + u.off, pre, lo, hi);
    lo = max(lo, split * per);
    hi = min(hi, (int)min((int64_t)u.lk, (int64_t)(split + 1) * per) - 1);
    const float *kb = p.k + (int64_t)b * u.lk * p.ldkv + (int64_t)hk * d, *vb = p.v + (int64_t)b * u.lk * p.ldkv + (int64_t)hk * d;
    for (int j0 = lo + st; j0 <= hi; j0 += kStreams * U) {
        floatx4 kx[U][NC], vx[U][NC];
        int kd[U];
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int j = min(j0 + kStreams * i, hi);
            load_row<NC, VEC>(kx[i], kb + (int64_t)j * p.ldkv, l16, d);
            load_row<NC, VEC>(vx[i], vb + (int64_t)j * p.ldkv, l16, d);
            kd[i] = u.kd ? u.kd[(int64_t)b * u.lk + j] : 0;
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            float x[U], top = m[r];
            bool see[U];
#pragma unroll
            for (int i = 0; i < U; i++) {
                const int j = j0 + kStreams * i, gap = pos[r] - j;
                see[i] = j <= hi && doc[r] >= 0 && doc[r] == kd[i] && in_reach(u, gap, j, pre);
                float th;
                x[i] = score(u, row_sum(dot<NC>(q[r], kx[i])), th);
                if (u.slopes) x[i] = __builtin_fmaf(-slope[r], (float)(gap < 0 ? -gap : gap), x[i]);
                if (see[i]) top = x[i] > top ? x[i] : top;
            }
            const float mu = top == -kInf ? 0.0f : top, alpha = exp2_hw(m[r] - mu);
            if (alpha != 1.0f) {
                l[r] *= alpha;
#pragma unroll
                for (int n = 0; n < NC; n++) acc[r][n] *= alpha;
            }
            m[r] = top;
#pragma unroll
            for (int i = 0; i < U; i++)
                if (see[i]) {
                    const float e = exp2_hw(x[i] - mu);
                    l[r] += e;
                    add_scaled<NC>(acc[r], e, vx[i]);
                }
        }
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
        if (l16 == 0) {
            sm[st][r] = m[r];
            sl[st][r] = l[r];
        }
#pragma unroll
        for (int n = 0; n < NC; n++) *reinterpret_cast<floatx4 *>(&sa[st][r][64 * n + 4 * l16]) = acc[r][n];
    }
    __syncthreads();
    const int64_t bh = (int64_t)b * u.Hk + hk, all = (int64_t)u.B * u.Hk * rows;
    for (int f = threadIdx.x; f < R * d; f += 256) {
        const int r = f / d, c = f - r * d;
        if (rr0 + r >= rows) break;
        float top = -kInf;
#pragma unroll
        for (int s = 0; s < kStreams; s++) top = sm[s][r] > top ? sm[s][r] : top;
        const float mu = top == -kInf ? 0.0f : top;
        float sum = 0.0f, a = 0.0f;
#pragma unroll
        for (int s = 0; s < kStreams; s++) {
            const float w = exp2_hw(sm[s][r] - mu);
            sum = __builtin_fmaf(w, sl[s][r], sum);
            a = __builtin_fmaf(w, sa[s][r][c], a);
        }
        const int64_t at = bh * rows + rr0 + r;
        if (part) {
            part[((int64_t)split * all + at) * d + c] = a;
            if (c == 0) {
                float *ms = part + (int64_t)nsplit * all * d + (int64_t)split * all + at;
                ms[0] = mu;
                ms[(int64_t)nsplit * all] = sum;
            }
        } else {
            const Row row = row_of(u, hk, rr0 + r);
            const float rl = sum == 0.0f ? 0.0f : 1.0f / sum;
            p.out[((int64_t)b * u.lq + row.t) * p.ldo + (int64_t)row.h * d + c] = rl == 0.0f && sum == 0.0f ? 0.0f : a * rl;
            if (c == 0 && p.stats) {
                const int64_t sr = stat_at(u, b, row);
                p.stats[sr] = mu;
                p.stats[all + sr] = rl;
            }
        }
    }
}

template <int NC, int R, bool VEC>
__global__ void __launch_bounds__(256) k_scored_fwd_rows(Rule u, Ptrs p, int blocks, int nsplit, int per, float *part) {
    OM_LDS_POISON();
    int i = blockIdx.x;
    const int rb = i % blocks;
    i /= blocks;
    const int split = i % nsplit;
    i /= nsplit;
    fwd_rows<NC, R, VEC>(u, p, i / u.Hk, i % u.Hk, rb * R, split, nsplit, per, part);
}

// Joins the splits: o = sum_s 2^(m_s - m) a_s / sum_s 2^(m_s - m) l_s, in split order; a thread per four values (or one,
// where d is no multiple of four). The loads of kAtOnce splits are issued together: a loop that waits for every split in
// turn took 33 us for 96 rows of 32 splits.
constexpr int kAtOnce = 8;
template <int W>
__global__ void __launch_bounds__(256) k_scored_join(Rule u, Ptrs p, int nsplit, const float *__restrict__ part) {
    OM_LDS_POISON();
    typedef float vec __attribute__((ext_vector_type(W), aligned(4)));
    const int rows = u.G * u.lq, d = u.d, per = d / W;
    const int64_t all = (int64_t)u.B * u.Hk * rows, f = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (f >= all * per) return;
    const int64_t at = f / per;
    const int c = (int)(f - at * per) * W;
    const float *ms = part + (int64_t)nsplit * all * d + at, *ls = ms + (int64_t)nsplit * all;
    float mu = -kInf, sum = 0.0f;  // of the splits so far
    vec a;
#pragma unroll
    for (int e = 0; e < W; e++) a[e] = 0.0f;
    for (int s0 = 0; s0 < nsplit; s0 += kAtOnce) {
        float m[kAtOnce], l[kAtOnce];
        vec x[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const int64_t s = min(s0 + i, nsplit - 1);
            m[i] = ms[s * all];
            l[i] = s0 + i < nsplit ? ls[s * all] : 0.0f;
            x[i] = *reinterpret_cast<const vec *>(part + (s * all + at) * d + c);
        }
        // a split without a visible key has l = 0 and stands at 0: it must not count
        float top = mu;
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) top = l[i] != 0.0f && m[i] > top ? m[i] : top;
        const float old = top == -kInf ? 1.0f : exp2_hw(mu - top);
        mu = top;
        sum *= old;
        a *= old;
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const float w = exp2_hw(m[i] - (top == -kInf ? 0.0f : top));
            sum = l[i] != 0.0f ? __builtin_fmaf(w, l[i], sum) : sum;
#pragma unroll
            for (int e = 0; e < W; e++) a[e] = l[i] != 0.0f ? __builtin_fmaf(w, x[i][e], a[e]) : a[e];
        }
    }
    if (mu == -kInf) mu = 0.0f;
    const int64_t bh = at / rows;
    const int b = (int)(bh / u.Hk);
    const Row row = row_of(u, (int)(bh % u.Hk), (int)(at - bh * rows));
    const float rl = sum == 0.0f ? 0.0f : 1.0f / sum;
    vec o;
#pragma unroll
    for (int e = 0; e < W; e++) o[e] = sum == 0.0f ? 0.0f : a[e] * rl;
    *reinterpret_cast<vec *>(p.out + ((int64_t)b * u.lq + row.t) * p.ldo + (int64_t)row.h * d + c) = o;
    if (c == 0 && p.stats) {
        const int64_t sr = stat_at(u, b, row);
        p.stats[sr] = mu;
        p.stats[all + sr] = rl;
    }
}

// Joins the streams' sums of R held rows in stream order and writes them (or adds them) to `rowp(r)`.
template <int NC, int R, typename F>
__device__ __forceinline__ void join_streams(float (&sa)[kStreams][R][NC * 64], const floatx4 (&a)[R][NC], int d, float w,
                                             int acc, F rowp) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, st = (threadIdx.x >> 6) * 4 + (lane >> 4);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int n = 0; n < NC; n++) *reinterpret_cast<floatx4 *>(&sa[st][r][64 * n + 4 * l16]) = a[r][n];
    __syncthreads();
    for (int f = threadIdx.x; f < R * d; f += 256) {
        const int r = f / d, c = f - r * d;
        float *to = rowp(r);
        if (!to) break;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kStreams; i++) s += sa[i][r][c];
        s *= w;
        to[c] = acc ? to[c] + s : s;
    }
}

// dQ of rows rr0 .. rr0 + R - 1: the keys stream past.
template <int NC, int R, bool VEC>
__device__ __forceinline__ void dq_rows(const Rule &u, const Ptrs &p, int b, int hk, int rr0,
                                        float (&sa)[kStreams][R][NC * 64]) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, st = (threadIdx.x >> 6) * 4 + (lane >> 4);
    const int rows = u.G * u.lq, d = u.d, pre = u.prefix ? u.prefix[b] : 0;
    const int64_t all = (int64_t)u.B * u.Hk * rows;
    floatx4 q[R][NC], g[R][NC], dq[R][NC];
    float m[R], rl[R], delta[R], slope[R];
    int pos[R], doc[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const Row row = row_of(u, hk, min(rr0 + r, rows - 1));
        const int64_t tok = (int64_t)b * u.lq + row.t, sr = stat_at(u, b, row);
        load_row<NC, VEC>(q[r], p.q + tok * p.ldq + (int64_t)row.h * d, l16, d);
        load_row<NC, VEC>(g[r], p.g + tok * p.ldg + (int64_t)row.h * d, l16, d);
        load_row<NC, VEC>(dq[r], p.o + tok * p.ldo + (int64_t)row.h * d, l16, d);
        delta[r] = row_sum(dot<NC>(g[r], dq[r]));
        m[r] = p.st[sr];
        rl[r] = p.st[all + sr];
        pos[r] = row.t + u.off;
        doc[r] = rr0 + r >= rows || rl[r] == 0.0f ? -1 : u.qd ? u.qd[tok] : 0;
        slope[r] = u.slopes ? u.slopes[row.h] * kLog2e : 0.0f;
#pragma unroll
        for (int n = 0; n < NC; n++) dq[r][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    int lo, hi;
    key_range(u, rr0 / u.G + u.off, (min(rr0 + R, rows) - 1) / u.G + u.off, pre, lo, hi);
    const float *kb = p.k + (int64_t)b * u.lk * p.ldkv + (int64_t)hk * d, *vb = p.v + (int64_t)b * u.lk * p.ldkv + (int64_t)hk * d;
    for (int j = lo + st; j <= hi; j += kStreams) {
        floatx4 kx[NC], vx[NC];
        load_row<NC, VEC>(kx, kb + (int64_t)j * p.ldkv, l16, d);
        load_row<NC, VEC>(vx, vb + (int64_t)j * p.ldkv, l16, d);
        const int kd = u.kd ? u.kd[(int64_t)b * u.lk + j] : 0;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int gap = pos[r] - j;
            if (doc[r] < 0 || doc[r] != kd || !in_reach(u, gap, j, pre)) continue;
            float th, x = score(u, row_sum(dot<NC>(q[r], kx)), th);
            if (u.slopes) x = __builtin_fmaf(-slope[r], (float)(gap < 0 ? -gap : gap), x);
            const float pr = exp2_hw(x - m[r]) * rl[r];
            const float ds = pr * (row_sum(dot<NC>(g[r], vx)) - delta[r]) * (1.0f - th * th);
            add_scaled<NC>(dq[r], ds, kx);
        }
    }
    join_streams<NC, R>(sa, dq, d, u.scale, p.acc, [&](int r) -> float * {
        if (rr0 + r >= rows) return nullptr;
        const Row row = row_of(u, hk, rr0 + r);
        return p.dq + ((int64_t)b * u.lq + row.t) * p.lddq + (int64_t)row.h * d;
    });
}

// dK and dV of keys j0 .. j0 + R - 1: the rows of the key head's whole group stream past.
template <int NC, int R, bool VEC>
__device__ __forceinline__ void dkv_keys(const Rule &u, const Ptrs &p, int b, int hk, int j0,
                                         float (&sa)[kStreams][R][NC * 64]) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, st = (threadIdx.x >> 6) * 4 + (lane >> 4);
    const int rows = u.G * u.lq, d = u.d, pre = u.prefix ? u.prefix[b] : 0;
    const int64_t all = (int64_t)u.B * u.Hk * rows;
    floatx4 k[R][NC], v[R][NC], dk[R][NC], dv[R][NC];
    int kd[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int64_t tok = (int64_t)b * u.lk + min(j0 + r, u.lk - 1);
        load_row<NC, VEC>(k[r], p.k + tok * p.ldkv + (int64_t)hk * d, l16, d);
        load_row<NC, VEC>(v[r], p.v + tok * p.ldkv + (int64_t)hk * d, l16, d);
        kd[r] = j0 + r >= u.lk ? -1 : u.kd ? u.kd[tok] : 0;
#pragma unroll
        for (int n = 0; n < NC; n++) dk[r][n] = dv[r][n] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    int r0, r1;
    row_range(u, j0, min(j0 + R, u.lk) - 1, pre, r0, r1);
    for (int rr = r0 + st; rr < r1; rr += kStreams) {
        const Row row = row_of(u, hk, rr);
        const int64_t tok = (int64_t)b * u.lq + row.t, sr = stat_at(u, b, row);
        floatx4 q[NC], g[NC], o[NC];
        load_row<NC, VEC>(q, p.q + tok * p.ldq + (int64_t)row.h * d, l16, d);
        load_row<NC, VEC>(g, p.g + tok * p.ldg + (int64_t)row.h * d, l16, d);
        load_row<NC, VEC>(o, p.o + tok * p.ldo + (int64_t)row.h * d, l16, d);
        const float m = p.st[sr], rl = p.st[all + sr], delta = row_sum(dot<NC>(g, o));
        const float slope = u.slopes ? u.slopes[row.h] * kLog2e : 0.0f;
        const int doc = rl == 0.0f ? -1 : u.qd ? u.qd[tok] : 0, pos = row.t + u.off;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int gap = pos - (j0 + r);
            if (doc < 0 || doc != kd[r] || !in_reach(u, gap, j0 + r, pre)) continue;
            float th, x = score(u, row_sum(dot<NC>(q, k[r])), th);
            if (u.slopes) x = __builtin_fmaf(-slope, (float)(gap < 0 ? -gap : gap), x);
            const float pr = exp2_hw(x - m) * rl;
            const float ds = pr * (row_sum(dot<NC>(g, v[r])) - delta) * (1.0f - th * th);
            add_scaled<NC>(dv[r], pr, g);
            add_scaled<NC>(dk[r], ds, q);
        }
    }
    auto to = [&](float *base) {
        return [=](int r) -> float * {
            return j0 + r < u.lk ? base + ((int64_t)b * u.lk + j0 + r) * p.lddkv + (int64_t)hk * d : nullptr;
        };
    };
    if (p.dk) join_streams<NC, R>(sa, dk, d, u.scale, p.acc, to(p.dk));
    if (p.dv) join_streams<NC, R>(sa, dv, d, 1.0f, p.acc, to(p.dv));
}

// Both halves in one launch: the first nq workgroups of each (batch, key head) take rows, the others keys.
template <int NC, int R, bool VEC>
__global__ void __launch_bounds__(256) k_scored_bwd_rows(Rule u, Ptrs p, int nq, int nk) {
    OM_LDS_POISON();
    __shared__ __attribute__((aligned(16))) float sa[kStreams][R][NC * 64];
    const int each = nq + nk, i = blockIdx.x / each, x = blockIdx.x - i * each;
    const int b = i / u.Hk, hk = i - b * u.Hk;
    if (x < nq) dq_rows<NC, R, VEC>(u, p, b, hk, x * R, sa);
    else dkv_keys<NC, R, VEC>(u, p, b, hk, (x - nq) * R, sa);
}

bool al16(const void *p) { return ((uintptr_t)p & 15) == 0; }

om_status make_rule(om_ctx *ctx, const char *what, const om_attention_scores *f, int B, int lq, int lk, int d, Rule &u) {
    OM_REQUIRE(ctx, f, "%s: scores is NULL", what);
    OM_REQUIRE(ctx, B >= 0 && lq >= 0 && lk >= 0 && d >= 1 && d <= 256, "%s: B=%d lq=%d lk=%d d=%d (d from 1 to 256)", what,
               B, lq, lk, d);
    OM_REQUIRE(ctx, f->heads >= 1 && f->kv_heads >= 1 && f->heads % f->kv_heads == 0,
               "%s: %d heads are not a multiple of %d key heads", what, f->heads, f->kv_heads);
    // 2^30 keeps every row, key and position index, and their sums with a tile or a window, inside 32 bits (not a key's
    // index times the group: row_range)
    constexpr int64_t kMost = 1 << 30;
    OM_REQUIRE(ctx, (int64_t)f->heads * d <= kMost && lq <= kMost && lk <= kMost && (int64_t)B * f->heads <= kMost &&
               (int64_t)B * f->heads * lq <= kMost && (int64_t)B * f->kv_heads * lk <= kMost, "%s: too many rows", what);
    OM_REQUIRE(ctx, std::isfinite(f->cap) && f->cap >= 0.0f, "%s: cap must be finite and not negative", what);
    OM_REQUIRE(ctx, !std::isinf(f->scale), "%s: scale must be finite", what);
    OM_REQUIRE(ctx, f->causal == 0 || f->causal == 1, "%s: causal=%d", what, f->causal);
    OM_REQUIRE(ctx, f->window >= 0, "%s: window=%d", what, f->window);
    OM_REQUIRE(ctx, !f->q_doc == !f->k_doc, "%s: documents need both q_doc and k_doc", what);
    u = Rule{};
    u.B = B;
    u.Hk = f->kv_heads;
    u.G = f->heads / f->kv_heads;
    u.lq = lq;
    u.lk = lk;
    u.d = d;
    u.off = lk - lq;
    u.causal = f->causal;
    // |i - j| is below the larger length, so a window that wide is none; a narrower one cannot take a position out of 32 bits
    u.window = f->window >= (lq > lk ? lq : lk) ? 0 : f->window;
    u.scale = f->scale == 0.0f || f->scale != f->scale ? 1.0f / sqrtf((float)d) : f->scale;
    u.cl2 = u.scale * kLog2e;
    if (f->cap > 0.0f) {
        u.icap = u.scale / f->cap;
        u.capl2 = f->cap * kLog2e;
        OM_REQUIRE(ctx, std::isfinite(u.icap) && std::isfinite(u.capl2) && u.icap != 0.0f, "%s: cap %g is out of range", what,
                   (double)f->cap);
    }
    u.slopes = f->slopes;
    u.qd = f->q_doc;
    u.kd = f->k_doc;
    u.prefix = f->prefix;
    return OM_OK;
}

om_status check_strides(om_ctx *ctx, const char *what, const Rule &u, const Ptrs &p) {
    const int64_t qw = (int64_t)u.Hk * u.G * u.d, kw = (int64_t)u.Hk * u.d;
    OM_REQUIRE(ctx, p.ldq >= qw && p.ldo >= qw && p.ldkv >= kw, "%s: row strides %lld / %lld / %lld below heads * d = %lld "
               "or kv_heads * d = %lld", what, (long long)p.ldq, (long long)p.ldo, (long long)p.ldkv, (long long)qw,
               (long long)kw);
    return OM_OK;
}

template <typename F>
void by_width(int d, bool vec, F f) {
    auto w = [&](auto nc) {
        if (vec) f(nc, std::true_type());
        else f(nc, std::false_type());
    };
    if (d <= 64) w(std::integral_constant<int, 1>());
    else if (d <= 128) w(std::integral_constant<int, 2>());
    else w(std::integral_constant<int, 4>());
}

void join(om_ctx *ctx, const Rule &u, const Ptrs &p, int nsplit, const float *part) {
    auto go = [&](auto kern, int w) {
        const int64_t values = (int64_t)u.B * u.Hk * u.G * u.lq * (u.d / w);
        hipLaunchKernelGGL(kern, dim3((unsigned)((values + 255) / 256)), dim3(256), 0, ctx->stream, u, p, nsplit, part);
    };
    u.d % 4 == 0 ? go(k_scored_join<4>, 4) : go(k_scored_join<1>, 1);
}

// The matrix kernels run where there is work enough: below, their splitting pass and half-filled tiles cost more than the row
// kernels' whole call. In us, forward / backward, by rows against by matrix: 4 heads of 31 | 32 rows, 512 keys of 64 values (64
// thousand pairs) 14 / 34, 21 / 41; 4096 keys (half a million) 42 / 297, 25 / 50; 96 heads of 64 keys (196 thousand) 19 / 22,
// 13 / 20; at 128 values 24 heads of 512 keys (380 thousand) 32 / 64, 33 / 72; of 4096 keys 173 / 485, 61 / 179. A forward of
// less than eight rows leaves most of a tile empty and runs faster by rows, 7 rows as above in 20 us; a backward does not,
// whose keys the row kernels do not split: 252 us.
// The matrix kernels' factors, scale or scale / cap times the operands' powers of two (2^-52 .. 2^28 each), have to stay fp32
// numbers: within 2^-40 .. 2^40 for a score that is not lost itself.
bool by_matrix(const Rule &u, int least) {
    const int64_t rows = (int64_t)u.G * u.lq;
    const float s = std::fabs(u.scale), c = std::fabs(u.icap);
    const bool fits = s >= 0x1p-40f && s <= 0x1p40f && (c == 0.0f || (c >= 0x1p-40f && c <= 0x1p40f));
    return fits && u.d <= 128 && rows >= least && rows * u.lk * u.B * u.Hk >= 1024 * (int64_t)((u.d + 31) / 32 * 32);
}

om_status fwd_by_rows(om_ctx *ctx, const Rule &u, const Ptrs &p) {
    const bool vec = u.d % 4 == 0 && p.ldq % 4 == 0 && p.ldkv % 4 == 0 && al16(p.q) && al16(p.k) && al16(p.v);
    const int rows = u.G * u.lq;
    om_status status = OM_OK;
    by_width(u.d, vec, [&](auto nc, auto v) {
        constexpr int NC = decltype(nc)::value;
        constexpr bool V = decltype(v)::value;
        auto launch = [&](auto rc) {
            constexpr int R = decltype(rc)::value;
            const int64_t blocks = (rows + R - 1) / R, wgs = blocks * u.B * u.Hk;
            // Split the keys until the chip has about four workgroups per CU, in pieces of at least 64 keys.
            int64_t ns = wgs >= 2 * ctx->num_cus ? 1 : 4 * ctx->num_cus / wgs;
            if (ns > (u.lk + 63) / 64) ns = (u.lk + 63) / 64;
            if (ns < 1) ns = 1;
            const int per = (int)((u.lk + ns - 1) / ns);
            if (per > 0) ns = (u.lk + per - 1) / per;
            if (wgs * ns > most_groups(256)) {
                status = om::fail(ctx, OM_E_ARG, "om_attention_fwd_scored: too many row blocks");
                return;
            }
            float *part = nullptr;
            const int64_t all = (int64_t)u.B * u.Hk * rows;
            if (ns > 1) {
                status = om::scratch2(ctx, sizeof(float) * (uint64_t)ns * all * (u.d + 2), &part);
                if (status) return;
            }
            hipLaunchKernelGGL((k_scored_fwd_rows<NC, R, V>), dim3((unsigned)(wgs * ns)), dim3(256), 0, ctx->stream, u, p,
                               (int)blocks, (int)ns, per, part);
            if (ns > 1) join(ctx, u, p, (int)ns, part);
        };
        // Three rows a pass over K and V: 4096 keys of 64 values, 16 x 12 heads, 7 rows in 227 us where six a pass take 311
        // (their registers leave half the wavefronts), 3 rows in 82 us; one row alone in 76 us where three a pass take 82.
        if (NC >= 4 || rows == 1) launch(std::integral_constant<int, 1>());
        else launch(std::integral_constant<int, 3>());
    });
    return status ? status : OM_LAUNCH_CHECK(ctx, "om_attention_fwd_scored");
}

om_status bwd_by_rows(om_ctx *ctx, const Rule &u, const Ptrs &p) {
    const bool vec = u.d % 4 == 0 && p.ldq % 4 == 0 && p.ldkv % 4 == 0 && p.ldo % 4 == 0 && p.ldg % 4 == 0 && al16(p.q) &&
                     al16(p.k) && al16(p.v) && al16(p.o) && al16(p.g);
    om_status status = OM_OK;
    by_width(u.d, vec, [&](auto nc, auto v) {
        constexpr int NC = decltype(nc)::value, R = NC == 1 ? 4 : NC == 2 ? 2 : 1;
        constexpr bool V = decltype(v)::value;
        const int64_t rows = (int64_t)u.G * u.lq, nq = p.dq ? (rows + R - 1) / R : 0;
        const int64_t nk = p.dk || p.dv ? (u.lk + R - 1) / R : 0, wgs = (nq + nk) * u.B * u.Hk;
        if (wgs == 0) return;
        if (wgs > most_groups(256)) {
            status = om::fail(ctx, OM_E_ARG, "om_attention_bwd_scored: too many row blocks");
            return;
        }
        hipLaunchKernelGGL((k_scored_bwd_rows<NC, R, V>), dim3((unsigned)wgs), dim3(256), 0, ctx->stream, u, p, (int)nq,
                           (int)nk);
    });
    return status ? status : OM_LAUNCH_CHECK(ctx, "om_attention_bwd_scored");
}

}  // namespace

extern "C" {

om_status om_attention_fwd_scored(om_ctx *ctx, const float *q, int ld_q, const float *k, const float *v, int ld_kv, float *o,
                                  int ld_o, float *stats, int B, int lq, int lk, int d, const om_attention_scores *scores) {
    OM_CHECK_CTX(ctx);
    const char *what = "om_attention_fwd_scored";
    Rule u;
    if (om_status s = make_rule(ctx, what, scores, B, lq, lk, d, u)) return s;
    Ptrs p = {};
    p.q = q;
    p.k = k;
    p.v = v;
    p.out = o;
    p.stats = stats;
    p.ldq = ld_q;
    p.ldkv = ld_kv;
    p.ldo = ld_o;
    if (om_status s = check_strides(ctx, what, u, p)) return s;
    if (B == 0 || lq == 0) return OM_OK;
    OM_REQUIRE(ctx, q && o && ((k && v) || lk == 0), "%s: NULL q/k/v/o", what);
    if (om_status s = om::use_device(ctx)) return s;
    if (!by_matrix(u, 8)) return fwd_by_rows(ctx, u, p);
    int joins;
    float *part;
    if (om_status s = fwd_by_matrix(ctx, u, p, &joins, &part)) return s;
    if (joins == 1) return OM_OK;
    join(ctx, u, p, joins, part);
    return OM_LAUNCH_CHECK(ctx, what);
}

om_status om_attention_bwd_scored(om_ctx *ctx, const float *q, int ld_q, const float *k, const float *v, int ld_kv,
                                  const float *o, int ld_o, const float *stats, const float *g, int ld_g, float *dq,
                                  int ld_dq, float *dk, float *dv, int ld_dkv, int B, int lq, int lk, int d,
                                  const om_attention_scores *scores, int acc) {
    OM_CHECK_CTX(ctx);
    const char *what = "om_attention_bwd_scored";
    Rule u;
    if (om_status s = make_rule(ctx, what, scores, B, lq, lk, d, u)) return s;
    Ptrs p = {};
    p.q = q;
    p.k = k;
    p.v = v;
    p.o = o;
    p.g = g;
    p.st = stats;
    p.dq = dq;
    p.dk = dk;
    p.dv = dv;
    p.ldq = ld_q;
    p.ldkv = ld_kv;
    p.ldo = ld_o;
    p.ldg = ld_g;
    p.lddq = ld_dq;
    p.lddkv = ld_dkv;
    p.acc = acc != 0;
    if (om_status s = check_strides(ctx, what, u, p)) return s;
    const int64_t qw = (int64_t)u.Hk * u.G * d, kw = (int64_t)u.Hk * d;
    OM_REQUIRE(ctx, ld_g >= qw && (!dq || ld_dq >= qw) && ((!dk && !dv) || ld_dkv >= kw),
               "%s: gradient row strides %d / %d / %d below heads * d = %lld or kv_heads * d = %lld", what, ld_g, ld_dq,
               ld_dkv, (long long)qw, (long long)kw);
    if (B == 0 || (!dq && !dk && !dv)) return OM_OK;
    OM_REQUIRE(ctx, (q && o && g && stats) || lq == 0, "%s: NULL q/o/stats/g", what);
    OM_REQUIRE(ctx, (k && v) || lk == 0, "%s: NULL k/v", what);
    if (om_status s = om::use_device(ctx)) return s;
    return by_matrix(u, 1) ? bwd_by_matrix(ctx, u, p) : bwd_by_rows(ctx, u, p);
}

}  // extern "C"
