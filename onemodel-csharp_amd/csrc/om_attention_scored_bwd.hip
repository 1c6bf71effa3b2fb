// Scored attention's backward on the matrix cores (operands: om_attention_scored_mm.hpp).
//
// With E = 2^(x - m) from the saved m, re the exponent of a row's gradient and w = 2^re / l:
//   D = E (g 2^-re . v - delta 2^-re) (1 - tanh^2),
//   dv_j = sum_i E_ij 2^ge (g_i 2^-ge / l_i),  dk_j = scale sum_i D_ij 2^ge (q_i 2^(re - ge) / l_i),  dq_i = scale w_i sum_j D_ij k_j,
// ge the exponent of g_i / l_i: an operand's row carries the row's factor up to a power of two, the weights carry that in fp32
// and are split at a running scale of each key's, so that weights of 1 / length and gradients of any size keep their bits in
// fp16 pairs.
//
// Two roles share a launch (their tails fill each other's): a workgroup of 128 keys holds K and V fragments and walks the rows
// of the key head's whole group, scores with a key in each lane; one of 128 rows holds Q and G and walks the keys, with a
// query in each lane. Either way a block of scores leaves the matrix unit in the order in which it is the next product's
// operand. Recomputing the scores for the second role costs two products of seven; partial dq from the first role would
// cost rows * keys / 32 values of traffic, more than that from about 2000 keys on, and atomics would lose the fixed order.
//
// Bound: as the forward. 12 heads of 64 values in 4 key heads, 4096 causal rows with a cap: 350 to 415 us over several runs, 382
// in the middle (matrix unit busy 40 % of the time, vector unit 62 %); 16 heads of 128 in 4, 8192 rows in a window of 1024: 1080
// to 1225 us (30 %, 33 %, one wavefront a SIMD).
#include <algorithm>

#include "om_attention_scored_split.hpp"

namespace {

using namespace osc;

constexpr int kKeys = 128;   // keys of a workgroup of the first role
// Wavefronts of a workgroup. Up to 64 values a head, four: each holds 32 keys' dk and dv, two or three workgroups a CU. Above,
// both and the fragments of K and V take more than half a SIMD's registers, and one wavefront a SIMD is left. Up to 96, eight
// share the stages instead: four hold K and dv and form the scores and the weights, four hold V and dk of the same keys, form
// g . v meanwhile, and take the weights over through LDS (777 rows of 80 values, prefix: 108 -> 95 us). At 128 that spills
// registers and is no faster than four (8192 rows in a window of 1024, timed side by side: 1157 us against 1152).
constexpr int waves_of(int dp) { return dp == 96 ? 8 : 4; }
constexpr int kStep = 32;    // rows (or keys) of a step
constexpr int kListed = 256; // blocks whose step data stands in LDS

struct BwdArgs {
    const char *kn, *kt, *vn;        // K in both forms, V in rows form
    const char *qn, *gn, *g2, *q2;   // RowsOut
    const float *v, *keys;           // the rows' records and the steps' words of the keys
    const Stats *ks, *vs;
    const RowStats *rs;
    int nt, nr;                      // blocks of 64 keys and rows of a head
    int kblocks, rblocks;            // workgroups along them
    int nsplit, qsplit;              // splits of each block of keys' rows for dk and dv, of each block of rows' keys for dq
    int keys_wgs, rows_wgs;          // workgroups of the roles
    int kperiod, rperiod;            // where the roles' sweeps begin: at multiples, in blocks of rows and in steps of keys
    float *part;                     // [split][B Hk][lk][2][d] (dk, dv), NULL for one split
    float *qpart;                    // [split][B Hk][G lq][d] (dq), NULL for one split
};

template <int DP, bool VEC>
__global__ void __launch_bounds__(256) k_scored_split_bwd(Rule u, Ptrs p, SplitOut ko, SplitOut vo, RowsOut ro, int nt, int nr) {
    OM_LDS_POISON();
    __shared__ __attribute__((aligned(16))) char lds[DP * 256];
    __shared__ uint32_t sh[48];
    const int keys = u.B * u.Hk * nt, rows = u.B * u.Hk * nr;
    int i = blockIdx.x;
    if (i < rows) {  // the longer jobs first
        const int bh = i / nr;
        split_rows<DP, VEC>(u, p, bh / u.Hk, bh % u.Hk, i % nr, i, ro, lds, sh);
    } else {
        i -= rows;
        const int at = i % keys, bh = at / nt;
        const bool v = i >= keys;
        split_keys<DP, VEC>(u, v ? p.v : p.k, p.ldkv, bh / u.Hk, bh % u.Hk, at % nt, at, v ? vo : ko, lds, sh);
    }
}

// What a row and a key make of each other by plain sums: p in *pr, d loss / d (q . k) / scale in *ds. 16 lanes hold the
// vectors.
template <int NC>
struct Pair {
    floatx4 q[NC], g[NC];
    float m, rl, delta, slope;
    int pos, doc;
    int64_t tok;
    int h;
    __device__ __forceinline__ void row(const Rule &u, const Ptrs &p, int b, int hk, int rr, int l16) {
        const Row r = row_of(u, hk, rr);
        tok = (int64_t)b * u.lq + r.t;
        h = r.h;
        const int64_t sr = stat_at(u, b, r), all = (int64_t)u.B * u.Hk * u.G * u.lq;
        float dot = 0.0f;
#pragma unroll
        for (int n = 0; n < NC; n++) {
            const int c = 64 * n + 4 * l16;
            q[n] = load4<false>(p.q + tok * p.ldq + (int64_t)h * u.d, c, u.d);
            g[n] = load4<false>(p.g + tok * p.ldg + (int64_t)h * u.d, c, u.d);
            const floatx4 o = load4<false>(p.o + tok * p.ldo + (int64_t)h * u.d, c, u.d);
#pragma unroll
            for (int e = 0; e < 4; e++) dot = __builtin_fmaf(g[n][e], o[e], dot);
        }
        delta = row_sum(dot);
        m = p.st[sr];
        rl = p.st[all + sr];
        pos = r.t + u.off;
        doc = rl == 0.0f ? -1 : u.qd ? u.qd[tok] : 0;
        slope = u.slopes ? u.slopes[h] * kLog2e : 0.0f;
    }
    __device__ __forceinline__ bool sees(const Rule &u, int j, int kd, int pre) const {
        return doc >= 0 && doc == kd && in_reach(u, pos - j, j, pre);
    }
    __device__ __forceinline__ void grads(const Rule &u, const floatx4 (&k)[NC], const floatx4 (&v)[NC], int j, float &pr,
                                          float &ds) const {
        float s = 0.0f, dp = 0.0f, th;
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s = __builtin_fmaf(q[n][e], k[n][e], s);
                dp = __builtin_fmaf(g[n][e], v[n][e], dp);
            }
        float x = score(u, row_sum(s), th);
        const int gap = pos - j;
        if (u.slopes) x = __builtin_fmaf(-slope, (float)(gap < 0 ? -gap : gap), x);
        pr = exp2_hw(x - m) * rl;
        ds = pr * (row_sum(dp) - delta) * (1.0f - th * th);
    }
};
// Sum of the four streams' values, the same in each.
__device__ __forceinline__ float join4(float v) {
    const int l16 = threadIdx.x & 15;
    float s = 0.0f;
    for (int o = 0; o < 4; o++) s += __shfl(v, l16 + 16 * o, 64);
    return s;
}

// dq of one row over keys lo .. hi by one wavefront, to `to`.
template <int DP>
__device__ __forceinline__ void plain_dq(const Rule &u, const Ptrs &p, int b, int hk, int rr, int lo, int hi, int pre, float *to,
                                         int acc) {
    constexpr int NC = (DP + 63) / 64;
    const int lane = threadIdx.x & 63, l16 = lane & 15, st = lane >> 4;
    Pair<NC> r;
    r.row(u, p, b, hk, rr, l16);
    floatx4 dq[NC], k[NC], v[NC];
#pragma unroll
    for (int n = 0; n < NC; n++) dq[n] = floatx4{0.f, 0.f, 0.f, 0.f};
    const int64_t base = (int64_t)b * u.lk;
    for (int j = lo + st; j <= hi; j += 4) {
        if (!r.sees(u, j, u.kd ? u.kd[base + j] : 0, pre)) continue;
#pragma unroll
        for (int n = 0; n < NC; n++) {
            k[n] = load4<false>(p.k + (base + j) * p.ldkv + (int64_t)hk * u.d, 64 * n + 4 * l16, u.d);
            v[n] = load4<false>(p.v + (base + j) * p.ldkv + (int64_t)hk * u.d, 64 * n + 4 * l16, u.d);
        }
        float pr, ds;
        r.grads(u, k, v, j, pr, ds);
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) dq[n][e] = __builtin_fmaf(ds, k[n][e], dq[n][e]);
    }
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float s = join4(dq[n][e]) * u.scale;
            const int c = 64 * n + 4 * l16 + e;
            if (st == 0 && c < u.d) to[c] = acc ? to[c] + s : s;
        }
}

// dk and dv of one key over rows r0 .. r1 - 1 by one wavefront; `pk` (dk) and `pv` (dv) are where they go.
template <int DP>
__device__ __forceinline__ void plain_dkv(const Rule &u, const Ptrs &p, int b, int hk, int j, int r0, int r1, int pre, float *pk,
                                          float *pv, int acc) {
    constexpr int NC = (DP + 63) / 64;
    const int lane = threadIdx.x & 63, l16 = lane & 15, st = lane >> 4;
    const int64_t key = (int64_t)b * u.lk + j;
    floatx4 dk[NC], dv[NC], k[NC], v[NC];
#pragma unroll
    for (int n = 0; n < NC; n++) {
        k[n] = load4<false>(p.k + key * p.ldkv + (int64_t)hk * u.d, 64 * n + 4 * l16, u.d);
        v[n] = load4<false>(p.v + key * p.ldkv + (int64_t)hk * u.d, 64 * n + 4 * l16, u.d);
        dk[n] = dv[n] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    const int kd = u.kd ? u.kd[key] : 0;
    for (int rr = r0 + st; rr < r1; rr += 4) {
        Pair<NC> r;
        r.row(u, p, b, hk, rr, l16);
        if (!r.sees(u, j, kd, pre)) continue;
        float pr, ds;
        r.grads(u, k, v, j, pr, ds);
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                dv[n][e] = __builtin_fmaf(pr, r.g[n][e], dv[n][e]);
                dk[n][e] = __builtin_fmaf(ds, r.q[n][e], dk[n][e]);
            }
    }
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float sk = join4(dk[n][e]) * u.scale, sv = join4(dv[n][e]);
            const int c = 64 * n + 4 * l16 + e;
            if (st == 0 && c < u.d) {
                if (pk) pk[c] = acc ? pk[c] + sk : sk;
                if (pv) pv[c] = acc ? pv[c] + sv : sv;
            }
        }
}

// D is split at a scale of its lane's own, a running 2^s like a softmax's maximum: a lane's sums all belong to one row (or
// key), so they move with it when a block's largest |D| outgrows 2^15 of it. What a row with small values or a key with small
// weights adds up then keeps its bits whatever its neighbours hold.
constexpr int kNoScale = -100;
__device__ __forceinline__ float ldexp_hw(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }
// The scale's exponent after a block whose largest magnitude is `top`.
__device__ __forceinline__ int grown(float top, int s) {
    const int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
    return e - s > 14 ? e - 10 : s;
}

// Four consecutive values of a result row, added to or written.
__device__ __forceinline__ void put4(float *to, int c, int d, floatx4 v, int acc) {
    if (c + 3 < d && (((uintptr_t)(to + c)) & 15) == 0) {
        floatx4 *t = reinterpret_cast<floatx4 *>(to + c);
        *t = acc ? *t + v : v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (c + e < d) to[c + e] = acc ? to[c + e] + v[e] : v[e];
    }
}

// ---------------------------------------------------------------------------------------------------- dk and dv
// Either role's tables in LDS, by blocks of the other side: whether the block is visited (documents).
struct Tables {
    uint32_t red[8][4];
    unsigned char see[kListed];
};
template <int DP, int PARTS>
__device__ __forceinline__ void keys_role(const Rule &u, const Ptrs &p, const BwdArgs &a, int i, char *sh, Tables &tab) {
    constexpr bool DOCS = PARTS & kDocs, CAP = PARTS & kCap, SLOPES = PARTS & kSlopes;
    constexpr int NW = waves_of(DP), S = DP / 16, ND = DP / 32, HALF = kStep * DP * 4, STAGE = 4 * HALF + 1024;  // the rows' record last
    auto &red = tab.red;
    const Place pl = place_of(i, u.B * u.Hk);
    const int item = pl.item, split = pl.block % a.nsplit, kb = pl.block / a.nsplit;
    const int b = item / u.Hk, hk = item - b * u.Hk;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const int pre = u.prefix ? u.prefix[b] : 0;
    const int first = kb * kKeys, last = min(first + kKeys, u.lk) - 1;
    const int own = first + 32 * (w & 3);  // the wavefront's keys; the second four of eight have those of the first
    const int j = own + (lane & 31);
    const bool live = own <= last;
    const int kd = j <= last ? (DOCS ? u.kd[(int64_t)b * u.lk + j] : 0) : -1;
    const int64_t kt0 = (int64_t)item * a.nt, rt0 = (int64_t)item * a.nr;
    // the wavefront's block of keys (a wavefront past the last key repeats it and stores nothing)
    const int t = min(own / kBlock, a.nt - 1);
    const Stats ks = a.ks[kt0 + t], vs = a.vs[kt0 + t];
    const int tb = min(first / kBlock + 1, a.nt - 1);
    const Stats v0 = a.vs[kt0 + first / kBlock], v1 = a.vs[kt0 + tb], k0 = a.ks[kt0 + first / kBlock], k1 = a.ks[kt0 + tb];
    bool bad = max(max(v0.top, v1.top), max(k0.top, k1.top)) > kMostBits;
    const int kdlo = min(k0.doc_lo, k1.doc_lo), kdhi = max(k0.doc_hi, k1.doc_hi);
    // documents of the wavefront's own keys (those past the last one aside)
    int wlo = 0, whi = 0;
    if (DOCS) {
        wlo = __builtin_amdgcn_readfirstlane(wave_imin(j <= last ? kd : INT32_MAX));
        whi = __builtin_amdgcn_readfirstlane(wave_imax(j <= last ? kd : INT32_MIN));
    }
    // the blocks of rows that may see them
    int r0, r1;  // r1: one past the last
    row_range(u, first, last, pre, r0, r1);
    const int t0 = r0 / kBlock, t1 = r1 <= r0 ? t0 - 1 : (r1 - 1) / kBlock;
    uint32_t qt = 0, ql = 0xFFFFFFFFu, qnorm = 0;
    RowStats mine = {};  // the thread's first
    for (int rt = t0 + (int)threadIdx.x, n = 0; rt <= t1; rt += 64 * NW, n++) {
        const RowStats r = a.rs[rt0 + rt];
        if (n == 0) mine = r;
        bad = bad || r.bad;
        qt = max(qt, r.q2_top);
        qnorm = max(qnorm, __float_as_uint(r.norm));
        if (r.q2_top) ql = min(ql, r.q2_top);
    }
    if (DOCS && threadIdx.x < kListed && t0 + (int)threadIdx.x <= t1) {
        static_assert(kListed == 256, "a thread's first block is its entry");
        tab.see[threadIdx.x] = mine.doc_hi >= max(kdlo, 0) && mine.doc_lo <= kdhi && (mine.g2_top || mine.q2_top);
    }
    qt = wave_umax(qt);
    ql = wave_umin(ql);
    qnorm = wave_umax(qnorm);
    const uint32_t wave_bad = __any(bad) ? 1 : 0;
    if (lane == 0) {
        red[w][0] = qt;
        red[w][1] = ql;
        red[w][2] = wave_bad;
        red[w][3] = qnorm;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NW; n++) {
        qt = max(qt, red[n][0]);
        ql = min(ql, red[n][1]);
        bad = bad || red[n][2];
        qnorm = max(qnorm, red[n][3]);
    }
    bad = bad || !scores_fit(u, __uint_as_float(qnorm), larger(k0.norm, k1.norm));
    // dk's sums move between the blocks' scales: keep the largest move inside fp32
    bad = bad || (qt && (qt >> 23) - (ql >> 23) > 60);
    auto dest = [&](int n, int jj) -> float * {  // dk (0) or dv (1) of key jj
        if (a.part) return a.part + (((int64_t)split * u.B * u.Hk + item) * u.lk + jj) * 2 * u.d + n * u.d;
        float *base = n ? p.dv : p.dk;
        return base ? base + ((int64_t)b * u.lk + jj) * p.lddkv + (int64_t)hk * u.d : nullptr;
    };
    const int acc = a.part ? 0 : p.acc;
    if (__builtin_amdgcn_readfirstlane(bad)) {
        constexpr int EACH = kKeys / NW;
        const int per = (t1 - t0 + a.nsplit) / a.nsplit * kBlock, s0 = t0 * kBlock + split * per;  // the split's equal share
        r1 = max(r0, min(r1, s0 + per));
        r0 = min(max(r0, s0), r1);
        for (int jj = first + EACH * w; jj <= min(last, first + EACH * w + EACH - 1); jj++)
            plain_dkv<DP>(u, p, b, hk, jj, r0, r1, pre, dest(0, jj), dest(1, jj), acc);
        return;
    }
    // K and V fragments of the wavefront's keys
    u32x4 kh[S], km[S], vh[NW == 4 ? S : 1], vm[NW == 4 ? S : 1];  // the second four of eight have V's in kh, km
    {
        const int half = (own / 32) & 1;
        const char *kf = a.kn + (kt0 + t) * plane_bytes(DP, 1) + half * HALF + lane * 16;
        const char *vf = a.vn + (kt0 + t) * plane_bytes(DP, 1) + half * HALF + lane * 16;
#pragma unroll
        for (int s = 0; s < S; s++) {
            const char *f = NW == 8 && w >= 4 ? vf : kf;
            kh[s] = *reinterpret_cast<const u32x4 *>(f + (2 * s) * 1024);
            km[s] = *reinterpret_cast<const u32x4 *>(f + (2 * s + 1) * 1024);
            if constexpr (NW == 4) {
                vh[s] = *reinterpret_cast<const u32x4 *>(vf + (2 * s) * 1024);
                vm[s] = *reinterpret_cast<const u32x4 *>(vf + (2 * s + 1) * 1024);
            }
        }
    }
    const Reach reach = rows_seeing(u, j, kd, pre);
    // sums of dk and dv; of eight wavefronts each has one of them, in `dk`
    floatx16 dk[ND], dv[ND];
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            dk[n][e] = 0.0f;
            dv[n][e] = 0.0f;
        }
    float q2cur = 1.0f;
    int sd = kNoScale, sv = kNoScale;  // dk's sums are in units of 2^sd q2cur, dv's in units of 2^sv
    // The split has every nsplit-th block. They are taken downwards, and from a multiple of `period` blocks on, round the
    // range's ends: workgroups of other keys that run meanwhile then read the same blocks, under a causal rule from the last
    // row on, in a window at the same remainder, and find them in their XCD's L2. (Each from its own first row, a window of
    // 1024 at 8192 rows of 4 heads of 128 missed L2 in two of three reads and was bound by that.)
    const int base = t0 * kBlock, nb = t1 - t0 + 1, first_step = (r0 - base) / kStep, last_step = r1 <= r0 ? -1 : (r1 - 1 - base) / kStep;
    const int cut = max((t1 + 1) / a.kperiod * a.kperiod - t0, 0);
    auto top = [&](int bl) { return 2 * (bl - (t0 + bl - split + a.nsplit) % a.nsplit) + 1; };  // the split's last step up to block bl
    int stop = 0;
    bool more = cut > 0;
    auto settle = [&](int it) {  // the first step from `it` on that is the split's to take; -1 behind the last
        while (true) {
            if (it < stop) {
                if (!more) return -1;
                more = false;
                it = top(nb - 1);
                stop = 2 * cut;
            } else if ((it > last_step) | (it < first_step) || (DOCS && it / 2 < kListed && !tab.see[it / 2])) {
                it = it & 1 ? it - 1 : it + 1 - 2 * a.nsplit;
            } else {
                return it;
            }
        }
    };
    auto next = [&](int it) { return settle(it & 1 ? it - 1 : it + 1 - 2 * a.nsplit); };
    const RowBand band(u, own, min(own + 31, last), pre);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)(sh + 256);
    auto stage = [&](int it, int buf) {
        const int64_t off = (rt0 + t0) * plane_bytes(DP, 1) + (int64_t)it * HALF + lane * 16;
        const uint32_t to = lds0 + (uint32_t)(buf * STAGE);
        auto one = [&](const char *src, int n) {
#pragma unroll
            for (int q = 0; q < HALF / 1024; q += NW)
                if (HALF / 1024 % NW == 0 || q + w < HALF / 1024)
                    load_to_lds(src + off + (q + w) * 1024, to + (uint32_t)(n * HALF + (q + w) * 1024));
        };
        one(a.qn, 0);
        one(a.gn, 1);
        one(a.g2, 2);
        one(a.q2, 3);
        if (w == 0) load_to_lds(a.v + row_value((rt0 + t0) * kBlock + (int64_t)it * kStep, 0) + 4 * lane, to + 4 * HALF);
    };
    int it = settle(top((more ? cut : nb) - 1)), buf = 0;
    if (it >= 0) stage(it, 0);
    while (it >= 0) {
        land<0>();
        const int nx = next(it);
        if (nx >= 0) stage(nx, buf ^ 1);
        const int f0 = base + it * kStep, f1 = f0 + kStep - 1;
        const char *qf = sh + 256 + buf * STAGE + lane * 16, *gf = qf + HALF, *g2f = gf + HALF, *q2f = g2f + HALF;
        const float *rec = reinterpret_cast<const float *>(sh + 256 + buf * STAGE + 4 * HALF), *rv = rec + 4 * g;
        const float *blk = rec + 32 * kRowBlock;
        bool some = live & band.some(f0, f1), one = true;
        if (DOCS) {
            const int dlo = __builtin_amdgcn_readfirstlane(__float_as_int(blk[2]));
            const int dhi = __builtin_amdgcn_readfirstlane(__float_as_int(blk[3]));
            some = some & (whi >= 0) & (dhi >= wlo) & (dlo <= whi);
            one = (wlo == whi) & (dlo == dhi) & (dlo == wlo) & (wlo >= 0);
        }
        floatx16 x, dp;
        const float sq = blk[0], sq2 = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(blk[1])));
        auto move = [&](float to) {  // dk's sums to another block's scale
            if (to == q2cur) return;
            const float c = q2cur / to;
#pragma unroll
            for (int n = 0; n < ND; n++) dk[n] *= c;
            q2cur = to;
        };
        auto fit = [&](floatx16(&sum)[ND], int &s, float top) {  // sums to a scale that holds `top`, the lane's and its pair's largest
            const int sn = grown(pair_max(top), s);
            if (__any(sn != s)) {
                const int by = s - sn;
#pragma unroll
                for (int n = 0; n < ND; n++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sum[n][e] = ldexp_hw(sum[n][e], by);
                s = sn;
            }
            return pow2(-s);
        };
        // scores as the forward summed them, bit for bit where the operands are
        auto products = [&](floatx16 &out, const char *f, const u32x4 *fh, const u32x4 *fm) {
#pragma unroll
            for (int e = 0; e < 16; e++) out[e] = 0.0f;
#pragma unroll
            for (int s = 0; s < S; s++)
                out = mma3_t(*reinterpret_cast<const u32x4 *>(f + (2 * s) * 1024),
                             *reinterpret_cast<const u32x4 *>(f + (2 * s + 1) * 1024), fh[s], fm[s], out);
        };
        // x from raw products to weights E 2^ge; `keep(e, w)` gets them times 1 - tanh^2
        auto weights = [&](auto keep) {
            const float cs = sq * ks.scale;
            const bool whole = band.all(f0, f1) & one;
            if (CAP) {
                const float ic = u.icap * cs;
                float big = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e++) big = fmaxf(big, __builtin_fabsf(x[e]));
                const bool small = !__any(big * __builtin_fabsf(ic) >= kTanhSmall);
#pragma unroll
                for (int e = 0; e < 16; e++) x[e] *= ic;
                if (small) {
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = tanh_small(x[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = tanh_any(x[e]);
                }
            }
            const float fx = CAP ? u.capl2 : u.cl2 * cs;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const floatx4 m4 = *reinterpret_cast<const floatx4 *>(rv + 32 * kRowM + 8 * q);
                floatx4 y;
#pragma unroll
                for (int r = 0; r < 4; r++) y[r] = SLOPES ? x[4 * q + r] * fx : __builtin_fmaf(x[4 * q + r], fx, m4[r]);
                if (SLOPES || !whole) {
                    const intx4 p4 = *reinterpret_cast<const intx4 *>(rv + 32 * kRowPos + 8 * q);
                    if (SLOPES) {  // each rounding as in the forward, so that a score that is mostly bias cancels with its maximum
                        const floatx4 s4 = *reinterpret_cast<const floatx4 *>(rv + 32 * kRowSlope + 8 * q);
#pragma unroll
                        for (int r = 0; r < 4; r++) y[r] = __builtin_fmaf(-s4[r], __builtin_fabsf((float)(p4[r] - j)), y[r]) + m4[r];
                    }
                    if (!whole) {
                        intx4 qd = {kd, kd, kd, kd};
                        if (DOCS) qd = *reinterpret_cast<const intx4 *>(rv + 32 * kRowDoc + 8 * q);
#pragma unroll
                        for (int r = 0; r < 4; r++) y[r] = (reach.has(p4[r]) & (qd[r] == kd)) ? y[r] : -3e38f;
                    }
                }
                const floatx4 w4 = *reinterpret_cast<const floatx4 *>(rv + 32 * kRowGrad + 8 * q);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int e = 4 * q + r;
                    const float ex = exp2_hw(y[r]) * w4[r], th = x[e];
                    x[e] = ex;
                    keep(e, CAP ? ex * __builtin_fmaf(-th, th, 1.0f) : ex);
                }
            }
        };
        // dp from g . v to D 2^ge, given E 2^ge (1 - tanh^2); what D is multiplied with before it is split
        auto gradient = [&](const floatx16 &e1) -> float {
            float top = 0.0f;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const floatx4 d4 = *reinterpret_cast<const floatx4 *>(rv + 32 * kRowDelta + 8 * q);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int e = 4 * q + r;
                    dp[e] = e1[e] * __builtin_fmaf(dp[e], vs.scale, -d4[r]);
                    top = fmaxf(top, __builtin_fabsf(dp[e]));
                }
            }
            return fit(dk, sd, top);
        };
        auto largest = [&]() {  // of the weights, which are not negative
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e++) top = fmaxf(top, x[e]);
            return top;
        };
        auto add_half = [&](floatx16(&sum)[ND], const char *f, const floatx16 &v, float by, int s) {  // 16 of the step's rows
            float e8[8];
            u32x4 h, m;
#pragma unroll
            for (int e = 0; e < 8; e++) e8[e] = v[8 * s + e] * by;
            split8(e8, h, m);
#pragma unroll
            for (int c = 0; c < ND; c++) {
                const char *at = f + ((s * ND + c) * 2) * 1024;
                sum[c] = mma3(*reinterpret_cast<const u32x4 *>(at), *reinterpret_cast<const u32x4 *>(at + 1024), h, m, sum[c]);
            }
        };
        if constexpr (NW == 4) {
            if (some) {
                move(sq2);
                products(x, qf, kh, km);
                products(dp, gf, vh, vm);
                floatx16 e1;
                weights([&](int e, float v) { e1[e] = v; });
                const float fe = fit(dv, sv, largest()), fd = gradient(e1);
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    add_half(dv, g2f, x, fe, s);
                    add_half(dk, q2f, dp, fd, s);
                }
            }
        } else {
            // a wavefront's and its partner's registers hold the same rows and key: the weights pass lane by lane
            floatx4 *pass = reinterpret_cast<floatx4 *>(sh + 256 + 2 * STAGE + (w & 3) * 4096) + lane;
            if (some && w < 4) {
                products(x, qf, kh, km);
                floatx4 e4;
                weights([&](int e, float v) {
                    e4[e & 3] = v;
                    if ((e & 3) == 3) pass[64 * (e >> 2)] = e4;
                });
            } else if (some) {
                products(dp, gf, kh, km);
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (some && w < 4) {
                const float fe = fit(dk, sv, largest());
#pragma unroll
                for (int s = 0; s < 2; s++) add_half(dk, g2f, x, fe, s);
            } else if (some) {
                move(sq2);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const floatx4 e4 = pass[64 * q];
#pragma unroll
                    for (int r = 0; r < 4; r++) x[4 * q + r] = e4[r];
                }
                const float fd = gradient(x);
#pragma unroll
                for (int s = 0; s < 2; s++) add_half(dk, q2f, dp, fd, s);
            }
        }
        it = nx;
        buf ^= 1;
    }
    if (j > last) return;
    const float fv = pow2(-kLift), fk = q2cur * pow2(-kLift) * u.scale;
    const bool has_v = NW == 4 || w < 4, has_k = NW == 4 || w >= 4;
    float *tk = has_k ? dest(0, j) : nullptr, *tv = has_v ? dest(1, j) : nullptr;
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int c = 32 * n + 8 * q + 4 * g;
            const floatx16 &dvn = dv[n];
            const floatx4 xk = floatx4{dk[n][4 * q], dk[n][4 * q + 1], dk[n][4 * q + 2], dk[n][4 * q + 3]};
            const floatx4 xv = NW == 4 ? floatx4{dvn[4 * q], dvn[4 * q + 1], dvn[4 * q + 2], dvn[4 * q + 3]} : xk;
            if (tk) {
                floatx4 y;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = ldexp_hw(xk[e], sd) * fk;
                put4(tk, c, u.d, y, acc);
            }
            if (tv) {
                floatx4 y;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = ldexp_hw(xv[e], sv) * fv;
                put4(tv, c, u.d, y, acc);
            }
        }
}

// ------------------------------------------------------------------------------------------------------------ dq
template <int DP, int PARTS>
__device__ __forceinline__ void rows_role(const Rule &u, const Ptrs &p, const BwdArgs &a, int i, char *sh, Tables &tab) {
    constexpr bool DOCS = PARTS & kDocs, CAP = PARTS & kCap, SLOPES = PARTS & kSlopes;
    constexpr int NW = waves_of(DP), ROWS = 32 * NW, S = DP / 16, ND = DP / 32, HALF = kStep * DP * 4, STAGE = 3 * HALF + 4 * kKeyWords;  // the step's words last
    auto &red = tab.red;
    const Place pl = place_of(i, u.B * u.Hk);
    const int item = pl.item, split = pl.block % a.qsplit, rb = a.rblocks - 1 - pl.block / a.qsplit;
    const int b = item / u.Hk, hk = item - b * u.Hk, rows = u.G * u.lq;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const int pre = u.prefix ? u.prefix[b] : 0;
    const int first = rb * ROWS, last = min(first + ROWS, rows) - 1;
    const int own = first + 32 * w, rr = own + (lane & 31);
    const Row row = row_of(u, hk, min(rr, rows - 1));
    const int64_t tok = (int64_t)b * u.lq + row.t;
    const int pos = row.t + u.off, doc = DOCS ? u.qd[tok] : 0;
    const float slope = SLOPES ? u.slopes[row.h] * kLog2e : 0.0f;
    const bool live = own <= last;
    const int64_t kt0 = (int64_t)item * a.nt, rt0 = (int64_t)item * a.nr;
    const int rt = min(own / kBlock, a.nr - 1);
    const RowStats rs = a.rs[rt0 + rt];
    bool bad = false;
    float qnorm = 0.0f;
    int qlo = INT32_MAX, qhi = INT32_MIN;
#pragma unroll
    for (int n = 0; n < ROWS / kBlock; n++) {
        const RowStats r = a.rs[rt0 + min(first / kBlock + n, a.nr - 1)];
        bad = bad || (r.bad & kBadRows);
        qnorm = larger(qnorm, r.norm);
        qlo = min(qlo, r.doc_lo);
        qhi = max(qhi, r.doc_hi);
    }
    int lo, hi;
    const int i0 = first / u.G + u.off, i1 = last / u.G + u.off;
    key_range(u, i0, i1, pre, lo, hi);
    // the split's equal share of the blocks
    const int c0 = lo / kBlock, c1 = hi < lo ? c0 - 1 : hi / kBlock, per = (c1 - c0 + a.qsplit) / a.qsplit;
    const int t0 = c0 + split * per, t1 = min(c1, t0 + per - 1);
    lo = max(lo, t0 * kBlock);
    hi = min(hi, t1 * kBlock + kBlock - 1);
    auto dest = [&](int r, const Row &to) {  // dq of row r
        return a.qpart ? a.qpart + (((int64_t)split * u.B * u.Hk + item) * rows + r) * u.d
                       : p.dq + ((int64_t)b * u.lq + to.t) * p.lddq + (int64_t)to.h * u.d;
    };
    const int acc = a.qpart ? 0 : p.acc;
    uint32_t kt = 0, vt = 0, kl = 0xFFFFFFFFu, knorm = 0;
    Stats mk = {};  // the thread's first
    for (int t = t0 + (int)threadIdx.x, n = 0; t <= t1; t += 64 * NW, n++) {
        const Stats sk = a.ks[kt0 + t], sv = a.vs[kt0 + t];
        if (n == 0) mk = sk;
        kt = max(kt, sk.columns ? sk.top : 0xFFFFFFFFu);
        knorm = max(knorm, __float_as_uint(sk.norm));
        kl = min(kl, sk.low);
        vt = max(vt, sv.top);
    }
    kt = wave_umax(kt);
    vt = wave_umax(vt);
    kl = wave_umin(kl);
    knorm = wave_umax(knorm);
    if (lane == 0) {
        red[w][0] = kt;
        red[w][1] = vt;
        red[w][2] = kl;
        red[w][3] = knorm;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NW; n++) {
        kt = max(kt, red[n][0]);
        vt = max(vt, red[n][1]);
        kl = min(kl, red[n][2]);
        knorm = max(knorm, red[n][3]);
    }
    bad = bad || !scores_fit(u, qnorm, __uint_as_float(knorm)) || kt > kMostBits || vt > kMostBits || !even_rows(kt, kl);
    if (__builtin_amdgcn_readfirstlane(bad)) {
        for (int r = own; r <= min(last, own + 31); r++) plain_dq<DP>(u, p, b, hk, r, lo, hi, pre, dest(r, row_of(u, hk, r)), acc);
        return;
    }
    const int ek = kt ? scale_exp(kt) : 0;
    int wlo = 0, whi = 0;  // documents of the wavefront's rows
    if (DOCS) {
        wlo = __builtin_amdgcn_readfirstlane(wave_imin(doc));
        whi = __builtin_amdgcn_readfirstlane(wave_imax(doc));
    }
    if (DOCS) {
        if (threadIdx.x < kListed && t0 + (int)threadIdx.x <= t1) {
            static_assert(kListed == 256, "a thread's first block is its entry");
            tab.see[threadIdx.x] = mk.doc_hi >= max(qlo, 0) && mk.doc_lo <= qhi;
        }
        __syncthreads();
    }
    // Q and G fragments of the wavefront's rows, and their values
    u32x4 qh[S], qm[S], gh[S], gm[S];
    {
        const int half = own / 32 & 1;
        const char *qf = a.qn + (rt0 + rt) * plane_bytes(DP, 1) + half * HALF + lane * 16;
        const char *gf = a.gn + (rt0 + rt) * plane_bytes(DP, 1) + half * HALF + lane * 16;
#pragma unroll
        for (int s = 0; s < S; s++) {
            qh[s] = *reinterpret_cast<const u32x4 *>(qf + (2 * s) * 1024);
            qm[s] = *reinterpret_cast<const u32x4 *>(qf + (2 * s + 1) * 1024);
            gh[s] = *reinterpret_cast<const u32x4 *>(gf + (2 * s) * 1024);
            gm[s] = *reinterpret_cast<const u32x4 *>(gf + (2 * s + 1) * 1024);
        }
    }
    const int64_t at = rt0 * kBlock + min(rr, a.nr * kBlock - 1);
    const float m = a.v[row_value(at, kRowM)], delta = a.v[row_value(at, kRowDelta)], wr = a.v[row_value(at, kRowW)];
    const Reach reach = keys_seen(u, pos, doc, pre);
    floatx16 dq[ND];
    int sd = kNoScale;  // dq's sums are in units of 2^sd
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int e = 0; e < 16; e++) dq[n][e] = 0.0f;
    const int wi0 = min(own, last) / u.G + u.off, wi1 = min(own + 31, last) / u.G + u.off;
    const int base = t0 * kBlock, steps = hi < lo ? 0 : (hi - base) / kStep + 1;
    const Band whole_wg(u, i0, i1, pre), mine(u, wi0, wi1, pre);
    // Keys upwards, in a window from a multiple of `period` steps on and round the range's end: see the keys' role.
    const int abs0 = base / kStep, up = (abs0 + a.rperiod - 1) / a.rperiod * a.rperiod - abs0, cut = up < steps ? up : 0;
    int stop = steps;
    bool more = cut > 0;
    auto settle = [&](int it) {  // the first step from `it` on to take; -1 behind the last
        while (true) {
            const int j0 = base + it * kStep;
            if (it >= stop) {
                if (!more) return -1;
                more = false;
                it = 0;
                stop = cut;
            } else if ((j0 >= whole_wg.pre) & (j0 + kStep <= whole_wg.some0)) {  // a window leaves a gap behind a prefix
                it = (whole_wg.some0 - base) / kStep;
            } else if (DOCS && it / 2 < kListed && !tab.see[it / 2]) {
                it++;
            } else {
                return it;
            }
        }
    };
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)(sh + 256);
    auto stage = [&](int it, int buf) {
        const int64_t off = (kt0 + t0) * plane_bytes(DP, 1) + (int64_t)it * HALF + lane * 16;
        const uint32_t to = lds0 + (uint32_t)(buf * STAGE);
        auto one = [&](const char *src, int n) {
#pragma unroll
            for (int q = 0; q < HALF / 1024; q += NW)
                if (HALF / 1024 % NW == 0 || q + w < HALF / 1024)
                    load_to_lds(src + off + (q + w) * 1024, to + (uint32_t)(n * HALF + (q + w) * 1024));
        };
        one(a.kn, 0);
        one(a.vn, 1);
        one(a.kt, 2);
        if (w == 0) load_to_lds4(a.keys + (2 * (kt0 + t0) + it) * kKeyWords + lane, to + 3 * HALF);
    };
    int it = settle(cut), buf = 0;
    if (it >= 0) stage(it, 0);
    while (it >= 0) {
        land<0>();
        const int nx = settle(it + 1);
        if (nx >= 0) stage(nx, buf ^ 1);
        const int j0 = base + it * kStep, j1 = j0 + kStep - 1;
        const char *kf = sh + 256 + buf * STAGE + lane * 16, *vf = kf + HALF, *ktf = vf + HALF;
        const int *words = reinterpret_cast<const int *>(sh + 256 + buf * STAGE + 3 * HALF);
        bool some = live & mine.some(j0, j1), one = true;
        if (DOCS) {
            const int dlo = __builtin_amdgcn_readfirstlane(words[kKeyDocLo]), dhi = __builtin_amdgcn_readfirstlane(words[kKeyDocHi]);
            some = some & (whi >= 0) & (dhi >= wlo) & (dlo <= whi);
            one = (wlo == whi) & (dlo == dhi) & (dlo == wlo) & (wlo >= 0);
        }
        const float sk = __int_as_float(words[kKeyScaleK]), sv = __int_as_float(words[kKeyScaleV]);
        floatx16 x, dp;
        auto products = [&](floatx16 &out, const char *f, const u32x4 *fh, const u32x4 *fm) {
#pragma unroll
            for (int e = 0; e < 16; e++) out[e] = 0.0f;
#pragma unroll
            for (int s = 0; s < S; s++)
                out = mma3(*reinterpret_cast<const u32x4 *>(f + (2 * s) * 1024),
                           *reinterpret_cast<const u32x4 *>(f + (2 * s + 1) * 1024), fh[s], fm[s], out);
        };
        // x from raw products to the weights E (1 - tanh^2)
        auto weights = [&]() {
            // K's exponent less the largest; a block of zeros may say anything
            const int step = min(max((words[kKeyScaleK] >> 23) - 127 - ek, -32), 0);
            const float cs = rs.q * sk;
            const bool whole = mine.all(j0, j1) & one;
            if (CAP) {
                const float ic = u.icap * cs;
                float big = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e++) big = fmaxf(big, __builtin_fabsf(x[e]));
                const bool small = !__any(big * __builtin_fabsf(ic) >= kTanhSmall);
#pragma unroll
                for (int e = 0; e < 16; e++) x[e] *= ic;
                if (small) {
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = tanh_small(x[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = tanh_any(x[e]);
                }
            }
            const float fx = CAP ? u.capl2 : u.cl2 * cs, mu = (float)step + m;
            const float gap0 = (float)(pos - j0 - 4 * g);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int o = 8 * (e >> 2) + (e & 3);
                float y = SLOPES ? __builtin_fmaf(-slope, __builtin_fabsf(gap0 - (float)o), x[e] * fx) + mu : __builtin_fmaf(x[e], fx, mu);
                if (!whole) y = (reach.has(j0 + 4 * g + o) & (!DOCS || words[kKeyDoc + 4 * g + o] == doc)) ? y : -3e38f;
                const float ex = exp2_hw(y);
                x[e] = CAP ? ex * __builtin_fmaf(-x[e], x[e], 1.0f) : ex;
            }
        };
        auto rescale = [&](int sn) {  // dq's sums to units of 2^sn
            if (__any(sn != sd)) {
                const int by = sd - sn;
#pragma unroll
                for (int n = 0; n < ND; n++)
#pragma unroll
                    for (int e = 0; e < 16; e++) dq[n][e] = ldexp_hw(dq[n][e], by);
                sd = sn;
            }
        };
        auto gradient = [&]() {  // dp from g . v to D
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                dp[e] = x[e] * __builtin_fmaf(dp[e], sv, -delta);
                top = fmaxf(top, __builtin_fabsf(dp[e]));
            }
            rescale(grown(pair_max(top), sd));
        };
        auto add_half = [&](int s) {  // 16 of the step's keys
            const float fd = pow2(-sd);
            float e8[8];
            u32x4 dh, dm;
#pragma unroll
            for (int e = 0; e < 8; e++) e8[e] = dp[8 * s + e] * fd;
            split8(e8, dh, dm);
#pragma unroll
            for (int c = 0; c < ND; c++) {
                const char *f = ktf + ((s * ND + c) * 2) * 1024;
                dq[c] = mma3(*reinterpret_cast<const u32x4 *>(f), *reinterpret_cast<const u32x4 *>(f + 1024), dh, dm, dq[c]);
            }
        };
        if (some) {
            products(x, kf, qh, qm);
            products(dp, vf, gh, gm);
            weights();
            gradient();
#pragma unroll
            for (int s = 0; s < 2; s++) add_half(s);
        }
        it = nx;
        buf ^= 1;
    }
    if (rr > last) return;
    const float f = u.scale * pow2(ek - kLift);
    float *to = dest(rr, row);
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const floatx4 v = floatx4{ldexp_hw(dq[n][4 * q], sd), ldexp_hw(dq[n][4 * q + 1], sd),
                                      ldexp_hw(dq[n][4 * q + 2], sd), ldexp_hw(dq[n][4 * q + 3], sd)} * f * wr;
            put4(to, 32 * n + 8 * q + 4 * g, u.d, v, acc);
        }
}

template <int DP, int PARTS>
__global__ void __launch_bounds__(64 * waves_of(DP), DP == 128 ? 1 : 2) k_scored_bwd_mm(Rule u, Ptrs p, BwdArgs a) {
    OM_LDS_POISON();
    __shared__ __attribute__((aligned(16))) char sh[256 + 2 * (4 * kStep * DP * 4 + 1024) + (waves_of(DP) == 8 ? 16384 : 0)];
    __shared__ Tables tab;
    // The roles' workgroups in proportion, each in its order of falling work: the longest of both start first. Eight ids a
    // turn, one on each XCD, so that a role's index keeps its remainder by eight and an XCD its items.
    const int64_t id = blockIdx.x >> 3, all = gridDim.x >> 3, kg = (a.keys_wgs + 7) / 8;
    const int k = (int)(id * kg / all), x = blockIdx.x & 7;
    if ((int)((id + 1) * kg / all) > k) {
        if (8 * k + x < a.keys_wgs) keys_role<DP, PARTS>(u, p, a, 8 * k + x, sh, tab);
    } else if (8 * ((int)id - k) + x < a.rows_wgs) {
        rows_role<DP, PARTS>(u, p, a, 8 * ((int)id - k) + x, sh, tab);
    }
}

// dk and dv (`dkv` values), then dq (`dq` values), from their splits' sums, in split order; a thread per four values (or one,
// where d is no multiple of four).
template <int W>
__global__ void __launch_bounds__(256) k_scored_join_bwd(Rule u, Ptrs p, int64_t dkv, int nsplit, const float *__restrict__ part,
                                                         int64_t dq, int qsplit, const float *__restrict__ qpart) {
    OM_LDS_POISON();
    typedef float vec __attribute__((ext_vector_type(W), aligned(4)));
    int64_t f = ((int64_t)blockIdx.x * 256 + threadIdx.x) * W;
    if (f >= dkv + dq) return;
    const bool q = f >= dkv;
    const int64_t each = q ? dq : dkv;
    const float *from = q ? qpart : part;
    const int n = q ? qsplit : nsplit;
    if (q) f -= dkv;
    const int64_t row = f / u.d;  // a row's query of a head, or dk, dv of a key in turn
    const int c = (int)(f - row * u.d);
    float *to;
    if (q) {
        const int64_t rows = (int64_t)u.G * u.lq, item = row / rows;
        const Row r = row_of(u, (int)(item % u.Hk), (int)(row - item * rows));
        to = p.dq + ((item / u.Hk) * u.lq + r.t) * p.lddq + (int64_t)r.h * u.d;
    } else {
        const int64_t key = row >> 1, item = key / u.lk;
        to = row & 1 ? p.dv : p.dk;
        if (!to) return;
        to += ((item / u.Hk) * u.lk + (key - item * u.lk)) * p.lddkv + (item % u.Hk) * u.d;
    }
    vec s = *reinterpret_cast<const vec *>(from + f);
    for (int i = 1; i < n; i++) s += *reinterpret_cast<const vec *>(from + i * each + f);
    vec *out = reinterpret_cast<vec *>(to + c);
    *out = p.acc ? *out + s : s;
}

}  // namespace

namespace osc {

om_status bwd_by_matrix(om_ctx *ctx, const Rule &u, const Ptrs &p) {
    const char *what = "om_attention_bwd_scored";
    const int64_t items = (int64_t)u.B * u.Hk, rows = (int64_t)u.G * u.lq;
    const int dp = u.d <= 32 ? 32 : u.d <= 64 ? 64 : u.d <= 96 ? 96 : 128;
    BwdArgs a = {};
    a.nt = (u.lk + kBlock - 1) / kBlock;
    a.nr = (int)((rows + kBlock - 1) / kBlock);
    a.kblocks = (u.lk + kKeys - 1) / kKeys;
    const int rows_wg = 32 * waves_of(dp);
    a.rblocks = (int)((rows + rows_wg - 1) / rows_wg);
    const bool keys = p.dk || p.dv;
    // Split the rows of dk and dv until there are eight wavefronts a CU, in pieces of at least eight blocks (below, a workgroup's
    // start of 5 us and the join cost what the shorter walk saves). Half as many: 644 us for 488 at 4096 causal rows of 64
    // values, 1557 for 1363 in the window of 128; half as many again: 501 and 1342; 777 rows of 80 values with twice as many:
    // 158 for 149.
    const int64_t want = 8 / waves_of(dp) * ctx->num_cus;
    int64_t ns = 1, wk = items * a.kblocks;
    if (wk < want) ns = want / wk;
    ns = ns > a.nr / 8 ? a.nr / 8 : ns;
    ns = ns < 1 ? 1 : ns;
    a.nsplit = (int)ns;
    wk = keys ? wk * a.nsplit : 0;
    // The keys of dq alike: 32 rows of 4 heads over 4096 keys of 64 values, 225 us for the call whole, 50 us in pieces.
    int64_t qs = 1, wr = items * a.rblocks;
    if (wr < want) qs = want / wr;
    qs = qs > a.nt / 8 ? a.nt / 8 : qs;
    qs = qs < 1 ? 1 : qs;
    a.qsplit = (int)qs;
    wr = p.dq ? wr * a.qsplit : 0;
    const int64_t jobs = items * (2 * (int64_t)a.nt + a.nr);
    OM_REQUIRE(ctx, wk + wr + 64 <= most_groups(64 * waves_of(dp)) && jobs <= most_groups(256), "%s: too many row blocks", what);
    a.keys_wgs = (int)wk;
    a.rows_wgs = (int)wr;
    // a window's whole range: of rows that see a workgroup's keys, in blocks a split; of keys that its rows see, in steps
    const int64_t sides = u.causal ? 1 : 2, none = INT32_MAX / 2;
    a.kperiod = (int)(u.window ? std::min(none, (sides * u.window + kKeys) * u.G / kBlock + 1) : none);
    a.rperiod = (int)(u.window ? std::min(none, (sides * u.window + rows_wg / u.G) / kStep + 2) : none);
    const int64_t kp = plane_bytes(dp, items * a.nt), rp = plane_bytes(dp, items * a.nr);
    const int64_t vals = items * a.nr * kBlock * kRowValues * (int64_t)sizeof(float);
    const int64_t words = 2 * items * a.nt * kKeyWords * (int64_t)sizeof(float);
    const int64_t qpart = p.dq && a.qsplit > 1 ? (int64_t)sizeof(float) * a.qsplit * items * rows * u.d : 0;
    const int64_t part = keys && a.nsplit > 1 ? (int64_t)sizeof(float) * a.nsplit * items * u.lk * 2 * u.d : 0;
    const int64_t stats = 2 * items * a.nt * (int64_t)sizeof(Stats) + items * a.nr * (int64_t)sizeof(RowStats);
    float *scr;
    if (om_status s = om::scratch2(ctx, (uint64_t)(3 * kp + 4 * rp + vals + words + stats + part + qpart), &scr)) return s;
    char *at = reinterpret_cast<char *>(scr);
    auto take = [&](int64_t bytes) {
        char *x = at;
        at += bytes;
        return x;
    };
    SplitOut ko = {}, vo = {};
    RowsOut ro = {};
    a.kn = ko.rows = take(kp);
    a.kt = ko.cols = take(kp);
    a.vn = vo.rows = take(kp);
    a.qn = ro.q = take(rp);
    a.gn = ro.g = take(rp);
    a.g2 = ro.g2 = take(rp);
    a.q2 = ro.q2 = take(rp);
    a.v = ro.v = reinterpret_cast<float *>(take(vals));
    float *kw = reinterpret_cast<float *>(take(words));
    a.keys = ko.keys = vo.keys = kw;
    vo.is_v = true;
    a.part = part ? reinterpret_cast<float *>(take(part)) : nullptr;
    a.qpart = qpart ? reinterpret_cast<float *>(take(qpart)) : nullptr;
    a.ks = ko.stats = reinterpret_cast<Stats *>(take(items * a.nt * (int64_t)sizeof(Stats)));
    a.vs = vo.stats = reinterpret_cast<Stats *>(take(items * a.nt * (int64_t)sizeof(Stats)));
    a.rs = ro.stats = reinterpret_cast<RowStats *>(take(items * a.nr * (int64_t)sizeof(RowStats)));
    auto al16 = [](const void *x) { return ((uintptr_t)x & 15) == 0; };
    const bool vec = u.d % 4 == 0 && p.ldq % 4 == 0 && p.ldkv % 4 == 0 && p.ldo % 4 == 0 && p.ldg % 4 == 0 && al16(p.q) &&
                     al16(p.k) && al16(p.v) && al16(p.o) && al16(p.g);
    by_depth(u.d, [&](auto dpc) {
        constexpr int DP = decltype(dpc)::value;
        auto split = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3((unsigned)jobs), dim3(256), 0, ctx->stream, u, p, ko, vo, ro, a.nt, a.nr);
        };
        vec ? split(k_scored_split_bwd<DP, true>) : split(k_scored_split_bwd<DP, false>);
        by_parts(parts_of(u), [&](auto pc) {
            hipLaunchKernelGGL((k_scored_bwd_mm<DP, decltype(pc)::value>), dim3((unsigned)(8 * ((wk + 7) / 8 + (wr + 7) / 8))), dim3(64 * waves_of(DP)), 0,
                               ctx->stream, u, p, a);
        });
    });
    if (part || qpart) {
        const int64_t dkv = part ? items * u.lk * 2 * u.d : 0, dq = qpart ? items * rows * u.d : 0;
        auto join = [&](auto kern, int w) {
            hipLaunchKernelGGL(kern, dim3((unsigned)(((dkv + dq) / w + 255) / 256)), dim3(256), 0, ctx->stream, u, p, dkv, a.nsplit,
                               a.part, dq, a.qsplit, a.qpart);
        };
        u.d % 4 == 0 ? join(k_scored_join_bwd<4>, 4) : join(k_scored_join_bwd<1>, 1);
    }
    return OM_LAUNCH_CHECK(ctx, what);
}

}  // namespace osc
