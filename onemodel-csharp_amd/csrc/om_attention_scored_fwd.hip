// Scored attention's forward on the matrix cores (operands: om_attention_scored_mm.hpp).
//
// A workgroup takes 128 rows of one key head's group (a wavefront 32: its lanes' queries) and walks the visible keys in
// steps of 32. S^T = K Q^T leaves a query's scores in its lane's registers; they become weights E = 2^(x - m) there, are
// split, and are the operand of O^T += V^T E^T as they stand. K and V come split from scratch, straight into LDS, a
// ring of steps, one barrier each. The running maximum m moves only when some lane's maximum grows by more than 2^2: E then
// stays below 2^14 with its 2^12 of headroom, and the accumulators are left alone in most steps.
//
// Bound: a wavefront's matrix instructions and its vector work (exponents, caps, masks, splits) follow each other, so a SIMD
// runs one of them only while another wavefront is in the other; 12 heads of 64 values in 4 key heads, 4096 causal rows with
// a cap: 107 to 123 us over several runs and 14 us for the joins, 210 to 240 TFLOP/s of fp32 products where three fp16 products
// for each reach about 380.
#include <algorithm>
#include <cmath>

#include "om_attention_scored_split.hpp"

namespace {

using namespace osc;

constexpr float kInf = __builtin_inff();
constexpr int kRows = 128;      // rows of a workgroup
constexpr float kSlack = 2.0f;  // how far a maximum may outgrow m before m moves
constexpr int kListed = 256;    // blocks of keys whose documents' look stands in LDS

template <int DP, bool VEC>
__global__ void __launch_bounds__(256) k_scored_split_kv(Rule u, Ptrs p, SplitOut ko, SplitOut vo, int nt) {
    OM_LDS_POISON();
    __shared__ __attribute__((aligned(16))) char lds[DP * 256];
    __shared__ uint32_t sh[48];
    const int items = u.B * u.Hk * nt;
    const int which = blockIdx.x / items, at = blockIdx.x - which * items;
    const int t = at % nt, bh = at / nt;
    split_keys<DP, VEC>(u, which ? p.v : p.k, p.ldkv, bh / u.Hk, bh % u.Hk, t, at, which ? vo : ko, lds, sh);
}

// One row by plain fp32 sums over the keys lo .. hi, by one wavefront: 16 lanes to a key, four keys at a time. For rows
// whose operands the split cannot hold.
template <int DP>
__device__ __forceinline__ void plain_row(const Rule &u, const Ptrs &p, int b, int hk, int rr, int lo, int hi, int split, int nsplit,
                                       float *part) {
    constexpr int NC = (DP + 63) / 64;
    const int lane = threadIdx.x & 63, l16 = lane & 15, st = lane >> 4, d = u.d;
    const int pre = u.prefix ? u.prefix[b] : 0;
    const Row row = row_of(u, hk, rr);
    const int64_t tok = (int64_t)b * u.lq + row.t;
    const int doc = u.qd ? u.qd[tok] : 0, pos = row.t + u.off;
    const float slope = u.slopes ? u.slopes[row.h] * kLog2e : 0.0f;
    floatx4 q[NC], acc[NC];
    float m = -kInf, l = 0.0f;
#pragma unroll
    for (int n = 0; n < NC; n++) {
        q[n] = load4<false>(p.q + tok * p.ldq + (int64_t)row.h * d, 64 * n + 4 * l16, d);
        acc[n] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    const int64_t base = (int64_t)b * u.lk;
    for (int j = lo + st; j <= hi; j += 4) {
        const int gap = pos - j;
        if (doc < 0 || (u.kd && u.kd[base + j] != doc) || !in_reach(u, gap, j, pre)) continue;
        const float *kr = p.k + (base + j) * p.ldkv + (int64_t)hk * d, *vr = p.v + (base + j) * p.ldkv + (int64_t)hk * d;
        float s = 0.0f, th;
#pragma unroll
        for (int n = 0; n < NC; n++) {
            const floatx4 k = load4<false>(kr, 64 * n + 4 * l16, d);
#pragma unroll
            for (int e = 0; e < 4; e++) s = __builtin_fmaf(q[n][e], k[e], s);
        }
        float x = score(u, row_sum(s), th);
        if (u.slopes) x = __builtin_fmaf(-slope, (float)(gap < 0 ? -gap : gap), x);
        const float top = x > m ? x : m, mu = top == -kInf ? 0.0f : top, alpha = exp2_hw(m - mu), e1 = exp2_hw(x - mu);
        m = top;
        l = l * alpha + e1;
#pragma unroll
        for (int n = 0; n < NC; n++) {
            const floatx4 v = load4<false>(vr, 64 * n + 4 * l16, d);
#pragma unroll
            for (int e = 0; e < 4; e++) acc[n][e] = __builtin_fmaf(e1, v[e], acc[n][e] * alpha);
        }
    }
    // join the four streams
    float top = m;
    for (int o = 16; o < 64; o += 16) {
        const float x = __shfl(m, (lane + o) & 63, 64);
        top = x > top ? x : top;
    }
    const float mu = top == -kInf ? 0.0f : top, w = exp2_hw(m - mu);
    auto joined = [&](float v) {
        float s = 0.0f;
        for (int o = 0; o < 4; o++) s += __shfl(v * w, l16 + 16 * o, 64);
        return s;
    };
    const float sum = joined(l);
    const int64_t rows = (int64_t)u.G * u.lq, all = (int64_t)u.B * u.Hk * rows, at = ((int64_t)b * u.Hk + hk) * rows + rr;
    const float rl = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float a = joined(acc[n][e]);
            const int c = 64 * n + 4 * l16 + e;
            if (st == 0 && c < d) {
                if (part) part[((int64_t)split * all + at) * d + c] = a;
                else p.out[tok * p.ldo + (int64_t)row.h * d + c] = sum == 0.0f ? 0.0f : a * rl;
            }
        }
    if (lane == 0) {
        if (part) {
            float *ms = part + (int64_t)nsplit * all * d + (int64_t)split * all + at;
            ms[0] = mu;
            ms[(int64_t)nsplit * all] = sum;
        } else if (p.stats) {
            const int64_t sr = stat_at(u, b, row);
            p.stats[sr] = mu;
            p.stats[all + sr] = rl;
        }
    }
}

struct FwdArgs {
    const char *kn, *vt;      // K in rows form, V in columns form
    const Stats *ks, *vs;     // their blocks' statistics
    const float *keys;        // the steps' words
    int nt;                   // blocks of 64 keys of a head
    int blocks;               // workgroups along a head's rows
    int nsplit;               // splits of each block of rows' keys
    float *part;              // the splits' sums (om_attention_scored.hip joins them), NULL for one split
    int vec;                  // q's rows are 16-byte aligned
};

template <int DP, int PARTS>
__global__ void __launch_bounds__(256, DP == 32 ? 4 : DP == 64 ? 3 : 2) k_scored_fwd_mm(Rule u, Ptrs p, FwdArgs a) {
    OM_LDS_POISON();
    constexpr bool DOCS = PARTS & kDocs, CAP = PARTS & kCap, SLOPES = PARTS & kSlopes;
    constexpr int KT = 32, S = DP / 16, ND = DP / 32, NST = DP == 128 ? 2 : 3;  // as many stages as leave two workgroups a CU
    constexpr int HALF = KT * DP * 4, STAGE = 2 * HALF + 4 * kKeyWords;  // K's planes, V's, the step's words
    constexpr int PER = 2 * (HALF / 4096) + 1;  // loads of a step per wavefront
    __shared__ __attribute__((aligned(16))) char sh[256 + NST * STAGE];  // no stage at LDS address 0
    __shared__ unsigned char visit[DOCS ? kListed : 1];  // whether some row may see the block
    __shared__ uint32_t red[4][8];
    const Place at = place_of(blockIdx.x, u.B * u.Hk);
    const int item = at.item, split = at.block % a.nsplit, rb = a.blocks - 1 - at.block / a.nsplit;
    const int b = item / u.Hk, hk = item - b * u.Hk, rows = u.G * u.lq;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const int pre = u.prefix ? u.prefix[b] : 0;
    const int first = rb * kRows, last = min(first + kRows, rows) - 1;
    const int rr = first + 32 * w + (lane & 31);
    const Row row = row_of(u, hk, min(rr, rows - 1));
    const int64_t tok = (int64_t)b * u.lq + row.t;
    const int pos = row.t + u.off, doc = DOCS ? u.qd[tok] : 0;
    const float slope = SLOPES ? u.slopes[row.h] * kLog2e : 0.0f;

    // The row's query: d = 16 s + 8 g + e.
    float x0[S][8];
    {
        const float *qr = p.q + tok * p.ldq + (int64_t)row.h * u.d;
#pragma unroll
        for (int s = 0; s < S; s++) {
            const floatx4 lo = a.vec ? load4<true>(qr, 16 * s + 8 * g, u.d) : load4<false>(qr, 16 * s + 8 * g, u.d);
            const floatx4 hi = a.vec ? load4<true>(qr, 16 * s + 8 * g + 4, u.d) : load4<false>(qr, 16 * s + 8 * g + 4, u.d);
#pragma unroll
            for (int e = 0; e < 4; e++) x0[s][e] = lo[e], x0[s][4 + e] = hi[e];
        }
    }

    // The blocks of keys this workgroup can see, and what their split found; a thread keeps the first round's.
    int lo, hi;
    const int i0 = first / u.G + u.off, i1 = last / u.G + u.off;
    key_range(u, i0, i1, pre, lo, hi);
    // this split's share of them, in blocks: equal shares, so that a block of rows is as many equal pieces
    const int c0 = lo / kBlock, c1 = hi < lo ? c0 - 1 : hi / kBlock, per = (c1 - c0 + a.nsplit) / a.nsplit;
    const int t0 = c0 + split * per, t1 = min(c1, t0 + per - 1);
    lo = max(lo, t0 * kBlock);
    hi = min(hi, t1 * kBlock + kBlock - 1);
    uint32_t ktop = 0, vtop = 0, vlow = 0xFFFFFFFFu, knorm = 0;
    const int64_t kt0 = (int64_t)item * a.nt;
    Stats mk = {};
    for (int t = t0 + (int)threadIdx.x, n = 0; t <= t1; t += 256, n++) {
        const Stats sk = a.ks[kt0 + t], sv = a.vs[kt0 + t];
        if (n == 0) mk = sk;
        ktop = max(ktop, sk.top);
        knorm = max(knorm, __float_as_uint(sk.norm));
        vtop = max(vtop, sv.top);
        vlow = min(vlow, sv.low);
    }
    // The query, scaled and split.
    u32x4 qh[S], qm[S];
    int eq;
    bool bad;
    uint32_t qnorm;
    {
        uint32_t top = 0;
        float norm = 0.0f;
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (doc < 0) x0[s][e] = 0.0f;
                top = max(top, __float_as_uint(x0[s][e]) & 0x7FFFFFFFu);
                norm = __builtin_fmaf(x0[s][e], x0[s][e], norm);
            }
        qnorm = __float_as_uint(pair_sum(norm));
        const auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);
        top = max(both[0], both[1]);
        bad = !in_range(top) || (SLOPES && !bias_fits(u, slope));
        eq = !in_range(top) || !top ? 0 : scale_exp(top);
        const float sc = u.scale < 0.0f ? -pow2(-eq) : pow2(-eq);
#pragma unroll
        for (int s = 0; s < S; s++) {
#pragma unroll
            for (int e = 0; e < 8; e++) x0[s][e] *= sc;
            split8(x0[s], qh[s], qm[s]);
        }
    }
    ktop = wave_umax(ktop);
    vtop = wave_umax(vtop);
    vlow = wave_umin(vlow);
    knorm = wave_umax(knorm);
    qnorm = wave_umax(qnorm);
    // documents of the wavefront's rows; a padded row sees nothing, whatever the others see
    int wqlo = 0, wqhi = 0;
    bool one_doc = true;
    if (DOCS) {
        wqlo = __builtin_amdgcn_readfirstlane(wave_imin(doc < 0 ? INT32_MAX : doc));
        wqhi = __builtin_amdgcn_readfirstlane(wave_imax(doc));
        one_doc = wqlo == wqhi && !__any(doc < 0);
    }
    const uint32_t wave_bad = __any(bad) ? 1 : 0;
    if (lane == 0) {
        red[w][0] = ktop;
        red[w][1] = vtop;
        red[w][2] = vlow;
        red[w][3] = (uint32_t)wqlo;
        red[w][4] = (uint32_t)wqhi;
        red[w][5] = wave_bad;
        red[w][6] = knorm;
        red[w][7] = qnorm;
    }
    __syncthreads();
    int qlo = wqlo, qhi = wqhi;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        ktop = max(ktop, red[i][0]);
        vtop = max(vtop, red[i][1]);
        vlow = min(vlow, red[i][2]);
        qlo = min(qlo, (int)red[i][3]);
        qhi = max(qhi, (int)red[i][4]);
        bad = bad || red[i][5];
        knorm = max(knorm, red[i][6]);
        qnorm = max(qnorm, red[i][7]);
    }
    bad = bad || !scores_fit(u, __uint_as_float(qnorm), __uint_as_float(knorm)) || ktop > kMostBits || vtop > kMostBits || !even_rows(vtop, vlow);
    if (__builtin_amdgcn_readfirstlane(bad)) {
        for (int r = first + 32 * w; r <= min(last, first + 32 * w + 31); r++)
            plain_row<DP>(u, p, b, hk, r, lo, hi, split, a.nsplit, a.part);
        return;
    }
    const int ev = vtop ? scale_exp(vtop) : 0;
    if (DOCS) {
        if (t0 + (int)threadIdx.x <= t1) {
            static_assert(kListed == 256, "a thread's first block is its entry");
            visit[threadIdx.x] = !(mk.doc_hi < qlo || mk.doc_lo > qhi);
        }
        __syncthreads();
    }

    const int base = t0 * kBlock, steps = hi < lo ? 0 : (hi - base) / KT + 1;
    const Band whole_wg(u, i0, i1, pre);
    auto next = [&](int it) {  // the next step with a key that some row may see
        it++;
        // a window leaves a gap behind a prefix
        const int j0 = base + it * KT;
        if ((j0 >= whole_wg.pre) & (j0 + KT <= whole_wg.some0)) it = (whole_wg.some0 - base) / KT;
        if (DOCS)
            while (it < steps && it / 2 < kListed && !visit[it / 2]) it++;
        return it < steps ? it : steps;
    };
    const char *kn = a.kn + (kt0 + t0) * plane_bytes(DP, 1), *vt = a.vt + (kt0 + t0) * plane_bytes(DP, 1);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)(sh + 256);
    auto stage = [&](int it, int slot) {
        const char *ka = kn + (int64_t)it * HALF + lane * 16, *va = vt + (int64_t)it * HALF + lane * 16;
        const uint32_t to = lds0 + (uint32_t)(slot * STAGE);
#pragma unroll
        for (int i = 0; i < PER / 2; i++) load_to_lds(ka + (4 * i + w) * 1024, to + (uint32_t)(4 * i + w) * 1024u);
#pragma unroll
        for (int i = 0; i < PER / 2; i++) load_to_lds(va + (4 * i + w) * 1024, to + HALF + (uint32_t)(4 * i + w) * 1024u);
        if (lane >> 4 == w)  // a quarter of the step's words each
            load_to_lds4(a.keys + (2 * (kt0 + t0) + it) * kKeyWords + lane, to + 2 * HALF);
    };

    const Reach reach = keys_seen(u, pos, doc, pre);
    floatx16 acc[ND];
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[n][e] = 0.0f;
    float m = -kInf, l = 0.0f;
    const int wi0 = min(first + 32 * w, last) / u.G + u.off, wi1 = min(first + 32 * w + 31, last) / u.G + u.off;
    const bool live = first + 32 * w <= last;
    const Band mine(u, wi0, wi1, pre);
    const float cq = __builtin_fabsf(u.cl2) * pow2(eq), icq = __builtin_fabsf(u.icap) * pow2(eq);

    int it = next(-1), nx = it < steps ? next(it) : steps, slot = 0;
    if (it < steps) stage(it, 0);
    if (NST == 3 && nx < steps) stage(nx, 1);
    while (it < steps) {
        // this step has landed (with three stages the next is in flight), and every wavefront is done with the one before
        if (NST == 2 || nx >= steps) land<0>();
        else land<PER>();
        const int nn = nx < steps ? next(nx) : steps;
        if (NST == 3 && nn < steps) stage(nn, slot == 0 ? 2 : slot - 1);
        if (NST == 2 && nx < steps) stage(nx, slot ^ 1);
        const int j0 = base + it * KT, j1 = j0 + KT - 1;
        const char *kf = sh + 256 + slot * STAGE + lane * 16, *vf = kf + HALF;
        const int *words = reinterpret_cast<const int *>(sh + 256 + slot * STAGE + 2 * HALF);
        // what the wavefront's 32 rows see of the step
        bool some = live & mine.some(j0, j1), one = true;
        if (DOCS) {
            const int dlo = __builtin_amdgcn_readfirstlane(words[kKeyDocLo]), dhi = __builtin_amdgcn_readfirstlane(words[kKeyDocHi]);
            some = some & (dhi >= wqlo) & (dlo <= wqhi);
            one = one_doc & (dlo == dhi) & (dlo == wqlo) & (dlo >= 0);
        }
        if (some) {
            const float ksc = __int_as_float(words[kKeyScaleK]);
            // V's exponent less the largest, in steps of 4; a block of zeros may say anything
            const int vst = min(max(((words[kKeyScaleV] >> 23) - 127 - ev) >> 2, -8), 0);
            floatx16 x;
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = 0.0f;
#pragma unroll
            for (int s = 0; s < S; s++) {
                const u32x4 kh = *reinterpret_cast<const u32x4 *>(kf + (2 * s) * 1024);
                const u32x4 km = *reinterpret_cast<const u32x4 *>(kf + (2 * s + 1) * 1024);
                x = mma3(kh, km, qh[s], qm[s], x);
            }
            // x * f is the score in log2 units
            float f = cq * ksc;
            if (CAP) {
                const float ic = icq * ksc;
                float big = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e++) big = fmaxf(big, __builtin_fabsf(x[e]));
                if (__any(big * ic >= kTanhSmall)) {
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = tanh_any(x[e] * ic);
                } else {
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = tanh_small(x[e] * ic);
                }
            f = u.capl2;
            }
            if (SLOPES) {
                const float gap0 = (float)(pos - j0 - 4 * g);
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const float gap = gap0 - (float)(8 * (e >> 2) + (e & 3));
                    x[e] = __builtin_fmaf(-slope, __builtin_fabsf(gap), x[e] * f);
                }
                f = 1.0f;
            }
            if (!(mine.all(j0, j1) & one)) {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    intx4 kd = {doc, doc, doc, doc};
                    if (DOCS) kd = *reinterpret_cast<const intx4 *>(words + kKeyDoc + 8 * q + 4 * g);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const bool ok = reach.has(j0 + 8 * q + 4 * g + r) & (kd[r] == doc);
                        x[4 * q + r] = ok ? x[4 * q + r] : -kInf;
                    }
                }
            }
            float top = -kInf;
#pragma unroll
            for (int e = 0; e < 16; e++) top = fmaxf(top, x[e]);
            top = pair_max(top) * f;
            if (__any(top > m + kSlack)) {
                const float mn = fmaxf(m, top), al = mn == -kInf ? 1.0f : exp2_hw(m - mn);
                m = mn;
                l *= al;
#pragma unroll
                for (int n = 0; n < ND; n++) acc[n] *= al;
            }
            const float lift = (float)kLift + 4.0f * (float)vst, mu = (m == -kInf ? 0.0f : -m) + lift;
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                x[e] = exp2_hw(__builtin_fmaf(x[e], f, mu));
                sum += x[e];
            }
            l = __builtin_fmaf(sum, pow2(-4 * vst), l);
#pragma unroll
            for (int s = 0; s < 2; s++) {
                float e8[8];
#pragma unroll
                for (int e = 0; e < 8; e++) e8[e] = x[8 * s + e];
                u32x4 ph, pm;
                split8(e8, ph, pm);
#pragma unroll
                for (int c = 0; c < ND; c++) {
                    const char *at = vf + ((s * ND + c) * 2) * 1024;
                    acc[c] = mma3(*reinterpret_cast<const u32x4 *>(at), *reinterpret_cast<const u32x4 *>(at + 1024), ph, pm, acc[c]);
                }
            }
        }
        it = nx;
        nx = nn;
        slot = slot == NST - 1 ? 0 : slot + 1;
    }

    l = pair_sum(l);
    if (rr > last) return;
    const int64_t all = (int64_t)u.B * u.Hk * rows, out = (int64_t)item * rows + rr;
    const float mu = m == -kInf ? 0.0f : m, rl = l == 0.0f ? 0.0f : 1.0f / l, unlift = pow2(-kLift);
    const float wgt = a.part ? pow2(ev) * unlift : pow2(ev) * rl;
    float *to = a.part ? a.part + ((int64_t)split * all + out) * u.d : p.out + tok * p.ldo + (int64_t)row.h * u.d;
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int c = 32 * n + 8 * q + 4 * g;
            floatx4 v = floatx4{acc[n][4 * q], acc[n][4 * q + 1], acc[n][4 * q + 2], acc[n][4 * q + 3]} * wgt;
            if (l == 0.0f) v = floatx4{0.f, 0.f, 0.f, 0.f};
            if (c + 3 < u.d && (((uintptr_t)(to + c)) & 15) == 0) {
                *reinterpret_cast<floatx4 *>(to + c) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (c + e < u.d) to[c + e] = v[e];
            }
        }
    if (g == 0) {
        if (a.part) {
            float *ms = a.part + (int64_t)a.nsplit * all * u.d + (int64_t)split * all + out;
            ms[0] = mu;
            ms[(int64_t)a.nsplit * all] = l * unlift;
        } else if (p.stats) {
            const int64_t sr = stat_at(u, b, row);
            p.stats[sr] = mu;
            p.stats[all + sr] = l == 0.0f ? 0.0f : rl * pow2(kLift);
        }
    }
}

}  // namespace

namespace osc {

// The forward by the matrix cores, d up to 128; *joins gets the number of splits left to join (1: none) and *part where
// they lie.
// Into how many pieces to split each row block's keys: the number whose time is least by what was measured of the parts. A
// workgroup takes 5 us before its first step of 32 keys; a step of 64 values a head takes 1.2 us alone on its CU and 0.25 us
// more for each neighbour there, in proportion for other widths; pieces are joined at 4 TB/s after another launch. Work that
// differs from block to block (a causal rule over many rows) fills the chip up to the longest piece, even work goes in rounds.
// 500 rows behind 4096 keys, 2 x 12 heads of 64: one round of 8 pieces 58 us with its join, two of 16 69 us. 512 x 512 in
// documents, 8 x 12 heads: whole rows 33 us, 2 pieces 42 us with their join.
static int64_t pieces(const om_ctx *ctx, const Rule &u, int dp, int64_t wgs, int64_t rows) {
    const int64_t most = std::min<int64_t>((u.lk + kBlock - 1) / kBlock / 4, 64);
    const double cus = ctx->num_cus, occ = dp == 32 ? 4 : dp == 64 ? 3 : 2, wide = dp / 64.0;
    const double seen = u.window ? std::min<double>(u.lk, (u.causal ? 1.0 : 2.0) * u.window + kRows / u.G) : u.lk;
    const double longest = seen / 32;
    const bool uneven = u.causal && !u.window && 2 * (int64_t)u.lq > u.lk;
    const double mean = uneven ? longest * (1.0 - 0.5 * u.lq / u.lk) : longest;
    int64_t best = 1;
    double least = 0.0;
    for (int64_t ns = 1; ns <= std::max<int64_t>(most, 1); ns++) {
        const double n = (double)wgs * ns, there = std::min(occ, std::ceil(n / cus));
        const double step = (1.2 + 0.25 * (there - 1.0)) * wide, one = 5.0 + step * longest / ns;
        double us = uneven ? std::max(one, n / (occ * cus) * (5.0 + step * mean / ns)) : std::ceil(n / (occ * cus)) * one;
        if (ns > 1) us += 4.0 + 2.0 * ns * rows * (u.d + 2) * sizeof(float) / 4e6;
        if (ns == 1 || us < least) {
            best = ns;
            least = us;
        }
    }
    return best;
}

om_status fwd_by_matrix(om_ctx *ctx, const Rule &u, const Ptrs &p, int *joins, float **part) {
    const int nt = (u.lk + kBlock - 1) / kBlock, rows = u.G * u.lq, blocks = (rows + kRows - 1) / kRows;
    const int64_t items = (int64_t)u.B * u.Hk, wgs = items * blocks, all = items * rows;
    const int dp = u.d <= 32 ? 32 : u.d <= 64 ? 64 : u.d <= 96 ? 96 : 128;
    const int64_t ns = pieces(ctx, u, dp, wgs, all);
    OM_REQUIRE(ctx, wgs * ns <= most_groups(256) && 2 * items * nt <= most_groups(256), "om_attention_fwd_scored: too many row blocks");
    const int64_t plane = plane_bytes(dp, items * nt), stats = items * nt * (int64_t)sizeof(Stats);
    const int64_t words = 2 * items * nt * kKeyWords * (int64_t)sizeof(float);
    const int64_t join = ns > 1 ? (int64_t)sizeof(float) * ns * all * (u.d + 2) : 0;
    float *scr;
    if (om_status s = om::scratch2(ctx, (uint64_t)(2 * plane + 2 * stats + words + join), &scr)) return s;
    char *base = reinterpret_cast<char *>(scr);
    FwdArgs a = {};
    a.kn = base;
    a.vt = base + plane;
    // 16-byte stores first, the statistics last
    float *keys = reinterpret_cast<float *>(base + 2 * plane);
    a.keys = keys;
    a.part = ns > 1 ? reinterpret_cast<float *>(base + 2 * plane + words) : nullptr;
    a.ks = reinterpret_cast<Stats *>(base + 2 * plane + words + join);
    a.vs = a.ks + items * nt;
    a.nt = nt;
    a.blocks = blocks;
    a.nsplit = (int)ns;
    auto al16 = [](const void *x) { return ((uintptr_t)x & 15) == 0; };
    a.vec = u.d % 4 == 0 && p.ldq % 4 == 0 && al16(p.q);
    const bool vec = u.d % 4 == 0 && p.ldkv % 4 == 0 && al16(p.k) && al16(p.v);
    const SplitOut ko = {base, nullptr, const_cast<Stats *>(a.ks), keys, false};
    const SplitOut vo = {nullptr, base + plane, const_cast<Stats *>(a.vs), keys, true};
    by_depth(u.d, [&](auto dpc) {
        constexpr int DP = decltype(dpc)::value;
        auto split = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3((unsigned)(2 * items * nt)), dim3(256), 0, ctx->stream, u, p, ko, vo, nt);
        };
        vec ? split(k_scored_split_kv<DP, true>) : split(k_scored_split_kv<DP, false>);
        by_parts(parts_of(u), [&](auto pc) {
            hipLaunchKernelGGL((k_scored_fwd_mm<DP, decltype(pc)::value>), dim3((unsigned)(wgs * ns)), dim3(256), 0, ctx->stream, u,
                               p, a);
        });
    });
    *joins = (int)ns;
    *part = a.part;
    return OM_LAUNCH_CHECK(ctx, "om_attention_fwd_scored");
}

}  // namespace osc
