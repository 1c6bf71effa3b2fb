// Rotary positions, forward and backward: pairs of each head's values turn by pos * f_i (a 2 x 2 rotation per pair,
// whose transpose, the turn by the opposite angle, is the backward).
//
// Bound: HBM, 8 bytes per value (one read, one write) plus 4 per token. The angle costs about 45 vector instructions
// per pair, which a CU hides eight times over under its share of the bandwidth (8 B per cycle), so nothing is tabulated
// and every thread forms its own: turns = pos * (f_i / 2 pi) in double with the product's rounding error beside it, the
// fractional part exactly, then sine and cosine of an eighth turn by their Taylor sums in fp32. What is left of an angle's error
// is f_i's one rounding, 2^-53 of the angle (2.4e-7 at 2^31), and the eighth turn's in fp32, 5e-8. (f_i as two doubles leaves
// only the latter, but their reads cost 3 % of a long call and a third of a short one.)
#include "om_internal.hpp"

#include <cmath>

namespace {

constexpr int kMaxPairs = 128;  // d up to 256
struct Turns {
    double f[kMaxPairs];  // turns per position of pair i
};

// (cos, sin)(2 pi pos f), each within 1.2e-7.
__device__ __forceinline__ void cos_sin(double pos, double f, float &c, float &s) {
    const double turns = pos * f, left = __builtin_fma(pos, f, -turns);  // the product, exactly
    const double r = turns - __builtin_rint(turns) + left;  // -1/2 .. 1/2, the difference exact
    const double q = __builtin_rint(4.0 * r);        // quarter turns: -2 .. 2
    const float y = (float)((r - 0.25 * q) * 6.283185307179586);  // |y| <= pi / 4
    const float z = y * y;
    // Taylor sums to y^9 and y^10; the next terms are below 2e-9 and 2e-10 there
    float ps = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    ps = __builtin_fmaf(z, ps, 8.3333333e-3f);
    ps = __builtin_fmaf(z, ps, -1.6666667e-1f);
    const float sy = __builtin_fmaf(y * z, ps, y);
    float pc = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    pc = __builtin_fmaf(z, pc, -1.3888889e-3f);
    pc = __builtin_fmaf(z, pc, 4.1666667e-2f);
    pc = __builtin_fmaf(z, pc, -0.5f);
    const float cy = __builtin_fmaf(z, pc, 1.0f);
    const int n = (int)q;
    const float a = (n & 1) ? sy : cy, b = (n & 1) ? cy : sy;
    c = ((n + 1) & 2) ? -a : a;
    s = (n & 2) ? -b : b;
}

typedef float floatx4 __attribute__((ext_vector_type(4)));

// One thread per slot of a head: a pair slot of W pairs (W = 4 half pairs or 2 interleaved ones in the vector form, 1
// in the scalar form) or a slot of values that pass through. Threads run over a row's slots first, so a wavefront reads
// consecutive memory.
template <bool HALF, bool VEC, bool ACC>
__global__ void __launch_bounds__(256) k_rope(const float *x, int64_t ldx, const int32_t *__restrict__ pos, int pos0,
                                              float *y, int64_t ldy, int64_t total, int seq, int heads, int d,
                                              int rot, int pair_slots, int slots, float amp, float sign, Turns tr) {
    OM_LDS_POISON();
    constexpr int W = !VEC ? 1 : HALF ? 4 : 2;
    const int per_row = heads * slots;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row;
        const int in = (int)(i - row * per_row), h = in / slots, sl = in - h * slots;
        const float *xr = x + row * ldx + h * d;
        float *yr = y + row * ldy + h * d;
        auto put = [&](int at, auto v) {
            if constexpr (ACC) v = v + *reinterpret_cast<const decltype(v) *>(yr + at);
            *reinterpret_cast<decltype(v) *>(yr + at) = v;
        };
        if (sl >= pair_slots) {  // passes through
            const int at = rot + (sl - pair_slots) * (VEC ? 4 : 1);
            if constexpr (VEC) put(at, *reinterpret_cast<const floatx4 *>(xr + at));
            else put(at, xr[at]);
            continue;
        }
        const int p0 = sl * W;
        const double ps = (double)(pos ? pos[row] : pos0 + (int)(row % seq));
        float c[W], s[W];
#pragma unroll
        for (int w = 0; w < W; w++) {
            cos_sin(ps, tr.f[p0 + w], c[w], s[w]);
            c[w] *= amp;
            s[w] *= amp * sign;
        }
        if constexpr (VEC && HALF) {
            const floatx4 a = *reinterpret_cast<const floatx4 *>(xr + p0);
            const floatx4 b = *reinterpret_cast<const floatx4 *>(xr + rot / 2 + p0);
            floatx4 u, v;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                u[w] = a[w] * c[w] - b[w] * s[w];
                v[w] = b[w] * c[w] + a[w] * s[w];
            }
            put(p0, u);
            put(rot / 2 + p0, v);
        } else if constexpr (VEC) {
            const floatx4 a = *reinterpret_cast<const floatx4 *>(xr + 2 * p0);
            floatx4 u;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                u[2 * w] = a[2 * w] * c[w] - a[2 * w + 1] * s[w];
                u[2 * w + 1] = a[2 * w + 1] * c[w] + a[2 * w] * s[w];
            }
            put(2 * p0, u);
        } else {
            const int ia = HALF ? p0 : 2 * p0, ib = HALF ? p0 + rot / 2 : 2 * p0 + 1;
            const float a = xr[ia], b = xr[ib];
            put(ia, a * c[0] - b * s[0]);
            put(ib, b * c[0] + a * s[0]);
        }
    }
}

om_status rope(om_ctx *ctx, const char *what, const float *x, int ldx, const int32_t *pos, int pos0, float *y, int ldy,
               int rows, int seq, int heads, int d, const om_rope *rp, int acc, float sign) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, rp, "%s: rope is NULL", what);
    OM_REQUIRE(ctx, rows >= 0 && heads >= 0 && d >= 2 && d <= 2 * kMaxPairs, "%s: rows=%d heads=%d d=%d (d from 2 to %d)",
               what, rows, heads, d, 2 * kMaxPairs);
    OM_REQUIRE(ctx, rp->layout == OM_ROPE_HALF || rp->layout == OM_ROPE_INTERLEAVED, "%s: layout %d", what, rp->layout);
    OM_REQUIRE(ctx, rp->scaling >= OM_ROPE_PLAIN && rp->scaling <= OM_ROPE_BANDS, "%s: scaling %d", what, rp->scaling);
    OM_REQUIRE(ctx, rp->rot >= 2 && rp->rot <= d && rp->rot % 2 == 0, "%s: rot=%d needs an even number from 2 to d=%d",
               what, rp->rot, d);
    OM_REQUIRE(ctx, std::isfinite(rp->base) && rp->base > 1.0 && std::isfinite(rp->amplitude),
               "%s: base must be finite and above 1, the amplitude finite", what);
    OM_REQUIRE(ctx, rp->scaling == OM_ROPE_PLAIN || (std::isfinite(rp->factor) && rp->factor >= 1.0),
               "%s: factor must be finite and at least 1", what);
    OM_REQUIRE(ctx, rp->scaling != OM_ROPE_NTK || rp->rot > 2, "%s: OM_ROPE_NTK needs rot above 2", what);
    OM_REQUIRE(ctx, rp->scaling != OM_ROPE_BANDS || (std::isfinite(rp->trained) && rp->trained > 0.0 &&
               std::isfinite(rp->low) && std::isfinite(rp->high) && rp->low < rp->high),
               "%s: bands need a positive trained length and low < high", what);
    OM_REQUIRE(ctx, (int64_t)heads * d <= INT32_MAX && ldx >= heads * d && ldy >= heads * d,
               "%s: row strides %d / %d below heads * d = %lld", what, ldx, ldy, (long long)heads * d);
    OM_REQUIRE(ctx, x != y || (ldx == ldy && !acc), "%s: in place needs equal strides and no accumulation", what);
    if (rows == 0 || heads == 0) return OM_OK;
    OM_REQUIRE(ctx, x && y, "%s: NULL pointer", what);
    OM_REQUIRE(ctx, pos || seq >= 1, "%s: seq=%d", what, seq);
    OM_REQUIRE(ctx, pos || (int64_t)pos0 + (seq < rows ? seq : rows) - 1 <= INT32_MAX, "%s: positions past 2^31 - 1", what);
    if (om_status s = om::use_device(ctx)) return s;
    const int rot = rp->rot;
    // In the host's 64-bit significands and rounded once, each speed from the one before: 128 products are 2^-56 of it off. (A
    // power for each took 8 us a call.)
    typedef long double wide;
    const wide base = rp->scaling == OM_ROPE_NTK ? rp->base * std::pow((wide)rp->factor, rot / (rot - (wide)2)) : (wide)rp->base;
    const wide step = std::pow(base, (wide)-2 / rot);
    wide plain = 1 / 6.283185307179586476925286766559L;
    Turns tr = {};
    for (int i = 0; i < rot / 2; i++, plain *= step) {
        wide f = plain;
        if (rp->scaling == OM_ROPE_LINEAR) f /= rp->factor;
        if (rp->scaling == OM_ROPE_BANDS) {
            wide keep = (f * rp->trained - rp->low) / ((wide)rp->high - rp->low);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f *= keep + (1 - keep) / rp->factor;
        }
        tr.f[i] = (double)f;
    }
    const bool half = rp->layout == OM_ROPE_HALF;
    // 16-byte slots where every one starts at a multiple of 16 bytes
    const bool vec = ldx % 4 == 0 && ldy % 4 == 0 && d % 4 == 0 && rot % (half ? 8 : 4) == 0 &&
                     (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
    const int pair_slots = rot / 2 / (!vec ? 1 : half ? 4 : 2), slots = pair_slots + (d - rot) / (vec ? 4 : 1);
    const int64_t total = (int64_t)rows * heads * slots;
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3(om::grid1d(total, 256, (int64_t)ctx->num_cus * 64)), dim3(256), 0, ctx->stream, x,
                           (int64_t)ldx, pos, pos0, y, (int64_t)ldy, total, seq < 1 ? 1 : seq, heads, d, rot, pair_slots,
                           slots, rp->amplitude, sign, tr);
    };
    auto pick = [&](auto h) {
        constexpr bool H = decltype(h)::value;
        if (vec) acc ? go(k_rope<H, true, true>) : go(k_rope<H, true, false>);
        else acc ? go(k_rope<H, false, true>) : go(k_rope<H, false, false>);
    };
    half ? pick(std::true_type()) : pick(std::false_type());
    return OM_LAUNCH_CHECK(ctx, what);
}

}  // namespace

extern "C" {

om_status om_rope_fwd(om_ctx *ctx, const float *x, int ld_x, const int32_t *pos, int pos0, float *y, int ld_y, int rows,
                      int seq, int heads, int d, const om_rope *rp) {
    return rope(ctx, "om_rope_fwd", x, ld_x, pos, pos0, y, ld_y, rows, seq, heads, d, rp, 0, 1.0f);
}
om_status om_rope_bwd(om_ctx *ctx, const float *g, int ld_g, const int32_t *pos, int pos0, float *dx, int ld_dx, int rows,
                      int seq, int heads, int d, const om_rope *rp, int acc) {
    return rope(ctx, "om_rope_bwd", g, ld_g, pos, pos0, dx, ld_dx, rows, seq, heads, d, rp, acc != 0, -1.0f);
}

}  // extern "C"
