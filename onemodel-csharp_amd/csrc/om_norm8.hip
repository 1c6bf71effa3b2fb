// LayerNorm that keeps its normalised rows in 8 bits (om_pack8.hpp has the format), forward and backward.
//
// Forward: mean and variance in 64 bits and rounded once each, so that the rows kept, xh = fl(fl(x - mean) * rstd), have bits
// of their own whatever order a row was summed in; y = xh gamma + beta, xh8 = pack(xh). Kept are the normalised rows and not
// x: a code is off by 2^-4 of its value, which of x would be 2^-4 of its mean as well. Backward, with h the value of xh8 and
// q = g gamma: dx = rstd (q - mean(q) - h mean(q h)), dgamma = sum of g h, dbeta = sum of g.
//
// Bound: HBM, 9 bytes a value each way (x or g 4, the packed rows 1, y or dx 4): 16384 x 4096 252 us both ways, 4.8 TB/s;
// 4096 x 384 15.2 us, three launches near their latency. A row is read once and stays in registers: one wavefront to a row of up
// to 1024 columns, then four, eight past 4096 and sixteen past 8192 (one row of 8192 forward 5.5 us by eight, 7.2 by four; 4096
// rows of 16384 141 us by sixteen, 173 by four), four values a lane at a time, so that 32 lanes hold a block of 128. Rows past
// 16384 columns (backward: 8192, whose column sums need the registers) are read again for each pass.
#include "om_pack8.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

using namespace om8;

// What NW wavefronts add up together: the totals in every lane, in a fixed order. `sh` holds NW values; the wavefronts meet
// before it is written, so calls may follow each other.
template <int NW, class T>
__device__ __forceinline__ T row_sum(T v, T *sh) {
    v = wave_sum8(v);
    if constexpr (NW == 1) {
        return v;
    } else {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        __syncthreads();
        T t = sh[0];
#pragma unroll
        for (int i = 1; i < NW; i++) t += sh[i];
        return t;
    }
}

__device__ __forceinline__ void put_codes(const Packed &p, int64_t row, int64_t blk, int64_t col, floatx4 xh) {
    const int s = scale_byte(max32(finite_bits4(xh)));
    *reinterpret_cast<uint32_t *>(p.q + row * p.ldq + col) = encode4(xh, inverse_of(s));
    if ((threadIdx.x & 31) == 0) p.s[row * p.lds + blk] = (uint8_t)s;
}

// NW wavefronts to a row (of one, four rows to a workgroup), NV quads of 64 NW lanes. NV = 0: any number, read again for each pass.
template <int NW, int NV>
__global__ void __launch_bounds__(NW == 1 ? 256 : 64 * NW) k_ln8(const float *x, const float *__restrict__ gamma, const float *__restrict__ beta,
                                             float *y, Packed p, float *__restrict__ rstd, int64_t rows, int64_t cols,
                                             float eps, double inv_n) {
    OM_LDS_POISON();
    __shared__ double sh[NW];
    constexpr int L = 64 * NW, KEEP = NV ? NV : 1;
    const int64_t row = NW == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= rows) return;  // whole rows leave; a row of more than one wavefront is its workgroup's only one
    const int t = threadIdx.x % L;
    const float *xr = x + row * cols;
    const int64_t quads = p.ldq / 4;  // up to the end of the last block
    const int nv = NV ? NV : (int)((quads + L - 1) / L);
    floatx4 v[KEEP];
    auto at = [&](int i) { return 4 * ((int64_t)i * L + t); };
    auto quad = [&](int i) { return at(i) < cols ? load4(xr + at(i), cols - at(i)) : floatx4{0.0f, 0.0f, 0.0f, 0.0f}; };
    // f(i, quad i), from registers or read again
    auto sweep = [&](auto f) {
        if constexpr (NV) {
#pragma unroll
            for (int i = 0; i < NV; i++) f(i, v[i]);
        } else {
            for (int i = 0; i < nv; i++) f(i, quad(i));
        }
    };
    if constexpr (NV) {
#pragma unroll
        for (int i = 0; i < NV; i++) v[i] = quad(i);
    }
    double sum = 0.0;
    sweep([&](int, floatx4 w) { sum += ((double)w[0] + (double)w[1]) + ((double)w[2] + (double)w[3]); });
    const double mean = row_sum<NW>(sum, sh) * inv_n;
    double ss = 0.0;
    sweep([&](int i, floatx4 w) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double d = (double)w[e] - mean;
            ss += at(i) + e < cols ? d * d : 0.0;
        }
    });
    // 1 / sqrt by the instruction's approximation (about 2^-26) and two Newton steps, 2^-52: the float nearest to it is the
    // exact value's but where that lies within 2^-28 of a step from a tie. (Zero and what is not finite by the division.)
    const double var = row_sum<NW>(ss, sh) * inv_n + (double)eps;
    double root = __builtin_amdgcn_rsq(var);
#pragma unroll
    for (int i = 0; i < 2; i++) root = root * __builtin_fma(-0.5 * var * root, root, 1.5);
    if (!(var > 1e-300 && var < 1e300)) root = 1.0 / sqrt(var);
    const float r = (float)root, m = (float)mean;
    if (t == 0) rstd[row] = r;
    sweep([&](int i, floatx4 xh) {
        const int64_t c = at(i);
        if (c >= p.ldq) return;  // whole blocks of 32 lanes leave together
#pragma unroll
        for (int e = 0; e < 4; e++) xh[e] = c + e < cols ? (xh[e] - m) * r : 0.0f;
        put_codes(p, row, c / 128, c, xh);
        if (c < cols) {
            const floatx4 ga = load4(gamma + c, cols - c), be = load4(beta + c, cols - c);
            floatx4 o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = xh[e] * ga[e] + be[e];
            store4(y + row * cols + c, cols - c, o);
        }
    });
    if (const int64_t b = p.ldq / 128; t < p.lds - b) p.s[row * p.lds + b + t] = 0;
}

// A workgroup takes `chunk` rows: sixteen wavefronts a row each (NW = 1; eight past 512 columns, whose sums need the
// registers), or four to a row (NW = 4). Every lane keeps the fp64 sums of its own columns and leaves them as one partial row
// of the workgroup's (added over its wavefronts through LDS in order where several share the columns). A workgroup that is the only one leaves the sums themselves, out (+)= sum.
struct Sums {
    double *part;  // the partial rows, or null
    float *out;
    int acc;
};
template <int NW, int NV>
constexpr int kBwdThreads = NW > 1 ? 64 * NW : NV <= 2 ? 1024 : 512;
template <int NW, int NV, bool ACC>
__global__ void __launch_bounds__((kBwdThreads<NW, NV>))
    k_ln8_bwd(const float *g, Packed p, const float *__restrict__ gamma, const float *__restrict__ rstd, float *dx, Sums dgamma,
              Sums dbeta, int64_t rows, int64_t cols, int chunk) {
    OM_LDS_POISON();
    constexpr int L = 64 * NW, WAVES = kBwdThreads<NW, NV> / 64, AT_ONCE = WAVES / NW;
    __shared__ float sh[NW];
    __shared__ double cs[NW == 1 ? 2 * NV * WAVES * 256 : 1];
    const int t = threadIdx.x % L, w = threadIdx.x >> 6;
    const int64_t r0 = (int64_t)blockIdx.x * chunk, r1 = min(rows, r0 + chunk);
    double sg[4 * NV], sb[4 * NV];
    floatx4 ga[NV];
    auto at = [&](int i) { return 4 * ((int64_t)i * L + t); };
#pragma unroll
    for (int i = 0; i < NV; i++) {
        ga[i] = at(i) < cols ? load4(gamma + at(i), cols - at(i)) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 4; e++) sg[4 * i + e] = sb[4 * i + e] = 0.0;
    }
    for (int64_t row = r0 + (NW == 1 ? w : 0); row < r1; row += AT_ONCE) {
        const float *gr = g + row * cols;
        floatx4 gv[NV], h[NV], old[ACC ? NV : 1];
        uint32_t q[NV];
        int s[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int64_t c = at(i);
            const bool in = c < cols;
            gv[i] = in ? load4(gr + c, cols - c) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            q[i] = in ? *reinterpret_cast<const uint32_t *>(p.q + row * p.ldq + c) : 0u;
            s[i] = in ? p.s[row * p.lds + c / 128] : 0;
            if constexpr (ACC) old[i] = in && dx ? load4(dx + row * cols + c, cols - c) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            h[i] = decode4(q[i], scale_of(s[i]));
#pragma unroll
            for (int e = 0; e < 4; e++) {
                sg[4 * i + e] = __builtin_fma((double)gv[i][e], (double)h[i][e], sg[4 * i + e]);
                sb[4 * i + e] += (double)gv[i][e];
                gv[i][e] *= ga[i][e];
                s1 += gv[i][e];
                s2 = __builtin_fmaf(gv[i][e], h[i][e], s2);
            }
        }
        if (dx) {
            const float m1 = row_sum<NW>(s1, sh) / (float)cols, m2 = row_sum<NW>(s2, sh) / (float)cols, r = rstd[row];
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int64_t c = at(i);
                if (c >= cols) break;
                floatx4 o;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    o[e] = r * ((gv[i][e] - m1) - h[i][e] * m2);
                    if constexpr (ACC) o[e] = old[i][e] + o[e];
                }
                store4(dx + row * cols + c, cols - c, o);
            }
        }
    }
    auto put = [&](const Sums &to, int64_t c, double v) {
        if (c >= cols) return;
        if (to.part) to.part[(int64_t)blockIdx.x * cols + c] = v;
        else if (to.out) to.out[c] = to.acc ? to.out[c] + (float)v : (float)v;
    };
    if constexpr (NW == 1) {  // value e of quad i of lane t at 256 i + 64 e + t, a row of them to each wavefront
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                cs[(256 * w + 64 * e + t) + 256 * WAVES * i] = sg[4 * i + e];
                cs[(256 * w + 64 * e + t) + 256 * WAVES * (NV + i)] = sb[4 * i + e];
            }
        __syncthreads();
        for (int q = threadIdx.x; q < 512 * NV; q += 64 * WAVES) {
            const double *from = cs + 256 * WAVES * (q >> 8) + (q & 255);
            double v = from[0];
#pragma unroll
            for (int k = 1; k < WAVES; k++) v += from[256 * k];
            const bool b = q >= 256 * NV;
            put(b ? dbeta : dgamma, 256 * (int64_t)((q >> 8) - (b ? NV : 0)) + 4 * (q & 63) + ((q >> 6) & 3), v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                put(dgamma, at(i) + e, sg[4 * i + e]);
                put(dbeta, at(i) + e, sb[4 * i + e]);
            }
    }
}

// dx alone for rows of any length: both passes over the row read it again.
template <bool ACC>
__global__ void __launch_bounds__(256) k_ln8_dx_long(const float *g, Packed p, const float *__restrict__ gamma,
                                                     const float *__restrict__ rstd, float *dx, int64_t cols) {
    OM_LDS_POISON();
    __shared__ float sh[4];
    const int64_t row = blockIdx.x;
    const float *gr = g + row * cols;
    auto value = [&](int64_t c) {
        return decode4(*reinterpret_cast<const uint32_t *>(p.q + row * p.ldq + c), scale_of(p.s[row * p.lds + c / 128]));
    };
    auto graded = [&](int64_t c) {
        floatx4 q = load4(gr + c, cols - c);
        const floatx4 ga = load4(gamma + c, cols - c);
#pragma unroll
        for (int e = 0; e < 4; e++) q[e] *= ga[e];
        return q;
    };
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t c = 4 * threadIdx.x; c < cols; c += 1024) {
        const floatx4 q = graded(c), h = value(c);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            s1 += q[e];
            s2 = __builtin_fmaf(q[e], h[e], s2);
        }
    }
    const float m1 = row_sum<4>(s1, sh) / (float)cols, m2 = row_sum<4>(s2, sh) / (float)cols, r = rstd[row];
    for (int64_t c = 4 * threadIdx.x; c < cols; c += 1024) {
        const floatx4 q = graded(c), h = value(c);
        const floatx4 old = ACC ? load4(dx + row * cols + c, cols - c) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        floatx4 o;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            o[e] = r * ((q[e] - m1) - h[e] * m2);
            if constexpr (ACC) o[e] = old[e] + o[e];
        }
        store4(dx + row * cols + c, cols - c, o);
    }
}
// dgamma's and dbeta's partials of such rows: a workgroup adds `chunk` rows of 1024 columns.
__global__ void __launch_bounds__(256) k_ln8_params_long(const float *__restrict__ g, Packed p, double *part_g, double *part_b,
                                                         int64_t rows, int64_t cols, int chunk) {
    OM_LDS_POISON();
    const int64_t c = 1024 * (int64_t)blockIdx.y + 4 * threadIdx.x;
    if (c >= cols) return;
    double sg[4] = {0.0, 0.0, 0.0, 0.0}, sb[4] = {0.0, 0.0, 0.0, 0.0};
    const int64_t r1 = min(rows, ((int64_t)blockIdx.x + 1) * chunk);
    for (int64_t row = (int64_t)blockIdx.x * chunk; row < r1; row++) {
        const floatx4 gv = load4(g + row * cols + c, cols - c);
        const floatx4 h =
            decode4(*reinterpret_cast<const uint32_t *>(p.q + row * p.ldq + c), scale_of(p.s[row * p.lds + c / 128]));
#pragma unroll
        for (int e = 0; e < 4; e++) {
            sg[e] = __builtin_fma((double)gv[e], (double)h[e], sg[e]);
            sb[e] += (double)gv[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (c + e < cols) {
            if (part_g) part_g[(int64_t)blockIdx.x * cols + c + e] = sg[e];
            if (part_b) part_b[(int64_t)blockIdx.x * cols + c + e] = sb[e];
        }
}

// Columns of a row that stay in registers: the forward keeps the values alone, the backward sums beside them.
constexpr int64_t kKeptFwd = 16384, kKeptBwd = 8192, kOneWave = 1024;  // kOneWave: a wavefront to a row
template <class F>
void by_width(int64_t cols, int64_t kept, F f) {
    if (cols > kept) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 0>());
#define OM_LN8(NW, NV) \
    if (cols <= 256 * NW * NV) return f(std::integral_constant<int, NW>(), std::integral_constant<int, NV>());
    OM_LN8(1, 1) OM_LN8(1, 2) OM_LN8(1, 3) OM_LN8(1, 4) OM_LN8(4, 2) OM_LN8(4, 3) OM_LN8(4, 4) OM_LN8(8, 4) OM_LN8(16, 4)
#undef OM_LN8
}

// Rows to a workgroup of the backward. Up to 1024 columns its eight or sixteen wavefronts take a row each and a CU holds one
// workgroup, so 256 of them are one round (8192 x 384 12.1 us, 512 of them 15.3), and up to 32 (24) rows one alone saves the
// second launch (24 x 384 5.3 us, 6.6 in three). Of longer rows a workgroup takes 0.7 to 2 us each, one after the other, and its
// sums are a row to write, read and add: the two together are least about sqrt(rows / 32) (64 x 4096: 11.3 us by two, 28.4 by
// sixteen; 4096 x 2048 25 us by eight, 29 by sixteen), with two workgroups a CU at most, or one past 4096 columns, of which a CU
// holds no more (8192 x 8192: 145 us by 32 rows, 165 by 16).
int rows_each(int64_t rows, int64_t cols, int cus) {
    if (cols <= kOneWave) {
        const int alone = cols <= 512 ? 32 : 24;
        return rows <= alone ? alone : (int)std::max<int64_t>(8, (rows + cus - 1) / cus);
    }
    if (rows <= 2) return 2;
    const int64_t most = cols > 4096 ? cus : 2 * cus;
    return (int)std::max<int64_t>((rows + most - 1) / most, (int64_t)std::sqrt((double)rows / 32));
}

}  // namespace

extern "C" {

om_status om_layernorm_fwd_x8(om_ctx *ctx, const float *x, const float *gamma, const float *beta, float *y, uint8_t *xh8,
                              float *rstd, int rows, int cols, float eps) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, rows >= 0 && cols > 0, "om_layernorm_fwd_x8: rows=%d cols=%d", rows, cols);
    OM_REQUIRE(ctx, aligned16(xh8), "om_layernorm_fwd_x8: packed tensors start at multiples of 16 bytes");
    if (rows == 0) return OM_OK;
    OM_REQUIRE(ctx, x && gamma && beta && y && xh8 && rstd, "om_layernorm_fwd_x8: NULL pointer");
    const Packed p = packed(xh8, rows, cols);
    om_status status = OM_OK;
    by_width(cols, kKeptFwd, [&](auto nw, auto nv) {
        constexpr int NW = decltype(nw)::value, NV = decltype(nv)::value, threads = NW == 1 ? 256 : 64 * NW;
        const int64_t groups = NW == 1 ? ((int64_t)rows + 3) / 4 : rows;
        status = launches(groups, threads) ? om::use_device(ctx)
                                           : om::fail(ctx, OM_E_ARG, "om_layernorm_fwd_x8: %d x %d is more than a launch takes", rows, cols);
        if (status) return;
        hipLaunchKernelGGL((k_ln8<NW, NV>), dim3((unsigned)groups), dim3(threads), 0, ctx->stream, x, gamma, beta, y, p, rstd,
                           (int64_t)rows, (int64_t)cols, eps, 1.0 / cols);
    });
    if (status) return status;
    return OM_LAUNCH_CHECK(ctx, "om_layernorm_fwd_x8");
}

om_status om_layernorm_bwd_x8(om_ctx *ctx, const float *g, const uint8_t *xh8, const float *gamma, const float *rstd,
                              float *dx, float *dgamma, float *dbeta, int rows, int cols, int acc_dx, int acc_params) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, rows >= 0 && cols > 0, "om_layernorm_bwd_x8: rows=%d cols=%d", rows, cols);
    OM_REQUIRE(ctx, aligned16(xh8), "om_layernorm_bwd_x8: packed tensors start at multiples of 16 bytes");
    OM_REQUIRE(ctx, rows == 0 || (g && xh8 && gamma && rstd), "om_layernorm_bwd_x8: NULL pointer");
    if (!dx && !dgamma && !dbeta) return OM_OK;
    OM_REQUIRE(ctx, cols <= 65535 * 1024 && (cols <= kKeptBwd || launches(rows, 256)),
               "om_layernorm_bwd_x8: %d x %d is more than a launch takes", rows, cols);
    if (rows == 0 && acc_params) return OM_OK;
    if (om_status s = om::use_device(ctx)) return s;
    if (rows == 0) {  // empty sums
        if (dgamma)
            if (om_status s = om_fill(ctx, dgamma, 0.0f, cols)) return s;
        return dbeta ? om_fill(ctx, dbeta, 0.0f, cols) : OM_OK;
    }
    const int chunk = rows_each(rows, cols, ctx->num_cus), chunks = (int)(((int64_t)rows + chunk - 1) / chunk);
    const bool one = chunks == 1 && cols <= kKeptBwd;
    double *pg = nullptr, *pb = nullptr;
    if (!one && (dgamma || dbeta)) {
        float *scr;
        if (om_status s = om::scratch(ctx, sizeof(double) * 2ull * (uint64_t)chunks * (uint64_t)cols, &scr)) return s;
        double *base = reinterpret_cast<double *>(scr);
        pg = dgamma ? base : nullptr;
        pb = dbeta ? base + (uint64_t)chunks * (uint64_t)cols : nullptr;
    }
    const Packed p = packed(xh8, rows, cols);
    by_width(cols, kKeptBwd, [&](auto nw, auto nv) {
        constexpr int NW = decltype(nw)::value, NV = decltype(nv)::value;
        if constexpr (NV && 256 * NW * NV <= kKeptBwd) {
            auto go = [&](auto kern) {
                hipLaunchKernelGGL(kern, dim3((unsigned)chunks), dim3(kBwdThreads<NW, NV>), 0, ctx->stream, g, p, gamma, rstd, dx,
                                   Sums{pg, one ? dgamma : nullptr, acc_params}, Sums{pb, one ? dbeta : nullptr, acc_params},
                                   (int64_t)rows, (int64_t)cols, chunk);
            };
            acc_dx ? go(k_ln8_bwd<NW, NV, true>) : go(k_ln8_bwd<NW, NV, false>);
        } else if constexpr (!NV) {
            auto go = [&](auto kern) {
                hipLaunchKernelGGL(kern, dim3((unsigned)rows), dim3(256), 0, ctx->stream, g, p, gamma, rstd, dx,
                                   (int64_t)cols);
            };
            if (pg || pb)
                hipLaunchKernelGGL(k_ln8_params_long, dim3((unsigned)chunks, (unsigned)((cols + 1023) / 1024)), dim3(256),
                                   0, ctx->stream, g, p, pg, pb, (int64_t)rows, (int64_t)cols, chunk);
            if (dx) acc_dx ? go(k_ln8_dx_long<true>) : go(k_ln8_dx_long<false>);  // last: dx may be g
        }
    });
    if (om_status s = OM_LAUNCH_CHECK(ctx, "om_layernorm_bwd_x8")) return s;
    if (one) return OM_OK;
    if (dgamma && dbeta) return om::chunk_final(ctx, pg, chunks, cols, dgamma, acc_params, pb, dbeta);
    if (dgamma) return om::chunk_final(ctx, pg, chunks, cols, dgamma, acc_params);
    return dbeta ? om::chunk_final(ctx, pb, chunks, cols, dbeta, acc_params) : OM_OK;
}

}  // extern "C"
