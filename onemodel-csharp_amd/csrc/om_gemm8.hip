// Products of packed tensors (om_pack8.hpp has the format): C[m, n] (+)= sum over k of A[m, k] B[n, k], both packed along k,
// and a Linear's weight gradient from an fp32 gradient and its packed input, dW[o, i] (+)= sum over rows of g[r, o] xt8[i, r].
//
// Arithmetic. An e4m3 code times a power of two is a bf16 value (4 significand bits of 8), so the codes are widened in
// registers, v_cvt_scalef32_pk_bf16_fp8 with the block's scale, and multiplied by v_mfma_f32_32x32x16_bf16: every product is
// exact and sums are fp32 (2-norm error 1e-7 at k = 4096). The 8-bit matrix instructions have up to twice the rate, but do
// not keep their sums: a 128-term dot product comes out 1.5e-5 off in the 2-norm (normal values; 5e-5 with all exponents in
// use), as their adder drops what is 2^-13 or so below its largest term. The conversion costs two to three vector
// instructions an MFMA at 64 x 64 to 128 x 64 values a wavefront and runs beside it (16 k of both: 15.4 ns an MFMA alone,
// 16.6 with six conversions to each).
#include "om_pack8.hpp"

#include <type_traits>

#include "om_split.hpp"

namespace {

using namespace om8;
using om8::floatx4;
using oms::floatx16;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t widen2(uint32_t w, float scale, std::false_type) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}
__device__ __forceinline__ uint32_t widen2(uint32_t w, float scale, std::true_type) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
}
// Eight codes to a fragment.
__device__ __forceinline__ u32x4 widen8(uint32_t w0, uint32_t w1, float scale) {
    return u32x4{widen2(w0, scale, std::false_type()), widen2(w0, scale, std::true_type()),
                 widen2(w1, scale, std::false_type()), widen2(w1, scale, std::true_type())};
}

// 16 (or 4) bytes a lane from `src` (this lane's address) to LDS at byte address lds + 16 (4) * lane, without registers. m0
// holds the address for this one instruction only; nothing else in these kernels reads it. land() waits until all of this
// wavefront's loads have landed and its own LDS reads are done, then meets the others.
__device__ __forceinline__ void load_to_lds(const void *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds4(const void *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void land() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

struct Gemm8 {
    Packed a, b;
    int m, n, blocks;       // blocks of 128 along k
    const float *bias;
    float *c;
    int64_t ldc;
    int acc;
    int splits, per;        // split s takes blocks [s * per, ..)
    float *ws;              // splits > 1: partial sums [split][m][n]
    int tiles_m, tiles_n;
};

// Workgroup -> (split, tile row, tile column). Each XCD (workgroups are dealt to the eight of them in turn) gets a run of
// neighbouring tiles, eight tile rows deep, so that what it reads is shared in its own L2.
__device__ __forceinline__ void tile_of(int tiles_m, int tiles_n, int total, int &split, int &tm, int &tn) {
    int lin = blockIdx.x;
    const int per = total >> 3, left = total & 7, x = lin & 7;
    lin = x * per + min(x, left) + (lin >> 3);
    const int area = tiles_m * tiles_n;
    split = lin / area;
    lin -= split * area;
    const int band = lin / (8 * tiles_n), rows = min(8, tiles_m - 8 * band), r = lin - band * 8 * tiles_n;
    tn = r / rows;
    tm = 8 * band + r % rows;
}

// LDS of one stage (128 k): rows of 128 bytes, the eight 16-byte pieces of a row permuted so that 16 neighbouring rows' equal
// pieces stand on distinct banks; behind the rows one dword of scale bytes each.
__device__ __forceinline__ int piece_at(int row, int piece) { return row * 128 + ((piece ^ (row >> 1)) & 7) * 16; }

// A tile's operand on its way into LDS: NW wavefronts, each instruction 64 pieces (eight rows). Rows past the last one
// load the last one again; what they give is not stored.
template <int ROWS, int NW>
struct Stage {
    static constexpr int PER = ROWS / 8 / NW;
    static_assert(ROWS % (8 * NW) == 0, "whole instructions to each wavefront");
    const uint8_t *src[PER];
    const uint8_t *sc;
    __device__ __forceinline__ Stage(const Packed &p, int r0, int rows, int wv, int lane) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int r = 8 * (wv * PER + i) + (lane >> 3), piece = (lane ^ (r >> 1)) & 7;
            src[i] = p.q + (int64_t)min(r0 + r, rows - 1) * p.ldq + 16 * piece;
        }
        sc = p.s + (int64_t)min(r0 + (wv * 64 + lane) % ROWS, rows - 1) * p.lds;
    }
    __device__ __forceinline__ void load(int blk, uint32_t lds, int wv) const {
#pragma unroll
        for (int i = 0; i < PER; i++) load_to_lds(src[i] + (int64_t)blk * 128, lds + (wv * PER + i) * 1024);
    }
    // The scale dword that holds block blk's byte, of every row.
    __device__ __forceinline__ void load_scales(int blk, uint32_t lds, int wv) const {
        if (wv < ROWS / 64) load_to_lds4(sc + (blk & ~3), lds + wv * 256);
    }
};

__device__ __forceinline__ float scale_in(uint32_t dword, int blk) { return scale_of((int)(dword >> (8 * (blk & 3))) & 255); }

// A workgroup of WM x WN wavefronts computes BM x BN of C in stages of 128 k, two of them in LDS: the next one's loads are
// issued as the current one begins. A lane's 16-byte piece g + 2 j (g = lane / 32) of a row feeds two MFMAs, which so see
// k = 32 j + 16 g + 8 t + e in place of their own order, alike for both operands.
template <int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) k_gemm8(Gemm8 p) {
    OM_LDS_POISON();
    constexpr int NW = WM * WN, MT = BM / WM / 32, NT = BN / WN / 32;
    constexpr int STAGE = (BM + BN) * 132, AS = BM * 128, BS = AS + BN * 128, SS = BS + BM * 4;
    __shared__ __attribute__((aligned(16))) char sh[2 * STAGE];
    const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int split, tm, tn;
    tile_of(p.tiles_m, p.tiles_n, gridDim.x, split, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN, wm = wv / WN * (BM / WM), wn = wv % WN * (BN / WN);
    const int b0 = split * p.per, b1 = min(p.blocks, b0 + p.per);
    const Stage<BM, NW> sa(p.a, m0, p.m, wv, lane);
    const Stage<BN, NW> sb(p.b, n0, p.n, wv, lane);
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)sh;
    auto issue = [&](int blk, uint32_t at) {
        sa.load(blk, at, wv);
        sb.load(blk, at + AS, wv);
        sa.load_scales(blk, at + BS, wv);
        sb.load_scales(blk, at + SS, wv);
    };
    floatx16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;
    if (b0 < b1) issue(b0, base);  // (k may be 0)
    for (int blk = b0; blk < b1; blk++) {
        const int at = ((blk - b0) & 1) * STAGE;
        land();
        if (blk + 1 < b1) issue(blk + 1, base + (STAGE - at));
        const char *cur = sh + at;
        float fa[MT], fb[NT];
#pragma unroll
        for (int i = 0; i < MT; i++) fa[i] = scale_in(*reinterpret_cast<const uint32_t *>(cur + BS + 4 * (wm + 32 * i + l32)), blk);
#pragma unroll
        for (int j = 0; j < NT; j++) fb[j] = scale_in(*reinterpret_cast<const uint32_t *>(cur + SS + 4 * (wn + 32 * j + l32)), blk);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            u32x4 a[MT], b[NT];
#pragma unroll
            for (int i = 0; i < MT; i++) a[i] = *reinterpret_cast<const u32x4 *>(cur + piece_at(wm + 32 * i + l32, 2 * q + g));
#pragma unroll
            for (int j = 0; j < NT; j++) b[j] = *reinterpret_cast<const u32x4 *>(cur + AS + piece_at(wn + 32 * j + l32, 2 * q + g));
#pragma unroll
            for (int t = 0; t < 2; t++) {
                u32x4 wa[MT], wb[NT];
#pragma unroll
                for (int i = 0; i < MT; i++) wa[i] = widen8(a[i][2 * t], a[i][2 * t + 1], fa[i]);
#pragma unroll
                for (int j = 0; j < NT; j++) wb[j] = widen8(b[j][2 * t], b[j][2 * t + 1], fb[j]);
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int j = 0; j < NT; j++) acc[i][j] = oms::mma(wa[i], wb[j], acc[i][j]);
            }
        }
    }
    // A register is one row, 32 neighbouring columns over the lanes: stores of whole 128-byte lines.
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int col = n0 + wn + 32 * j + l32;
        if (col >= p.n) continue;
        const float bias = p.bias ? p.bias[col] : 0.0f;
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int row = m0 + wm + 32 * i + 8 * (e >> 2) + 4 * g + (e & 3);
                if (row >= p.m) continue;
                float v = acc[i][j][e];
                if (p.splits > 1) {
                    p.ws[((int64_t)split * p.m + row) * p.n + col] = v;
                    continue;
                }
                float *c = p.c + row * p.ldc + col;
                if (p.bias) v = v + bias;
                if (p.acc) v = *c + v;
                *c = v;
            }
    }
}

// Adds the splits' sums in order, then bias and C.
__global__ void __launch_bounds__(256) k_gemm8_join(Gemm8 p) {
    OM_LDS_POISON();
    const int64_t total = (int64_t)p.m * p.n, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        float v = p.ws[i];
#pragma unroll 4
        for (int s = 1; s < p.splits; s++) v += p.ws[s * total + i];
        const int64_t row = i / p.n, col = i - row * p.n;
        if (p.bias) v = v + p.bias[col];
        float *c = p.c + row * p.ldc + col;
        *c = p.acc ? *c + v : v;
    }
}

om_status gemm8(om_ctx *ctx, const char *what, Gemm8 p) {
    const int64_t big = (int64_t)((p.m + 255) / 256) * ((p.n + 255) / 256);
    const int bm = big >= ctx->num_cus ? 256 : 128;
    p.tiles_m = (p.m + bm - 1) / bm;
    p.tiles_n = (p.n + bm - 1) / bm;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    int splits = 1;
    if (tiles < ctx->num_cus) splits = (int)(ctx->num_cus / tiles);
    if (splits > p.blocks) splits = p.blocks;
    p.per = splits > 1 ? (p.blocks + splits - 1) / splits : p.blocks;
    p.splits = splits > 1 ? (p.blocks + p.per - 1) / p.per : 1;
    OM_REQUIRE(ctx, tiles * p.splits <= INT32_MAX, "%s: %d x %d is more than a launch takes", what, p.m, p.n);
    if (p.splits > 1)
        if (om_status s = om::scratch(ctx, sizeof(float) * (uint64_t)p.splits * (uint64_t)p.m * (uint64_t)p.n, &p.ws)) return s;
    const unsigned grid = (unsigned)(tiles * p.splits);
    if (bm == 256) hipLaunchKernelGGL((k_gemm8<256, 256, 2, 4>), dim3(grid), dim3(512), 0, ctx->stream, p);
    else hipLaunchKernelGGL((k_gemm8<128, 128, 2, 2>), dim3(grid), dim3(256), 0, ctx->stream, p);
    if (p.splits > 1)
        hipLaunchKernelGGL(k_gemm8_join, dim3(om::grid1d((int64_t)p.m * p.n, 256, (int64_t)ctx->num_cus * 8)), dim3(256), 0,
                           ctx->stream, p);
    return OM_LAUNCH_CHECK(ctx, what);
}

// ------------------------------------------------------------------------------------------------- weight gradient
// dW = g^T x with x packed along the rows and g as it is. g is split into three bf16 parts that hold all of its bits (h + m +
// l), a value of x is one part, so a product is three MFMAs (six with x in fp32) and as exact as those. A wavefront owns 32
// rows of dW (columns of g) and all BN columns; it loads its g straight into fragments, 32 lanes to a row of g, and splits
// them in registers. Sums that come out infinite or NaN (an infinite g, whose parts are NaN; a g that rounds up past bf16's
// range) are formed again on the fp32 instruction.
struct Dw8 {
    const float *g;         // [rows, m]
    Packed x;               // [n, rows]
    int rows, m, n, blocks;
    float *dw, *db;
    int acc_dw, acc_db;
    int splits, per;
    float *ws;              // splits > 1: [split][m][n], behind them (8-byte aligned) the column sums [split][m]
    double *cs;
    int tiles_m, tiles_n;
};

__device__ __forceinline__ void split3(float x0, float x1, uint32_t &h, uint32_t &m, uint32_t &l) {
    h = oms::pack2(x0, x1);
    asm("" : "+v"(h));  // else the compiler converts x0 a second time instead of shifting h
    const float r0 = x0 - __uint_as_float(h << 16), r1 = x1 - __uint_as_float(h & 0xFFFF0000u);
    m = oms::pack2(r0, r1);
    asm("" : "+v"(m));
    l = oms::pack2(r0 - __uint_as_float(m << 16), r1 - __uint_as_float(m & 0xFFFF0000u));
}

template <int BN, int MG>
__global__ void __launch_bounds__(64 * MG) k_dw8(Dw8 p) {
    OM_LDS_POISON();
    constexpr int BM = 32 * MG, NT = BN / 32, STAGE = BN * 132, SS = BN * 128;
    __shared__ __attribute__((aligned(16))) char sh[2 * STAGE];
    const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int split, tm, tn;
    tile_of(p.tiles_m, p.tiles_n, gridDim.x, split, tm, tn);
    const int m0 = tm * BM + 32 * wv, n0 = tn * BN;
    const int b0 = split * p.per, b1 = min(p.blocks, b0 + p.per);
    const Stage<BN, MG> sb(p.x, n0, p.n, wv, lane);
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)sh;
    auto issue = [&](int blk, uint32_t at) {
        sb.load(blk, at, wv);
        sb.load_scales(blk, at + SS, wv);
    };
    // a wavefront past the last row of dW loads the last one; nothing of it is stored
    const float *gp = p.g + min(m0 + l32, p.m - 1);
    const bool sums = p.db && tn == 0;
    double cs = 0.0;
    floatx16 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[j][e] = 0.0f;
    float raw[16];
    // The 16 values of g that chunk q (32 k) of block blk takes in this lane; rows past the last are zero.
    auto fetch = [&](int blk, int q) {
        const int64_t k0 = (int64_t)blk * 128 + 32 * q + 16 * g;
        if ((int64_t)blk * 128 + 128 <= p.rows) {
#pragma unroll
            for (int e = 0; e < 16; e++) raw[e] = gp[(k0 + e) * p.m];
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float v = gp[min(k0 + e, (int64_t)p.rows - 1) * p.m];
                raw[e] = k0 + e < p.rows ? v : 0.0f;
            }
        }
    };
    issue(b0, base);
    fetch(b0, 0);
    for (int blk = b0; blk < b1; blk++) {
        const int at = ((blk - b0) & 1) * STAGE;
        land();
        if (blk + 1 < b1) issue(blk + 1, base + (STAGE - at));
        const char *cur = sh + at;
        float fb[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) fb[j] = scale_in(*reinterpret_cast<const uint32_t *>(cur + SS + 4 * (32 * j + l32)), blk);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            u32x4 fa[2][3];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t h, m, l;
                    split3(raw[8 * t + 2 * e], raw[8 * t + 2 * e + 1], h, m, l);
                    fa[t][0][e] = h;
                    fa[t][1][e] = m;
                    fa[t][2][e] = l;
                }
            if (sums) {
#pragma unroll
                for (int e = 0; e < 16; e++) cs += (double)raw[e];
            }
            if (q < 3) fetch(blk, q + 1);
            else if (blk + 1 < b1) fetch(blk + 1, 0);
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const u32x4 b = *reinterpret_cast<const u32x4 *>(cur + piece_at(32 * j + l32, 2 * q + g));
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const u32x4 w = widen8(b[2 * t], b[2 * t + 1], fb[j]);
                    acc[j] = oms::mma(fa[t][2], w, acc[j]);
                    acc[j] = oms::mma(fa[t][1], w, acc[j]);
                    acc[j] = oms::mma(fa[t][0], w, acc[j]);
                }
            }
        }
    }
    unsigned big = 0;
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) oms::note(acc[j][e], big);
    if (oms::beyond(big)) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int64_t col = min(n0 + 32 * j + l32, p.n - 1);
            const uint8_t *xq = p.x.q + col * p.x.ldq, *xs = p.x.s + col * p.x.lds;
            floatx16 t;
#pragma unroll
            for (int e = 0; e < 16; e++) t[e] = 0.0f;
            const int k1 = (int)min((int64_t)b1 * 128, (int64_t)p.rows);
#pragma unroll 1
            for (int k0 = b0 * 128; k0 < k1; k0 += 2) {
                const int k = min(k0 + g, k1 - 1);
                const bool in = k0 + g < k1;
                const float x = decode4(xq[k], scale_of(xs[k / 128]))[0];
                const float gv = gp[(int64_t)k * p.m];
                t = __builtin_amdgcn_mfma_f32_32x32x2f32(in ? gv : 0.0f, in ? x : 0.0f, t, 0, 0, 0);
            }
            oms::take_beyond(acc[j], t);
        }
    }
    if (sums) {
        cs += __shfl_xor(cs, 32, 64);
        const int row = m0 + l32;
        if (g == 0 && row < p.m) {
            if (p.splits > 1) {
                p.cs[(int64_t)split * p.m + row] = cs;
            } else {
                const float v = (float)cs;
                p.db[row] = p.acc_db ? p.db[row] + v : v;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int col = n0 + 32 * j + l32;
        if (col >= p.n) continue;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int row = m0 + 8 * (e >> 2) + 4 * g + (e & 3);
            if (row >= p.m) continue;
            if (p.splits > 1) {
                p.ws[((int64_t)split * p.m + row) * p.n + col] = acc[j][e];
                continue;
            }
            float *c = p.dw + (int64_t)row * p.n + col;
            *c = p.acc_dw ? *c + acc[j][e] : acc[j][e];
        }
    }
}

__global__ void __launch_bounds__(256) k_dw8_join(Dw8 p) {
    OM_LDS_POISON();
    const int64_t total = (int64_t)p.m * p.n, step = (int64_t)gridDim.x * 256, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t i = at; i < total; i += step) {
        float v = p.ws[i];
#pragma unroll 4
        for (int s = 1; s < p.splits; s++) v += p.ws[s * total + i];
        p.dw[i] = p.acc_dw ? p.dw[i] + v : v;
    }
    if (!p.db) return;
    for (int64_t i = at; i < p.m; i += step) {
        double c = p.cs[i];
        for (int s = 1; s < p.splits; s++) c += p.cs[(int64_t)s * p.m + i];
        p.db[i] = p.acc_db ? p.db[i] + (float)c : (float)c;
    }
}

om_status dw8(om_ctx *ctx, Dw8 p) {
    const int64_t big = (int64_t)((p.m + 255) / 256) * ((p.n + 127) / 128);
    const int bm = big >= ctx->num_cus ? 256 : 128;
    p.tiles_m = (p.m + bm - 1) / bm;
    p.tiles_n = (p.n + 127) / 128;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    int splits = 1;
    if (tiles < ctx->num_cus) splits = (int)(ctx->num_cus / tiles);
    if (splits > p.blocks) splits = p.blocks;
    p.per = (p.blocks + splits - 1) / splits;
    p.splits = (p.blocks + p.per - 1) / p.per;
    OM_REQUIRE(ctx, tiles * p.splits <= INT32_MAX, "om_linear_bwd_x8: in=%d out=%d is more than a launch takes", p.n, p.m);
    if (p.splits > 1) {
        const uint64_t sums = ((uint64_t)p.splits * p.m * p.n + 1) / 2 * 2;
        if (om_status s = om::scratch(ctx, 4 * sums + 8ull * p.splits * p.m, &p.ws)) return s;
        p.cs = reinterpret_cast<double *>(p.ws + sums);
    }
    const unsigned grid = (unsigned)(tiles * p.splits);
    if (bm == 256) hipLaunchKernelGGL((k_dw8<128, 8>), dim3(grid), dim3(512), 0, ctx->stream, p);
    else hipLaunchKernelGGL((k_dw8<128, 4>), dim3(grid), dim3(256), 0, ctx->stream, p);
    if (p.splits > 1)
        hipLaunchKernelGGL(k_dw8_join, dim3(om::grid1d((int64_t)p.m * p.n, 256, (int64_t)ctx->num_cus * 8)), dim3(256), 0,
                           ctx->stream, p);
    return OM_LAUNCH_CHECK(ctx, "om_linear_bwd_x8");
}

}  // namespace

extern "C" {

om_status om_gemm8(om_ctx *ctx, int m, int n, int k, const uint8_t *a8, const uint8_t *b8, const float *bias, float *c,
                   int ldc, int acc) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, m >= 0 && n >= 0 && k >= 0 && ldc >= n, "om_gemm8: m=%d n=%d k=%d ldc=%d", m, n, k, ldc);
    OM_REQUIRE(ctx, aligned16(a8) && aligned16(b8), "om_gemm8: packed tensors start at multiples of 16 bytes");
    if (m == 0 || n == 0) return OM_OK;
    OM_REQUIRE(ctx, c && (k == 0 || (a8 && b8)), "om_gemm8: NULL pointer");
    if (om_status s = om::use_device(ctx)) return s;
    Gemm8 p = {};
    p.a = packed(a8, m, k);
    p.b = packed(b8, n, k);
    p.m = m, p.n = n, p.blocks = (int)blocks8(k);
    p.bias = bias, p.c = c, p.ldc = ldc, p.acc = acc;
    return gemm8(ctx, "om_gemm8", p);
}

om_status om_linear_bwd_x8(om_ctx *ctx, const float *g, const uint8_t *xt8, const float *w, float *dx, float *dw, float *db,
                           int rows, int in, int out, int acc_dx, int acc_dw, int acc_db) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, rows >= 0 && in > 0 && out > 0, "om_linear_bwd_x8: rows=%d in=%d out=%d", rows, in, out);
    OM_REQUIRE(ctx, aligned16(xt8), "om_linear_bwd_x8: packed tensors start at multiples of 16 bytes");
    OM_REQUIRE(ctx, rows == 0 || (g && (!dx || w) && (!dw || xt8)), "om_linear_bwd_x8: a needed tensor is NULL");
    if (om_status s = om::use_device(ctx)) return s;
    if (rows > 0 && dx)
        if (om_status s = om_linear_bwd(ctx, g, nullptr, w, dx, nullptr, nullptr, rows, in, out, acc_dx, 0, 0)) return s;
    if (rows == 0) {  // empty sums
        if (dw && !acc_dw)
            if (om_status s = om_fill(ctx, dw, 0.0f, (int64_t)in * out)) return s;
        return db && !acc_db ? om_fill(ctx, db, 0.0f, out) : OM_OK;
    }
    if (!dw) return db ? om_colsum(ctx, g, db, rows, out, acc_db) : OM_OK;
    Dw8 p = {};
    p.g = g;
    p.x = packed(xt8, in, rows);
    p.rows = rows, p.m = out, p.n = in, p.blocks = (int)blocks8(rows);
    p.dw = dw, p.db = db, p.acc_dw = acc_dw, p.acc_db = acc_db;
    return dw8(ctx, p);
}

}  // extern "C"
