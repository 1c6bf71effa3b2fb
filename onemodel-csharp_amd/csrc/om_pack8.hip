// Tensors to 8 bits and back (om_pack8.hpp has the format), and GELU with its input kept so.
//
// All of these are bound by HBM: packing reads 4 bytes a value and writes 1 to each packed form, unpacking the reverse.
// A block of 128 neighbouring values is one half-wavefront, four values (16 bytes) a lane, so its largest value is one
// reduction over 32 lanes and its codes are one 128-byte line.
#include "om_pack8.hpp"

#include <type_traits>

namespace {

using namespace om8;

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // blocks of one half-wavefront in flight

// Walks the blocks of [rows, cols]: half-wavefront h of the grid takes blocks h, h + halves, ..., kUnroll of them at a time;
// `load(u, row, col)` for each first, then `use(u, row, block, col)`.
// (The host checks that there are fewer than 2^31 blocks.)
template <class Load, class Use>
__device__ __forceinline__ void each_block(int64_t rows, int blocks, Load load, Use use) {
    const uint32_t total = (uint32_t)(rows * blocks), halves = gridDim.x * (kThreads / 32);
    const int at = 4 * (threadIdx.x & 31);
    for (uint32_t b0 = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); b0 < total; b0 += halves * kUnroll) {
        int64_t row[kUnroll];
        int blk[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const uint32_t b = b0 + u * halves, r = b / (uint32_t)blocks;
            row[u] = r;
            blk[u] = (int)(b - r * (uint32_t)blocks);
            if (b < total) load(u, row[u], blk[u], (int64_t)blk[u] * 128 + at);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; u++)
            if (b0 + u * halves < total) use(u, row[u], blk[u], (int64_t)blk[u] * 128 + at);
    }
}

// A lane's four values of a block into the packed row, and the row's scale bytes.
__device__ __forceinline__ void put_block(const Packed &p, int64_t row, int blk, int blocks, int64_t col, floatx4 v) {
    const int s = scale_byte(max32(finite_bits4(v)));
    *reinterpret_cast<uint32_t *>(p.q + row * p.ldq + col) = encode4(v, inverse_of(s));
    const int l = threadIdx.x & 31;
    if (l == 0) p.s[row * p.lds + blk] = (uint8_t)s;
    if (blk == blocks - 1 && l > 0 && blk + l < p.lds) p.s[row * p.lds + blk + l] = 0;
}

__global__ void __launch_bounds__(kThreads) k_pack8(const float *__restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                                    int blocks, Packed p) {
    OM_LDS_POISON();
    floatx4 v[kUnroll];
    each_block(rows, blocks, [&](int u, int64_t r, int, int64_t c) { v[u] = load4(x + r * ld + c, cols - c); },
               [&](int u, int64_t r, int b, int64_t c) { put_block(p, r, b, blocks, c, v[u]); });
}

// The transpose packed (and the tensor itself where ROWS): a workgroup takes 128 rows x 128 columns, so that both kinds
// of blocks are whole. Thread t holds rows 16 (t / 32) .. + 15 of columns 4 (t % 32) .. + 3. Codes of the transpose go
// through LDS, so that they leave as whole 128-byte lines; the 16-byte pieces of a column stand permuted by column there.
template <bool ROWS>
__global__ void __launch_bounds__(kThreads) k_pack8_t(const float *__restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                                      int rblocks, int cblocks, Packed p, Packed t) {
    OM_LDS_POISON();
    __shared__ uint32_t tops[8][128];
    __shared__ __attribute__((aligned(16))) uint8_t tr[128 * 128];
    const int l = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int rb = (int)(blockIdx.x / cblocks), cb = (int)(blockIdx.x % cblocks);
    const int64_t r0 = (int64_t)rb * 128, c0 = (int64_t)cb * 128, c = c0 + 4 * l;
    floatx4 v[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int64_t r = r0 + 16 * g + i;
        v[i] = r < rows ? load4(x + r * ld + c, cols - c) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    uint32_t top[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) top[e] = max(top[e], finite_bits(v[i][e]));
    *reinterpret_cast<u32x4 *>(&tops[g][4 * l]) = u32x4{top[0], top[1], top[2], top[3]};
    if constexpr (ROWS) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int64_t r = r0 + 16 * g + i;
            if (r < rows) put_block(p, r, cb, cblocks, c, v[i]);
        }
    }
    __syncthreads();
    int s[4];
#pragma unroll
    for (int e = 0; e < 4; e++) s[e] = 0;
#pragma unroll
    for (int q = 0; q < 8; q++) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(&tops[q][4 * l]);
#pragma unroll
        for (int e = 0; e < 4; e++) top[e] = max(top[e], w[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        s[e] = scale_byte(top[e]);
        const float inv = inverse_of(s[e]);
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[i] = encode4(floatx4{v[4 * i][e], v[4 * i + 1][e], v[4 * i + 2][e], v[4 * i + 3][e]}, inv);
        *reinterpret_cast<u32x4 *>(tr + (4 * l + e) * 128 + ((g ^ l) & 7) * 16) = w;
    }
    if (g == 0) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (c + e < cols) {
                uint8_t *d = t.s + (c + e) * t.lds + rb;
                d[0] = (uint8_t)s[e];
                if (rb == rblocks - 1)
                    for (int z = 1; rb + z < t.lds; z++) d[z] = 0;
            }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int col = 32 * i + (threadIdx.x >> 3), piece = threadIdx.x & 7;
        if (c0 + col < cols)
            *reinterpret_cast<u32x4 *>(t.q + (c0 + col) * t.ldq + r0 + 16 * piece) =
                *reinterpret_cast<const u32x4 *>(tr + col * 128 + ((piece ^ (col >> 2)) & 7) * 16);
    }
}

template <bool ACC>
__global__ void __launch_bounds__(kThreads) k_unpack8(Packed p, float *y, int64_t ld, int64_t rows, int64_t cols, int blocks) {
    OM_LDS_POISON();
    uint32_t q[kUnroll];
    int s[kUnroll];
    floatx4 old[kUnroll];
    each_block(rows, blocks,
               [&](int u, int64_t r, int b, int64_t c) {
                   q[u] = *reinterpret_cast<const uint32_t *>(p.q + r * p.ldq + c);
                   s[u] = p.s[r * p.lds + b];
                   if constexpr (ACC) old[u] = load4(y + r * ld + c, cols - c);
               },
               [&](int u, int64_t r, int, int64_t c) {
                   floatx4 v = decode4(q[u], scale_of(s[u]));
                   if constexpr (ACC) v = old[u] + v;
                   store4(y + r * ld + c, cols - c, v);
               });
}

// GELU that keeps its input packed: 4 bytes read and 5 written a value, the erf under their shadow.
template <bool REF>
__global__ void __launch_bounds__(kThreads) k_gelu8(const float *x, float *y, int64_t rows, int64_t cols, int blocks,
                                                    Packed p) {
    OM_LDS_POISON();
    floatx4 v[kUnroll];
    each_block(rows, blocks, [&](int u, int64_t r, int, int64_t c) { v[u] = load4(x + r * cols + c, cols - c); },
               [&](int u, int64_t r, int b, int64_t c) {
                   put_block(p, r, b, blocks, c, v[u]);
                   floatx4 a;
#pragma unroll
                   for (int e = 0; e < 4; e++) a[e] = REF ? omd::gelu(v[u][e]) : omd::gelu_fast(v[u][e]);
                   store4(y + r * cols + c, cols - c, a);
               });
}
template <bool REF, bool ACC>
__global__ void __launch_bounds__(kThreads) k_gelu8_bwd(const float *g, Packed p, float *dx, int64_t rows, int64_t cols,
                                                        int blocks) {
    OM_LDS_POISON();
    uint32_t q[kUnroll];
    int s[kUnroll];
    floatx4 gv[kUnroll], old[kUnroll];
    each_block(rows, blocks,
               [&](int u, int64_t r, int b, int64_t c) {
                   q[u] = *reinterpret_cast<const uint32_t *>(p.q + r * p.ldq + c);
                   s[u] = p.s[r * p.lds + b];
                   gv[u] = load4(g + r * cols + c, cols - c);
                   if constexpr (ACC) old[u] = load4(dx + r * cols + c, cols - c);
               },
               [&](int u, int64_t r, int, int64_t c) {
                   const floatx4 h = decode4(q[u], scale_of(s[u]));
                   floatx4 d;
#pragma unroll
                   for (int e = 0; e < 4; e++) {
                       d[e] = REF ? omd::gelu_grad(gv[u][e], h[e]) : omd::gelu_grad_fast(gv[u][e], h[e]);
                       if constexpr (ACC) d[e] = old[u][e] + d[e];
                   }
                   store4(dx + r * cols + c, cols - c, d);
               });
}

// Workgroups for a walk over rows * blocks half-wavefronts' blocks: each then has up to kUnroll of them, and eight
// workgroups stand on a CU.
constexpr int64_t kMostBlocks = INT32_MAX;
unsigned walk_grid(const om_ctx *ctx, int64_t rows, int64_t blocks) {
    return om::grid1d(rows * blocks, kThreads / 32 * kUnroll, (int64_t)ctx->num_cus * 8);
}

}  // namespace

extern "C" {

uint64_t om_pack8_bytes(int rows, int cols) { return rows > 0 && cols > 0 ? bytes8(rows, cols) : 0; }

om_status om_pack8(om_ctx *ctx, const float *x, int ld_x, int rows, int cols, uint8_t *x8, uint8_t *xt8) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, rows >= 0 && cols >= 0 && ld_x >= cols, "om_pack8: rows=%d cols=%d ld_x=%d", rows, cols, ld_x);
    OM_REQUIRE(ctx, x8 || xt8, "om_pack8: x8 and xt8 are both NULL");
    OM_REQUIRE(ctx, aligned16(x8) && aligned16(xt8), "om_pack8: packed tensors start at multiples of 16 bytes");
    if (rows == 0 || cols == 0) return OM_OK;
    OM_REQUIRE(ctx, x, "om_pack8: NULL x");
    const int64_t rb = blocks8(rows), cb = blocks8(cols);
    OM_REQUIRE(ctx, (xt8 ? rb : (int64_t)rows) * cb <= kMostBlocks, "om_pack8: %d x %d is more than a launch takes", rows, cols);
    if (om_status s = om::use_device(ctx)) return s;
    const Packed p = packed(x8, rows, cols), t = packed(xt8, cols, rows);
    if (!xt8)
        hipLaunchKernelGGL(k_pack8, dim3(walk_grid(ctx, rows, cb)), dim3(kThreads), 0, ctx->stream, x, (int64_t)ld_x,
                           (int64_t)rows, (int64_t)cols, (int)cb, p);
    else if (x8)
        hipLaunchKernelGGL(k_pack8_t<true>, dim3((unsigned)(rb * cb)), dim3(kThreads), 0, ctx->stream, x, (int64_t)ld_x,
                           (int64_t)rows, (int64_t)cols, (int)rb, (int)cb, p, t);
    else
        hipLaunchKernelGGL(k_pack8_t<false>, dim3((unsigned)(rb * cb)), dim3(kThreads), 0, ctx->stream, x, (int64_t)ld_x,
                           (int64_t)rows, (int64_t)cols, (int)rb, (int)cb, p, t);
    return OM_LAUNCH_CHECK(ctx, "om_pack8");
}

om_status om_unpack8(om_ctx *ctx, const uint8_t *x8, float *y, int ld_y, int rows, int cols, int acc) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, rows >= 0 && cols >= 0 && ld_y >= cols, "om_unpack8: rows=%d cols=%d ld_y=%d", rows, cols, ld_y);
    OM_REQUIRE(ctx, aligned16(x8), "om_unpack8: packed tensors start at multiples of 16 bytes");
    if (rows == 0 || cols == 0) return OM_OK;
    OM_REQUIRE(ctx, x8 && y, "om_unpack8: NULL pointer");
    const int64_t cb = blocks8(cols);
    OM_REQUIRE(ctx, rows * cb <= kMostBlocks, "om_unpack8: %d x %d is more than a launch takes", rows, cols);
    if (om_status s = om::use_device(ctx)) return s;
    const Packed p = packed(x8, rows, cols);
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3(walk_grid(ctx, rows, cb)), dim3(kThreads), 0, ctx->stream, p, y, (int64_t)ld_y,
                           (int64_t)rows, (int64_t)cols, (int)cb);
    };
    acc ? go(k_unpack8<true>) : go(k_unpack8<false>);
    return OM_LAUNCH_CHECK(ctx, "om_unpack8");
}

om_status om_gelu_fwd_x8(om_ctx *ctx, const float *x, float *y, uint8_t *x8, int rows, int cols) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, rows >= 0 && cols >= 0, "om_gelu_fwd_x8: rows=%d cols=%d", rows, cols);
    OM_REQUIRE(ctx, aligned16(x8), "om_gelu_fwd_x8: packed tensors start at multiples of 16 bytes");
    if (rows == 0 || cols == 0) return OM_OK;
    OM_REQUIRE(ctx, x && y && x8, "om_gelu_fwd_x8: NULL pointer");
    const int64_t cb = blocks8(cols);
    OM_REQUIRE(ctx, rows * cb <= kMostBlocks, "om_gelu_fwd_x8: %d x %d is more than a launch takes", rows, cols);
    if (om_status s = om::use_device(ctx)) return s;
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3(walk_grid(ctx, rows, cb)), dim3(kThreads), 0, ctx->stream, x, y, (int64_t)rows,
                           (int64_t)cols, (int)cb, packed(x8, rows, cols));
    };
    ctx->gelu_mode == OM_GELU_REFERENCE ? go(k_gelu8<true>) : go(k_gelu8<false>);
    return OM_LAUNCH_CHECK(ctx, "om_gelu_fwd_x8");
}

om_status om_gelu_bwd_x8(om_ctx *ctx, const float *g, const uint8_t *x8, float *dx, int rows, int cols, int acc) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, rows >= 0 && cols >= 0, "om_gelu_bwd_x8: rows=%d cols=%d", rows, cols);
    OM_REQUIRE(ctx, aligned16(x8), "om_gelu_bwd_x8: packed tensors start at multiples of 16 bytes");
    if (rows == 0 || cols == 0) return OM_OK;
    OM_REQUIRE(ctx, g && x8 && dx, "om_gelu_bwd_x8: NULL pointer");
    const int64_t cb = blocks8(cols);
    OM_REQUIRE(ctx, rows * cb <= kMostBlocks, "om_gelu_bwd_x8: %d x %d is more than a launch takes", rows, cols);
    if (om_status s = om::use_device(ctx)) return s;
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3(walk_grid(ctx, rows, cb)), dim3(kThreads), 0, ctx->stream, g, packed(x8, rows, cols),
                           dx, (int64_t)rows, (int64_t)cols, (int)cb);
    };
    if (ctx->gelu_mode == OM_GELU_REFERENCE) acc ? go(k_gelu8_bwd<true, true>) : go(k_gelu8_bwd<true, false>);
    else acc ? go(k_gelu8_bwd<false, true>) : go(k_gelu8_bwd<false, false>);
    return OM_LAUNCH_CHECK(ctx, "om_gelu_bwd_x8");
}

}  // extern "C"
