// Tensors to 8 bits and back (om_pack8.hpp has the format), and GELU with its input kept so.
//
// All of these are bound by HBM: packing reads 4 bytes a value and writes 1 to each packed form, unpacking the reverse
// (16384 x 4096 packed and unpacked 134.8 us, 5.0 TB/s, where a copy reaches 5.1; small tensors take 2.6 to 2.9 us, a launch).
// A block of 128 neighbouring values is one half-wavefront, four values (16 bytes) a lane, so its largest value is one
// reduction over 32 lanes and its codes are one 128-byte line. Two blocks of a row make a wavefront's item; its row and place
// are scalar values.
#include "om_pack8.hpp"

#include <type_traits>

namespace {

using namespace om8;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
constexpr int kThreads = 256;
// Items of one wavefront in flight. Four give the same times on large tensors (61.7 and 61.6 us to pack 16384 x 4096, call behind
// call on one x, which the caches hold in part: 78 us where it comes from HBM, at 5.1 TB/s 65) and take
// longer on small ones (3.5 and 2.9 us for 64 x 256, 4.8 and 3.6 with GELU).
constexpr int kUnroll = 2;

// A wavefront's share of a walk over [rows, cols]: 256 columns of one row, two blocks, four values a lane; of a tensor of one
// block (PAIR) two rows. Row and segment are the same for all lanes, so their arithmetic is scalar.
struct Item {
    int64_t row;  // this lane's
    int64_t col;  // first of this lane's four values
    int blk;      // block of col; the lane has no part in it where blk >= blocks or the row does not exist
    bool in;
    bool whole;   // no lane's values end early (the same for all lanes)
};
// The wavefront's kUnroll neighbouring items: `load(u, item)` for each, then `mid()`, then `use(u, item)`. What mid does for
// all of them at once (the reductions) is not held up by their conditions.
template <bool PAIR, class Load, class Mid, class Use>
__device__ __forceinline__ void each_item(uint32_t wg, int64_t rows, int64_t cols, int blocks, Load load, Mid mid, Use use) {
    const int lane = threadIdx.x & 63;
    const uint32_t segs = PAIR ? 1u : (uint32_t)(blocks + 1) / 2, total = PAIR ? (uint32_t)((rows + 1) / 2) : (uint32_t)rows * segs;
    const uint32_t w = (wg * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kUnroll;
    uint32_t r = w / segs, k = w - r * segs;
    Item it[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
        if constexpr (PAIR) {
            it[u].row = 2 * (int64_t)r + (lane >> 5);
            it[u].col = 4 * (lane & 31);
            it[u].blk = 0;
            it[u].in = w + u < total && it[u].row < rows;
            it[u].whole = cols == 128;
        } else {
            it[u].row = r;
            it[u].col = (int64_t)k * 256 + 4 * lane;
            it[u].blk = 2 * (int)k + (lane >> 5);
            it[u].whole = (int64_t)k * 256 + 256 <= cols;
            it[u].in = w + u < total && (it[u].whole || it[u].blk < blocks);
        }
        if (it[u].in) load(u, it[u]);
        if (++k == segs) {
            k = 0;
            r++;
        }
    }
    mid();
#pragma unroll
    for (int u = 0; u < kUnroll; u++)
        if (it[u].in) use(u, it[u]);
}
__device__ __forceinline__ floatx4 take(const float *p, int64_t ld, int64_t cols, const Item &it) {
    return load4(p + it.row * ld + it.col, it.whole ? 4 : cols - it.col);
}
__device__ __forceinline__ void give(float *p, int64_t ld, int64_t cols, const Item &it, floatx4 v) {
    store4(p + it.row * ld + it.col, it.whole ? 4 : cols - it.col, v);
}
__device__ __forceinline__ floatx4 value_of(const Packed &p, const Item &it) {
    return decode4(*reinterpret_cast<const uint32_t *>(p.q + it.row * p.ldq + it.col), scale_of(p.s[it.row * p.lds + it.blk]));
}

// A lane's four values of a block into the packed row by the block's scale byte s, and the row's scale bytes.
__device__ __forceinline__ void put_block(const Packed &p, int64_t row, int blk, int blocks, int64_t col, floatx4 v, int s) {
    *reinterpret_cast<uint32_t *>(p.q + row * p.ldq + col) = encode4(v, inverse_of(s));
    const int l = threadIdx.x & 31;
    if (l == 0) p.s[row * p.lds + blk] = (uint8_t)s;
    if (blk == blocks - 1 && l > 0 && blk + l < p.lds) p.s[row * p.lds + blk + l] = 0;
}
// Scale bytes of N blocks, a lane's values of each in v.
template <int N>
__device__ __forceinline__ void scales_of(const floatx4 (&v)[N], int (&s)[N]) {
#pragma unroll
    for (int u = 0; u < N; u++) s[u] = scale_byte(max32(finite_bits4(v[u])));
}

template <bool PAIR>
__device__ __forceinline__ void pack_rows(uint32_t wg, const float *__restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                          int blocks, const Packed &p) {
    floatx4 v[kUnroll] = {};
    int s[kUnroll];
    each_item<PAIR>(wg, rows, cols, blocks, [&](int u, const Item &it) { v[u] = take(x, ld, cols, it); },
                    [&] { scales_of(v, s); },
                    [&](int u, const Item &it) { put_block(p, it.row, it.blk, blocks, it.col, v[u], s[u]); });
}
template <bool PAIR>
__global__ void __launch_bounds__(kThreads) k_pack8(const float *__restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                                    int blocks, Packed p) {
    OM_LDS_POISON();
    pack_rows<PAIR>(blockIdx.x, x, ld, rows, cols, blocks, p);
}

// Both forms of a small tensor: the transpose by tiles of 128 rows x 32 columns, and from workgroup `tiles` on the rows, from a
// reading of their own. Four times as many and smaller workgroups than one for 128 x 128 of both, and two barriers in place of
// three: 777 x 1000 4.1 us and 5.1, 2304 x 768 4.7 and 5.4; at 4096 x 768 the second reading costs more (6.2 and 6.0 us), at
// 16384 x 4096 half as much again (121 and 82). Thread t of a tile holds rows 4 (t / 8) .. + 3 of columns 4 (t % 8) .. + 3.
constexpr int64_t kSmall = 1 << 21;
template <bool PAIR>
__global__ void __launch_bounds__(kThreads) k_pack8_small(const float *__restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                                          int blocks, int rblocks, uint32_t tiles, int ctiles, Packed p, Packed t) {
    OM_LDS_POISON();
    if (blockIdx.x >= tiles) return pack_rows<PAIR>(blockIdx.x - tiles, x, ld, rows, cols, blocks, p);
    __shared__ __attribute__((aligned(16))) uint32_t tops[4][32];
    __shared__ __attribute__((aligned(16))) uint32_t tr[32 * 34];  // 34 to a column: the lanes that write meet on no bank
    const int l = threadIdx.x & 7, g = threadIdx.x >> 3, w = threadIdx.x >> 6;
    const int rb = (int)(blockIdx.x / ctiles), ct = (int)(blockIdx.x % ctiles);
    const int64_t r0 = (int64_t)rb * 128 + 4 * g, c0 = (int64_t)ct * 32, c = c0 + 4 * l;
    floatx4 v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = r0 + i < rows ? load4(x + (r0 + i) * ld + c, cols - c) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 top;
#pragma unroll
    for (int e = 0; e < 4; e++) {  // over the eight lanes of the wavefront that have these columns
        uint32_t m = top_of(v[0][e], v[1][e], v[2][e], v[3][e]);
        m = max(m, lane_of16<kRotate8>(m));
        auto o = __builtin_amdgcn_permlane16_swap(m, m, false, false);
        m = max(o[0], o[1]);
        o = __builtin_amdgcn_permlane32_swap(m, m, false, false);
        top[e] = max(o[0], o[1]);
    }
    if ((threadIdx.x & 56) == 0) *reinterpret_cast<u32x4 *>(&tops[w][4 * l]) = top;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const u32x4 o = *reinterpret_cast<const u32x4 *>(&tops[q][4 * l]);
#pragma unroll
        for (int e = 0; e < 4; e++) top[e] = max(top[e], o[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int s = scale_byte(top[e]);
        tr[(4 * l + e) * 34 + g] = encode4(floatx4{v[0][e], v[1][e], v[2][e], v[3][e]}, inverse_of(s));
        if (g == e && c + e < cols) {
            uint8_t *d = t.s + (c + e) * t.lds + rb;
            d[0] = (uint8_t)s;
            if (rb == rblocks - 1)
                for (int z = 1; rb + z < t.lds; z++) d[z] = 0;
        }
    }
    __syncthreads();
    const int col = threadIdx.x >> 3, piece = threadIdx.x & 7;
    if (c0 + col >= cols) return;
    const u32x2 *s = reinterpret_cast<const u32x2 *>(tr + col * 34 + 4 * piece), a = s[0], b = s[1];
    *reinterpret_cast<u32x4 *>(t.q + (c0 + col) * t.ldq + (int64_t)rb * 128 + 16 * piece) = u32x4{a[0], a[1], b[0], b[1]};
}

// The transpose of any tensor (and the tensor itself where ROWS): a workgroup takes 128 rows x 128 columns, so that both kinds
// of blocks are whole. Thread t holds rows 4 (t / 32) .. + 3 of columns 4 (t % 32) .. + 3; sixteen wavefronts, since a small
// tensor has few such tiles and its time is one tile's. Codes of the transpose go through LDS, four rows of a column in a
// dword, so that they leave as whole 128-byte lines; dword g of a column stands at g ^ (column / 4), so that neither the
// lanes that write nor those that read 16 bytes meet on a bank. 16384 x 4096: 82 us with the rows (4.9 TB/s), 67 without.
constexpr int kTile = 1024;
template <bool ROWS>
__global__ void __launch_bounds__(kTile) k_pack8_t(const float *__restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                                   int rblocks, int cblocks, Packed p, Packed t) {
    OM_LDS_POISON();
    __shared__ uint32_t tops[16][128];
    __shared__ float inv[128];
    __shared__ __attribute__((aligned(16))) uint32_t tr[128 * 32];
    const int l = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int rb = (int)(blockIdx.x / cblocks), cb = (int)(blockIdx.x % cblocks);
    const int64_t r0 = (int64_t)rb * 128 + 4 * g, c0 = (int64_t)cb * 128, c = c0 + 4 * l;
    floatx4 v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = r0 + i < rows ? load4(x + (r0 + i) * ld + c, cols - c) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 top;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t m = top_of(v[0][e], v[1][e], v[2][e], v[3][e]);
        const auto o = __builtin_amdgcn_permlane32_swap(m, m, false, false);  // the wavefront's other four rows
        top[e] = max(o[0], o[1]);
    }
    if ((g & 1) == 0) *reinterpret_cast<u32x4 *>(&tops[g >> 1][4 * l]) = top;
    if constexpr (ROWS) {
        int s[4];
        scales_of(v, s);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (r0 + i < rows) put_block(p, r0 + i, cb, cblocks, c, v[i], s[i]);
    }
    __syncthreads();
    if (threadIdx.x < 128) {
        uint32_t m = 0;
#pragma unroll
        for (int q = 0; q < 16; q++) m = max(m, tops[q][threadIdx.x]);
        const int s = scale_byte(m);
        inv[threadIdx.x] = inverse_of(s);
        if (c0 + threadIdx.x < cols) {
            uint8_t *d = t.s + (c0 + threadIdx.x) * t.lds + rb;
            d[0] = (uint8_t)s;
            if (rb == rblocks - 1)
                for (int z = 1; rb + z < t.lds; z++) d[z] = 0;
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; e++)
        tr[(4 * l + e) * 32 + (g ^ l)] = encode4(floatx4{v[0][e], v[1][e], v[2][e], v[3][e]}, inv[4 * l + e]);
    __syncthreads();
    const int col = threadIdx.x >> 3, piece = threadIdx.x & 7, k = col >> 2;
    if (c0 + col < cols) {
        u32x4 w = *reinterpret_cast<const u32x4 *>(tr + col * 32 + 4 * (piece ^ (k >> 2)));
        if (k & 1) w = u32x4{w[1], w[0], w[3], w[2]};
        if (k & 2) w = u32x4{w[2], w[3], w[0], w[1]};
        *reinterpret_cast<u32x4 *>(t.q + (c0 + col) * t.ldq + (int64_t)rb * 128 + 16 * piece) = w;
    }
}

template <bool PAIR, bool ACC>
__global__ void __launch_bounds__(kThreads) k_unpack8(Packed p, float *y, int64_t ld, int64_t rows, int64_t cols, int blocks) {
    OM_LDS_POISON();
    floatx4 v[kUnroll], old[kUnroll];
    each_item<PAIR>(blockIdx.x, rows, cols, blocks,
                    [&](int u, const Item &it) {
                        v[u] = value_of(p, it);
                        if constexpr (ACC) old[u] = take(y, ld, cols, it);
                    },
                    [] {},
                    [&](int u, const Item &it) {
                        if constexpr (ACC) v[u] = old[u] + v[u];
                        give(y, ld, cols, it, v[u]);
                    });
}

// GELU that keeps its input packed: 4 bytes read and 5 written a value, the erf under their shadow (16001 x 1999 forward and
// backward 111.5 us, 5.2 TB/s).
template <bool PAIR, bool REF>
__global__ void __launch_bounds__(kThreads) k_gelu8(const float *x, float *y, int64_t rows, int64_t cols, int blocks,
                                                    Packed p) {
    OM_LDS_POISON();
    floatx4 v[kUnroll] = {};
    int s[kUnroll];
    each_item<PAIR>(blockIdx.x, rows, cols, blocks, [&](int u, const Item &it) { v[u] = take(x, cols, cols, it); },
                    [&] { scales_of(v, s); },
                    [&](int u, const Item &it) {
                        put_block(p, it.row, it.blk, blocks, it.col, v[u], s[u]);
                        floatx4 a;
#pragma unroll
                        for (int e = 0; e < 4; e++) a[e] = REF ? omd::gelu(v[u][e]) : omd::gelu_fast(v[u][e]);
                        give(y, cols, cols, it, a);
                    });
}
template <bool PAIR, bool REF, bool ACC>
__global__ void __launch_bounds__(kThreads) k_gelu8_bwd(const float *g, Packed p, float *dx, int64_t rows, int64_t cols,
                                                        int blocks) {
    OM_LDS_POISON();
    floatx4 h[kUnroll], gv[kUnroll], old[kUnroll];
    each_item<PAIR>(blockIdx.x, rows, cols, blocks,
                    [&](int u, const Item &it) {
                        h[u] = value_of(p, it);
                        gv[u] = take(g, cols, cols, it);
                        if constexpr (ACC) old[u] = take(dx, cols, cols, it);
                    },
                    [] {},
                    [&](int u, const Item &it) {
                        floatx4 d;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            d[e] = REF ? omd::gelu_grad(gv[u][e], h[u][e]) : omd::gelu_grad_fast(gv[u][e], h[u][e]);
                            if constexpr (ACC) d[e] = old[u][e] + d[e];
                        }
                        give(dx, cols, cols, it, d);
                    });
}

// Workgroups of a walk over [rows, cols]; f(whether the tensor is one block wide, grid) for it.
int64_t walk_groups(int64_t rows, int64_t blocks) {
    const int64_t items = blocks == 1 ? (rows + 1) / 2 : rows * ((blocks + 1) / 2), per = kThreads / 64 * kUnroll;
    return (items + per - 1) / per;
}
template <class F>
void walk(int64_t rows, int64_t blocks, F f) {
    const dim3 grid((unsigned)walk_groups(rows, blocks));
    blocks == 1 ? f(std::true_type(), grid) : f(std::false_type(), grid);
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
    OM_REQUIRE(ctx, xt8 ? launches(rb * cb, kTile) : launches(walk_groups(rows, cb), kThreads),
               "om_pack8: %d x %d is more than a launch takes", rows, cols);
    if (om_status s = om::use_device(ctx)) return s;
    const Packed p = packed(x8, rows, cols), t = packed(xt8, cols, rows);
    if (!xt8)
        walk(rows, cb, [&](auto pair, dim3 grid) {
            hipLaunchKernelGGL(k_pack8<decltype(pair)::value>, grid, dim3(kThreads), 0, ctx->stream, x, (int64_t)ld_x,
                               (int64_t)rows, (int64_t)cols, (int)cb, p);
        });
    else if (x8 && (int64_t)rows * cols <= kSmall) {
        const int ct = (int)(((int64_t)cols + 31) / 32);
        const uint32_t tiles = (uint32_t)(rb * ct);
        walk(rows, cb, [&](auto pair, dim3 grid) {
            hipLaunchKernelGGL(k_pack8_small<decltype(pair)::value>, dim3(grid.x + tiles), dim3(kThreads), 0, ctx->stream, x,
                               (int64_t)ld_x, (int64_t)rows, (int64_t)cols, (int)cb, (int)rb, tiles, ct, p, t);
        });
    } else if (x8)
        hipLaunchKernelGGL(k_pack8_t<true>, dim3((unsigned)(rb * cb)), dim3(kTile), 0, ctx->stream, x, (int64_t)ld_x,
                           (int64_t)rows, (int64_t)cols, (int)rb, (int)cb, p, t);
    else
        hipLaunchKernelGGL(k_pack8_t<false>, dim3((unsigned)(rb * cb)), dim3(kTile), 0, ctx->stream, x, (int64_t)ld_x,
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
    OM_REQUIRE(ctx, launches(walk_groups(rows, cb), kThreads), "om_unpack8: %d x %d is more than a launch takes", rows,
               cols);
    if (om_status s = om::use_device(ctx)) return s;
    const Packed p = packed(x8, rows, cols);
    walk(rows, cb, [&](auto pair, dim3 grid) {
        constexpr bool P = decltype(pair)::value;
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, ctx->stream, p, y, (int64_t)ld_y, (int64_t)rows, (int64_t)cols,
                               (int)cb);
        };
        acc ? go(k_unpack8<P, true>) : go(k_unpack8<P, false>);
    });
    return OM_LAUNCH_CHECK(ctx, "om_unpack8");
}

om_status om_gelu_fwd_x8(om_ctx *ctx, const float *x, float *y, uint8_t *x8, int rows, int cols) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, rows >= 0 && cols >= 0, "om_gelu_fwd_x8: rows=%d cols=%d", rows, cols);
    OM_REQUIRE(ctx, aligned16(x8), "om_gelu_fwd_x8: packed tensors start at multiples of 16 bytes");
    if (rows == 0 || cols == 0) return OM_OK;
    OM_REQUIRE(ctx, x && y && x8, "om_gelu_fwd_x8: NULL pointer");
    const int64_t cb = blocks8(cols);
    OM_REQUIRE(ctx, launches(walk_groups(rows, cb), kThreads), "om_gelu_fwd_x8: %d x %d is more than a launch takes", rows,
               cols);
    if (om_status s = om::use_device(ctx)) return s;
    walk(rows, cb, [&](auto pair, dim3 grid) {
        constexpr bool P = decltype(pair)::value;
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, ctx->stream, x, y, (int64_t)rows, (int64_t)cols, (int)cb,
                               packed(x8, rows, cols));
        };
        ctx->gelu_mode == OM_GELU_REFERENCE ? go(k_gelu8<P, true>) : go(k_gelu8<P, false>);
    });
    return OM_LAUNCH_CHECK(ctx, "om_gelu_fwd_x8");
}

om_status om_gelu_bwd_x8(om_ctx *ctx, const float *g, const uint8_t *x8, float *dx, int rows, int cols, int acc) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, rows >= 0 && cols >= 0, "om_gelu_bwd_x8: rows=%d cols=%d", rows, cols);
    OM_REQUIRE(ctx, aligned16(x8), "om_gelu_bwd_x8: packed tensors start at multiples of 16 bytes");
    if (rows == 0 || cols == 0) return OM_OK;
    OM_REQUIRE(ctx, g && x8 && dx, "om_gelu_bwd_x8: NULL pointer");
    const int64_t cb = blocks8(cols);
    OM_REQUIRE(ctx, launches(walk_groups(rows, cb), kThreads), "om_gelu_bwd_x8: %d x %d is more than a launch takes", rows,
               cols);
    if (om_status s = om::use_device(ctx)) return s;
    walk(rows, cb, [&](auto pair, dim3 grid) {
        constexpr bool P = decltype(pair)::value;
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, ctx->stream, g, packed(x8, rows, cols), dx, (int64_t)rows,
                               (int64_t)cols, (int)cb);
        };
        if (ctx->gelu_mode == OM_GELU_REFERENCE) acc ? go(k_gelu8_bwd<P, true, true>) : go(k_gelu8_bwd<P, true, false>);
        else acc ? go(k_gelu8_bwd<P, false, true>) : go(k_gelu8_bwd<P, false, false>);
    });
    return OM_LAUNCH_CHECK(ctx, "om_gelu_bwd_x8");
}

}  // extern "C"
