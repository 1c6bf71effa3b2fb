// Products of packed tensors (om_pack8.hpp has the format): C[m, n] (+)= sum over k of A[m, k] B[n, k], both packed along k,
// and a Linear's weight gradient from an fp32 gradient and its packed input, dW[o, i] (+)= sum over rows of g[r, o] xt8[i, r].
//
// Arithmetic. An e4m3 code times a power of two is a bf16 value (4 significand bits of 8), so the codes are widened in
// registers, v_cvt_scalef32_pk_bf16_fp8 with the block's scale, and multiplied by v_mfma_f32_32x32x16_bf16: every product is
// exact and sums are fp32 (2-norm error 1e-7 at k = 4096). The 8-bit matrix instructions have up to twice the rate (bare
// instructions, scaled 32x32x64 4590 TFLOP/s, bf16 32x32x16 2170), but do not keep their sums: a dot product comes out 1.2e-5 off
// in the 2-norm over 32 terms, 1.5e-5 over 128 and over 4096 (normal values; 4e-5 to 5e-5 with all exponents in use), as if their
// adder dropped what is 2^-13 or so below its largest term. That does not grow with k: to keep exact products and fp32 sums is a
// choice, paid with up to half the rate of large products. The conversion costs two to three vector
// instructions an MFMA at 64 x 64 to 128 x 64 values a wavefront and runs beside it (16 k of both: 15.4 ns an MFMA alone,
// 16.6 with six conversions to each).
//
// Bound: large products by the clock that the card keeps under matrix work (4096^3 107 to 111 us, 1240 to 1285 TFLOP/s; without
// the loads 101, without the conversions 104; the library's bf16 product, which converts nothing and reads twice the bytes,
// 105 to 112); small ones by the launch and one chain of loads, 3 to 6 us.
#include "om_gemm8_choose.hpp"
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

// 16 (or 4) bytes a lane from base (uniform) + off (this lane's) to LDS at byte address lds + 16 (4) * lane, without registers. m0
// holds the address for this one instruction only, which needs a wait state (s_nop 0) between the write and its read; nothing else
// in these kernels reads it. Loads land in the order of their issue; land<N>() waits until at most this wavefront's last N are in
// flight and its own LDS reads are done, then meets the others.
__device__ __forceinline__ void load_to_lds(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds4(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
// The same with an address to each lane.
__device__ __forceinline__ void load_to_lds4(const void *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void land() {
    static_assert(N <= 63, "vmcnt holds at most 63");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

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
// load the last one again; what they give is not stored. Offsets inside a tile stay in 32 bits (the host checks).
template <int ROWS, int NW>
struct Stage {
    static constexpr int PER = ROWS / 8 / NW;
    static_assert(ROWS % (8 * NW) == 0, "whole instructions to each wavefront");
    const uint8_t *q, *s;  // of the tile's first row
    uint32_t off[PER], soff;
    __device__ __forceinline__ Stage(const Packed &p, int r0, int rows, int wv, int lane) {
        q = p.q + (int64_t)r0 * p.ldq;
        s = p.s + (int64_t)r0 * p.lds;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int r = 8 * (wv * PER + i) + (lane >> 3), piece = (lane ^ (r >> 1)) & 7;
            off[i] = (uint32_t)min(r, rows - 1 - r0) * (uint32_t)p.ldq + 16 * piece;
        }
        soff = (uint32_t)min((wv * 64 + lane) % ROWS, rows - 1 - r0) * (uint32_t)p.lds;
    }
    __device__ __forceinline__ void load(int blk, uint32_t lds, int wv) const {
#pragma unroll
        for (int i = 0; i < PER; i++) load_to_lds(q + (int64_t)blk * 128, off[i], lds + (wv * PER + i) * 1024);
    }
    // The scale dword that holds block blk's byte, of every row.
    __device__ __forceinline__ void load_scales(int blk, uint32_t lds, int wv) const {
        if (wv < (ROWS + 63) / 64) load_to_lds4(s + (blk & ~3), soff, lds + wv * 256);
    }
};

__device__ __forceinline__ float scale_in(uint32_t dword, int blk) { return scale_of((int)(dword >> (8 * (blk & 3))) & 255); }

// One half chunk (16 k) of a wavefront's MT x NT blocks: its MFMAs from the widened operands w, and between them, in this
// order, the conversions of the half that comes next and what `beside` has to do: the matrix pipe takes 32 cycles an MFMA,
// the four to six instructions after it go under those. (Left to itself the compiler gathers the conversions, and the two
// pipes take turns.)
template <int MT, int NT, class Raw, class Scale, class Beside>
__device__ __forceinline__ void half_chunk(floatx16 (&acc)[MT][NT], const u32x4 (&w)[MT + NT], u32x4 (&next)[MT + NT], Raw raw,
                                           Scale scale, Beside beside) {
    constexpr int M = MT * NT, V = 2 * (MT + NT);  // conversions in pairs
#pragma unroll
    for (int f = 0; f < M; f++) {
        acc[f / NT][f % NT] = oms::mma(w[f / NT], w[MT + f % NT], acc[f / NT][f % NT]);
        beside(f);
#pragma unroll
        for (int v = f * V / M; v < (f + 1) * V / M; v++) {
            const int o = v / 2, h = v & 1;
            const uint32_t c = raw(o, h);
            next[o][2 * h] = widen2(c, scale(o), std::false_type());
            next[o][2 * h + 1] = widen2(c, scale(o), std::true_type());
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Where finished sums go: a split's own partial sums, or C with the bias (-0, which changes nothing, where there is none).
struct Out {
    float *base;
    int64_t ld;
    const float *bias;
    bool acc;
    __device__ __forceinline__ Out(const Gemm8 &p, int split) {
        const bool part = p.splits > 1;
        base = part ? p.ws + (int64_t)split * p.m * p.n : p.c;
        ld = part ? p.n : p.ldc;
        bias = part ? nullptr : p.bias;
        acc = !part && p.acc;
    }
    __device__ __forceinline__ float bias_of(int col) const { return bias ? bias[col] : -0.0f; }
    __device__ __forceinline__ void put(int row, int col, float v, float bias) const {
        float *c = base + row * ld + col;
        v = v + bias;
        *c = acc ? *c + v : v;
    }
};

// A workgroup of WM x WN wavefronts computes BM x BN of C in stages of 128 k, two of them in LDS: the next one's loads are
// issued as the current one begins. Products of few stages gain from more and smaller workgroups on a CU, not from more stages
// in LDS (4096 x 1536 x 384: 128 x 64 with two stages and three workgroups a CU 11.3 us, with three and two 13.5, with six and
// one 18.9). A lane's 16-byte piece g + 2 j (g = lane / 32) of a row feeds two MFMAs, which so see
// k = 32 j + 16 g + 8 t + e in place of their own order, alike for both operands.
template <int BM, int BN, int WM, int WN, int WAVES>
__global__ void __launch_bounds__(64 * WM * WN, WAVES) k_gemm8(Gemm8 p) {
    OM_LDS_POISON();
    constexpr int NW = WM * WN, MT = BM / WM / 32, NT = BN / WN / 32;
    constexpr int AS = BM * 128, BS = AS + BN * 128, SS = BS + (BM + 63) / 64 * 256, STAGE = SS + (BN + 63) / 64 * 256;
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
    // A stage is four chunks of 32 k, a chunk two halves of 16. Operands 0 .. MT - 1 are A's blocks, the others B's. A chunk's
    // codes are read a chunk ahead, a half's are widened a half ahead. The barrier stands before a stage's last chunk, whose
    // codes are in registers by then, so that the next stage's first ones follow without a gap and the stage just read is
    // free for the loads of the one after the next.
    u32x4 raw[2][MT + NT], w[2][MT + NT];
    float sc[2][MT + NT];
    auto row_at = [&](int o) { return o < MT ? (wm + 32 * o + l32) : BM + wn + 32 * (o - MT) + l32; };
    auto read = [&](int h, const char *cur, int q, int o) {
        raw[h][o] = *reinterpret_cast<const u32x4 *>(cur + piece_at(row_at(o), 2 * q + g));
    };
    auto read_scale = [&](const char *cur, int o) { return *reinterpret_cast<const uint32_t *>(cur + BS + 4 * row_at(o)); };
    auto first_half = [&](int q, const char *cur, int nq) {  // reads chunk nq of `cur` meanwhile
        half_chunk<MT, NT>(acc, w[0], w[1], [&](int o, int h) { return raw[q & 1][o][2 + h]; }, [&](int o) { return sc[0][o]; },
                           [&](int f) {
#pragma unroll
                               for (int o = f * (MT + NT) / (MT * NT); o < (f + 1) * (MT + NT) / (MT * NT); o++)
                                   read((q + 1) & 1, cur, nq, o);
                           });
    };
    auto second_half = [&](int q, int s) {
        half_chunk<MT, NT>(acc, w[1], w[0], [&](int o, int h) { return raw[(q + 1) & 1][o][h]; },
                           [&](int o) { return sc[s][o]; }, [](int) {});
    };
    if (b0 < b1) {  // (k may be 0)
        issue(b0, base);
        land<0>();
        if (b0 + 1 < b1) issue(b0 + 1, base + STAGE);
#pragma unroll
        for (int o = 0; o < MT + NT; o++) {
            read(0, sh, 0, o);
            sc[0][o] = sc[1][o] = scale_in(read_scale(sh, o), b0);
            w[0][o] = widen8(raw[0][o][0], raw[0][o][1], sc[0][o]);
        }
        for (int blk = b0; blk < b1; blk++) {
            const int at = ((blk - b0) & 1) * STAGE;
#pragma unroll
            for (int q = 0; q < 3; q++) {
                first_half(q, sh + at, q + 1);
                second_half(q, 0);
            }
            if (blk + 1 < b1) {
                land<0>();
                if (blk + 2 < b1) issue(blk + 2, base + at);
#pragma unroll
                for (int o = 0; o < MT + NT; o++) sc[1][o] = scale_in(read_scale(sh + (STAGE - at), o), blk + 1);
            }
            first_half(3, sh + (STAGE - at), 0);  // (past the last stage what the other buffer holds, for nothing)
            second_half(3, 1);
#pragma unroll
            for (int o = 0; o < MT + NT; o++) sc[0][o] = sc[1][o];
        }
    }
    // A register is one row, 32 neighbouring columns over the lanes: stores of whole 128-byte lines.
    const Out to(p, split);
    const bool whole = m0 + BM <= p.m;
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int col = n0 + wn + 32 * j + l32;
        if (col >= p.n) continue;
        const float bias = to.bias_of(col);
#pragma unroll
        for (int i = 0; i < MT; i++) {
            const int row = m0 + wm + 32 * i + 4 * g;
            float *c = to.base + row * to.ld + col;
            float old[16];
            if (to.acc) {
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int r = 8 * (e >> 2) + (e & 3);
                    if (whole || row + r < p.m) old[e] = c[r * to.ld];
                }
#pragma unroll
                for (int e = 0; e < 16; e++) acc[i][j][e] = old[e] + (acc[i][j][e] + bias);
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++) acc[i][j][e] += bias;
            }
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int r = 8 * (e >> 2) + (e & 3);
                if (whole || row + r < p.m) c[r * to.ld] = acc[i][j][e];
            }
        }
    }
}

// Few tiles: the NW wavefronts of a workgroup share one tile of 32 x 32 and take every NW-th block of 128 k each, alone: the next
// block is on its way into a wavefront's own part of LDS while this one is multiplied, and nothing meets before the sums do, in
// LDS and in order. (Four wavefronts on quarters of each block, with a barrier a block and four blocks in flight: 777 x 333 x 1000
// 6.2 us, so 5.2; 4096 x 384 x 1536 13.9 and 11.3; 100 x 4096 x 4096 11.7 and 9.4.)
template <int NW>
__global__ void __launch_bounds__(64 * NW) k_gemm8_few(Gemm8 p) {
    OM_LDS_POISON();
    constexpr int SLOT = 64 * 128 + 256, LD = 33, OUT = NW * 32 * LD * 4, LDS = NW * SLOT > OUT ? NW * SLOT : OUT;
    __shared__ __attribute__((aligned(16))) char sh[LDS];
    const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int split, tm, tn;
    tile_of(p.tiles_m, p.tiles_n, gridDim.x, split, tm, tn);
    const int m0 = 32 * tm, n0 = 32 * tn;
    const int b0 = split * p.per, b1 = min(p.blocks, b0 + p.per);
    // Rows 0 .. 31 of a block are A's, the others B's, eight a load; rows past the last one load it again, and what they give is
    // not stored.
    const uint8_t *qa = p.a.q + (int64_t)m0 * p.a.ldq, *qb = p.b.q + (int64_t)n0 * p.b.ldq;
    uint32_t off[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = 8 * i + (lane >> 3), piece = (lane ^ (r >> 1)) & 7;
        const bool a = i < 4;
        off[i] = (uint32_t)min(a ? r : r - 32, (a ? p.m - m0 : p.n - n0) - 1) * (uint32_t)(a ? p.a.ldq : p.b.ldq) + 16 * piece;
    }
    const uint8_t *ss = g ? p.b.s + (int64_t)min(n0 + l32, p.n - 1) * p.b.lds : p.a.s + (int64_t)min(m0 + l32, p.m - 1) * p.a.lds;
    const char *mine = sh + wv * SLOT;
    const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)sh + (uint32_t)wv * SLOT;
    auto issue = [&](int k) {
#pragma unroll
        for (int i = 0; i < 8; i++) load_to_lds((i < 4 ? qa : qb) + (int64_t)k * 128, off[i], at + 1024 * i);
        load_to_lds4(ss + (k & ~3), at + 64 * 128);
    };
    floatx16 acc[1][1];
#pragma unroll
    for (int e = 0; e < 16; e++) acc[0][0][e] = 0.0f;
    if (b0 + wv < b1) {
        issue(b0 + wv);
        for (int blk = b0 + wv; blk < b1; blk += NW) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            u32x4 raw[4][2], w[2][2];
            float sc[2];
#pragma unroll
            for (int o = 0; o < 2; o++) {
                sc[o] = scale_in(*reinterpret_cast<const uint32_t *>(mine + 64 * 128 + 4 * (32 * o + l32)), blk);
#pragma unroll
                for (int q = 0; q < 4; q++) raw[q][o] = *reinterpret_cast<const u32x4 *>(mine + piece_at(32 * o + l32, 2 * q + g));
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read, so the next may be loaded over it
            if (blk + NW < b1) issue(blk + NW);
#pragma unroll
            for (int o = 0; o < 2; o++) w[0][o] = widen8(raw[0][o][0], raw[0][o][1], sc[o]);
#pragma unroll
            for (int h = 0; h < 8; h++)  // (the last half converts its own codes again, for nothing)
                half_chunk<1, 1>(acc, w[h & 1], w[(h & 1) ^ 1],
                                 [&](int o, int t) { return raw[min(h + 1, 7) / 2][o][2 * (min(h + 1, 7) & 1) + t]; },
                                 [&](int o) { return sc[o]; }, [](int) {});
        }
    }
    __syncthreads();
    float *out = reinterpret_cast<float *>(sh);
#pragma unroll
    for (int e = 0; e < 16; e++) out[(wv * 32 + 8 * (e >> 2) + 4 * g + (e & 3)) * LD + l32] = acc[0][0][e];
    __syncthreads();
    const Out to(p, split);
    constexpr int EACH = 16 / NW;  // values a thread
    const int c = threadIdx.x % 32, col = n0 + c;
    if (col >= p.n) return;
    const float bias = to.bias_of(col);
    float v[EACH];
#pragma unroll
    for (int u = 0; u < EACH; u++) {
        const int r = threadIdx.x / 32 + u * 2 * NW;
        v[u] = out[r * LD + c];
#pragma unroll
        for (int w = 1; w < NW; w++) v[u] += out[(w * 32 + r) * LD + c];
    }
#pragma unroll
    for (int u = 0; u < EACH; u++) {
        const int row = m0 + threadIdx.x / 32 + u * 2 * NW;
        if (row < p.m) to.put(row, col, v[u], bias);
    }
}

// At most 16 MR rows of A: a workgroup computes 16 columns on v_mfma_f32_16x16x32_bf16, its NW wavefronts a share of k each.
// Each wavefront goes through its blocks of 128 k alone, the next one on its way into its own part of LDS while this one is
// multiplied (whole 128-byte rows; loaded straight into fragments, 64 bytes of 16 rows at a time, they take three times as
// long), so nothing meets before the sums do. More wavefronts hide a block's latency better than more blocks in flight (17 x 2048
// x 2048: eight 4.1 us, four with two blocks each 4.45) until a CU has several workgroups (17 x 8192 x 4096: eight 9.2, four 8.2).
// Bound: latency, then B's bytes (16 x 4096 x 4096 5.2 us, 3.2 TB/s).
template <int NW, int MR>
__global__ void __launch_bounds__(64 * NW) k_gemm8_thin(Gemm8 p) {
    OM_LDS_POISON();
    typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
    constexpr int ROWS = 16 * (MR + 1), SLOT = ROWS * 128 + 256;
    static_assert(ROWS <= 64, "one load of scales");
    constexpr int AT_B = MR * 2048, AT_S = ROWS * 128, OUT = NW * MR * 1024, LDS = NW * SLOT > OUT ? NW * SLOT : OUT;
    __shared__ __attribute__((aligned(16))) char sh[LDS];
    const int lane = threadIdx.x & 63, row = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per = (p.blocks + NW - 1) / NW, b0 = wv * per, b1 = min(p.blocks, b0 + per);
    // Rows and columns past the last one are the last one again; what they give is not stored.
    uint32_t oa[2 * MR], ob[2];
#pragma unroll
    for (int i = 0; i < 2 * MR; i++) {
        const int r = 8 * i + (lane >> 3), piece = (lane ^ (r >> 1)) & 7;
        oa[i] = (uint32_t)min(r, p.m - 1) * (uint32_t)p.a.ldq + 16 * piece;
        if (i < 2) ob[i] = (uint32_t)min(r, p.n - 1 - n0) * (uint32_t)p.b.ldq + 16 * piece;
    }
    const uint8_t *qb = p.b.q + (int64_t)n0 * p.b.ldq;
    // scale dwords: A's rows, then B's, and B's again
    const uint8_t *ss =
        lane < 16 * MR ? p.a.s + (int64_t)min(lane, p.m - 1) * p.a.lds : p.b.s + (int64_t)min(n0 + row, p.n - 1) * p.b.lds;
    const char *mine = sh + wv * SLOT;
    const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)sh + (uint32_t)wv * SLOT;
    auto issue = [&](int k) {
#pragma unroll
        for (int i = 0; i < 2 * MR; i++) load_to_lds(p.a.q + (int64_t)k * 128, oa[i], at + 1024 * i);
#pragma unroll
        for (int i = 0; i < 2; i++) load_to_lds(qb + (int64_t)k * 128, ob[i], at + AT_B + 1024 * i);
        load_to_lds4(ss + (k & ~3), at + AT_S);
    };
    floatx4 acc[MR];
#pragma unroll
    for (int i = 0; i < MR; i++) acc[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    if (b0 < b1) {
        issue(b0);
        for (int blk = b0; blk < b1; blk++) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            u32x4 a[MR + 1][2];  // B's last
            float f[MR + 1];
#pragma unroll
            for (int i = 0; i <= MR; i++) {
#pragma unroll
                for (int j = 0; j < 2; j++) a[i][j] = *reinterpret_cast<const u32x4 *>(mine + 2048 * i + piece_at(row, 4 * j + g));
                f[i] = scale_in(*reinterpret_cast<const uint32_t *>(mine + AT_S + 4 * (16 * i + row)), blk);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read, so the next may be loaded over it
            if (blk + 1 < b1) issue(blk + 1);
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const auto b = __builtin_bit_cast(bf16x8, widen8(a[MR][j][2 * t], a[MR][j][2 * t + 1], f[MR]));
#pragma unroll
                    for (int i = 0; i < MR; i++)
                        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            __builtin_bit_cast(bf16x8, widen8(a[i][j][2 * t], a[i][j][2 * t + 1], f[i])), b, acc[i], 0, 0, 0);
                }
        }
    }
    __syncthreads();
    float *out = reinterpret_cast<float *>(sh);
#pragma unroll
    for (int i = 0; i < MR; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) out[(wv * MR + i) * 256 + (4 * g + e) * 16 + row] = acc[i][e];
    __syncthreads();
    const Out to(p, 0);
    const int col = n0 + (threadIdx.x & 15);
    if (col >= p.n) return;
    const float bias = to.bias_of(col);
#pragma unroll
    for (int i = threadIdx.x >> 4; i < 16 * MR; i += 4 * NW) {
        if (i >= p.m) break;
        const int at = 16 * i + (threadIdx.x & 15);
        float v = out[at];
#pragma unroll
        for (int w = 1; w < NW; w++) v += out[256 * MR * w + at];
        to.put(i, col, v, bias);
    }
}

// The sum of `parts` values `stride` apart, in order, eight loads in flight.
template <class T>
__device__ __forceinline__ T add_parts(const T *p, int64_t stride, int parts) {
    T v = p[0];
    for (int s0 = 1; s0 < parts; s0 += 8) {
        T w[8];
#pragma unroll
        for (int u = 0; u < 8; u++) w[u] = s0 + u < parts ? p[(s0 + u) * stride] : T(0);
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (s0 + u < parts) v += w[u];
    }
    return v;
}

// Adds the splits' sums in order, then bias and C.
__global__ void __launch_bounds__(256) k_gemm8_join(Gemm8 p) {
    OM_LDS_POISON();
    const int64_t total = (int64_t)p.m * p.n, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        float v = add_parts(p.ws + i, total, p.splits);
        const int64_t row = i / p.n, col = i - row * p.n;
        if (p.bias) v = v + p.bias[col];
        float *c = p.c + row * p.ldc + col;
        *c = p.acc ? *c + v : v;
    }
}

om_status gemm8(om_ctx *ctx, Gemm8 p) {
    if (const Thin t = choose_thin(ctx->num_cus, p.m, p.n, p.blocks); t.mr) {
        OM_REQUIRE(ctx, launches(t.groups, 64 * t.nw), "om_gemm8: n=%d is more than a launch takes", p.n);
        if (om_status s = om::use_device(ctx)) return s;
        p.splits = 1;
        auto go = [&](auto eight, auto four) {
            hipLaunchKernelGGL(t.nw == 8 ? eight : four, dim3((unsigned)t.groups), dim3(64 * t.nw), 0, ctx->stream, p);
        };
        switch (t.mr) {
            case 1: go(k_gemm8_thin<8, 1>, k_gemm8_thin<4, 1>); break;
            case 2: go(k_gemm8_thin<8, 2>, k_gemm8_thin<4, 2>); break;
            default: go(k_gemm8_thin<8, 3>, k_gemm8_thin<4, 3>); break;
        }
        return OM_LAUNCH_CHECK(ctx, "om_gemm8");
    }
    const Choice ch = choose_product(ctx->num_cus, p.m, p.n, p.blocks, p.a.ldq);
    OM_REQUIRE(ctx, ch.tile >= 0, "om_gemm8: k is more than a launch takes");
    const Tile &c = kTiles[ch.tile];
    p.tiles_m = (int)(((int64_t)p.m + c.bm - 1) / c.bm);
    p.tiles_n = (int)(((int64_t)p.n + c.bn - 1) / c.bn);
    split_blocks(p.blocks, ch.splits, p.per, p.splits);
    const int64_t wgs = (int64_t)p.tiles_m * p.tiles_n * p.splits;
    const int threads = ch.tile == 0 || ch.tile == 5 ? 512 : 256;
    OM_REQUIRE(ctx, launches(wgs, threads), "om_gemm8: %d x %d is more than a launch takes", p.m, p.n);
    if (om_status s = om::use_device(ctx)) return s;
    if (p.splits > 1)
        if (om_status s = om::scratch(ctx, sizeof(float) * (uint64_t)p.splits * (uint64_t)p.m * (uint64_t)p.n, &p.ws)) return s;
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(threads), 0, ctx->stream, p); };
    switch (ch.tile) {
        case 0: go(k_gemm8<256, 256, 2, 4, 2>); break;
        case 1: go(k_gemm8<128, 128, 2, 2, 2>); break;
        case 2: go(k_gemm8<128, 64, 2, 2, 3>); break;
        case 3: go(k_gemm8<64, 64, 2, 2, 4>); break;
        case 4: go(k_gemm8_few<4>); break;
        default: go(k_gemm8_few<8>); break;
    }
    if (p.splits > 1)
        hipLaunchKernelGGL(k_gemm8_join, dim3(om::grid1d((int64_t)p.m * p.n, 256, (int64_t)ctx->num_cus * 8)), dim3(256), 0,
                           ctx->stream, p);
    return OM_LAUNCH_CHECK(ctx, "om_gemm8");
}

// ------------------------------------------------------------------------------------------------- weight gradient
// dW = g^T x with x packed along the rows and g as it is. g is split into three bf16 parts that hold all of its bits (h + m +
// l; parts below 2^-126, which only values below 2^-103 have, may count as zero), a value of x is one part, so a product is three MFMAs (six with x in fp32)
// and as exact as those. A wavefront owns 32 rows of dW (columns of g) and all BN columns, so g is split once; 16384 x 4096 x
// 4096 takes 1470 us, 1120 TFLOP/s of bf16 products and 85 to 90 % of the library's rate, with six vector instructions beside
// each MFMA (64 x 128 by two such groups, x widened for both: 1490 us; 32 x 256: 1503). Sums that come out infinite or NaN (an
// infinite g, whose parts are NaN; a g that rounds up past bf16's range) are formed again on the fp32 instruction.
struct Dw8 {
    const float *g;         // [rows, m]
    Packed x;               // [n, rows]
    int rows, m, n, blocks;
    int full;               // pieces of 128 (k_dw8_few: 64) whole rows that are loaded four columns at a time
    float *dw, *db;
    int acc_dw, acc_db;
    int splits, per;
    float *ws;              // splits > 1: [split][m][n], behind them (8-byte aligned) the column sums [split][m]
    double *cs;
    int tiles_m, tiles_n;
};

// The parts of two values, in two steps: the first part and what it leaves (x), then the other two.
__device__ __forceinline__ uint32_t split_first(float &x0, float &x1) {
    uint32_t h = oms::pack2(x0, x1);
    asm("" : "+v"(h));  // else the compiler converts x0 a second time instead of shifting h
    x0 -= __uint_as_float(h << 16);
    x1 -= __uint_as_float(h & 0xFFFF0000u);
    return h;
}
__device__ __forceinline__ void split_rest(float r0, float r1, uint32_t &m, uint32_t &l) {
    m = oms::pack2(r0, r1);
    asm("" : "+v"(m));
    l = oms::pack2(r0 - __uint_as_float(m << 16), r1 - __uint_as_float(m & 0xFFFF0000u));
}

// t + the products of `count` rows from k0 on with this lane's column of x (codes cq, scales cx) and of g, on the fp32
// instruction, two rows at a time.
__device__ __forceinline__ floatx16 add_rows8(const Dw8 &p, const uint8_t *cq, const uint8_t *cx, int gc, int k0, int count, floatx16 t) {
    const int g = (threadIdx.x >> 5) & 1;
#pragma unroll 1
    for (int end = min(k0 + count, p.rows); k0 < end; k0 += 2) {
        const int k = min(k0 + g, p.rows - 1);
        const bool in = k0 + g < p.rows;
        const float x = decode4(cq[k], scale_of(cx[k >> 7]))[0], gv = p.g[(int64_t)k * p.m + gc];
        t = __builtin_amdgcn_mfma_f32_32x32x2f32(in ? gv : 0.0f, in ? x : 0.0f, t, 0, 0, 0);
    }
    return t;
}

// The end of a workgroup whose NW wavefronts have a share of k each: their column sums and sums meet in LDS (at least NW * 32 *
// (32 NT + 1) floats of it, free once all have come here) and are added in order.
template <int NT, int NW>
__device__ __forceinline__ void finish_dw8(const Dw8 &p, int split, int tn, int m0, int n0, const floatx16 (&acc)[NT], double cs, char *sh) {
    constexpr int BN = 32 * NT, LD = BN + 1;
    const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5, wv = threadIdx.x >> 6;
    const bool sums = p.db && tn == 0;
    __syncthreads();
    if (sums) {
        cs += __shfl_xor(cs, 32, 64);
        double *shd = reinterpret_cast<double *>(sh);
        if (g == 0) shd[wv * 32 + l32] = cs;
        __syncthreads();
        const int row = m0 + l32;
        if (wv == 0 && g == 0 && row < p.m) {
#pragma unroll
            for (int i = 1; i < NW; i++) cs += shd[i * 32 + l32];
            if (p.splits > 1) {
                p.cs[(int64_t)split * p.m + row] = cs;
            } else {
                const float v = (float)cs;
                p.db[row] = p.acc_db ? p.db[row] + v : v;
            }
        }
        __syncthreads();
    }
    float *out = reinterpret_cast<float *>(sh);
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) out[(wv * 32 + 8 * (e >> 2) + 4 * g + (e & 3)) * LD + 32 * j + l32] = acc[j][e];
    __syncthreads();
    constexpr int STEP = 64 * NW / BN, EACH = 32 / STEP;
    static_assert(64 * NW % BN == 0 && 32 % STEP == 0, "whole rows to a pass of the threads");
    const int c = threadIdx.x % BN, col = n0 + c;
    if (col >= p.n) return;
    const bool part = p.splits > 1;
    float *to = part ? p.ws + (int64_t)split * p.m * p.n : p.dw;
    const bool keep = !part && p.acc_dw;
#pragma unroll 4
    for (int u = 0; u < EACH; u++) {
        const int r = threadIdx.x / BN + u * STEP, row = m0 + r;
        const float *s = out + r * LD + c;
        float v = s[0];
#pragma unroll
        for (int w = 1; w < NW; w++) v += s[w * 32 * LD];
        if (row < p.m) {
            float *d = to + (int64_t)row * p.n + col;
            *d = keep ? *d + v : v;
        }
    }
}

// A workgroup computes 32 x (32 NT) of dW with four wavefronts: wavefront q has all of it over the q-th 32 k of every block of
// 128. g and x come through LDS, D blocks and one more in registers, by loads of 16 bytes a lane (a dword a lane into registers,
// as g's layout would have it, keeps the load path busy as long for a quarter of the data: 210 us against 140 of products at
// 16384 x 768 x 2304). The next half's (16 k) splits and conversions stand between a half's MFMAs. At the end the wavefronts'
// sums meet in LDS and are added in order.
template <int NT, int D>
__global__ void __launch_bounds__(256, 2) k_dw8(Dw8 p) {
    OM_LDS_POISON();
    constexpr int BN = 32 * NT, SS = BN * 128, GS = SS + (BN + 63) / 64 * 256;  // a scale load fills 64 dwords
    constexpr int STAGE = GS + 4 * 4096, LD = BN + 1, OUT = 4 * 32 * LD * 4, LDS = D * STAGE > OUT ? D * STAGE : OUT;
    constexpr int LOADS = NT + 4;
    static_assert(BN <= 256, "scales by one load of each wavefront");
    __shared__ __attribute__((aligned(16))) char sh[LDS];
    const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
    const int q = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int split, tm, tn;
    tile_of(p.tiles_m, p.tiles_n, gridDim.x, split, tm, tn);
    const int m0 = 32 * tm, n0 = tn * BN;
    // blocks of 128 rows, and (in the last split) the rows behind the last that is taken as one
    const int b0 = split * p.per, b1 = min(p.full, b0 + p.per), count = max(b1 - b0, 0);
    const bool tail = split == p.splits - 1 && p.full < p.blocks;
    const uint8_t *xq = p.x.q + (int64_t)n0 * p.x.ldq;
    uint32_t off[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) {
        const int r = 8 * (q * NT + i) + (lane >> 3), piece = (lane ^ (r >> 1)) & 7;
        off[i] = (uint32_t)min(r, p.n - 1 - n0) * (uint32_t)p.x.ldq + 16 * piece;
    }
    const uint8_t *xs = p.x.s + (int64_t)min(n0 + (q * 64 + lane) % BN, p.n - 1) * p.x.lds;
    // g: this wavefront's own 32 rows x 32 columns of a stage, eight rows a load, four columns a lane. Columns past the last
    // four start there: column c then stands at c - (m - 4) of its four. (Of fewer than four columns the loads run on into
    // the next rows, which is why the last block is not loaded so then.)
    const int first4 = max(p.m - 4, 0), gc = min(m0 + l32, p.m - 1);
    const uint32_t goff = 4u * ((uint32_t)(lane >> 3) * (uint32_t)p.m + (uint32_t)min(m0 + 4 * (lane & 7), first4));
    const int gat = GS + q * 4096 + 2048 * g + 4 * ((l32 & ~3) + min(gc - min(m0 + (l32 & ~3), first4), 3));
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)sh;
    // Loads past the last block load that one again, into slots that nothing reads.
    auto issue = [&](int st) {
        const uint32_t at = base + (uint32_t)(st % D) * STAGE;
        const int blk = b0 + min(st, count - 1);
#pragma unroll
        for (int i = 0; i < NT; i++) load_to_lds(xq + (int64_t)blk * 128, off[i], at + (q * NT + i) * 1024);
        if (q * 64 < BN) load_to_lds4(xs + (blk & ~3), at + SS + q * 256);
#pragma unroll
        for (int i = 0; i < 4; i++)
            load_to_lds(p.g + ((int64_t)blk * 128 + 32 * q + 8 * i) * p.m, goff, at + GS + q * 4096 + i * 1024);
    };
    float raw[2][16];
    floatx16 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[j][e] = 0.0f;
    const bool sums = p.db && tn == 0;
    double cs = 0.0;
    u32x4 xr[2][NT], wa[2][3], wb[2][NT];
    float sc[2][NT];
    auto read = [&](int h, int st) {
        const char *cur = sh + (st % D) * STAGE;
#pragma unroll
        for (int j = 0; j < NT; j++) {
            sc[h][j] = scale_in(*reinterpret_cast<const uint32_t *>(cur + SS + 4 * (32 * j + l32)), b0 + st);
            xr[h][j] = *reinterpret_cast<const u32x4 *>(cur + piece_at(32 * j + l32, 2 * q + g));
        }
#pragma unroll
        for (int e = 0; e < 16; e++) raw[h][e] = *reinterpret_cast<const float *>(cur + gat + 128 * e);
    };
    // Step v of the operands of half t of the stage in set h: four pairs of g in two steps each, then the blocks of x; four to
    // six instructions each, which go under an MFMA's 32 cycles.
    constexpr int STEPS = 8 + NT;
    float left[2];
    auto prepare = [&](int t, int h, int v) {
        if (v >= 8) {
            wb[t][v - 8] = widen8(xr[h][v - 8][2 * t], xr[h][v - 8][2 * t + 1], sc[h][v - 8]);
        } else if (v % 2 == 0) {
            left[0] = raw[h][8 * t + v];
            left[1] = raw[h][8 * t + v + 1];
            wa[t][0][v / 2] = split_first(left[0], left[1]);
        } else {
            uint32_t m, l;
            split_rest(left[0], left[1], m, l);
            wa[t][1][v / 2] = m;
            wa[t][2][v / 2] = l;
        }
    };
    auto half = [&](int t, int h) {  // half t's products; the next half is t ^ 1, of set h
#pragma unroll
        for (int f = 0; f < 3 * NT; f++) {
            acc[f % NT] = oms::mma(wa[t][2 - f / NT], wb[t][f % NT], acc[f % NT]);
#pragma unroll
            for (int v = f * STEPS / (3 * NT); v < (f + 1) * STEPS / (3 * NT); v++) prepare(t ^ 1, h, v);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto add_sums = [&](int h) {
        if (sums) {  // four chains
            double part[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
            for (int e = 0; e < 16; e++) part[e & 3] += (double)raw[h][e];
            cs += (part[0] + part[1]) + (part[2] + part[3]);
        }
    };
    // Stage st from registers, the next one read meanwhile, its own slot loaded anew.
    auto turn = [&](int h, int st) {
        land<(D - 2) * LOADS>();
        issue(st + D);
        read(h ^ 1, st + 1);
        add_sums(h);
        half(0, h);
        half(1, h ^ 1);
    };
    if (count > 0) {
#pragma unroll
        for (int st = 0; st < D; st++) issue(st);
        land<(D - 1) * LOADS>();
        read(0, 0);
#pragma unroll
        for (int v = 0; v < STEPS; v++) prepare(0, 0, v);
        for (int st = 0; st < count; st += 2) {
            turn(0, st);
            if (st + 1 < count) turn(1, st + 1);
        }
        land<0>();  // the loads past the last stage, too, before LDS is used again
    }
#pragma unroll 1
    for (int blk = tail ? p.full : p.blocks; blk < p.blocks; blk++) {  // the rows behind, straight from memory
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int k = blk * 128 + 32 * q + 16 * g + e;
            const float v = p.g[(int64_t)min(k, p.rows - 1) * p.m + gc];
            raw[0][e] = k < p.rows ? v : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int64_t col = min(n0 + 32 * j + l32, p.n - 1);
            xr[0][j] = *reinterpret_cast<const u32x4 *>(p.x.q + col * p.x.ldq + (int64_t)blk * 128 + 32 * q + 16 * g);
            sc[0][j] = scale_of(p.x.s[col * p.x.lds + blk]);
        }
        add_sums(0);
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int v = 0; v < STEPS; v++) prepare(t, 0, v);
#pragma unroll
            for (int f = 0; f < 3 * NT; f++) acc[f % NT] = oms::mma(wa[t][2 - f / NT], wb[t][f % NT], acc[f % NT]);
        }
    }
    unsigned big = 0;
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int e = 0; e < 16; e++) oms::note(acc[j][e], big);
    if (oms::beyond(big)) {  // this wavefront's k again, two at a time
#pragma unroll 1
        for (int j = 0; j < NT; j++) {
            const int64_t col = min(n0 + 32 * j + l32, p.n - 1);
            const uint8_t *cq = p.x.q + col * p.x.ldq, *cx = p.x.s + col * p.x.lds;
            floatx16 t;
#pragma unroll
            for (int e = 0; e < 16; e++) t[e] = 0.0f;
            auto block = [&](int blk) { t = add_rows8(p, cq, cx, gc, blk * 128 + 32 * q, 32, t); };
#pragma unroll 1
            for (int blk = b0; blk < b1; blk++) block(blk);
            if (tail)
#pragma unroll 1
                for (int blk = p.full; blk < p.blocks; blk++) block(blk);
#pragma unroll
            for (int i = 0; i < NT; i++)
                if (i == j) oms::take_beyond(acc[i], t);
        }
    }
    finish_dw8<NT, 4>(p, split, tn, m0, n0, acc, cs, sh);
}

// The same for few tiles: 32 x 32 of dW, all of it to each of NW wavefronts, over every NW-th piece of 64 rows, alone: the next
// piece of g and x is on its way into a wavefront's own part of LDS while this one is multiplied, and nothing meets before the
// sums do. (300 x 300 x 300: 5.2 us, by the kernel above 6.1; 512 x 512 x 512 5.2 and 6.3; of more columns those above split g for
// more of x: 1000 x 1000 x 1000 21.6, 13.4 by 32 x 128.)
template <int NW>
__global__ void __launch_bounds__(64 * NW) k_dw8_few(Dw8 p) {
    OM_LDS_POISON();
    constexpr int SS = 2048, GS = SS + 256, SLOT = GS + 8192;  // x, its scales (a load fills 64 dwords), g
    constexpr int OUT = NW * 32 * 33 * 4, LDS = NW * SLOT > OUT ? NW * SLOT : OUT, STEPS = 9;
    __shared__ __attribute__((aligned(16))) char sh[LDS];
    const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int split, tm, tn;
    tile_of(p.tiles_m, p.tiles_n, gridDim.x, split, tm, tn);
    const int m0 = 32 * tm, n0 = 32 * tn;
    // pieces of 64 rows, and (in the last split) the rows behind the last that is taken as one
    const int full = p.full, last = (p.rows + 63) / 64, c0 = 2 * split * p.per, c1 = min(full, c0 + 2 * p.per), count = max(c1 - c0, 0);
    const bool tail = split == p.splits - 1 && full < last && wv == count % NW;
    // x: 16 rows of 64 bytes a load, the four 16-byte pieces of a row permuted so that 16 neighbouring rows' equal pieces stand on
    // distinct banks. g as above, eight rows a load.
    const uint8_t *xq = p.x.q + (int64_t)n0 * p.x.ldq, *xs = p.x.s + (int64_t)min(n0 + l32, p.n - 1) * p.x.lds;
    uint32_t off[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = 16 * i + (lane >> 2), piece = (lane ^ (r >> 2)) & 3;
        off[i] = (uint32_t)min(r, p.n - 1 - n0) * (uint32_t)p.x.ldq + 16 * piece;
    }
    const int first4 = max(p.m - 4, 0), gc = min(m0 + l32, p.m - 1);
    const uint32_t goff = 4u * ((uint32_t)(lane >> 3) * (uint32_t)p.m + (uint32_t)min(m0 + 4 * (lane & 7), first4));
    const int gat = GS + 2048 * g + 4 * ((l32 & ~3) + min(gc - min(m0 + (l32 & ~3), first4), 3));
    const char *mine = sh + wv * SLOT;
    const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)sh + (uint32_t)wv * SLOT;
    auto issue = [&](int c) {
#pragma unroll
        for (int i = 0; i < 2; i++) load_to_lds(xq + (int64_t)c * 64, off[i], at + 1024 * i);
        load_to_lds4(xs + ((c >> 1) & ~3), at + SS);
#pragma unroll
        for (int i = 0; i < 8; i++) load_to_lds(p.g + ((int64_t)c * 64 + 8 * i) * p.m, goff, at + GS + i * 1024);
    };
    floatx16 acc[1];
#pragma unroll
    for (int e = 0; e < 16; e++) acc[0][e] = 0.0f;
    const bool sums = p.db && tn == 0;
    double cs = 0.0;
    float raw[2][16], sc, left[2];
    u32x4 xr[2], wa[2][3], wb[2];
    // Step v of the operands of half h (16 rows) of a piece: four pairs of g in two steps each, then x.
    auto prepare = [&](int h, int v) {
        const int c = h >> 1, t = h & 1;
        if (v == 8) {
            wb[t] = widen8(xr[c][2 * t], xr[c][2 * t + 1], sc);
        } else if (v % 2 == 0) {
            left[0] = raw[c][8 * t + v];
            left[1] = raw[c][8 * t + v + 1];
            wa[t][0][v / 2] = split_first(left[0], left[1]);
        } else {
            uint32_t m, l;
            split_rest(left[0], left[1], m, l);
            wa[t][1][v / 2] = m;
            wa[t][2][v / 2] = l;
        }
    };
    auto multiply = [&] {  // the piece in registers
        if (sums) {  // four chains
            double part[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
            for (int e = 0; e < 32; e++) part[e & 3] += (double)raw[e >> 4][e & 15];
            cs += (part[0] + part[1]) + (part[2] + part[3]);
        }
#pragma unroll
        for (int v = 0; v < STEPS; v++) prepare(0, v);
#pragma unroll
        for (int h = 0; h < 4; h++)
#pragma unroll
            for (int f = 0; f < 3; f++) {
                acc[0] = oms::mma(wa[h & 1][2 - f], wb[h & 1], acc[0]);
                if (h < 3)
#pragma unroll
                    for (int v = f * STEPS / 3; v < (f + 1) * STEPS / 3; v++) prepare(h + 1, v);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    if (wv < count) {
        issue(c0 + wv);
        for (int c = c0 + wv; c < c1; c += NW) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            sc = scale_in(*reinterpret_cast<const uint32_t *>(mine + SS + 4 * l32), c >> 1);
#pragma unroll
            for (int q = 0; q < 2; q++) xr[q] = *reinterpret_cast<const u32x4 *>(mine + 64 * l32 + (((2 * q + g) ^ (l32 >> 2)) & 3) * 16);
#pragma unroll
            for (int e = 0; e < 32; e++) raw[e >> 4][e & 15] = *reinterpret_cast<const float *>(mine + gat + 4096 * (e >> 4) + 128 * (e & 15));
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read, so the next may be loaded over it
            if (c + NW < c1) issue(c + NW);
            multiply();
        }
    }
    const int64_t xcol = min(n0 + l32, p.n - 1);
    const uint8_t *cq = p.x.q + xcol * p.x.ldq, *cx = p.x.s + xcol * p.x.lds;
#pragma unroll 1
    for (int c = tail ? full : last; c < last; c++) {  // the rows behind, straight from memory
#pragma unroll
        for (int e = 0; e < 32; e++) {
            const int k = c * 64 + 32 * (e >> 4) + 16 * g + (e & 15);
            const float v = p.g[(int64_t)min(k, p.rows - 1) * p.m + gc];
            raw[e >> 4][e & 15] = k < p.rows ? v : 0.0f;
        }
#pragma unroll
        for (int q = 0; q < 2; q++) xr[q] = *reinterpret_cast<const u32x4 *>(cq + (int64_t)c * 64 + 32 * q + 16 * g);
        sc = scale_of(cx[c >> 1]);
        multiply();
    }
    unsigned big = 0;
#pragma unroll
    for (int e = 0; e < 16; e++) oms::note(acc[0][e], big);
    if (oms::beyond(big)) {  // this wavefront's k again
        floatx16 t;
#pragma unroll
        for (int e = 0; e < 16; e++) t[e] = 0.0f;
#pragma unroll 1
        for (int c = c0 + wv; c < c1; c += NW) t = add_rows8(p, cq, cx, gc, c * 64, 64, t);
        if (tail) t = add_rows8(p, cq, cx, gc, full * 64, (last - full) * 64, t);
        oms::take_beyond(acc[0], t);
    }
    finish_dw8<1, NW>(p, split, tn, m0, n0, acc, cs, sh);
}

// Adds the parts in order: dW's, and by the workgroups from `tiles` on the column sums'.
__global__ void __launch_bounds__(256) k_dw8_join(Dw8 p, unsigned tiles) {
    OM_LDS_POISON();
    if (blockIdx.x >= tiles) {
        const int64_t i = (int64_t)(blockIdx.x - tiles) * 256 + threadIdx.x;
        if (i >= p.m) return;
        const float v = (float)add_parts(p.cs + i, (int64_t)p.m, p.splits);
        p.db[i] = p.acc_db ? p.db[i] + v : v;
        return;
    }
    const int64_t total = (int64_t)p.m * p.n, step = (int64_t)tiles * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const float v = add_parts(p.ws + i, total, p.splits);
        p.dw[i] = p.acc_dw ? p.dw[i] + v : v;
    }
}

// Chooses the kernel for p (its tile in `tile`) and fills in the tiles and splits.
om_status plan_dw8(om_ctx *ctx, Dw8 &p, int &tile) {
    const Choice ch = choose_dw(ctx->num_cus, p.m, p.n, p.blocks, p.x.ldq);
    OM_REQUIRE(ctx, ch.tile >= 0 && p.rows <= INT32_MAX - 255 && p.m < 1 << 26,
               "om_linear_bwd_x8: rows=%d in=%d out=%d is more than a launch takes", p.rows, p.n, p.m);
    const Tile &c = kTilesDw[tile = ch.tile];
    p.tiles_m = (int)(((int64_t)p.m + c.bm - 1) / c.bm);
    p.tiles_n = (int)(((int64_t)p.n + c.bn - 1) / c.bn);
    split_blocks(p.blocks, ch.splits, p.per, p.splits);
    const int piece = tile == 3 ? 64 : 128;
    p.full = p.m >= 4 ? p.rows / piece : p.rows > 3 ? (p.rows - 3) / piece : 0;  // four of fewer columns end up to three rows on
    OM_REQUIRE(ctx, launches((int64_t)p.tiles_m * p.tiles_n * p.splits, tile == 3 ? 512 : 256),
               "om_linear_bwd_x8: in=%d out=%d is more than a launch takes", p.n, p.m);
    return OM_OK;
}

om_status dw8(om_ctx *ctx, Dw8 p, int tile) {
    if (p.splits > 1) {
        const uint64_t sums = ((uint64_t)p.splits * p.m * p.n + 1) / 2 * 2;
        if (om_status s = om::scratch(ctx, 4 * sums + 8ull * p.splits * p.m, &p.ws)) return s;
        p.cs = reinterpret_cast<double *>(p.ws + sums);
    }
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3((unsigned)((int64_t)p.tiles_m * p.tiles_n * p.splits)), dim3(tile == 3 ? 512 : 256), 0, ctx->stream, p);
    };
    switch (tile) {
        case 0: go(k_dw8<4, 2>); break;
        case 1: go(k_dw8<2, 2>); break;
        case 2: go(k_dw8<1, 3>); break;
        default: go(k_dw8_few<8>); break;
    }
    if (p.splits > 1) {
        const unsigned tiles = om::grid1d((int64_t)p.m * p.n, 256, (int64_t)ctx->num_cus * 8), sums = p.db ? (p.m + 255) / 256 : 0;
        hipLaunchKernelGGL(k_dw8_join, dim3(tiles + sums), dim3(256), 0, ctx->stream, p, tiles);
    }
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
    Gemm8 p = {};
    p.a = packed(a8, m, k);
    p.b = packed(b8, n, k);
    p.m = m, p.n = n, p.blocks = (int)blocks8(k);
    p.bias = bias, p.c = c, p.ldc = ldc, p.acc = acc;
    return gemm8(ctx, p);
}

om_status om_linear_bwd_x8(om_ctx *ctx, const float *g, const uint8_t *xt8, const float *w, float *dx, float *dw, float *db,
                           int rows, int in, int out, int acc_dx, int acc_dw, int acc_db) {
    OM_CHECK_CTX(ctx);
    OM_REQUIRE(ctx, rows >= 0 && in > 0 && out > 0, "om_linear_bwd_x8: rows=%d in=%d out=%d", rows, in, out);
    OM_REQUIRE(ctx, aligned16(xt8), "om_linear_bwd_x8: packed tensors start at multiples of 16 bytes");
    OM_REQUIRE(ctx, rows == 0 || (g && (!dx || w) && (!dw || xt8)), "om_linear_bwd_x8: a needed tensor is NULL");
    if (!dx && !dw && !db) return OM_OK;
    if (rows == 0) {  // empty sums
        if (acc_dw) dw = nullptr;
        if (acc_db) db = nullptr;
        if (!dw && !db) return OM_OK;
        if (om_status s = om::use_device(ctx)) return s;
        if (dw)
            if (om_status s = om_fill(ctx, dw, 0.0f, (int64_t)in * out)) return s;
        return db ? om_fill(ctx, db, 0.0f, out) : OM_OK;
    }
    Dw8 p = {};
    int tile = 0;
    if (dw) {
        p.g = g;
        p.x = packed(xt8, in, rows);
        p.rows = rows, p.m = out, p.n = in, p.blocks = (int)blocks8(rows);
        p.dw = dw, p.db = db, p.acc_dw = acc_dw, p.acc_db = acc_db;
        if (om_status s = plan_dw8(ctx, p, tile)) return s;
    }
    if (om_status s = om::use_device(ctx)) return s;
    if (dx)
        if (om_status s = om_linear_bwd(ctx, g, nullptr, w, dx, nullptr, nullptr, rows, in, out, acc_dx, 0, 0)) return s;
    if (!dw) return db ? om_colsum(ctx, g, db, rows, out, acc_db) : OM_OK;
    return dw8(ctx, p, tile);
}

}  // extern "C"
