// Scored attention on the matrix cores: the operand form that the forward and backward kernels share.
//
// fp32 products as three fp16 products. A block of 64 rows of an operand is scaled by a power of two that brings its
// largest value to 2^11 .. 2^15 and split into x = h + m + r, h and m fp16 (11 + 11 significand bits, |r| below 2^-22 |x|,
// or 2^-36 of the block's largest value where m is subnormal); a product keeps hh, hm, mh. The dropped terms are together
// about 2^-23 of |x||y|, so a sum of products keeps fp32's accuracy, at a third of the fp16 matrix rate (840 TFLOP/s
// where v_mfma_f32_16x16x4_f32 has 157 and the six-term bf16 split of om_split.hpp 419), and a split takes two vector
// operations a value where the bf16 one takes six. What fp16's range does not hold is found beforehand (Stats, RowStats): a
// block with an infinity, a NaN or a largest magnitude outside 2^-40 .. 2^40, or rows or columns whose largest values are more
// than 2^14 apart. A workgroup that would use such a block computes its rows by plain fp32 sums instead (plain_row in
// om_attention_scored_fwd.hip, plain_dq and plain_dkv in om_attention_scored_bwd.hip), and so does one whose scores may pass
// kMostScore: a score is held to 2^-22 of itself, so its weight to as much of the score, and past 2^24 the weights' 2^kLift is
// lost in the rounding of their exponents. Scores are bounded by the longest row's length times the longest key's.
//
// Operands lie in scratch in fragment order: v_mfma_f32_32x32x16_f16 takes, from lane l, eight values of row l % 32 at
// contraction indices of group g = l / 32, and a fragment of 64 lanes x 16 bytes is 1 KB of consecutive memory, so
// staging is a straight copy into LDS and a fragment read is one conflict-free ds_read_b128.
//   rows form (sums over d):    [block of 64 rows][32 rows][16 d][plane][lane][8], d = 16 s + 8 g + e;
//   columns form (sums over rows): [block of 64 rows][16 rows][32 d][plane][lane][8], lane % 32 the d, and element e of group
//     g row 16 s + 8 (e / 4) + 4 g + e % 4: the order in which a 32 x 32 result's registers hold its rows, so that a
//     block of weights goes from one product's result straight into the next one's operand.
#pragma once

#include "om_attention_scored.hpp"

namespace osc {

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 64;  // rows of an operand that share a scale

// What the split found in a block: the largest magnitude (bits; at or above infinity's if the split cannot hold the block),
// the smallest nonzero row maximum (bits), whether its columns keep their bits too, 2^e of its scale, the range of its document
// ids, and the largest sum of a row's squares.
struct Stats {
    uint32_t top, low, columns;
    float scale;
    int32_t doc_lo, doc_hi;
    float norm;
};
// What a step of 32 keys carries along with its operands, staged with them: 64 words.
enum { kKeyDoc = 0, kKeyScaleK = 32, kKeyScaleV, kKeyDocLo, kKeyDocHi, kKeyWords = 64 };
constexpr uint32_t kMostBits = (127u + 40) << 23, kLeastBits = (127u - 40) << 23;  // 2^40, 2^-40
constexpr float kMostScore = 1024.0f;  // in log2 units

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
// The exponent e of a scale 2^-e that brings `top` (bits of a magnitude in range) to 2^11 .. 2^15; steps of 2^4, so that
// neighbouring blocks mostly share it.
__device__ __forceinline__ int scale_exp(uint32_t top) {
    const int e = (int)(top >> 23) - 127 - 14;
    return (e + 3) & ~3;
}
__device__ __forceinline__ bool in_range(uint32_t top) { return top == 0 || (top >= kLeastBits && top <= kMostBits); }
// Whether the smallest nonzero row maximum is within 2^14 of the largest: every row then keeps its 22 bits but the last one
// or two.
__device__ __forceinline__ bool even_rows(uint32_t top, uint32_t low) { return top == 0 || (top >> 23) - (low >> 23) <= 14; }
// Whether scores of rows and keys with these largest sums of squares stay below kMostScore (no, if one is a NaN). A cap does not
// help: what goes into its tanh is held to 2^-36 of the largest.
__device__ __forceinline__ bool scores_fit(const Rule &u, float q_norm, float k_norm) {
    return __builtin_amdgcn_sqrtf(q_norm) * __builtin_amdgcn_sqrtf(k_norm) * __builtin_fabsf(u.cl2) < kMostScore;
}
// Whether a row's distance biases leave a score's last bits below a half: further out its weight may outgrow the 2^kLift.
__device__ __forceinline__ bool bias_fits(const Rule &u, float slope) {
    return __builtin_fabsf(slope) * ((float)u.lq + (float)u.lk) < 0x1p22f;
}

// Two values split into packed fp16 pairs: a packed conversion, the two remainders with the halves taken as they lie
// (v_fma_mix_f32 reads either half of a register as fp16), a packed conversion. Left to itself the compiler converts each
// value a second time to get its half alone: eight instructions where four do.
__device__ __forceinline__ void split2(float a, float b, uint32_t &h, uint32_t &m) {
    const half2 hh = {(_Float16)a, (_Float16)b};
    h = __builtin_bit_cast(uint32_t, hh);
    asm("" : "+v"(h));
    float ra, rb;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(h), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(h), "v"(b));
    const half2 mm = {(_Float16)ra, (_Float16)rb};
    m = __builtin_bit_cast(uint32_t, mm);
}
// Eight values as one lane's part of a fragment.
__device__ __forceinline__ void split8(const float *x, u32x4 &h, u32x4 &m) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t a, b;
        split2(x[2 * i], x[2 * i + 1], a, b);
        h[i] = a;
        m[i] = b;
    }
}
__device__ __forceinline__ floatx16 mma(u32x4 a, u32x4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
// One step of 16 terms: a's rows are the result's registers (8 q + 4 g + r in register 4 q + r), b's its lanes.
__device__ __forceinline__ floatx16 mma3(u32x4 ah, u32x4 am, u32x4 bh, u32x4 bm, floatx16 c) {
    c = mma(am, bh, c);
    c = mma(ah, bm, c);
    return mma(ah, bh, c);
}
// The same sum in the same order with the operands' roles exchanged: mma3_t(a, b) has the bits of mma3(b, a).
__device__ __forceinline__ floatx16 mma3_t(u32x4 ah, u32x4 am, u32x4 bh, u32x4 bm, floatx16 c) {
    c = mma(ah, bm, c);
    c = mma(am, bh, c);
    return mma(ah, bh, c);
}

// The other half-wavefront's value beside this one's: (lanes 0-31's, lanes 32-63's) of the lane's pair.
__device__ __forceinline__ void both_halves(float v, float &lo, float &hi) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    lo = __uint_as_float(p[0]);
    hi = __uint_as_float(p[1]);
}
__device__ __forceinline__ float pair_max(float v) {
    float a, b;
    both_halves(v, a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float pair_sum(float v) {
    float a, b;
    both_halves(v, a, b);
    return a + b;
}

// Largest of a value over the wavefront's 64 lanes, in every lane: four rotations inside a row of 16, then the rows' swaps.
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    auto turn = [&](auto ctrl) {
        v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, true));
    };
    turn(std::integral_constant<int, 0x128>());
    turn(std::integral_constant<int, 0x124>());
    turn(std::integral_constant<int, 0x122>());
    turn(std::integral_constant<int, 0x121>());
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(p[0], p[1]);
    const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(q[0], q[1]);
}
__device__ __forceinline__ uint32_t wave_umin(uint32_t v) { return ~wave_umax(~v); }
// The same for signed values.
__device__ __forceinline__ int wave_imax(int v) { return (int)(wave_umax((uint32_t)v ^ 0x80000000u) ^ 0x80000000u); }
__device__ __forceinline__ int wave_imin(int v) { return ~wave_imax(~v); }

// 16 (or 4) bytes per lane from `src` (this lane's address) to LDS at byte address lds + 16 (4) * lane, without registers. m0
// holds the address for this one instruction only; nothing else in these kernels reads it. Loads land in the order of
// their issue; land<N>() waits until at most this wavefront's last N are in flight and its own LDS reads are done, then
// meets the others.
__device__ __forceinline__ void load_to_lds(const void *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds4(const void *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void land() {
    static_assert(N <= 63, "vmcnt holds at most 63");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Bytes of one operand's two planes for `blocks` blocks of 64 rows.
inline __host__ __device__ int64_t plane_bytes(int dp, int64_t blocks) { return blocks * kBlock * dp * 4; }

// Which of the rule's parts a kernel is compiled for; the others cost it nothing, not a branch in its loop.
enum { kDocs = 1, kCap = 2, kSlopes = 4 };
inline int parts_of(const Rule &u) { return (u.qd ? kDocs : 0) | (u.icap != 0.0f ? kCap : 0) | (u.slopes ? kSlopes : 0); }
template <typename F>
void by_parts(int parts, F f) {
    switch (parts) {
    case 0: return f(std::integral_constant<int, 0>());
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, 3>());
    case 4: return f(std::integral_constant<int, 4>());
    case 5: return f(std::integral_constant<int, 5>());
    case 6: return f(std::integral_constant<int, 6>());
    default: return f(std::integral_constant<int, 7>());
    }
}
template <typename F>
void by_depth(int d, F f) {
    if (d <= 32) f(std::integral_constant<int, 32>());
    else if (d <= 64) f(std::integral_constant<int, 64>());
    else if (d <= 96) f(std::integral_constant<int, 96>());
    else f(std::integral_constant<int, 128>());
}

// What positions i0 .. i1 see of the keys, documents aside, as intervals: all of them see `all0 .. all1`, some may see
// `some0 .. some1`; and all see the keys below pre.
struct Band {
    int all0, all1, some0, some1, pre;
    __host__ __device__ __forceinline__ Band(const Rule &u, int i0, int i1, int prefix) {
        all0 = some0 = 0;
        all1 = some1 = u.lk - 1;
        if (u.causal) {
            all1 = min(all1, i0);
            some1 = min(some1, i1);
        }
        if (u.window) {
            all0 = max(0, i1 - u.window + 1);
            some0 = max(0, i0 - u.window + 1);
            all1 = min(all1, i0 + u.window - 1);
            some1 = min(some1, i1 + u.window - 1);
        }
        pre = min(prefix, u.lk);
    }
    // bitwise throughout: a chain of scalar branches costs more than the arithmetic it saves
    __host__ __device__ __forceinline__ bool all(int j0, int j1) const { return ((j0 >= all0) & (j1 <= all1)) | (j1 < pre); }
    __host__ __device__ __forceinline__ bool some(int j0, int j1) const { return ((j0 <= some1) & (j1 >= some0)) | (j0 < pre); }
};

// The same from the keys' side, in rows of the group: rows all0 .. all1 see all of keys j0 .. j1, rows some0 .. some1 some.
struct RowBand {
    int all0, all1, some0, some1;
    __host__ __device__ __forceinline__ RowBand(const Rule &u, int j0, int j1, int prefix) {
        int a0 = u.off, a1 = INT32_MAX, s0 = u.off, s1 = INT32_MAX;  // positions
        if (j1 >= prefix) {
            if (u.causal) a0 = max(a0, j1);
            if (u.window) {
                a0 = max(a0, j1 - u.window + 1);
                a1 = j0 + u.window - 1;
            }
        }
        if (j0 >= prefix) {
            if (u.causal) s0 = max(s0, j0);
            if (u.window) {
                s0 = max(s0, j0 - u.window + 1);
                s1 = j1 + u.window - 1;
            }
        }
        // positions cut to the queries' and one more on either side: a distance of lk times G may pass 32 bits
        auto row = [&](int pos) { return (min(max(pos, u.off - 1), u.lk) - u.off) * u.G; };
        all0 = row(a0);
        some0 = row(s0);
        all1 = a1 >= u.lk - 1 ? INT32_MAX : row(a1 + 1) - 1;
        some1 = s1 >= u.lk - 1 ? INT32_MAX : row(s1 + 1) - 1;
    }
    __host__ __device__ __forceinline__ bool all(int r0, int r1) const { return (r0 >= all0) & (r1 <= all1); }
    __host__ __device__ __forceinline__ bool some(int r0, int r1) const { return (r1 >= some0) & (r0 <= some1); }
};

// Workgroup id -> item and block. Ids are dealt round-robin over the 8 XCDs, each with its own L2, so the items come
// innermost: an XCD then works on few heads' operands (one in eight of them where their number is a multiple of eight), an
// even share of every block, and blocks are started in their order, which is by falling work under a causal rule, so that
// the short ones fill up behind the long ones. (Whole heads in consecutive ids per XCD gave some XCDs the long rows and
// others the short ones; taking blocks from both ends in turn gave some CUs two long ones: 450 -> 587 us in the backward
// of 4096 causal rows of 12 heads.)
struct Place {
    int item, block;
};
__device__ __forceinline__ Place place_of(int id, int items) { return Place{id % items, id / items}; }

}  // namespace osc
