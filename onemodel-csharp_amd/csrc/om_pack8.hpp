// Tensors held in 8 bits: the layout of a packed tensor and the conversions, shared by the pack and element kernels
// (om_pack8.hip), LayerNorm's (om_norm8.hip) and the products' (om_gemm8.hip).
//
// A packed tensor of [rows, cols] holds e4m3 codes, rows of stride8(cols) bytes (cols rounded up to 128, zeros behind the last
// column), and behind them the scale bytes, rows of scales8(cols) bytes (one to a block of 128 columns, rounded up to four,
// zeros behind the last block). A scale byte s stands for 2^(s - 127); a block takes the least s >= 0 that brings its largest
// finite value to 448, e4m3's largest, or below. A power of two, so the division is exact and a code is the one rounding
// (to nearest, ties to even) of its value; infinities and NaN become NaN codes.
#pragma once

#include <type_traits>

#include "om_internal.hpp"

namespace om8 {

inline int64_t blocks8(int64_t cols) { return (cols + 127) / 128; }
inline int64_t stride8(int64_t cols) { return blocks8(cols) * 128; }
inline int64_t scales8(int64_t cols) { return (blocks8(cols) + 3) / 4 * 4; }
inline uint64_t bytes8(int64_t rows, int64_t cols) { return (uint64_t)rows * (uint64_t)(stride8(cols) + scales8(cols)); }

// A packed tensor's parts.
struct Packed {
    uint8_t *q, *s;
    int64_t ldq, lds;
};
inline Packed packed(const uint8_t *p, int64_t rows, int64_t cols) {
    uint8_t *q = const_cast<uint8_t *>(p);
    return Packed{q, q ? q + rows * stride8(cols) : nullptr, stride8(cols), scales8(cols)};
}
// A launch takes fewer than 2^32 threads.
inline bool launches(int64_t groups, int threads) { return groups <= INT64_C(0xFFFFFFFF) / threads; }
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));  // rows of any alignment: the hardware takes 4 bytes
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// |x| as ordered bits, 0 where x is not finite.
__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
    return u < 0x7F800000u ? u : 0u;
}
// The largest of four. One look for all lanes whether anything is not finite spares the common case the selections.
__device__ __forceinline__ uint32_t top_of(float a, float b, float c, float d) {
    auto bits = [](float x) { return __float_as_uint(x) & 0x7FFFFFFFu; };
    uint32_t u = max(max(bits(a), bits(b)), max(bits(c), bits(d)));
    if (__any(u >= 0x7F800000u)) u = max(max(finite_bits(a), finite_bits(b)), max(finite_bits(c), finite_bits(d)));
    return u;
}
__device__ __forceinline__ uint32_t finite_bits4(floatx4 v) { return top_of(v[0], v[1], v[2], v[3]); }
// The scale byte of a block from its largest value's bits. 448 = 1.75 * 2^8: the exponent less 8, one more where the
// significand is above 1.75 (the sum carries), and 0 where that would be negative.
__device__ __forceinline__ int scale_byte(uint32_t top) { return max((int)((top + 0x1FFFFFu) >> 23) - 8, 0); }
// 2^(127 - s) and 2^(s - 127); s is at most 247 (top at most 2^128 (1 - 2^-24)).
__device__ __forceinline__ float inverse_of(int s) { return __uint_as_float((uint32_t)(254 - s) << 23); }
__device__ __forceinline__ float scale_of(int s) { return __uint_as_float(s ? (uint32_t)s << 23 : 1u << 22); }
// Four codes. The instruction rounds to nearest even and makes NaN codes of infinities and NaN.
__device__ __forceinline__ uint32_t encode4(floatx4 v, float inv) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, w, true);
}
__device__ __forceinline__ floatx4 decode4(uint32_t w, float scale) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return floatx4{a[0] * scale, a[1] * scale, b[0] * scale, b[1] * scale};
}
// The value of another lane of the 16 (CTRL: a DPP control).
template <int CTRL>
__device__ __forceinline__ uint32_t lane_of16(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
}
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;  // quad_perm [1,0,3,2], [2,3,0,1]; rows of 16
constexpr int kRotate8 = 0x128;  // of 16
// Largest of 32 neighbouring lanes, in all of them: five steps on the vector pipe, four inside 16 lanes and one across.
__device__ __forceinline__ uint32_t max32(uint32_t v) {
    v = max(v, lane_of16<kSwap1>(v));
    v = max(v, lane_of16<kSwap2>(v));
    v = max(v, lane_of16<kHalfMirror>(v));
    v = max(v, lane_of16<kMirror>(v));
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);  // the other 16 lanes' in one of the two
    return max(r[0], r[1]);
}
// Sum over the wavefront, in all lanes, by the same pairs (through LDS a step takes ten times as long, and a row's statistics
// are a chain of twelve).
__device__ __forceinline__ float wave_sum8(float v) {
    auto add = [](float x, uint32_t o) { return x + __uint_as_float(o); };
    v = add(v, lane_of16<kSwap1>(__float_as_uint(v)));
    v = add(v, lane_of16<kSwap2>(__float_as_uint(v)));
    v = add(v, lane_of16<kHalfMirror>(__float_as_uint(v)));
    v = add(v, lane_of16<kMirror>(__float_as_uint(v)));
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ double wave_sum8(double v) {
    auto join = [](uint32_t lo, uint32_t hi) { return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo); };
    auto step = [&](auto ctrl) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        v += join(lane_of16<decltype(ctrl)::value>((uint32_t)u), lane_of16<decltype(ctrl)::value>((uint32_t)(u >> 32)));
    };
    step(std::integral_constant<int, kSwap1>());
    step(std::integral_constant<int, kSwap2>());
    step(std::integral_constant<int, kHalfMirror>());
    step(std::integral_constant<int, kMirror>());
    auto across = [&](auto swap) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const auto lo = swap((uint32_t)u), hi = swap((uint32_t)(u >> 32));
        v = join(lo[0], hi[0]) + join(lo[1], hi[1]);
    };
    across([](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
    across([](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
    return v;
}

// Four neighbouring values of a row that ends at `left` more values (any number), zeros behind it.
__device__ __forceinline__ floatx4 load4(const float *p, int64_t left) {
    if (left >= 4) {
        const f4u v = *reinterpret_cast<const f4u *>(p);
        return floatx4{v[0], v[1], v[2], v[3]};
    }
    floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 3; e++)
        if (e < left) v[e] = p[e];
    return v;
}
__device__ __forceinline__ void store4(float *p, int64_t left, floatx4 v) {
    if (left >= 4) {
        *reinterpret_cast<f4u *>(p) = f4u{v[0], v[1], v[2], v[3]};
        return;
    }
#pragma unroll
    for (int e = 0; e < 3; e++)
        if (e < left) p[e] = v[e];
}

}  // namespace om8
