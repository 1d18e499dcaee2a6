// Device pieces of the serving attention kernels (fa_serving.hip): the two
// 16-bit element types on the gfx950 matrix cores, the LDS layout of a 32-key
// K or V tile, and the row arithmetic of an online softmax held per lane.
//
// Layouts (v_mfma_f32_32x32x16): S^T = K . Q^T leaves lane l with query l % 32
// and, in accumulator element r, key 8*(r/4) + 4*(l/32) + r%4 of the tile. O^T =
// V^T . P^T takes the weights of elements 8m .. 8m+7 as its B operand without
// moving them; its A operand, 8 keys of one head dim per lane in the same key
// order, comes from the row-major V tile through ds_read_b64_tr_b16.
#pragma once

#include "fa_common.hpp"

namespace fa::serving {

constexpr int kTileKeys = 32;  // keys per LDS tile

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

// An element type: its 8-wide operand, its matrix product, the sum of a pair
// of weights in 32 bits, and the bias of the weights' exponent. The sums use
// the rounded weights, the same the matrix product uses.
template <typename T>
struct Elem;

template <>
struct Elem<__bf16>
{
    using x8 = bf16x8;
    static constexpr uint32_t kExponent = 0x7f80;  // all ones: infinite or NaN
    // bf16 has fp32's range: the largest weight of a row is 1.
    static constexpr float kBias = 0.0f;
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float add_pair(__bf16 a, __bf16 b, float sum)
    {
        const bf16x2 pair = {a, b};
        const bf16x2 ones = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
        return __builtin_amdgcn_fdot2_f32_bf16(pair, ones, sum, false);
    }
};

template <>
struct Elem<_Float16>
{
    using x8 = f16x8;
    static constexpr uint32_t kExponent = 0x7c00;
    // fp16 ends at 2^-24 (spacing of its subnormals): with the largest weight
    // at 2^8 instead of 1 a key keeps all 11 bits down to 2^-22 of the
    // largest, and is lost only below 2^-33 of it. 2^8 is far from fp16's
    // 65504, and the factor cancels in the division by the row sum.
    static constexpr float kBias = 8.0f;
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float add_pair(_Float16 a, _Float16 b, float sum)
    {
        const f16x2 pair = {a, b};
        const f16x2 ones = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
        return __builtin_amdgcn_fdot2(pair, ones, sum, false);
    }
};

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b)
{
    typedef T t2 __attribute__((ext_vector_type(2)));
    const t2 v = {static_cast<T>(a), static_cast<T>(b)};
    return __builtin_bit_cast(uint32_t, v);
}

// 16-byte-chunk XOR swizzles of a tile's rows: the 16 rows of a K read's phase,
// and the 4 rows x 2 chunks of a V read's 16 lanes, fall on distinct banks.
template <int D>
__device__ __forceinline__ int swz_k(int row)
{
    return D == 128 ? (row & 15) : ((row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int swz_v(int row)
{
    return D == 128 ? (2 * (row & 3) + 8 * (row & 1)) : (2 * (row & 3));
}

// How kWaves waves share the copies of a K or V tile: 1 KiB each, 64 lanes of 16
// bytes.
template <int D, int kWaves>
struct TileCopy
{
    static constexpr int kChunks = D / 8;  // 16-byte chunks per row
    static constexpr int kBytes = 1024;
    static constexpr int kRows = 64 / kChunks;                     // rows one copy covers
    static constexpr int kIssues = kTileKeys / (kRows * kWaves);  // copies per wave and tile
    static_assert(kIssues >= 1 && kIssues * kRows * kWaves == kTileKeys, "a tile splits evenly over the waves");
    static_assert(16 % kRows == 0, "a copy lies in one half of the tile");
};

__device__ __forceinline__ void barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The value of lane l ^ 32 beside the lane's own, in either order
// (v_permlane32_swap of two copies; both registers are outputs, and the s_nop
// gives the wait states a VALU write needs before the swap reads it).
__device__ __forceinline__ void row_halves(float x, float& a, float& b)
{
    uint32_t lo = __builtin_bit_cast(uint32_t, x);
    uint32_t hi = lo;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(lo), "+v"(hi));
#pragma clang diagnostic pop
    a = __builtin_bit_cast(float, lo);
    b = __builtin_bit_cast(float, hi);
}

// Largest raw score of the lane's query over the tile (NaN wins).
__device__ __forceinline__ float row_max_raw(const f32x16& s)
{
    auto max3 = [](float a, float b, float c) {
        return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
    };
    const float a0 = max3(s[0], s[1], s[2]);
    const float a1 = max3(s[3], s[4], s[5]);
    const float a2 = max3(s[6], s[7], s[8]);
    const float a3 = max3(s[9], s[10], s[11]);
    const float a4 = max3(s[12], s[13], s[14]);
    const float mx = __builtin_elementwise_maximum(max3(a0, a1, a2), max3(a3, a4, s[15]));
    float a, b;
    row_halves(mx, a, b);
    return __builtin_elementwise_maximum(a, b);
}

// Scores of keys at or past `limit` become -inf; `limit` is the first dead key
// offset within the tile for the lane's query, minus 4*(lane/32).
__device__ __forceinline__ void mask_tile(f32x16& s, int limit)
{
#pragma unroll
    for (int r = 0; r < 16; ++r)
    {
        const float x = s[r];
        s[r] = (8 * (r >> 2) + (r & 3) < limit) ? x : -INFINITY;
    }
}

// Whether one of an operand's values is infinite or NaN: bits 15 and 31 of the
// result (an exponent of ones carries into them; nothing else does).
template <typename T>
__device__ __forceinline__ uint32_t not_finite(typename Elem<T>::x8 v)
{
    constexpr uint32_t kMask = Elem<T>::kExponent * 0x10001u;
    constexpr uint32_t kOne = (0x8000u - Elem<T>::kExponent) * 0x10001u;
    const i32x4 bits = __builtin_bit_cast(i32x4, v);
    uint32_t found = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) found |= (static_cast<uint32_t>(bits[e]) & kMask) + kOne;
    return found & 0x80008000u;
}

// The exponent base of a row that has seen no key: every finite scaled score is
// at least as large, so the updates need no special case.
constexpr float kEmptyBase = -3.40282347e38f;  // -FLT_MAX

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint32_t uniform(uint32_t x)
{
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
}
__device__ __forceinline__ uint64_t uniform(uint64_t x)
{
    return (static_cast<uint64_t>(uniform(static_cast<uint32_t>(x >> 32))) << 32) | uniform(static_cast<uint32_t>(x));
}

}  // namespace fa::serving
