// The 4-bit latent cache's queries and rows, as the attention and the weight-sum kernels take them.
//
// A cached position is 512 latent values as MXFP4 (256 bytes of E2M1 codes, element 2i in the low
// nibble of byte i, and 16 E8M0 scale bytes, one per 32 values) and 64 rotary values in bf16.
//
// Scores.  The matrix cores take the codes as they are: v_mfma_scale_f32_16x16x128_f8f6f4 reads an
// E2M1 operand with one E8M0 byte per row and 32 columns, which is the cache's own layout: lane
// (row r, quarter q) holds 16 bytes, group 4 q + s in step s of four (the order of a sum's columns is free, and
// in this one the lane's four scale bytes are one dword of the row).  The absorbed query qa (fp32) enters as a sum of E2M3
// terms (6 bits: 1 + 2 + 3) that share the other operand's place, each with an E8M0 byte per 32 columns:
//     qa = t1 + t2 + t3 (+ t4 + t5),   |t1| <= 7.5 s, the next terms' units s / 16, s / 2^9, s / 2^14, s / 2^19
// Each term rounds what is left to nearest; E2M3's step below 4 is at most 1/4, so a term leaves at most
// 1/8 of its unit (the first, up to 7.5: 1/4): 2^-12 s after three terms, 2^-22 s after five, where the group's
// largest magnitude is above 3.75 s.  Three (2^-14 of the largest at worst) are taken where the result is rounded to
// bf16 (2^-8), five where it is fp32 or the weights are summed.  An E2M1 x E2M3 product of 16 x 16 x 128 takes the time of a bf16
// one of 16 x 16 x 32 (19.5 against 18 cycles in a dependent chain), so five terms cost 1.25 bf16 products and need no decoded keys;
// two bf16 terms (2^-17) would cost two products and the decoding.  The rotary columns are bf16 on both sides: bf16 queries are
// one term, fp32 ones two or three.
//
// Values.  The second product's operands are fp16: E2M1 times 2^-23 .. 2^13 (scale bytes 104 .. 140) is exact in it,
// and its 11 bits make one term of a probability enough for a bf16 result (2^-11 each, independent, below the
// result's own 2^-8) and two for fp32 (2^-22), where bf16 would need two and three.  Probabilities are 2^kLift times those of the
// row's reference maximum, so fp16's last bit, 2^-24, is 2^-34 of the largest, and a probability is off by up to half of that whatever
// its size: n positions below 2^-35 beside one that takes all lose n 2^-35 of the context at most (2^-20 over 32,768; the divisor, in
// fp32, counts them).  A block that has come upon a scale
// byte outside that range goes over its positions again with bf16 operands, exact for every byte, and one term more.
//
// Query operands of 16 rows (a row: one head of one query), `terms` latent and `rterms` rotary terms:
//     [term][step]                  64 lanes x 16 bytes, then 64 x 8: the lane's 32 codes, 192 bits
//     [term]                        64 lanes x 4 bytes: the lane's scale byte of every step
//     [rotary term][step of 32]     64 lanes x 16 bytes: 8 bf16 columns
// where lane (q, r) = 16 q + r holds row r, columns 32 (4 q + step) .. +32 (rotary: 32 step + 8 q .. +8).
#pragma once

#include "k3_common.h"

namespace k3 {
namespace {

constexpr int kQ4Lat = 512, kQ4Rope = 64, kQ4Steps = kQ4Lat / 128;
constexpr float kLift = 10.f, kSlack = 5.f;              // log2: probabilities stay under 2^15, fp16's largest is 2^16 - 32
constexpr uint32_t kHalfLow = 104, kHalfHigh = 140;      // scale bytes whose values are exact in fp16
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x32_t __attribute__((ext_vector_type(32)));

__host__ __device__ constexpr int q4_tile_bytes(int terms, int rterms) { return terms * 6400 + rterms * 2048; }
__host__ __device__ constexpr int q4_code_at(int term, int step) { return (term * kQ4Steps + step) * 1536; }
__host__ __device__ constexpr int q4_scale_at(int terms, int term) { return terms * 6144 + term * 256; }
__host__ __device__ constexpr int q4_rope_at(int terms, int rterm, int step) {
    return terms * 6400 + (rterm * 2 + step) * 1024;
}

// Where sequence b's query t (of its first `count`, the last of them at position length - 1) may look: positions
// 0 .. sees - 1.
__device__ __forceinline__ int q4_sees(int t, int count, int length) {
    return t < count ? max(0, length - count + t + 1) : 0;
}

// scores of 16 positions (rows of A: codes and scale bytes) against 16 query rows, 128 columns
template <int STEP>
__device__ __forceinline__ f32x4 q4_mfma(u32x4 k, int kscale, u32x4 qlo, u32x2 qhi, int qscale, f32x4 c) {
    const i32x8 a = {static_cast<int>(k.x), static_cast<int>(k.y), static_cast<int>(k.z), static_cast<int>(k.w), 0, 0, 0, 0};
    const i32x8 b = {static_cast<int>(qlo.x), static_cast<int>(qlo.y), static_cast<int>(qlo.z), static_cast<int>(qlo.w),
                     static_cast<int>(qhi.x), static_cast<int>(qhi.y), 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4 /* E2M1 */, 2 /* E2M3 */, STEP, kscale, STEP, qscale);
}

__device__ __forceinline__ f32x4 q4_mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 q4_mfma_f16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Sum / max over the four 16-lane rows of the wave (lanes l, l^16, l^32, l^48), in every lane.
__device__ __forceinline__ float q4_rows_sum(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float q4_rows_max(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Sum over the 16 lanes of a row, in every lane of it.
__device__ __forceinline__ float q4_row16_sum(float v) {
    auto turned = [&](auto ctrl) __attribute__((always_inline)) {
        return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    v += turned(std::integral_constant<int, 0xb1>{});    // quad_perm [1,0,3,2]
    v += turned(std::integral_constant<int, 0x4e>{});    // quad_perm [2,3,0,1]
    v += turned(std::integral_constant<int, 0x124>{});   // row_ror:4
    v += turned(std::integral_constant<int, 0x128>{});   // row_ror:8
    return v;
}

// bf16 pair (RNE, hardware conversion) of (a, b): low half a
__device__ __forceinline__ uint32_t q4_pack_bf16(float a, float b) {
    const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t q4_pack_f16(float a, float b) {
    const f16x2 v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}
// eight E2M1 codes (of eight positions) times their scales, eight fp16 powers of two: exact
__device__ __forceinline__ u32x4 q4_values_f16(uint32_t codes, u32x4 scales) {
    // (as scalars: a bit cast of a vector's element reads its first one)
    const uint32_t h[4] = {scales.x, scales.y, scales.z, scales.w};
    const f16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 3)};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_bit_cast(uint32_t, v[i] * __builtin_bit_cast(f16x2, h[i]));
    return u32x4{o[0], o[1], o[2], o[3]};
}
__device__ __forceinline__ float q4_lo(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float q4_hi(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }
// the same in bf16
__device__ __forceinline__ u32x4 q4_values_bf16(uint32_t codes, u32x4 scales) {
    const f32x2 c[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3)};
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = hi16x2(__float_as_uint(c[i].x * q4_lo(scales[i])), __float_as_uint(c[i].y * q4_hi(scales[i])));
    return v;
}

}  // namespace
}  // namespace k3
