// New latents into the 4-bit cache: c [B, T, 512] and r [B, T, 64] (bf16 or fp32) become the MXFP4 codes, scale
// bytes and bf16 rotary rows of positions start[b] .. start[b] + counts[b] - 1.
//
// A group of 32 values x with largest magnitude m gets the scale 2^e, e = floor(log2 m) - 2, one more where
// m > 7 * 2^e: the magnitudes then end at 7, which rounds to 6, the format's largest, and is as far from it as the
// midpoint of 4 and 6 from either; the usual rule (never one more) would clip up to 8.  The byte is e + 127 held to 2..252, the
// range the rest of the library takes; codes round to nearest, ties to even.  A group of zeros gets
// byte 127, one with a NaN or an infinity 255, which makes the position NaN to every query that sees it.
//
// With norm weights the row is RMS-normalised first, in fp32 (the decode step's latent).
//
// A wave takes one position: 64 lanes x 8 values, a group is four lanes, its maximum two lane swaps, and a lane's eight
// codes are one dword, so loads and stores are whole lines.  One token 1.9 us: the launch.  Four
// sequences of 1024 to 8192 tokens, bf16: 21 MB in 9.4 us, 2.3 TB/s, where a copy reaches 5.1: blocks of four positions, many of them past
// their sequence's end, and one row's load in flight a wave.
#include "mla_q4.h"

namespace k3 {
namespace {

struct AppendArgs {
    const void *c, *r;
    int64_t c_b, c_t, r_b, r_t;          // elements
    uint8_t *packed, *scales;
    uint16_t *rot;
    int64_t p_b, p_t, s_b, s_t, o_b, o_t;  // elements of each buffer
    const int32_t *start, *counts;       // [B] or null
    int64_t start0;
    float *weight;                       // [B] rows of w_b floats, or null: the written positions' is zeroed
    int64_t w_b;
    const float *norm;                   // [512] or null
    float eps;
    int64_t T, cap;
};

template <int CTRL>
__device__ __forceinline__ uint32_t umax_dpp(uint32_t v) {
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false)));
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    if constexpr (std::is_same<T, float>::value) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = q4_lo(w[i]), v[2 * i + 1] = q4_hi(w[i]);
    }
}

template <typename CT, typename RT>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    const int lane = threadIdx.x & 63, b = blockIdx.y;
    const int64_t i = (static_cast<int64_t>(blockIdx.z) * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int64_t n = a.counts ? min(static_cast<int64_t>(a.counts[b]), a.T) : a.T;
    const int64_t at = (a.start ? a.start[b] : a.start0) + i;
    if (i >= n || at < 0 || at >= a.cap) return;
    float v[8];
    load8(static_cast<const CT *>(a.c) + b * a.c_b + i * a.c_t + lane * 8, v);
    if (a.norm) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
        const float rs = 1.0f / sqrtf(wave_sum_all(ss) / static_cast<float>(kQ4Lat) + a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * rs * a.norm[lane * 8 + j];
    }
    uint32_t top = 0;   // magnitudes compare as their bits do; infinities and NaNs are the largest
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    top = umax_dpp<0xb1>(top);   // quad_perm [1,0,3,2]
    top = umax_dpp<0x4e>(top);   // quad_perm [2,3,0,1]
    // biased exponent of m, less two, one more above 7/8 of the next power of two (1.75 x 2^floor(log2 m))
    int byte = static_cast<int>(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    byte = top >= 0x7f800000u ? 255 : top == 0u ? 127 : min(max(byte, 2), 252);
    uint32_t code = 0;
    if (byte < 255) {
        const float s = __uint_as_float(static_cast<uint32_t>(byte) << 23);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[0], v[1], s, 0);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[2], v[3], s, 1);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[4], v[5], s, 2);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, v[6], v[7], s, 3);
    }
    *reinterpret_cast<uint32_t *>(a.packed + b * a.p_b + at * a.p_t + lane * 4) = code;
    if (a.weight && lane == 0) a.weight[b * a.w_b + at] = 0.f;
    if ((lane & 3) == 0) a.scales[b * a.s_b + at * a.s_t + (lane >> 2)] = static_cast<uint8_t>(byte);
    const RT *r = static_cast<const RT *>(a.r) + b * a.r_b + i * a.r_t + lane;
    uint16_t o;
    if constexpr (std::is_same<RT, float>::value)
        o = f32_to_bf16(*r);
    else
        o = *r;
    a.rot[b * a.o_b + at * a.o_t + lane] = o;
}

}  // namespace

int mla_q4_append(const void *c, int64_t c_b, int64_t c_t, int c_dtype, const void *r, int64_t r_b, int64_t r_t, int r_dtype,
                  const float *norm, float eps, void *packed, int64_t p_b, int64_t p_t, void *scales, int64_t s_b, int64_t s_t,
                  void *rot, int64_t o_b, int64_t o_t, const int32_t *start, int64_t start0, const int32_t *counts,
                  float *weight, int64_t w_b, int64_t B, int64_t T, int64_t cap, hipStream_t st) {
    const AppendArgs a{c,   r,   c_b, c_t, r_b, r_t,   static_cast<uint8_t *>(packed), static_cast<uint8_t *>(scales),
                       static_cast<uint16_t *>(rot), p_b, p_t, s_b, s_t, o_b, o_t, start, counts, start0, weight, w_b, norm, eps, T, cap};
    // (a row of blocks has at most 2^32 - 1 threads, and a launch of more goes out short without an error)
    const int64_t blocks = cdiv(T, 4), rows = cdiv(blocks, 1 << 23);
    const dim3 grid(static_cast<unsigned>(cdiv(blocks, rows)), static_cast<unsigned>(B), static_cast<unsigned>(rows));
    if (c_dtype == K3_F32)
        r_dtype == K3_F32 ? append_kernel<float, float><<<grid, 256, 0, st>>>(a) : append_kernel<float, uint16_t><<<grid, 256, 0, st>>>(a);
    else
        r_dtype == K3_F32 ? append_kernel<uint16_t, float><<<grid, 256, 0, st>>>(a)
                          : append_kernel<uint16_t, uint16_t><<<grid, 256, 0, st>>>(a);
    return check_hip(hipGetLastError(), "mla q4 append launch");
}

}  // namespace k3

using namespace k3;

extern "C" int k3_mla_q4_append(const void *c, int64_t c_batch, int64_t c_row, int c_dtype, const void *r, int64_t r_batch,
                                int64_t r_row, int r_dtype, void *packed, int64_t p_batch, int64_t p_row, void *scales,
                                int64_t s_batch, int64_t s_row, void *rot, int64_t rot_batch, int64_t rot_row,
                                const int32_t *start, int64_t start0, const int32_t *counts, float *weight, int64_t w_batch,
                                int64_t B, int64_t T, int64_t cap, int64_t kv_lora_rank, int64_t rope_dim, void *stream) {
    if (B == 0 || T == 0) return K3_OK;
    if (!c || !r || !packed || !scales || !rot) return set_error(K3_ERR_NULL, "mla q4 append: null pointer");
    if ((c_dtype != K3_F32 && c_dtype != K3_BF16) || (r_dtype != K3_F32 && r_dtype != K3_BF16))
        return set_error(K3_ERR_DTYPE, "mla q4 append: dtype %d, %d", c_dtype, r_dtype);
    if (kv_lora_rank != kQ4Lat || rope_dim != kQ4Rope)
        return set_error(K3_ERR_SHAPE, "mla q4 append: kv_lora_rank=%lld rope=%lld; the cache takes 512 and 64",
                         (long long)kv_lora_rank, (long long)rope_dim);
    if (B < 0 || B > 65535 || T < 0 || T > (1 << 30) || cap < 0 || cap > (1 << 30) || (!start && (start0 < 0 || start0 + T > cap)))
        return set_error(K3_ERR_SHAPE, "mla q4 append: %lld tokens at %lld do not fit %lld positions (batch %lld)", (long long)T,
                         (long long)start0, (long long)cap, (long long)B);
    const int64_t unit = c_dtype == K3_F32 ? 4 : 8;
    if (c_batch % unit || c_row % unit || c_row < 0 || r_row < 0 || p_row < kQ4Lat / 2 || s_row < kQ4Lat / 32 || rot_row < kQ4Rope ||
        p_row % 4 || p_batch % 4)
        return set_error(K3_ERR_SHAPE, "mla q4 append: a row pitch is too small or not a multiple of 16 bytes");
    if (!blocks_apart(B, p_batch, cap, p_row, kQ4Lat / 2) || !blocks_apart(B, s_batch, cap, s_row, kQ4Lat / 32) ||
        !blocks_apart(B, rot_batch, cap, rot_row, kQ4Rope) || (weight && !blocks_apart(B, w_batch, 1, cap, cap)))
        return set_error(K3_ERR_SHAPE, "mla q4 append: sequences overlap in a buffer that is written");
    if (!aligned16(c) || (reinterpret_cast<uintptr_t>(packed) & 3u))
        return set_error(K3_ERR_ALIGN, "mla q4 append: c must be 16-byte and packed 4-byte aligned");
    return mla_q4_append(c, c_batch, c_row, c_dtype, r, r_batch, r_row, r_dtype, nullptr, 0.f, packed, p_batch, p_row, scales, s_batch,
                         s_row, rot, rot_batch, rot_row, start, start0, counts, weight, w_batch, B, T, cap, static_cast<hipStream_t>(stream));
}
