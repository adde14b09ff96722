// New latents into the pages of a batch: token m's latent row, RMS-normed if asked for, and its rotary row are rounded into row
// slots[m] of the pool (page slots[m] / page_size).
//
//     lat[slot] = round(norm * c * rsqrt(mean(c^2) + eps)),   rot[slot] = round(r)
//
// The sum of squares and the products are fp32, one rounding to nearest at the end (the cache's type).  A wave takes a token: 8 latent
// columns and one rotary column a lane, so a row is read and written as whole 128-byte lines.  A block is four tokens; slots outside the pool
// are left out.  Bound by memory: 8 prompts of up to 4096 fp32 tokens 13.0 us, 48 MB at 3.7 TB/s (a large copy 4.8); 64 tokens 3.2, the launch.
#include <type_traits>

#include "k3_common.h"

namespace k3 {
namespace {

constexpr int kLat = 512, kRot = 64;
constexpr int64_t kMaxRow = 1 << 23;         // blocks of a row of the grid
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct AppendArgs {
    const void *c, *r;
    int64_t c_b, c_t, r_b, r_t;             // elements
    const float *norm;
    float eps;
    const int32_t *slots;
    uint16_t *lat, *rot;
    int64_t lat_page, lat_row, rot_page, rot_row;
    int64_t rows;                           // of the pool
    int64_t M;
    int T, shift;
};

template <typename T>
__device__ __forceinline__ float read(const T *p) {
    if constexpr (std::is_same<T, float>::value)
        return *p;
    else
        return bf16_to_f32(*p);
}

template <bool F16>
__device__ __forceinline__ uint16_t rounded(float v) {
    if constexpr (F16)
        return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
    else
        return f32_to_bf16(v);
}

template <typename CT, typename RT, bool F16>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t m = (blockIdx.y * static_cast<int64_t>(gridDim.x) + blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (m >= a.M) return;
    const int64_t slot = a.slots[m];
    if (slot < 0 || slot >= a.rows) return;
    const int64_t b = m / a.T, t = m - b * a.T;
    const CT *c = static_cast<const CT *>(a.c) + b * a.c_b + t * a.c_t + lane * 8;
    const float rot = read(static_cast<const RT *>(a.r) + b * a.r_b + t * a.r_t + lane);
    float v[8];
    if constexpr (std::is_same<CT, float>::value) {
        const f32x4 x = *reinterpret_cast<const f32x4 *>(c), y = *reinterpret_cast<const f32x4 *>(c + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = x[j], v[4 + j] = y[j];
    } else {
        const u32x4 x = *reinterpret_cast<const u32x4 *>(c);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(x[j] << 16), v[2 * j + 1] = __uint_as_float(x[j] & 0xffff0000u);
    }
    if (a.norm) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
        const float rs = 1.0f / sqrtf(wave_sum_all(ss) / static_cast<float>(kLat) + a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = a.norm[lane * 8 + j] * (v[j] * rs);
    }
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = rounded<F16>(v[2 * j]) | static_cast<uint32_t>(rounded<F16>(v[2 * j + 1])) << 16;
    const int64_t page = slot >> a.shift, off = slot & ((1ll << a.shift) - 1);
    *reinterpret_cast<u32x4 *>(a.lat + page * a.lat_page + off * a.lat_row + lane * 8) = u32x4{o[0], o[1], o[2], o[3]};
    a.rot[page * a.rot_page + off * a.rot_row + lane] = rounded<F16>(rot);
}

template <typename CT, typename RT>
int launch(const AppendArgs &a, bool f16, hipStream_t st) {
    // (a row of blocks has at most 2^32 - 1 threads, and a launch of more goes out short without an error)
    const int64_t blocks = cdiv(a.M, 4), rows = cdiv(blocks, kMaxRow);
    const dim3 grid(static_cast<unsigned>(cdiv(blocks, rows)), static_cast<unsigned>(rows));
    if (f16)
        paged_append_kernel<CT, RT, true><<<grid, 256, 0, st>>>(a);
    else
        paged_append_kernel<CT, RT, false><<<grid, 256, 0, st>>>(a);
    return check_hip(hipGetLastError(), "mla paged append: launch");
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" int k3_mla_paged_append(const void *c, int64_t c_batch, int64_t c_row, int c_dtype, const void *r, int64_t r_batch, int64_t r_row,
                                   int r_dtype, const float *norm, float eps, const int32_t *slots, void *lat, int64_t lat_page,
                                   int64_t lat_row, void *rot, int64_t rot_page, int64_t rot_row, int cache_dtype, int64_t pages,
                                   int64_t page_size, int64_t B, int64_t T, int64_t kv_lora_rank, int64_t rope_dim, void *stream) {
    if (B == 0 || T == 0 || pages == 0) return K3_OK;
    if (!c || !r || !slots || !lat || !rot) return set_error(K3_ERR_NULL, "mla paged append: null pointer");
    if ((c_dtype != K3_F32 && c_dtype != K3_BF16) || (r_dtype != K3_F32 && r_dtype != K3_BF16))
        return set_error(K3_ERR_DTYPE, "mla paged append: dtype %d, %d", c_dtype, r_dtype);
    if (cache_dtype != K3_F16 && cache_dtype != K3_BF16) return set_error(K3_ERR_DTYPE, "mla paged append: cache dtype %d", cache_dtype);
    if (kv_lora_rank != kLat || rope_dim != kRot)
        return set_error(K3_ERR_SHAPE, "mla paged append: kv_lora_rank=%lld rope=%lld; the cache takes 512 and 64", (long long)kv_lora_rank,
                         (long long)rope_dim);
    if (page_size < 1 || page_size > (1 << 16) || (page_size & (page_size - 1)))
        return set_error(K3_ERR_SHAPE, "mla paged append: page_size=%lld must be a power of two up to 65536", (long long)page_size);
    if (B < 0 || T < 0 || T >= (1ll << 31) || B >= (1ll << 31) || B * T > (1ll << 32) || pages < 0 || pages >= (1ll << 31))
        return set_error(K3_ERR_SHAPE, "mla paged append: B=%lld, T=%lld or %lld pages out of range", (long long)B, (long long)T, (long long)pages);
    const int64_t unit = c_dtype == K3_F32 ? 4 : 8;
    if (c_batch % unit || c_row % unit || lat_row % 8 || lat_page % 8)
        return set_error(K3_ERR_SHAPE, "mla paged append: row pitches of c and lat must be whole 16 bytes");
    if (lat_row < kLat || rot_row < kRot || !blocks_apart(pages, lat_page, page_size, lat_row, kLat) ||
        !blocks_apart(pages, rot_page, page_size, rot_row, kRot))
        return set_error(K3_ERR_SHAPE, "mla paged append: rows or pages of the pool overlap");
    if (!aligned16(c) || !aligned16(lat)) return set_error(K3_ERR_ALIGN, "mla paged append: c and lat must be 16-byte aligned");
    int shift = 0;
    while ((1ll << shift) < page_size) ++shift;
    const AppendArgs a{c, r, c_batch, c_row, r_batch, r_row, norm, eps, slots, static_cast<uint16_t *>(lat), static_cast<uint16_t *>(rot), lat_page,
                       lat_row, rot_page, rot_row, pages * page_size, B * T, static_cast<int>(T), shift};
    auto st = static_cast<hipStream_t>(stream);
    const bool f16 = cache_dtype == K3_F16;
    if (c_dtype == K3_F32) return r_dtype == K3_F32 ? launch<float, float>(a, f16, st) : launch<float, uint16_t>(a, f16, st);
    return r_dtype == K3_F32 ? launch<uint16_t, float>(a, f16, st) : launch<uint16_t, uint16_t>(a, f16, st);
}
