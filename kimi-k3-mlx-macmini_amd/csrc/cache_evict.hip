// Eviction from a cache by accumulated attention weight: of a sequence's n positions the first `sink`, the last `recent` and,
// of those between, the ones with the largest weights stay, `keep` in all (all n where n <= keep), and move to the
// front of new buffers in their order.
//
// Two launches.  select (a block per sequence): the weights become keys that order as whole numbers do (NaN below
// all, -0 as 0) and stay in registers (up to 32,768 positions; beyond that every pass reads them again); the key of the
// last one to stay is found 11, 11 and 10 bits at a time from a histogram of the keys that still match, in LDS (four
// copies, by lane, for weights that are alike; sixteen took 22.9 us for 21.3), and no further than a bin that stays whole.  Of the
// positions with exactly that key the lowest stay.  A wave's ballot over 64 neighbours counts them in order, and one scan over those
// counts gives each kept position its place: no atomics on the result.  gather: rows of every buffer, 16 bytes a thread.
// Bound by a block's passes (select: 5.8 us for 1025 positions, 20 for 32,768, of which loading and the first histogram 8, the
// places 6), by HBM or the launch (gather: 53 MB in 10 us).
#include <algorithm>

#include "k3_common.h"

namespace k3 {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048, kCopies = 4, kMaxBuffers = 8;

struct SelectArgs {
    const float *weight;
    int64_t ld;
    const int32_t *lengths;
    int length, cap, keep, sink, recent;
    int32_t *index, *kept;
};

__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;               // NaN
    if (u == 0x80000000u) return 0x80000000u;                     // -0 as 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// inclusive prefix of v over the wave: within rows of 16 lanes, then across them
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);    // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);    // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);    // row_bcast:31 into rows 2 and 3
    return v;
}

// exclusive prefix of v over the block's threads, and the total
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t *sums, uint32_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t s = wave_prefix(v);
    if (lane == 63) sums[wave] = s;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        const uint32_t x = sums[w];
        before += w < wave ? x : 0u;
        total += x;
    }
    __syncthreads();
    return before + s - v;
}

// lanes below this one whose bit is set
__device__ __forceinline__ int below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// VPT keys a thread, position (j * kWaves + wave) * 64 + lane of a chunk of kThreads * VPT
template <int VPT>
__global__ __launch_bounds__(kThreads) void select_kernel(SelectArgs a) {
    __shared__ int hist[kBins * kCopies];
    __shared__ int2 counts[VPT * kWaves];   // of 64 neighbours: keys above the threshold, keys at it
    __shared__ uint32_t sums[kWaves];
    __shared__ int found[3];
    constexpr int kChunk = kThreads * VPT;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
    const int n = a.lengths ? min(max(a.lengths[b], 0), a.cap) : a.length;
    int32_t *index = a.index + static_cast<int64_t>(b) * a.keep;
    const int nk = min(n, a.keep);
    if (tid == 0) a.kept[b] = nk;
    for (int i = nk + tid; i < a.keep; i += kThreads) index[i] = -1;
    if (n <= a.keep) {
        for (int i = tid; i < n; i += kThreads) index[i] = i;
        return;
    }
    // the middle positions sink .. sink + mid - 1, `need` of them stay
    const int mid = n - a.recent - a.sink;
    int need = a.keep - a.sink - a.recent;
    for (int i = tid; i < a.sink; i += kThreads) index[i] = i;
    for (int i = tid; i < a.recent; i += kThreads) index[a.keep - a.recent + i] = n - a.recent + i;
    if (need == 0) return;
    const float *w = a.weight + b * a.ld + a.sink;
    // (Behind the last position keys of 0, the lowest there is: they come after all that are there, so wherever they are counted among
    // the positions at the threshold, `need` are found before them.)
    uint32_t key[VPT];
    auto load = [&](int c0) {
        float f[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int i = c0 + j * kThreads + tid;
            f[j] = i < mid ? w[i] : __builtin_nanf("");
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) key[j] = order_key(f[j]);
    };
    if (mid <= kChunk) load(0);
    uint32_t prefix = 0;     // the bits of the threshold key found so far
    int shift = 32;
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass == 2 ? 10 : 11;
        shift -= bits;
#pragma unroll
        for (int i = 0; i < kBins * kCopies / kThreads; ++i) hist[i * kThreads + tid] = 0;
        __syncthreads();
        for (int c0 = 0; c0 < mid; c0 += kChunk) {
            if (mid > kChunk) load(c0);
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                if (c0 + j * kThreads >= mid) break;
                const uint32_t k = key[j];
                if (pass == 0 || (k >> (shift + bits)) == prefix)
                    atomicAdd(&hist[((k >> shift) & ((1 << bits) - 1)) * kCopies + (tid & (kCopies - 1))], 1);
            }
        }
        __syncthreads();
        // thread t counts bins 2 t' and 2 t' + 1, t' = 1023 - t: from the top down
        const int top = kThreads - 1 - tid;
        int c[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int4 v = *reinterpret_cast<const int4 *>(&hist[(2 * top + x) * kCopies]);
            c[x] = (v.x + v.y) + (v.z + v.w);
        }
        uint32_t total;
        const int above = static_cast<int>(block_prefix(static_cast<uint32_t>(c[0] + c[1]), sums, total));   // keys in higher bins
#pragma unroll
        for (int x = 1, over = above; x >= 0; over += c[x], --x)
            if (over < need && over + c[x] >= need) found[0] = 2 * top + x, found[1] = need - over, found[2] = c[x];
        __syncthreads();
        prefix = (prefix << bits) | static_cast<uint32_t>(found[0]);
        need = found[1];
        const bool whole = found[1] == found[2];
        __syncthreads();
        if (whole) break;
    }
    // keys whose leading bits are above the prefix stay, and the first `need` of those that match (the largest key, +infinity's, leaves
    // room above it)
    const uint32_t low = prefix << shift, high = (prefix + 1) << shift;
    int at = a.sink, same_seen = 0;
    for (int c0 = 0; c0 < mid; c0 += kChunk) {
        if (mid > kChunk) load(c0);
        // lane j: how many of the wave's j-th 64 neighbours are above (high half) and at the threshold (a chunk has 2^15 at most)
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const uint64_t more = __ballot(key[j] >= high), same = __ballot(key[j] >= low) & ~more;
            mine = lane == j ? (static_cast<uint32_t>(__popcll(more)) << 16) + static_cast<uint32_t>(__popcll(same)) : mine;
        }
        if (lane < VPT) counts[lane * kWaves + wave].x = static_cast<int>(mine);
        __syncthreads();
        const uint32_t v = tid < VPT * kWaves ? static_cast<uint32_t>(counts[tid].x) : 0u;
        uint32_t total;
        const uint32_t before = block_prefix(v, sums, total);
        const int same_before = same_seen + static_cast<int>(before & 0xffffu), same_after = same_seen + static_cast<int>(total & 0xffffu);
        // of the positions at the threshold the first `need` stay
        const int stayed = min(same_seen, need);
        if (tid < VPT * kWaves) counts[tid] = make_int2(at + static_cast<int>(before >> 16) + min(same_before, need) - stayed, same_before);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const uint64_t more = __ballot(key[j] >= high), same = __ballot(key[j] >= low) & ~more;
            const int2 o = counts[j * kWaves + wave];
            const uint64_t stays = more | (same & __ballot(o.y + below(same) < need));
            if ((stays >> lane) & 1) index[o.x + below(stays)] = a.sink + c0 + j * kThreads + tid;
        }
        at += static_cast<int>(total >> 16) + min(same_after, need) - stayed, same_seen = same_after;
        __syncthreads();
    }
}

struct GatherArgs {
    const char *src[kMaxBuffers];
    char *dst[kMaxBuffers];
    int64_t src_b[kMaxBuffers], src_r[kMaxBuffers], dst_b[kMaxBuffers], dst_r[kMaxBuffers];   // bytes
    int units[kMaxBuffers], unit[kMaxBuffers];                                                // of a row; bytes of a unit: 16, 4 or 1
    const int32_t *index;
    int buffers, keep, rows, per;   // rows a block takes
};
constexpr int kGatherRows = 64;

template <typename U>
__device__ __forceinline__ void copy_rows(const GatherArgs &a, int x, int b, int r0, int nrows, const int *at) {
    const int units = a.units[x];
    const char *src = a.src[x] + b * a.src_b[x];
    char *dst = a.dst[x] + b * a.dst_b[x] + r0 * a.dst_r[x];
    for (int i = threadIdx.x; i < nrows * units; i += 256) {
        const int r = i / units, u = i % units, s = at[r];
        U v{};
        if (s >= 0) v = *reinterpret_cast<const U *>(src + s * a.src_r[x] + u * static_cast<int>(sizeof(U)));
        *reinterpret_cast<U *>(dst + r * a.dst_r[x] + u * static_cast<int>(sizeof(U))) = v;
    }
}

__global__ __launch_bounds__(256) void gather_kernel(GatherArgs a) {
    __shared__ int at[kGatherRows];
    const int b = blockIdx.y, r0 = blockIdx.x * a.per, nrows = min(a.per, a.rows - r0);
    if (static_cast<int>(threadIdx.x) < nrows) {
        const int r = r0 + threadIdx.x;
        at[threadIdx.x] = r < a.keep ? a.index[static_cast<int64_t>(b) * a.keep + r] : -1;
    }
    __syncthreads();
    for (int x = 0; x < a.buffers; ++x) {
        if (a.unit[x] == 16)
            copy_rows<uint4>(a, x, b, r0, nrows, at);
        else if (a.unit[x] == 4)
            copy_rows<uint32_t>(a, x, b, r0, nrows, at);
        else
            copy_rows<uint8_t>(a, x, b, r0, nrows, at);
    }
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" int k3_cache_evict(const float *weight, int64_t w_batch, const int32_t *lengths, int64_t max_length, int64_t B, int64_t keep,
                              int64_t sink, int64_t recent, int32_t *index, int32_t *kept, int64_t buffers, const void *const *src,
                              const int64_t *src_batch, const int64_t *src_row, void *const *dst, const int64_t *dst_batch,
                              const int64_t *dst_row, const int64_t *row_bytes, int64_t dst_rows, void *stream) {
    if (B == 0) return K3_OK;
    if (!kept || (keep > 0 && !index) || (max_length > 0 && !weight) ||
        (buffers > 0 && (!src || !src_batch || !src_row || !dst || !dst_batch || !dst_row || !row_bytes)))
        return set_error(K3_ERR_NULL, "cache evict: null pointer");
    if (B < 0 || B > 65535 || max_length < 0 || max_length > (1 << 30) || keep < 0 || keep > (1 << 30) || sink < 0 || recent < 0 ||
        sink + recent > keep || w_batch < 0)
        return set_error(K3_ERR_SHAPE, "cache evict: B=%lld, length=%lld, keep=%lld with sink=%lld and recent=%lld", (long long)B,
                         (long long)max_length, (long long)keep, (long long)sink, (long long)recent);
    if (buffers < 0 || buffers > kMaxBuffers || dst_rows < (buffers > 0 ? keep : 0) || dst_rows > (1 << 30))
        return set_error(K3_ERR_SHAPE, "cache evict: %lld buffers (at most %d) of %lld rows for %lld kept", (long long)buffers, kMaxBuffers,
                         (long long)dst_rows, (long long)keep);
    GatherArgs g{};
    for (int64_t x = 0; x < buffers; ++x) {
        if (row_bytes[x] < 0 || row_bytes[x] > (1 << 20) || (row_bytes[x] > 0 && dst_rows > 0 && (!dst[x] || (max_length > 0 && !src[x]))))
            return set_error(K3_ERR_SHAPE, "cache evict: buffer %lld", (long long)x);
        if (src_row[x] < row_bytes[x] || dst_row[x] < row_bytes[x])
            return set_error(K3_ERR_SHAPE, "cache evict: rows of buffer %lld overlap", (long long)x);
        if (!blocks_apart(B, dst_batch[x], dst_rows, dst_row[x], row_bytes[x]))
            return set_error(K3_ERR_SHAPE, "cache evict: sequences of buffer %lld's result overlap", (long long)x);
        const int64_t all = row_bytes[x] | src_batch[x] | src_row[x] | dst_batch[x] | dst_row[x] |
                            static_cast<int64_t>(reinterpret_cast<uintptr_t>(src[x]) | reinterpret_cast<uintptr_t>(dst[x]));
        g.unit[x] = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
        g.units[x] = static_cast<int>(row_bytes[x] / g.unit[x]);
        g.src[x] = static_cast<const char *>(src[x]), g.dst[x] = static_cast<char *>(dst[x]);
        g.src_b[x] = src_batch[x], g.src_r[x] = src_row[x], g.dst_b[x] = dst_batch[x], g.dst_r[x] = dst_row[x];
    }
    auto st = static_cast<hipStream_t>(stream);
    const SelectArgs s{weight, w_batch, lengths, static_cast<int>(max_length), static_cast<int>(max_length), static_cast<int>(keep),
                       static_cast<int>(sink), static_cast<int>(recent), index, kept};
    const dim3 grid(static_cast<unsigned>(B));
    if (max_length <= 4 * kThreads)
        select_kernel<4><<<grid, kThreads, 0, st>>>(s);
    else if (max_length <= 16 * kThreads)
        select_kernel<16><<<grid, kThreads, 0, st>>>(s);
    else
        select_kernel<32><<<grid, kThreads, 0, st>>>(s);
    int rc = check_hip(hipGetLastError(), "cache evict: select launch");
    if (rc || buffers == 0 || dst_rows == 0) return rc;
    g.index = index, g.buffers = static_cast<int>(buffers), g.keep = static_cast<int>(keep), g.rows = static_cast<int>(dst_rows);
    g.per = kGatherRows;      // fewer rows to a block until there are two blocks a CU
    while (g.per > 4 && cdiv(dst_rows, g.per) * B < 512) g.per /= 2;
    gather_kernel<<<dim3(static_cast<unsigned>(cdiv(dst_rows, g.per)), static_cast<unsigned>(B)), 256, 0, st>>>(g);
    return check_hip(hipGetLastError(), "cache evict: gather launch");
}
