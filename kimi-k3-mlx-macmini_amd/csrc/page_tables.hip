// Block tables of a batch of requests over a common pool of pages, and the rows that their new tokens go to.
//
// Request b holds lengths[b] positions, ceil(lengths[b] / page) pages, named by the first entries of its row of the table; it
// is to hold target[b].  The free list's entries from `used` on are the pages that nobody holds.
//   returns  a request that shrinks gives back its pages from max(pages of the target, shared[b]) on; all of them, in the batch's
//            order, go in front of the list's free entries, which then begin at base = used - returned
//   takes    a request that grows takes its pages from base on, one request after the other; the first that the list does not
//            hold enough for, and every later one that needs pages, stays as it is (so the ones that get theirs are those whose running
//            sum of needs fits: one prefix sum answers for all of them)
//            Pages that it takes in the places of shared ones are its own: shared[b] comes down to the pages before them
//   slots    new token i of request b -> its row in the pool, page * page_size + position % page_size, or -1
// A page taken from below `used` is one that was just given back: it is looked up in the giver's own row (by a binary search of the
// running sums), so nothing waits for the list to be written.
//
// One block plans: a thread takes neighbouring requests, a prefix sum over the block's 1024 threads orders them.  Few tokens
// (kAlone) are then done by the same block, more by a second launch.  Both are bound by latency: dependent loads of lengths, table
// and list (about 1 us each) and the launch itself.  64 requests of a token each 4.4 us; 48 prompts of up to 8192 tokens 3.4 + 6.8, where a copy
// would write the 1.6 MB of slots in 0.3.
// One launch / two, us a call in a graph: 1 request of 2048 tokens 4.0 / 5.8, 4096 4.8 / 5.8, 8192 6.4 / 5.9; 16 of 256 6.0 / 6.5, of 512 7.1 / 6.9; 64 of one
// 4.8 / 6.5, of 16 5.1 / 6.8.  The rule counts tokens alone: where many requests have few each one launch is the longer (its sixteen waves move
// the requests' pages one after the other): 64 of 64 12.1 / 8.7, 512 of one 10.3 / 7.8, 2048 of one 26.3 / 11.7.
#include <algorithm>

#include "k3_common.h"

namespace k3 {
namespace {

constexpr int64_t kMaxRequests = 65535;
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
static_assert((kMaxRequests + kPlanThreads - 1) / kPlanThreads <= 64, "a bit for each of a thread's requests");
constexpr int kLdsRequests = 2048;      // the plan's records of so many requests fit in LDS
constexpr int64_t kAlone = 4096;        // tokens (requests x new tokens) that the planning block does itself

struct Record {
    int len, to;                        // positions before and after
    int before, give;                   // pages given back by earlier requests, and by this one
    int at;                             // the first of its new pages in the list
};

struct TablesArgs {
    int32_t *table;
    int64_t ld;
    const int32_t *lengths, *target;
    int32_t *shared, *free_list;
    const int32_t *used;
    int32_t *new_lengths, *new_used, *slots;
    Record *records;                    // [B], and behind them base and used
    int B, W, N, shift, tokens;
};

__device__ __forceinline__ int pages_of(int positions, int shift) { return (positions + (1 << shift) - 1) >> shift; }

// page k of the request with record r, whose first `have` are in its row
__device__ __forceinline__ int page_at(const TablesArgs &a, const Record *rec, const int32_t *row, const Record &r, int have, int base, int used, int k) {
    if (k < have) return row[k];
    const int j = r.at + (k - have);
    if (j >= used) return a.free_list[j];
    const int rank = j - base;          // it is the rank-th of those given back
    int b = 0;
    for (int step = 1 << (31 - __clz(max(a.B - 1, 1))); step; step >>= 1)
        if (b + step < a.B && rec[b + step].before <= rank) b += step;
    const Record &g = rec[b];
    return a.table[b * a.ld + (pages_of(g.len, a.shift) - g.give) + (rank - g.before)];
}

// the pages that request b gives back and takes, by `lanes` threads
__device__ __forceinline__ void move_pages(const TablesArgs &a, const Record *rec, int b, int base, int used, int lane, int lanes) {
    const Record r = rec[b];
    int32_t *row = a.table + b * a.ld;
    const int have = pages_of(r.len, a.shift), want = pages_of(r.to, a.shift);
    for (int i = lane; i < r.give; i += lanes)
        if (base + r.before + i < used) a.free_list[base + r.before + i] = row[have - r.give + i];
    for (int k = have + lane; k < want; k += lanes) row[k] = page_at(a, rec, row, r, have, base, used, k);
}

__device__ __forceinline__ int slot_of(const TablesArgs &a, const Record *rec, int b, int i, int base, int used) {
    const Record r = rec[b];
    if (i >= r.to - r.len) return -1;
    const int pos = r.len + i, page = page_at(a, rec, a.table + b * a.ld, r, pages_of(r.len, a.shift), base, used, pos >> a.shift);
    const int64_t slot = (static_cast<int64_t>(page) << a.shift) + (pos & ((1 << a.shift) - 1));
    return page < 0 || slot > INT32_MAX ? -1 : static_cast<int>(slot);
}

// sum over the threads before this one, and over all
struct Sum2 {
    int x, y;
};
__device__ __forceinline__ Sum2 scan(Sum2 own, Sum2 *waves, Sum2 &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sum2 in = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(in.x, o), y = __shfl_up(in.y, o);
        if (lane >= o) in.x += x, in.y += y;
    }
    if (lane == 63) waves[wave] = in;
    __syncthreads();
    Sum2 before{in.x - own.x, in.y - own.y};
    total = Sum2{0, 0};
    for (int w = 0; w < kPlanWaves; ++w) {
        const Sum2 s = waves[w];
        if (w < wave) before.x += s.x, before.y += s.y;
        total.x += s.x, total.y += s.y;
    }
    return before;
}

template <bool ALONE>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(TablesArgs a) {
    __shared__ Record lds[ALONE ? kLdsRequests : 1];
    __shared__ Sum2 waves[kPlanWaves];
    __shared__ int granted;
    Record *const rec = ALONE ? lds : a.records;
    const int tid = threadIdx.x, per = (a.B + kPlanThreads - 1) / kPlanThreads, first = tid * per, last = min(a.B, first + per);
    const int most = a.W << a.shift;
    const int used = min(max(a.used[0], 0), a.N);
    if (tid == 0) granted = 0;
    uint64_t below = 0;                 // of this thread's requests (64 at most): those that grow from below their shared pages
    Sum2 own{0, 0};                     // given back, needed
    for (int b = first; b < last; ++b) {
        const int len = min(max(a.lengths[b], 0), most), target = max(a.target[b], 0);
        const int have = pages_of(len, a.shift);
        const bool fits = target <= most;
        const int want = fits ? pages_of(target, a.shift) : have;
        const int shared = a.shared ? a.shared[b] : 0, keep = max(want, shared);
        if (want > have && shared > have) below |= 1ull << (b - first);
        const int give = want < have ? max(have - keep, 0) : 0;
        rec[b] = Record{len, fits ? target : len, own.x, give, own.y};
        own.x += give, own.y += max(want - have, 0);
    }
    Sum2 total;
    const Sum2 before = scan(own, waves, total);
    const int base = max(used - total.x, 0), left = a.N - base;
    int got = 0;
    for (int b = first; b < last; ++b) {
        Record r = rec[b];
        const int need = max(pages_of(r.to, a.shift) - pages_of(r.len, a.shift), 0), at = before.y + r.at;
        if (need && at + need > left) r.to = r.len;
        else got = max(got, need ? at + need : 0);
        if ((below >> (b - first) & 1) && r.to != r.len) a.shared[b] = pages_of(r.len, a.shift);
        r.before += before.x, r.at = base + at;
        rec[b] = r;
        a.new_lengths[b] = r.to;
    }
    if (got) atomicMax(&granted, got);  // (those that got theirs are the first ones: their last sum is the largest)
    __syncthreads();
    if (tid == 0) {
        a.new_used[0] = base + granted;
        if (!ALONE) a.records[a.B].len = base, a.records[a.B].to = used;
    }
    if (!ALONE) return;
    for (int b = tid >> 6; b < a.B; b += kPlanWaves) move_pages(a, rec, b, base, used, tid & 63, 64);
    __syncthreads();                    // the list is written only where page_at does not read it, the rows where slot_of's k < have is not
    for (int j = tid; j < a.B * a.tokens; j += kPlanThreads) {
        const int b = j / a.tokens;
        a.slots[j] = slot_of(a, rec, b, j - b * a.tokens, base, used);
    }
}

constexpr int kFillThreads = 256, kFillTokens = 4 * kFillThreads;

// grid (ceil(tokens / kFillTokens) or 1, B)
__global__ __launch_bounds__(kFillThreads) void fill_kernel(TablesArgs a) {
    const int b = blockIdx.y, base = a.records[a.B].len, used = a.records[a.B].to;
    if (blockIdx.x == 0) move_pages(a, a.records, b, base, used, threadIdx.x, kFillThreads);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int i = blockIdx.x * kFillTokens + u * kFillThreads + threadIdx.x;
        if (i < a.tokens) a.slots[static_cast<int64_t>(b) * a.tokens + i] = slot_of(a, a.records, b, i, base, used);
    }
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" int64_t k3_page_tables_workspace_size(int64_t B) { return B <= 0 ? 0 : (B + 1) * static_cast<int64_t>(sizeof(Record)); }

extern "C" int k3_page_tables(int32_t *table, int64_t table_row, int64_t blocks, const int32_t *lengths, const int32_t *target,
                              int32_t *shared, int32_t *free_list, int64_t pages, const int32_t *used, int64_t page_size, int64_t B,
                              int64_t tokens, int32_t *new_lengths, int32_t *new_used, int32_t *slots, void *workspace,
                              int64_t workspace_bytes, void *stream) {
    if (B == 0) return K3_OK;
    if (!lengths || !target || !used || !new_lengths || !new_used || !workspace || (blocks > 0 && !table) || (pages > 0 && !free_list) ||
        (tokens > 0 && !slots))
        return set_error(K3_ERR_NULL, "page tables: null pointer");
    if (page_size < 1 || page_size > (1 << 16) || (page_size & (page_size - 1)))
        return set_error(K3_ERR_SHAPE, "page tables: page_size=%lld must be a power of two up to 65536", (long long)page_size);
    if (B < 0 || B > kMaxRequests || blocks < 0 || blocks * page_size >= (1ll << 31) || B * blocks >= (1ll << 31) || pages < 0 || pages >= (1ll << 31) ||
        tokens < 0 || tokens >= (1ll << 31) || B * tokens >= (1ll << 40))
        return set_error(K3_ERR_SHAPE, "page tables: B=%lld, %lld blocks of %lld, %lld pages or %lld tokens out of range", (long long)B,
                         (long long)blocks, (long long)page_size, (long long)pages, (long long)tokens);
    if (B > 1 && table_row < blocks)
        return set_error(K3_ERR_SHAPE, "page tables: the table's rows overlap, %lld apart", (long long)table_row);
    if (workspace_bytes < k3_page_tables_workspace_size(B))
        return set_error(K3_ERR_WORKSPACE, "page tables: workspace %lld < %lld bytes", (long long)workspace_bytes,
                         (long long)k3_page_tables_workspace_size(B));
    if (reinterpret_cast<uintptr_t>(workspace) & 3u) return set_error(K3_ERR_ALIGN, "page tables: workspace must be 4-byte aligned");
    int shift = 0;
    while ((1ll << shift) < page_size) ++shift;
    const TablesArgs a{table, table_row, lengths, target, shared, free_list, used, new_lengths, new_used, slots, static_cast<Record *>(workspace),
                       static_cast<int>(B), static_cast<int>(blocks), static_cast<int>(pages), shift, static_cast<int>(tokens)};
    auto st = static_cast<hipStream_t>(stream);
    if (B <= kLdsRequests && B * tokens <= kAlone) {
        plan_kernel<true><<<1, kPlanThreads, 0, st>>>(a);
        return check_hip(hipGetLastError(), "page tables: launch");
    }
    plan_kernel<false><<<1, kPlanThreads, 0, st>>>(a);
    const int rc = check_hip(hipGetLastError(), "page tables: plan launch");
    if (rc) return rc;
    fill_kernel<<<dim3(static_cast<unsigned>(std::max<int64_t>(1, cdiv(tokens, kFillTokens))), static_cast<unsigned>(B)), kFillThreads, 0, st>>>(a);
    return check_hip(hipGetLastError(), "page tables: fill launch");
}
