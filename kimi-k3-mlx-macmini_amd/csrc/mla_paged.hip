// Latent (MLA) attention of a batch over a paged cache, in the absorbed form: one token or several of each of B sequences, the
// positions of a common prefix read and multiplied once for all of them.
//
//     qa[b,t,h]  = q_nope[b,t,h] W_UK[h]                                             [512]
//     s[b,t,h,j] = scale (qa[b,t,h] . lat_j + q_rot[b,t,h] . rot_j)                   j < sees(b, t)
//     p = softmax_j(s);   o[b,t,h] = W_UV[h] (sum_j p[b,t,h,j] lat_j)
//
// A row is one head of one query.  Every row reads the same 1152 bytes of a position, so a set of rows over a range of positions is two
// matrix products, 2176 flops a pair: for a sequence its own T x H rows, for the prefix the rows of all sequences.  Launches:
//   qa       q_nope W_UK on the bf16 matrix cores (fp32 queries as three bf16 terms), rounded into the terms that attend multiplies; a block
//            more makes the list of items
//   attend   an item a block: a tile of rows x a range of positions; the maximum and sum run with the positions
//   uv       the items' records joined (those of the prefix and the sequence's own alike), the context times W_UV, the output gate
//
// Numerics.  fp16 pages multiply as fp16: 11 bits make one term of a query or probability enough for a bf16 result (off by 2^-11 at most,
// independent errors below the result's own 2^-8) and two for fp32 (2^-22); bf16 terms would need two and three.  The absorbed query's 128
// columns of a quarter, and its rotary columns, are scaled by a power of two of their own that puts the largest at 2^13 .. 2^14 (a block
// of the query launch has one of them), and all to the row's largest scale as attend takes them in, so fp16's range is no question of the
// queries' size: what falls below fp16's last bit then is 2^-38 of the row's largest.  Probabilities are 2^kLiftP times those of the row's
// reference, which moves when one would exceed 2^kTop: so fp16 holds them, and its last bit is 2^-31 of the largest.  With one term an item's
// context, over its sum, goes to the join as fp16 (2^-11, and no finer than 2^-25, as the pages' own values), else as fp32.  bf16 pages multiply
// as bf16, exact, against two terms of both for a bf16 result (2^-16), three for fp32 (2^-24).
//
// Measured, us (qa + attend + uv):  1 request over 17 positions, 96 heads 7 + 9 + 6; 32 over up to 8192, 64 heads 9 + 20 + 13; 64 behind a prefix
// of 8192 and up to 1024 of their own 9 + 80 + 9; 120 behind 32,768 14 + 480 + 12 (535 when the card is warm).
#include <algorithm>
#include <type_traits>

#include "mla_q4.h"

namespace k3 {
namespace {

typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4_t *lds_s4;

constexpr int kLat = 512, kRot = 64;
constexpr int kSteps = (kLat + kRot) / 32;      // 18 steps of 32 columns of a score
constexpr int kParts = 5;                       // scales of a row: four quarters of 128 columns, the rotary columns
constexpr int kFrag = 1024;                     // bytes of an operand of 16 rows and 32 columns: 64 lanes x 16
constexpr float kLiftP = 7.f, kTop = 15.f;     // log2 of a probability at the row's reference, and of the largest there may be

// The order of a sequence's rows: by query (row = t H + h: few queries fill the groups of 16) or by head (row = h Tp + t, Tp = T rounded up
// to 16: a group is 16 queries of one head, so a block of the query launch, which takes one head's matrix, writes whole operands).
struct Rows {
    int T, H, Tp;                   // Tp 0: by query
    __host__ __device__ int count() const { return Tp ? H * Tp : T * H; }
    __device__ __forceinline__ int of(int t, int h) const { return Tp ? h * Tp + t : t * H + h; }
    __device__ __forceinline__ int query(int row) const { return Tp ? row % Tp : row / H; }     // may be >= T: no row
};

// ------------------------------------------------------------------ items
// Rows in groups of 16: group g of sequence b holds its rows 16 g .. +16.  A block takes an item: a tile of GT groups over a range of
// positions.  Positions below `split`, all of the prefix, are taken by tiles of any GT neighbours (ranges of one length, every tile's first range,
// then every tile's second ..), those from there on by tiles of one sequence (its ranges one after the other).  Where a sequence's groups fill whole
// tiles both are the same tiles, and the split may lie before the prefix's end: no range is cut there.
struct Item {
    int seq;            // the sequence, or -1: of all
    int tile;           // the first group is GT tile (of the sequence, or of all)
    int begin, end;     // positions
};
struct Head {           // of the list
    int ranges;         // below the split: its items are range r of tile i at r tiles + i
    int low, high;      // items below and above the split
};
struct Lists {
    const int32_t *lengths, *counts;
    Head *head;
    int2 *seq;          // [B]: first item above the split, ranges of each of its tiles
    Item *item;
    int B, T, t0, Tall, cap, prefix;        // prefix: positions
    int tiles, ptiles;  // of a sequence, of all
    int most;           // items there is room for
    int turns;          // items a CU may have
    int aligned;        // a sequence's groups fill whole tiles
};

// what query t (of its sequence's first n = counts[b]) sees
__device__ __forceinline__ int sees_of(const Lists &a, int b, int t) {
    const int len = min(max(a.lengths[b], 0), a.cap), n = a.counts ? min(max(a.counts[b], 0), a.Tall) : a.Tall;
    return q4_sees(t, n, len);
}
// .. the last query of the pass
__device__ __forceinline__ int sees_last(const Lists &a, int b) {
    const int n = a.counts ? min(max(a.counts[b], 0), a.Tall) : a.Tall, t = min(a.t0 + a.T, n) - 1;
    return t < a.t0 ? 0 : sees_of(a, b, t);
}

constexpr int kSearched = 1024;         // sequences up to which the ranges' length is searched for
constexpr int kCandidates = 64;         // lengths: from a share of the most turns of the card's 256 CUs to 1.6 shares of one, evenly by their logarithm
constexpr int kTurns = 8;
constexpr int kRound = 32;              // positions of a round of the attention
constexpr int kStart = 256;             // what an item's start and end cost, in positions
constexpr int kListLds = (kSearched + 4 * 4 * kCandidates + 16) * 4;

// n / d, 1 / d given.  Exact for n < 2^25 (a length and a range's, both up to 2^24) with n / d < 2^21 (ranges are of 32 positions at least,
// items fewer): n, 1 / d and the product are rounded, 2^-24 each, so the estimate is off by less than 1/2 and one step puts it right.
__device__ __forceinline__ int divide(int n, int d, float inverse) {
    int c = static_cast<int>(static_cast<float>(n) * inverse);
    return c + ((c + 1) * d <= n ? 1 : c * d > n ? -1 : 0);
}

// By one block of 256 threads.  All ranges are of one length, the candidate that costs least by this account of an XCD's 32 CUs and its eighth of the
// items: the full ranges in whole turns; the others (m positions at a mean, mx at most) where there is room in these, several to a CU if none but the
// prefix's ranges are full, else in turns of their own; and no less than all there is to do shared out.  (The schedule that the card then runs,
// worked out on the host for 120 draws of batches, prefixes and lengths, takes 0.8 % longer than at the best candidate, 38 % at worst; with
// half a range for mx and m and no account of XCDs 2.8 and 64 %.)  The list takes 4 to 7 us beside the queries' blocks, which take 6 and
// more.  (Equal shares of all positions to every block, items cut where a share ends: slower, 120 requests behind 32,768 positions by a fifth.
// Blocks that are at different places of the prefix miss in L2.)
__device__ __forceinline__ void list_items(const Lists &a, int *lds) {
    int *const own = lds, *const part = lds + kSearched, *const sh = part + 4 * 4 * kCandidates;    // own: what a sequence's last query sees
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int lp = 0;
    float sum = 0.f;
    for (int b = tid; b < a.B; b += 256) {
        const int n = sees_last(a, b);
        if (b < kSearched) own[b] = n;
        lp = max(lp, min(n, a.prefix));
        sum += static_cast<float>(a.aligned ? n : max(n - a.prefix, 0));
    }
    lp = static_cast<int>(wave_max_all(static_cast<float>(lp)));        // (at most 2^24: exact)
    sum = wave_sum_all(sum);
    if (lane == 0) sh[wave] = lp, sh[4 + wave] = __float_as_int(sum);
    __syncthreads();
    lp = max(max(sh[0], sh[1]), max(sh[2], sh[3]));
    sum = (__int_as_float(sh[4]) + __int_as_float(sh[5])) + (__int_as_float(sh[6]) + __int_as_float(sh[7]));
    const float work = static_cast<float>(a.tiles) * sum + (a.aligned ? 0.f : static_cast<float>(a.ptiles) * lp);
    int Ts = 1 << 24;                   // (all of a sequence: what always fits)
    // (a candidate a lane, a quarter of the sequences a wave)
    if (a.B <= kSearched) {
        const float least_want = 0.97f * work / (256.f * a.turns), step = log2f(1.6f / 0.97f * a.turns) / (kCandidates - 1);
        const float want = least_want * exp2f(step * lane);
        const int T1 = (static_cast<int>(fminf(want, 8388608.f)) / kRound + 1) * kRound;
        const float inv = 1.0f / T1;
        const int r0 = a.aligned ? lp / T1 : (lp + T1 - 1) / T1, split = a.aligned ? r0 * T1 : a.prefix;
        int full = 0, rest = 0, mx = 0;         // full ranges, others, the longest of these
        float spent = 0.f;                      // positions of the others
        for (int b = wave; b < a.B; b += 4) {
            const int o = max(own[b] - split, 0), c = divide(o, T1, inv), left = o - c * T1;
            full += c, rest += left > 0, mx = max(mx, left), spent += static_cast<float>(left);
        }
        reinterpret_cast<int4 *>(part)[wave * kCandidates + lane] = make_int4(full, rest, mx, __float_as_int(spent));
        __syncthreads();
        full = rest = mx = 0, spent = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int4 v = reinterpret_cast<const int4 *>(part)[i * kCandidates + lane];
            full += v.x, rest += v.y, mx = max(mx, v.z), spent += __int_as_float(v.w);
        }
        const int whole = full * a.tiles + r0 * a.ptiles, others = rest * a.tiles, items = whole + others;
        const float L = static_cast<float>(T1 + kStart), M = static_cast<float>(mx + kStart), m = spent / max(rest, 1) + kStart;
        const int mine = (whole + 7) >> 3, turns = (mine + 31) >> 5, room = (turns * 32 - mine) * (full ? 1 : max(1, static_cast<int>(L / M)));
        const int more = (max(((others + 7) >> 3) - room, 0) + 31) >> 5;
        float cost = turns * L + (more ? (more - 1) * m + M : 0.f);
        cost = fmaxf(cost, (work + static_cast<float>(items) * kStart) * (1.0f / 256.f));
        if (items > a.most) cost = INFINITY;
        // (cost, lane) least
        float least = cost;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) least = fminf(least, __shfl_xor(least, o));
        if (least < INFINITY) Ts = __builtin_amdgcn_readlane(T1, __builtin_ctzll(__ballot(cost == least)));
    }
    const int ranges = a.ptiles == 0 ? 0 : a.aligned ? lp / Ts : (lp + Ts - 1) / Ts, split = a.aligned ? ranges * Ts : a.prefix;
    const int low = ranges * a.ptiles;
    const float inv_p = 1.0f / max(a.ptiles, 1), inv_t = 1.0f / a.tiles, inv_T = 1.0f / Ts;
    for (int j = tid; j < low; j += 256) {
        const int r = divide(j, a.ptiles, inv_p);
        a.item[j] = Item{-1, j - r * a.ptiles, r * Ts, min((r + 1) * Ts, lp)};
    }
    // the sequences' items, 256 sequences at a time: their first items' places, then their items, a thread each
    int done = low;
    for (int b0 = 0; b0 < a.B; b0 += 256) {
        const int b = b0 + tid, nb = min(a.B - b0, 256);
        const int o = b >= a.B ? 0 : max((b < kSearched ? own[b] : sees_last(a, b)) - split, 0);
        const int c = divide(o + Ts - 1, Ts, inv_T), n = c * a.tiles;
        int at = n;
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) {
            const int x = __shfl_up(at, k);
            if (lane >= k) at += x;
        }
        __syncthreads();                // sh and part are free
        if (lane == 63) sh[wave] = at;
        __syncthreads();
        at -= n;
        for (int i = 0; i < wave; ++i) at += sh[i];
        if (b < a.B) a.seq[b] = make_int2(done + at, c);
        const int total = sh[0] + sh[1] + sh[2] + sh[3];
        part[tid] = at;
        if (b0 < kSearched) {
            __syncthreads();
            for (int j = tid; j < total; j += 256) {
                int q = 0;              // the last sequence that starts at or before j (one of several that start there has items: the last)
#pragma unroll
                for (int step = 128; step; step >>= 1)
                    if (q + step < nb && part[q + step] <= j) q += step;
                const int x = j - part[q], r = divide(x, a.tiles, inv_t), len = own[b0 + q];
                a.item[done + j] = Item{b0 + q, x - r * a.tiles, split + r * Ts, min(split + (r + 1) * Ts, len)};
            }
            __syncthreads();
        } else {
            for (int j = 0; j < n; ++j) {
                const int r = divide(j, a.tiles, inv_t);
                a.item[done + at + j] = Item{b, j - r * a.tiles, split + r * Ts, min(split + (r + 1) * Ts, split + o)};
            }
        }
        done += total;
    }
    if (tid == 0) *a.head = Head{ranges, low, done - low};
}

// ------------------------------------------------------------------ qa
struct QaArgs {
    const void *q_nope, *q_rot;
    int64_t n_b, n_t, n_h, r_b, r_t, r_h;       // strides in elements (batch, query, head)
    const uint16_t *w_uk;                       // [H, nope, 512]
    char *qop;                                  // [group][term][step] operands
    float *scales;                              // [group][kParts][16]
    int H, nope, M, T, t0, G;                   // M = B T queries of the pass; G groups a sequence
    Rows rows;
    Lists lists;
};

constexpr int kWLd = 272;                       // LDS bytes per staged weight row (128 columns + 16 bytes)
constexpr int kFLd = 132;                       // floats per staged result row

__device__ __forceinline__ void three_terms(const float (&v)[8], u32x4 (&f)[3]) {
    uint32_t t[3][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) split3_near<false>(v[i], t[0][i], t[1][i], t[2][i]);
#pragma unroll
    for (int x = 0; x < 3; ++x)
        f[x] = u32x4{hi16x2(t[x][0], t[x][1]), hi16x2(t[x][2], t[x][3]), hi16x2(t[x][4], t[x][5]), hi16x2(t[x][6], t[x][7])};
}

// 8 query values of a lane, columns 8 q4 .. +8 of a step of 32 of query r16.  They are loaded four lanes to a query (neighbouring lanes that read from
// 16 queries take the load path four times as long: 4 x 200 tokens 32 us for 28.5) and change lanes as they are used.
typedef u32x4 __attribute__((aligned(8))) u32x4_8;
template <typename QT>
struct Query {
    static constexpr int kWords = sizeof(QT) * 2;   // of 4 bytes
    u32x4 x[kWords / 4];
    __device__ __forceinline__ void load(const QT *q, bool there) {     // q: columns 8 (lane % 4) of query lane / 4
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) x[i] = there ? reinterpret_cast<const u32x4_8 *>(q)[i] : u32x4{};
    }
    __device__ __forceinline__ void terms(int from, u32x4 (&f)[3]) const {     // from: 4 times the lane that holds this lane's
        uint32_t v[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) v[i] = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(from, static_cast<int>(x[i / 4][i % 4])));
        if constexpr (std::is_same<QT, float>::value) {
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __uint_as_float(v[i]);
            three_terms(w, f);
        } else {
            f[0] = u32x4{v[0], v[1], v[2], v[3]};
        }
    }
};

// the operand terms of 8 neighbouring columns, scaled by s
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    return F16 ? q4_pack_f16(a, b) : q4_pack_bf16(a, b);
}
template <bool F16>
__device__ __forceinline__ void unpack2(uint32_t p, float &a, float &b) {
    if constexpr (F16) {
        const f16x2 v = __builtin_bit_cast(f16x2, p);
        a = static_cast<float>(v[0]), b = static_cast<float>(v[1]);
    } else {
        a = q4_lo(p), b = q4_hi(p);
    }
}
template <bool F16, int NT>
__device__ __forceinline__ void store_terms(float (&v)[8], float s, char *at) {     // at: the first term's operand, the lane's 16 bytes
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= s;
#pragma unroll
    for (int x = 0; x < NT; ++x) {
        u32x4 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = pack2<F16>(v[2 * i], v[2 * i + 1]);
            if (x + 1 < NT) {
                float a, b;
                unpack2<F16>(p[i], a, b);
                v[2 * i] -= a, v[2 * i + 1] -= b;
            }
        }
        *reinterpret_cast<u32x4 *>(at + x * (kSteps * kFrag)) = p;
    }
}
// the power of two that puts a magnitude (its bits) at 2^13 .. 2^14, and its inverse; 1 for infinities and NaNs, and for zeros, whose
// inverse is given as 0: they have no part in the row's scale
template <bool F16>
__device__ __forceinline__ void scale_of(uint32_t top, float &s, float &inverse) {
    if constexpr (!F16) {               // (bf16 terms need none)
        s = inverse = 1.f;
        return;
    }
    const int e = top == 0u || top >= 0x7f800000u ? 13 : min(max(static_cast<int>(top >> 23) - 127, -100), 120);
    s = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
    inverse = top == 0u ? 0.f : __uint_as_float(static_cast<uint32_t>(127 - 13 + e) << 23);
}

// A block: queries 16 MT y .. of head h, latent columns 128 z .. +128, all heads of a (y, z) after one another; and before them all
// one for the list of items.  Blocks b % 8 run on one XCD.  Rows by query: an eighth of the blocks in a row goes to each, so the heads that share an
// operand's 128-byte lines meet in one L2 (64 requests of 64 heads 10.7 -> 9.0 us, 120 16.0 -> 13.9); by head every head is on one XCD, with its matrix.
// MT 1: few queries, a wave to 32 of the columns; MT 4: a wave to 16 of the queries.  A block's 32 KB of weights are read and turned once
// for its queries; 64 heads' take 8.4 MB, 1.8 us at a copy's rate, and the launch 9 us for 32 and 64 queries: the first loads, one barrier,
// the products, another, the stores, one after the other, and no second block on the CU to hide them behind.
template <typename QT, bool F16, int NT, int MT>
__global__ __launch_bounds__(256) void qa_kernel(QaArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float *const fs = reinterpret_cast<float *>(lds);                   // [16 MT][kFLd], after the products
    constexpr int kTerms = std::is_same<QT, float>::value ? 3 : 1, kAhead = 4, kTiles = MT == 1 ? 2 : 8;    // column tiles of a wave
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, q4 = lane >> 4;
    const int blocks = gridDim.x - 1;
    if (blockIdx.x == 0) {
        list_items(a.lists, reinterpret_cast<int *>(lds));
        return;
    }
    const int id = static_cast<int>(blockIdx.x) - 1, b = blocks % 8 || a.rows.Tp ? id : (id & 7) * (blocks >> 3) + (id >> 3);
    const int h = b % a.H, m0 = b / a.H / 4 * 16 * MT, quarter = b / a.H % 4;
    const int steps = (a.nope + 31) >> 5;
    const uint16_t *w = a.w_uk + static_cast<int64_t>(h) * a.nope * kLat + quarter * 128;
    const int qt = MT == 1 ? 0 : wave, col = MT == 1 ? wave * 32 : 0, mine = m0 + 16 * qt + (lane >> 2);    // the wave's queries and columns
    const bool live = mine < a.M;
    const int qb = live ? mine / a.T : 0, qt0 = live ? a.t0 + mine - qb * a.T : 0;
    const QT *q = static_cast<const QT *>(a.q_nope) + qb * a.n_b + qt0 * a.n_t + h * a.n_h + 8 * (lane & 3);
    const int own = a.nope - 8 * (lane & 3), from = 16 * r16 + 4 * q4;
    Query<QT> ahead[kAhead];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) ahead[s].load(q + 32 * s, live && 32 * s < own);
    for (int i0 = 0; i0 < 2 * steps; i0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = (i0 + u) * 256 + tid, n = i >> 4;
            v[u] = n < a.nope ? *reinterpret_cast<const uint4 *>(w + static_cast<int64_t>(n) * kLat + (i & 15) * 8) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = (i0 + u) * 256 + tid, n = i >> 4;
            if (n < 32 * steps) *reinterpret_cast<uint4 *>(lds + n * kWLd + (i & 15) * 16) = v[u];
        }
    }
    f32x4 acc[kTiles];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    auto step = [&](int s, const Query<QT> &raw) __attribute__((always_inline)) {
        const char *wr = lds + (32 * s + 8 * q4 + (r16 >> 2)) * kWLd + (r16 & 3) * 8 + col * 2;
        u32x4 qf[3];
        raw.terms(from, qf);
#pragma unroll
        for (int j0 = 0; j0 < kTiles; j0 += 2) {
            u32x4 wf[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const s4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(wr + (j0 + j) * 32));
                const s4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(wr + (j0 + j) * 32 + 4 * kWLd));
                wf[j] = __builtin_bit_cast(u32x4, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
            }
#pragma unroll
            for (int k = kTerms - 1; k >= 0; --k)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[j0 + j] = q4_mfma_bf16(wf[j], qf[k], acc[j0 + j]);
        }
    };
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
        if (s < steps) step(s, ahead[s]);
    for (int s = kAhead; s < steps; ++s) {
        Query<QT> raw;
        raw.load(q + 32 * s, live && 32 * s < own);
        step(s, raw);
    }
    __syncthreads();   // the weights are read
#pragma unroll
    for (int j = 0; j < kTiles; ++j) *reinterpret_cast<f32x4 *>(fs + (16 * qt + r16) * kFLd + col + j * 16 + 4 * q4) = acc[j];
    __syncthreads();
    // where row (query m, head h)'s operands are
    auto place = [&](int m, int &r) -> int64_t {
        const int b = m / a.T, row = a.rows.of(m - b * a.T, h);
        r = row & 15;
        return static_cast<int64_t>(b) * a.G + (row >> 4);
    };
    if (tid < 64 * MT) {                // four threads to a query, a step of 32 columns each
        const int i = tid >> 2, k = tid & 3, m = m0 + i;
        float v[4][8];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(fs + i * kFLd + k * 32 + 4 * j);
#pragma unroll
            for (int y = 0; y < 4; ++y) v[j >> 1][(j & 1) * 4 + y] = x[y], top = max(top, __float_as_uint(x[y]) & 0x7fffffffu);
        }
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1)));
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2)));
        if (m < a.M) {
            float s, inverse;
            scale_of<F16>(top, s, inverse);
            int r;
            const int64_t g = place(m, r);
            char *const at = a.qop + (g * (NT * kSteps) + quarter * 4 + k) * kFrag + r * 16;
#pragma unroll
            for (int c = 0; c < 4; ++c) store_terms<F16, NT>(v[c], s, at + c * 256);
            if (k == 0) a.scales[(g * kParts + quarter) * 16 + r] = inverse;
        }
    }
    if (quarter != 0) return;
    // rotary columns 8 c .. +8 of a query, eight threads a query
    for (int j = tid; j < 128 * MT; j += 256) {
        const int i = j >> 3, m = m0 + i, c = j & 7;
        float v[8];
        uint32_t top = 0;
        const int b = min(m, a.M - 1) / a.T, t = min(m, a.M - 1) - b * a.T;
        const QT *qr = static_cast<const QT *>(a.q_rot) + b * a.r_b + (a.t0 + t) * a.r_t + h * a.r_h + c * 8;
        if constexpr (std::is_same<QT, float>::value) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(qr), y = *reinterpret_cast<const f32x4 *>(qr + 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = x[k], v[4 + k] = y[k];
        } else {
            const u32x2 x = *reinterpret_cast<const u32x2 *>(qr), y = *reinterpret_cast<const u32x2 *>(qr + 4);
            const uint32_t p[4] = {x.x, x.y, y.x, y.y};
#pragma unroll
            for (int k = 0; k < 4; ++k) v[2 * k] = q4_lo(p[k]), v[2 * k + 1] = q4_hi(p[k]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
#pragma unroll
        for (int k = 1; k < 8; k <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), k)));
        if (m >= a.M) continue;
        float s, inverse;
        scale_of<F16>(top, s, inverse);
        int r;
        const int64_t g = place(m, r);
        store_terms<F16, NT>(v, s, a.qop + (g * (NT * kSteps) + 16 + (c >> 2)) * kFrag + ((c & 3) * 16 + r) * 16);
        if (c == 0) a.scales[(g * kParts + 4) * 16 + r] = inverse;
    }
}

// ------------------------------------------------------------------ attend
struct AttendArgs {
    const char *qop;
    const float *scales;
    const char *lat, *rot;
    int64_t lat_page, rot_page;                 // bytes
    uint32_t lat_row, rot_row;
    const int32_t *table, *prefix;
    int64_t table_row;
    int pages, shift;
    Lists lists;
    void *part;                                 // [item][Mrec][512]: contexts (fp32), or contexts over their sums (fp16: with one term)
    float2 *ml;                                 // [item][Mrec]
    int G, groups, Mrec;                        // groups: of all sequences
    Rows rows;
    float c;                                    // scale * log2(e)
};

constexpr int kLatLd = 1056;                    // LDS bytes of a staged latent row: 1024 + 32
constexpr int kSlotBytes = kRound * (kLatLd + 128);
constexpr int kSlots = 4;
constexpr int kPBytes = 4 * kFrag;              // probabilities of 64 (row, term)s and a round
constexpr int attend_lds() { return kSlots * kSlotBytes + 2 * kPBytes; }

template <bool F16>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return F16 ? q4_mfma_f16(a, b, c) : q4_mfma_bf16(a, b, c);
}

// Infinities and NaNs of a pair to zero.
template <bool F16>
__device__ __forceinline__ uint32_t finite2(uint32_t p) {
    constexpr uint32_t e = F16 ? 0x7c00u : 0x7f80u;
    if ((p & e) == e) p &= 0xffff0000u;
    if ((p & (e << 16)) == (e << 16)) p &= 0xffffu;
    return p;
}

// 16 bytes a lane from offset `off` of a buffer straight into LDS, lane l's at to + 16 l; what lies outside the buffer arrives as zeros.  Not
// tracked by the compiler (nor is m0, which nothing else here uses): a wave waits for its own loads (arrived) and meets the others at a barrier
// before anything is read.  (As an instruction of the compiler's it made every read of LDS wait for all loads in flight.  No register is
// written, so none can be reused under it; its operands are read as it issues.)
__device__ __forceinline__ void load_to_lds(u32x4 rsrc, uint32_t off, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(rsrc), "s"(to) : "memory");
}
// All but the last LEFT loads have arrived, LDS is written and read; then all waves of the block are here.
template <int LEFT, bool LDS = true>
__device__ __forceinline__ void arrived_barrier() {
    if constexpr (LDS)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
    else
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// the largest of three, a NaN aside (fmaxf makes its operands canonical first)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

__device__ __forceinline__ void block_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// An item a block: eight waves, two to a SIMD.  Rounds of 32 positions are staged in LDS as they lie in the pages (latent rows 1024
// bytes of 1056, rotary rows 128 with the 16-byte columns of row r at c ^ (r & 7)).
//   score waves (0 .. 3): S^T[position][row], 16 positions of a round and two operands each (two groups of 16 rows, or a group's two terms), so
//           every row of keys is read from LDS twice; the queries' operands stay in registers.  A lane has four positions of a row, half of what
//           it holds as an operand of the second product.  The two waves of a row keep one reference: a wave that finds a score too far above
//           it says so, and at the start of the next round all waves know, and wait while the round's probabilities are formed again.
//   context waves (4 .. 7): ctx^T[column][row] += rows^T P^T, 128 columns each, from transposed reads of the staged rows.
// What bounds it: at 64 (row, term)s a round's products take 1088 cycles of a SIMD's matrix unit and the round 1960, 55 %: 960 to 1100 TFLOP/s
// (a large library product reaches 1205 in fp16).  No one part does: 120 requests behind 32,768 positions take 489 us, without the context's products 446,
// without the scores' 409, without the loads 461, without the exponentials 466; a round of nothing but its barrier, address and flag reads takes 890 cycles, and
// products keep the card near its power limit (the same call 550 to 650 us when repeated on random data).  Waves' priorities, operands
// read further ahead and other item costs than kStart are within the noise.
// GT = 4 / NT groups of 16 rows: with more terms the probabilities' further terms are rows of their own for the context waves, and the context
// is their sum.  With three, the scores of the queries' third terms are formed by the other two score waves and join the others through LDS.
template <bool F16, int NT>
__global__ __launch_bounds__(512, 1) void attend_kernel(AttendArgs a) {
    constexpr int GT = 4 / NT, VG = GT * NT, kRows = 16 * GT, GR = NT == 1 ? 2 : 1;      // GR: groups of rows of a score wave
    constexpr int kRecRow = kLat * (NT == 1 ? 2 : 4), kRecLd = kRecRow + 16;    // bytes of a record's row
    static_assert(kRows * kRecLd <= kSlots * kSlotBytes && kRows * kRecRow % (8 * 1024) == 0, "the records fit the rounds' room");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int limits[64];
    __shared__ float xm[2][2][64];              // largest exponents [parity][half of the round][row], where a reference has to move
    __shared__ f32x4 xs[NT == 3 ? 2 : 1][64];   // the third terms' scores [half of the round][lane]
    __shared__ float xf[64];                    // factors of the rows whose reference moved
    __shared__ __attribute__((aligned(16))) int need[4][4];     // [round % 4][score wave]: a reference has to move
    char *const pbuf = lds + kSlots * kSlotBytes;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, q4 = lane >> 4;
    // blocks b % 8 share an XCD and its L2: neighbours in the list, which read the same positions, go to one, and an eighth of both kinds to each
    const Head head = *a.lists.head;
    const int low = __builtin_amdgcn_readfirstlane(head.low), high = __builtin_amdgcn_readfirstlane(head.high);
    const int x = static_cast<int>(blockIdx.x & 7), j = static_cast<int>(blockIdx.x >> 3);
    const int l0 = static_cast<int>(static_cast<int64_t>(low) * x >> 3), l1 = static_cast<int>(static_cast<int64_t>(low) * (x + 1) >> 3);
    const int h0 = static_cast<int>(static_cast<int64_t>(high) * x >> 3), h1 = static_cast<int>(static_cast<int64_t>(high) * (x + 1) >> 3);
    if (j >= l1 - l0 + h1 - h0) return;
    const int at = j < l1 - l0 ? l0 + j : low + h0 + j - (l1 - l0);
    const Item it = a.lists.item[at];
    const int seq = __builtin_amdgcn_readfirstlane(it.seq), tile = __builtin_amdgcn_readfirstlane(it.tile);
    const int t_begin = __builtin_amdgcn_readfirstlane(it.begin), end = __builtin_amdgcn_readfirstlane(it.end);
    // the page of a lane's round of 64 (a round lies in one page): positions below `to` are in the table
    const int32_t *const pages = a.table + max(seq, 0) * a.table_row;
    auto page_of = [&](int rd, int to) __attribute__((always_inline)) {
        const int pos = t_begin + rd * kRound;
        return pos < to ? (pos < a.lists.prefix ? a.prefix : pages)[pos >> a.shift] : -1;
    };
    const int first_page = page_of(lane, end);      // (asked for beside the lengths)
    // ---- what the rows see
    if (tid < kRows) {
        const int g = tile * GT + (tid >> 4);
        const int b = seq >= 0 ? seq : g / a.G, row = (g - (seq >= 0 ? 0 : b * a.G)) * 16 + (tid & 15), t = a.rows.query(row);
        const bool there = b < a.lists.B && row < a.rows.count() && t < a.lists.T && (seq < 0 || g < a.G);
        limits[tid] = there ? min(sees_of(a.lists, b, a.lists.t0 + t), end) : 0;
    }
    __syncthreads();
    const int mine = lane < kRows ? limits[lane] : 0;
    const int t_end = static_cast<int>(wave_max_all(static_cast<float>(mine)));
    const int t_all = -static_cast<int>(wave_max_all(-static_cast<float>(mine > t_begin ? mine : 1 << 24)));     // what every row sees (of those that see any)
    float2 *const ml = a.ml + static_cast<int64_t>(at) * a.Mrec;
    if (t_end <= t_begin) {
        if (tid < a.Mrec) ml[tid] = make_float2(-INFINITY, 0.f);
        return;
    }
    const int nr = (t_end - t_begin + kRound - 1) / kRound;

    // ---- staging: round rd into slot rd % kSlots, by all waves: four latent rows each, the context waves eight rotary rows as well.
    // A lane keeps, for one of 64 rounds, where its rows are and how many bytes there are from there on: none for a page outside the pool.
    uint64_t my_lat, my_rot;
    uint32_t my_latb, my_rotb;
    auto place = [&](int rd, int p) __attribute__((always_inline)) {
        const int pos = t_begin + rd * kRound, off = pos & ((1 << a.shift) - 1);
        const bool in = rd < nr && p >= 0 && p < a.pages;
        const uint32_t rows = static_cast<uint32_t>(min(t_end - pos, kRound)) - 1u;
        p = in ? p : 0;
        my_lat = reinterpret_cast<uint64_t>(a.lat) + p * a.lat_page + static_cast<uint64_t>(off) * a.lat_row;
        my_rot = reinterpret_cast<uint64_t>(a.rot) + p * a.rot_page + static_cast<uint64_t>(off) * a.rot_row;
        my_latb = in ? rows * a.lat_row + 1024u : 0u;
        my_rotb = in ? rows * a.rot_row + 128u : 0u;
    };
    auto look_up = [&](int first) __attribute__((always_inline)) { place(first + lane, page_of(first + lane, t_end)); };
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)lds));
    const int rrow = 8 * (wave & 3) + (lane >> 3);
    const uint32_t lat_off = static_cast<uint32_t>(4 * wave) * a.lat_row + lane * 16u;
    const uint32_t rot_off = static_cast<uint32_t>(rrow) * a.rot_row + ((lane & 7) ^ (rrow & 7)) * 16u;
    auto rsrc_of = [&](uint64_t at, uint32_t bytes, int rd) __attribute__((always_inline)) {
        const int l = rd & 63;
        return u32x4{static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at), l)),
                     static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at >> 32), l)) & 0xffffu,
                     static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(bytes), l)), 0x00020000u};
    };
    // prepare(rd), then a row at a time: a load takes 16 cycles of the CU's path to LDS, so they are spread over a round
    u32x4 r_lat, r_rot;
    uint32_t to_slot;
    auto prepare = [&](int rd, bool context) __attribute__((always_inline)) {
        to_slot = lds0 + (rd & (kSlots - 1)) * kSlotBytes;
        r_lat = rsrc_of(my_lat, my_latb, rd);
        if (context) r_rot = rsrc_of(my_rot, my_rotb, rd);
    };
    auto stage_row = [&](int i) __attribute__((always_inline)) { load_to_lds(r_lat, lat_off + i * a.lat_row, to_slot + (4 * wave + i) * kLatLd); };
    auto stage_rot = [&]() __attribute__((always_inline)) { load_to_lds(r_rot, rot_off, to_slot + kRound * kLatLd + (wave & 3) * 1024); };
    auto stage = [&](int rd, bool context) __attribute__((always_inline)) {
        prepare(rd, context);
#pragma unroll
        for (int i = 0; i < 4; ++i) stage_row(i);
        if (context) stage_rot();
    };
    bool in0, in1;              // whether the pages of this round and the next are in the pool; r_lat says it of the one after that
    place(lane, first_page);

    // Iteration t = -1 .. nr - 1: round t + 3 is sent for, the score waves take round t + 1, the context waves round t; then round t + 2 is
    // waited for.  A slot is written again three iterations after its scores, two after its context.
    // The score waves leave in need[round % 4] whether a row's reference has to move for it: then its probabilities are formed again, by all
    // score waves, before they are used, and the block waits for it.  (One reading lane's word for the usual answer, that none has.)
    if (tid < 16) need[tid >> 2][tid & 3] = 0;
    auto needed = [&](int rd) __attribute__((always_inline)) { return *reinterpret_cast<const u32x4 *>(need[rd & 3]); };
    auto any_of = [&](u32x4 n) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(n.x | n.y | n.z | n.w) != 0; };

    if (wave < 4) {
        // ================= score waves
        constexpr int kAhead = 6;
        const int rg = wave & 1, pt = wave >> 1;            // operands 2 rg and 2 rg + 1; positions 16 pt .. +16 of a round
        const bool main = NT < 3 || rg == 0;                // (three terms: the third's waves give their scores to the others')
        stage(0, false);
        in0 = r_lat.z != 0;
        stage(1, false);
        in1 = r_lat.z != 0;
        u32x4 q[2][kSteps];                                 // [operand]: two groups of rows, or a group's two terms
        float fac[GR];
        int limit[GR];
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            const int grp = NT == 3 ? 0 : (2 * rg + o) / NT, term = NT == 3 ? 2 * rg + o : NT == 2 ? o : 0;
            const int gidx = min((seq >= 0 ? seq * a.G : 0) + tile * GT + grp, a.groups - 1);
            const char *qp = a.qop + (static_cast<int64_t>(gidx) * NT + min(term, NT - 1)) * (kSteps * kFrag) + lane * 16;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) q[o][k] = *reinterpret_cast<const u32x4 *>(qp + k * kFrag);
            if (NT == 3 && term == 3) {
#pragma unroll
                for (int k = 0; k < kSteps; ++k) q[o][k] = u32x4{0, 0, 0, 0};
            }
            float top = 1.f;
            if constexpr (F16) {        // to the row's one scale: exact, but for what comes below fp16's last bit
                float part[kParts];
                top = 0.f;
#pragma unroll
                for (int j = 0; j < kParts; ++j) {
                    part[j] = a.scales[(static_cast<int64_t>(gidx) * kParts + j) * 16 + r16];
                    top = fmaxf(top, part[j]);
                }
                const float inv = top > 0.f ? 1.0f / top : 0.f;     // (a power of two)
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    const _Float16 d = static_cast<_Float16>(part[k / 4] * inv);
                    const f16x2 d2 = {d, d};
                    const uint32_t w[4] = {q[o][k].x, q[o][k].y, q[o][k].z, q[o][k].w};
                    uint32_t v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w[i]) * d2);
                    q[o][k] = u32x4{v[0], v[1], v[2], v[3]};
                }
            }
            fac[o % GR] = top * a.c;
            limit[o % GR] = limits[grp * 16 + r16];
        }
        // (all of it is here before the loop: a wait for it there would wait for the rounds in flight)
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int k = 0; k < kSteps; ++k) asm volatile("" : "+v"(q[o][k]));
#pragma unroll
        for (int g = 0; g < GR; ++g) asm volatile("" : "+v"(fac[g]));
        // exponents of the last round's probabilities, 2^e with e = score - from (a row's reference less kLiftP); top: above it the reference
        // moves (kTop, or anything for a row that has none yet)
        float e[GR][4], from[GR], top[GR], l_run[GR], l_new[GR];
#pragma unroll
        for (int g = 0; g < GR; ++g) from[g] = 0.f, top[g] = -INFINITY, l_run[g] = l_new[g] = 0.f;
        const char *const krow = lds + (pt * 16 + r16) * kLatLd + q4 * 16;
        const char *const rrow0 = lds + kRound * kLatLd + (pt * 16 + r16) * 128;
        auto frag = [&](int slot, int k) __attribute__((always_inline)) {
            return *reinterpret_cast<const u32x4 *>(k < 16 ? krow + slot + k * 64 : rrow0 + slot + ((((k - 16) * 4 + q4) ^ (r16 & 7)) * 16));
        };
        // probabilities of a round, as operands of the second product
        auto publish = [&](int rd) __attribute__((always_inline)) {
            char *const to = pbuf + (rd & 1) * kPBytes + 2 * rg * kFrag + lane * 16 + pt * 8;
#pragma unroll
            for (int g = 0; g < GR; ++g) {
                float pr[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) pr[i] = __builtin_amdgcn_exp2f(e[g][i]);
                if constexpr (!F16 || NT == 2) l_new[g] = (pr[0] + pr[1]) + (pr[2] + pr[3]);
#pragma unroll
                for (int y = 0; y < NT; ++y) {
                    u32x2 o;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        o[i] = pack2<F16>(pr[2 * i], pr[2 * i + 1]);
                        if (y + 1 < NT) {
                            float u, w;
                            unpack2<F16>(o[i], u, w);
                            pr[2 * i] -= u, pr[2 * i + 1] -= w;
                        }
                    }
                    *reinterpret_cast<u32x2 *>(to + (NT == 1 ? g : y) * kFrag) = o;
                    if constexpr (F16 && NT == 1) {     // (the sum of what is multiplied: the roundings of a probability that takes all cancel)
                        const f16x2 one = {1, 1};
                        l_new[g] = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, static_cast<uint32_t>(o.x)), one,
                                                          __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, static_cast<uint32_t>(o.y)), one, 0.f, false), false);
                    }
                }
            }
        };
        arrived_barrier<4>();
        for (int rd = 0; rd <= nr; ++rd) {
            if (((rd + 2) & 63) == 0) look_up(rd + 2);
            const int slot = (rd & (kSlots - 1)) * kSlotBytes;
            u32x4 ring[kAhead];                             // operands on their way (of a round too many: of an old slot)
#pragma unroll
            for (int k = 0; k < kAhead; ++k) ring[k] = frag(slot, k);
            const u32x4 raw = needed(rd - 1);
            f32x4 acc[2];                                   // [operand]
            bool again = false;
            if (rd == nr) {
                again = any_of(raw);
            } else {
                __builtin_amdgcn_s_setprio(2);
                acc[0] = acc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    const u32x4 x = ring[k % kAhead];
#pragma unroll
                    for (int o = 0; o < 2; ++o) acc[o] = mfma<F16>(x, q[o][k], acc[o]);
                    if (k + kAhead < kSteps) ring[k % kAhead] = frag(slot, k + kAhead);
                    __builtin_amdgcn_sched_barrier(0);
                    if (k == 0) prepare(rd + 2, false);
                    if (k == 2) again = rd > 0 && any_of(raw);
                    if (k >= 4 && k % 3 == 1 && k < 16) stage_row(k / 3 - 1);
                }
            }
            {
                if (again && !main) {
                    block_barrier();
                } else if (again) {
                    const u32x4 n = needed(rd - 1);
                    const bool me = (pt ? (rg ? n.w : n.z) : (rg ? n.y : n.x)) != 0, other = (pt ? (rg ? n.y : n.x) : (rg ? n.w : n.z)) != 0;
#pragma unroll
                    for (int g = 0; g < GR; ++g) {
                        const int row = (GR * rg + g) * 16 + r16;
                        float t = other ? xm[(rd - 1) & 1][1 - pt][row] : -INFINITY, f = 1.f;
                        if (me) t = fmaxf(t, xm[(rd - 1) & 1][pt][row]);
                        if (t > top[g]) {
                            const float d = t - kLiftP;
                            f = top[g] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-d);
                            from[g] += d, top[g] = kTop;
#pragma unroll
                            for (int i = 0; i < 4; ++i) e[g][i] -= d;
                        }
                        l_run[g] *= f;
                        if (pt == 0 && q4 == 0) xf[row] = f;
                    }
                    publish(rd - 1);
                    block_barrier();
                }
#pragma unroll
                for (int g = 0; g < GR; ++g) l_run[g] += l_new[g];
            }
            if (rd < nr) {
                if constexpr (NT == 3) {
                    if (!main) xs[pt][lane] = acc[0];
                    block_barrier();
                    if (main) acc[1] += xs[pt][lane];
                }
                if (main) {
                    const int base = t_begin + rd * kRound + 16 * pt + 4 * q4;
                    const bool mixed = !in0 || t_begin + (rd + 1) * kRound > t_all;
#pragma unroll
                    for (int g = 0; g < GR; ++g)
#pragma unroll
                        for (int i = 0; i < 4; ++i) e[g][i] = fmaf(NT > 1 ? acc[0][i] + acc[1][i] : acc[g][i], fac[g], -from[g]);
                    if (mixed) {
#pragma unroll
                        for (int g = 0; g < GR; ++g)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                // (where values are cleaned for the sake of rows that do not see them, an infinite score has to make its row NaN by itself)
                                if (!(fabsf(e[g][i]) < INFINITY)) e[g][i] = NAN;
                                e[g][i] = in0 && base + i < limit[g] ? e[g][i] : -INFINITY;
                            }
                    }
                    bool above = false;
#pragma unroll
                    for (int g = 0; g < GR; ++g) above |= max3(max3(e[g][0], e[g][1], e[g][2]), e[g][3], top[g]) > top[g];
                    if (__any(above)) {
                        if (lane == 0) need[rd & 3][wave] = 1;
#pragma unroll
                        for (int g = 0; g < GR; ++g) {
                            const float t = q4_rows_max(fmaxf(fmaxf(e[g][0], e[g][1]), fmaxf(e[g][2], e[g][3])));
                            if (q4 == 0) xm[rd & 1][pt][(GR * rg + g) * 16 + r16] = t;
                        }
                    }
                    publish(rd);
                }
                __builtin_amdgcn_s_setprio(0);
            }
            in0 = in1, in1 = r_lat.z != 0;
            arrived_barrier<4>();
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int g = 0; g < GR; ++g) {
            const float l = q4_rows_sum(l_run[g]);
            if (main && q4 == 0) (pt ? xf : xm[0][0])[(GR * rg + g) * 16 + r16] = l;
            l_run[g] = l;
        }
        block_barrier();
        // (a row that sees nothing of the range was not masked where all others see all: its record counts for nothing)
#pragma unroll
        for (int g = 0; g < GR; ++g) {
            const int row = (GR * rg + g) * 16 + r16;
            if (main && pt == 0 && q4 == 0 && row < a.Mrec) {
                // (nor does one whose positions are all on pages outside the pool: it has no reference, and 0 might be far above the others')
                const float l = l_run[g] + xf[row];
                ml[row] = limit[g] > t_begin && l != 0.f ? make_float2(from[g], l) : make_float2(-INFINITY, 0.f);
            }
        }
    } else {
        // ================= context waves
        constexpr int kAhead = 5;
        const int cw = wave - 4;
        f32x4 acc[8][VG];                       // [16 columns][16 (row, term)s]
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int g = 0; g < VG; ++g) acc[n][g] = f32x4{0.f, 0.f, 0.f, 0.f};
        stage(0, true);
        in0 = r_lat.z != 0;
        stage(1, true);
        in1 = r_lat.z != 0;
        arrived_barrier<5>();
        s4_t ring[kAhead][2];                   // operands on their way: 16 columns of the positions 0 .. 16 and 16 .. 32
        const char *const src0 = lds + (4 * q4 + (r16 >> 2)) * kLatLd + cw * 256 + (r16 & 3) * 8;
        auto columns = [&](int rd, int n, s4_t (&x)[2]) __attribute__((always_inline)) {
            const char *src = src0 + (rd & (kSlots - 1)) * kSlotBytes;
            x[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(src + n * 32));
            x[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(src + n * 32 + 16 * kLatLd));
        };
        for (int rd = 0; rd <= nr; ++rd) {      // (as the score waves count: round rd - 1 is taken here)
            if (((rd + 2) & 63) == 0) look_up(rd + 2);
            if (rd == 0) {
                stage(2, true);
            } else {
                const char *const pb = pbuf + ((rd - 1) & 1) * kPBytes + lane * 16;
                const u32x4 raw = needed(rd - 1);
                u32x4 p[VG];
#pragma unroll
                for (int g = 0; g < VG; ++g) p[g] = *reinterpret_cast<const u32x4 *>(pb + g * kFrag);
                if (any_of(raw)) {
                    block_barrier();
#pragma unroll
                    for (int g = 0; g < VG; ++g) p[g] = *reinterpret_cast<const u32x4 *>(pb + g * kFrag);
#pragma unroll
                    for (int g = 0; g < VG; ++g) {
                        const float f = xf[g / NT * 16 + r16];
#pragma unroll
                        for (int n = 0; n < 8; ++n) acc[n][g] *= f;
                    }
                }
                if (wave == 4 && lane == 0) *reinterpret_cast<u32x4 *>(need[(rd + 1) & 3]) = u32x4{0, 0, 0, 0};
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const s4_t x = ring[n % kAhead][0], y = ring[n % kAhead][1];
                    if (n + kAhead < 8) columns(rd - 1, n + kAhead, ring[n % kAhead]);
                    const u32x4 v = __builtin_bit_cast(u32x4, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int g = 0; g < VG; ++g) acc[n][g] = mfma<F16>(v, p[g], acc[n][g]);
                    __builtin_amdgcn_sched_barrier(0);
                    if (n == 0) prepare(rd + 2, true);
                    if (n >= 1 && n < 5) stage_row(n - 1);
                    if (n == 5) stage_rot();
                }
            }
            if (NT == 3 && rd < nr) block_barrier();        // (the third terms' scores)
            // round rd's rows, which the score waves have: their first operands, while this wave would wait
            if (rd < nr && (!in0 || t_begin + (rd + 1) * kRound > t_all)) {
                // some row does not see all of it: what it does not see must not reach it, not even as 0 x infinity
                arrived_barrier<5>();           // (the scores are taken from the values as they are)
                char *const slot = lds + (rd & (kSlots - 1)) * kSlotBytes;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    u32x4 *const x = reinterpret_cast<u32x4 *>(slot + (4 * i + q4) * kLatLd + cw * 256 + r16 * 16);
                    u32x4 v = *x;
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = finite2<F16>(v[j]);
                    *x = v;
                }
#pragma unroll
                for (int n = 0; n < kAhead; ++n) columns(rd, n, ring[n]);
            } else {
#pragma unroll
                for (int n = 0; n < kAhead; ++n) columns(rd, n, ring[n]);
                // (nothing that this wave wrote is waited for but need[], which its reads since then came after)
                arrived_barrier<5, false>();
            }
            in0 = in1, in1 = r_lat.z != 0;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // (what still arrives must not fall into the records, nor into LDS that the block has left)
        block_barrier();
        // the rows go through LDS (the rounds are done), so that they leave it as whole rows
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            const int row = g * 16 + r16;
            char *const to = lds + row * kRecLd + (cw * 128 + 4 * q4) * (NT == 1 ? 2 : 4);
            if constexpr (NT == 1) {
                const float l = xm[0][0][row] + xf[row], inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const f32x4 o = acc[n][g] * inv;
                    *reinterpret_cast<u32x2 *>(to + n * 32) = u32x2{q4_pack_f16(o[0], o[1]), q4_pack_f16(o[2], o[3])};
                }
            } else {
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    f32x4 o = acc[n][g * NT] + acc[n][g * NT + 1];
                    if constexpr (NT == 3) o += acc[n][2];
                    *reinterpret_cast<f32x4 *>(to + n * 64) = o;
                }
            }
        }
    }
    block_barrier();
    {
        char *const to = static_cast<char *>(a.part) + static_cast<int64_t>(at) * a.Mrec * kRecRow;
        constexpr int kOf = kRecRow / 1024;         // 1 KB a wave and store
#pragma unroll
        for (int i = 0; i < kRows * kOf / 8; ++i) {
            const int piece = i * 8 + wave, row = piece / kOf, off = piece % kOf * 1024 + lane * 16;
            if (row < a.Mrec)
                *reinterpret_cast<u32x4 *>(to + static_cast<int64_t>(row) * kRecRow + off) = *reinterpret_cast<const u32x4 *>(lds + row * kRecLd + off);
        }
    }
}

// ------------------------------------------------------------------ uv
struct UvArgs {
    const void *part;
    const float2 *ml;
    const Head *head;
    const int2 *seq;
    const uint16_t *w_uv;       // [H, V, 512]
    void *out;                  // [B, Tall, H, V]
    const float *gate;          // the same, or null
    int H, V, M, T, t0, Tall, G, GT, tiles, ptiles, Mrec, out_bf16, half;       // half: the records are fp16
    Rows rows;
};

constexpr int kCLd = 1040;      // LDS bytes of a context row's term: 1024 + 16

// A row's records: those of its tile below the split, then its sequence's.
struct Records {
    int first, low, n, step, tiles, in, pin, Mrec;
    __device__ __forceinline__ Records(const UvArgs &a, int m, int h) {
        const int b = m / a.T, row = a.rows.of(m - b * a.T, h), g = row >> 4, pg = b * a.G + g;
        const int2 mine = a.seq[b];
        low = a.head->ranges, n = low + mine.y;
        first = mine.x + g / a.GT, step = a.ptiles, tiles = a.tiles, Mrec = a.Mrec;
        in = (g % a.GT) * 16 + (row & 15), pin = pg / a.GT * a.Mrec + (pg % a.GT) * 16 + (row & 15);
    }
    // the place of record k (at most 2^31 rows: of items of at least 1 KB a row, 2 TB)
    __device__ __forceinline__ int at(int k) const { return k < low ? k * step * Mrec + pin : (first + (k - low) * tiles) * Mrec + in; }
};

// The lanes of a whose bit is set, and those of b whose bit is not, change places; CTRL pairs the lanes (xor 1: 0xb1, xor 2: 0x4e).
template <int CTRL>
__device__ __forceinline__ void exchange(u32x4 &a, u32x4 &b, bool set) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const uint32_t x = a[d], y = b[d];
        const uint32_t to_a = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(y), CTRL, 0xf, 0xf, true));
        const uint32_t to_b = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xf, 0xf, true));
        a[d] = set ? to_a : x, b[d] = set ? y : to_b;
    }
}

// Bound by the records, 64 KB an item, and W_UV, behind the launch itself: 64 queries of 64 heads behind a prefix read 40 MB in 9 us.
// grid (H, ceil(M / PER)), eight waves: PER queries of head x.  A wave joins the records of a query (PER 1: eight waves every eighth record of 64), eight
// columns a lane, and leaves the context in LDS as TERMS bf16 terms; then a wave takes 16 output columns of all queries, its rows of W_UV as they lie.
template <int TERMS, int PER>
__global__ __launch_bounds__(512, PER == 8 ? 2 : 4) void uv_kernel(UvArgs a) {
    static_assert(PER == 1 || PER % 8 == 0, "waves to a query, or queries to a wave");
    constexpr int kTiles = (PER + 15) / 16, kRows = PER < 16 ? PER : 16, kSide = PER == 8 ? 12 : 4;  // kSide: records on their way
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float seen[PER];                                 // a query's sum: 0 where it sees nothing
    char *const ctx = lds;                                      // [TERMS][PER][kCLd]
    float *const sums = reinterpret_cast<float *>(lds + TERMS * PER * kCLd);    // PER 1: [8][512]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, q4 = lane >> 4;
    const int h = blockIdx.x, m0 = blockIdx.y * PER;
    const int vtiles = (a.V + 15) / 16;
    const auto rw = make_rsrc(a.w_uv + static_cast<int64_t>(h) * a.V * kLat, static_cast<uint32_t>(a.V) * (2 * kLat));
    // An operand's 16 neighbouring lanes are 16 rows of W_UV, and loaded like that take the load path three to four times as long as 64 bytes of
    // four rows do (4 x 200 tokens 54 us for 44, 6 long requests 15 for 11).  So load 4 J + i is of rows i, 4 + i, 8 + i and 12 + i, 256 bytes of
    // each, and turned() exchanges the lanes of a quad with the four loads: then operand 4 J + i is columns 128 J + 32 q4 + 8 i .. +8 of row r16.
    u32x4 w[16];
    auto weights = [&](int vt) __attribute__((always_inline)) {         // (rows past the head's last are outside and load zeros)
        const uint32_t at = static_cast<uint32_t>(vt * 16 + (r16 & 12)) * (2 * kLat) + q4 * 64 + (r16 & 3) * 16;
#pragma unroll
        for (int k = 0; k < 16; ++k) w[k] = __builtin_bit_cast(u32x4, buf_load16(rw, at + (k & 3) * (2 * kLat) + (k >> 2) * 256));
    };
    auto turned = [&]() __attribute__((always_inline)) {
        const bool odd = lane & 1, high = lane & 2;
#pragma unroll
        for (int J = 0; J < 16; J += 4) {
            exchange<0xb1>(w[J], w[J + 1], odd), exchange<0xb1>(w[J + 2], w[J + 3], odd);
            exchange<0x4e>(w[J], w[J + 2], high), exchange<0x4e>(w[J + 1], w[J + 3], high);
        }
    };
    // the context of columns 8 lane .. +8 (fp16 records: 16 bytes a lane), or of 4 lane .. +4 and 256 + 4 lane .. +4
    const bool half = TERMS == 2 && a.half;
    auto store = [&](int i, f32x4 x, f32x4 y) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
            const u32x2 p = {q4_pack_bf16(x[0], x[1]), q4_pack_bf16(x[2], x[3])}, o = {q4_pack_bf16(y[0], y[1]), q4_pack_bf16(y[2], y[3])};
            *reinterpret_cast<u32x2 *>(ctx + (t * PER + i) * kCLd + lane * (half ? 16 : 8)) = p;
            *reinterpret_cast<u32x2 *>(ctx + (t * PER + i) * kCLd + (half ? lane * 16 + 8 : 512 + lane * 8)) = o;
            x -= f32x4{q4_lo(p.x), q4_hi(p.x), q4_lo(p.y), q4_hi(p.y)};
            y -= f32x4{q4_lo(o.x), q4_hi(o.x), q4_lo(o.y), q4_hi(o.y)};
        }
    };
    // the row's records, and the maxima and sums of its first 64: sent for while the query before is joined
    auto stats = [&](const Records &rec, int k) __attribute__((always_inline)) { return k < rec.n ? a.ml[rec.at(k)] : make_float2(-INFINITY, 0.f); };
    auto query = [&](int i) __attribute__((always_inline)) { return Records(a, min(m0 + i, a.M - 1), h); };
    Records next = query(PER == 1 ? 0 : wave);
    float2 v_next = stats(next, lane);
    if constexpr (PER <= 8) weights(wave);      // (behind what the join waits for; with more queries, two blocks a CU: the registers are the joins')
#pragma unroll 1
    for (int i = PER == 1 ? 0 : wave; i < PER; i += 8) {
        f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
        float l = 0.f;
        const Records rec = next;
        float2 v = v_next;
        if (PER > 8 && i + 8 < PER) next = query(i + 8), v_next = stats(next, lane);
        if (m0 + i < a.M) {
            // (the weight of a record that the row sees nothing of is zero, and what is written there does not matter)
            float mx = v.x;
            for (int k0 = 64; k0 < rec.n; k0 += 64) mx = fmaxf(mx, stats(rec, k0 + lane).x);
            mx = wave_max_all(mx);
            for (int k0 = 0; k0 < rec.n; k0 += 64) {
                if (k0) v = stats(rec, k0 + lane);
                const int at = rec.at(min(k0 + lane, rec.n - 1)), n = min(rec.n - k0, 64);
                const float f = v.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(v.x - mx);
                if (PER > 1 || wave == 0) l = fmaf(f, v.y, l);
                // (fp16 records are contexts over their sums)
                const float weight = half ? f * v.y : f;
                for (int j0 = PER == 1 ? wave * kSide : 0; j0 < n; j0 += PER == 1 ? 8 * kSide : kSide) {
                    float g[kSide];
                    int from[kSide];
#pragma unroll
                    for (int j = 0; j < kSide; ++j) {
                        from[j] = __builtin_amdgcn_readlane(at, (j0 + j) & 63);
                        g[j] = j0 + j < n ? readlane_f(weight, (j0 + j) & 63) : 0.f;
                    }
                    if (half) {
                        u32x4 c[kSide] = {};
#pragma unroll
                        for (int j = 0; j < kSide; ++j) {
                            const uint16_t *p = static_cast<const uint16_t *>(a.part) + static_cast<int64_t>(from[j]) * kLat + 8 * lane;
                            if (g[j] != 0.f) c[j] = *reinterpret_cast<const u32x4 *>(p);
                        }
#pragma unroll
                        for (int j = 0; j < kSide; ++j) {
                            float u[8];
#pragma unroll
                            for (int k = 0; k < 4; ++k) unpack2<true>(c[j][k], u[2 * k], u[2 * k + 1]);
#pragma unroll
                            for (int k = 0; k < 4; ++k) x[k] = fmaf(g[j], u[k], x[k]), y[k] = fmaf(g[j], u[4 + k], y[k]);
                        }
                    } else {
                        f32x4 c[kSide][2] = {};
#pragma unroll
                        for (int j = 0; j < kSide; ++j) {
                            const float *p = static_cast<const float *>(a.part) + static_cast<int64_t>(from[j]) * kLat + 4 * lane;
                            if (j0 + j < n) c[j][0] = *reinterpret_cast<const f32x4 *>(p), c[j][1] = *reinterpret_cast<const f32x4 *>(p + 256);
                        }
#pragma unroll
                        for (int j = 0; j < kSide; ++j)
                            if (g[j] != 0.f) x += g[j] * c[j][0], y += g[j] * c[j][1]; 
                    }
                }
            }
            l = wave_sum_all(l);
        }
        if constexpr (PER > 1) {
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            if (lane == 0) seen[i] = l;
            store(i, x * inv, y * inv);
        } else {
            *reinterpret_cast<f32x4 *>(sums + wave * kLat + 4 * lane) = x;
            *reinterpret_cast<f32x4 *>(sums + wave * kLat + 256 + 4 * lane) = y;
            if (wave == 0 && lane == 0) seen[0] = l;
            __syncthreads();
            if (wave == 0) {
                const float all = seen[0], inv = all == 0.f ? 0.f : 1.0f / all;
#pragma unroll
                for (int k = 1; k < 8; ++k) {
                    x += *reinterpret_cast<const f32x4 *>(sums + k * kLat + 4 * lane);
                    y += *reinterpret_cast<const f32x4 *>(sums + k * kLat + 256 + 4 * lane);
                }
                store(0, x * inv, y * inv);
            }
        }
    }
    __syncthreads();
    for (int vt = wave; vt < vtiles; vt += 8) {
        if (PER > 8 || vt != wave) weights(vt);
        turned();
        f32x4 o[kTiles], o2[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) o[t] = o2[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int y = TERMS - 1; y >= 0; --y)
#pragma unroll
            for (int k = 0; k < 16; ++k)
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    f32x4 &to = k & 1 ? o2[t] : o[t];
                    const char *c = ctx + (y * PER + t * 16 + r16 % kRows) * kCLd + (k >> 2) * 256 + q4 * 64 + (k & 3) * 16;
                    to = q4_mfma_bf16(w[k], *reinterpret_cast<const u32x4 *>(c), to);
                }
#pragma unroll
        for (int t = 0; t < kTiles; ++t) o[t] += o2[t];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int m = m0 + t * 16 + r16, v = vt * 16 + 4 * q4;
            if (r16 >= kRows || m >= a.M || v >= a.V) continue;
            const int b = m / a.T, tq = a.t0 + m - b * a.T;
            const int64_t to = ((static_cast<int64_t>(b) * a.Tall + tq) * a.H + h) * a.V + v;
            if (a.gate) {
                const f32x4 g = *reinterpret_cast<const f32x4 *>(a.gate + to);
                const bool any = seen[t * 16 + r16] != 0.f;     // (the gate of a query that sees nothing may be anything: a row of padding's)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][i] = any ? o[t][i] / (1.0f + expf(-g[i])) : 0.f;
            }
            if (a.out_bf16)
                *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + to) = u32x2{q4_pack_bf16(o[t][0], o[t][1]), q4_pack_bf16(o[t][2], o[t][3])};
            else
                *reinterpret_cast<f32x4 *>(static_cast<float *>(a.out) + to) = o[t];
        }
    }
}

// ------------------------------------------------------------------ host side
constexpr int64_t kPassRows = 1 << 16;      // rows (heads x queries, all sequences) of one pass over the queries

struct Plan {
    int NT, GT, T, G, tiles, ptiles, Mrec, most, turns;     // T: queries of a sequence in a pass
    Rows rows;
    int64_t groups, qop, scales, part, ml, head, seq, item, total;
};

// By head where that adds a tenth of rows at most.
Rows rows_of(int64_t T, int64_t H) {
    const int64_t Tp = cdiv(T, 16) * 16;
    return Rows{static_cast<int>(T), static_cast<int>(H), 10 * Tp <= 11 * T ? static_cast<int>(Tp) : 0};
}

// What the launches are cut into; a function of its arguments alone.
Plan plan_of(int64_t B, int64_t T, int64_t H, int64_t max_length, int64_t prefix, int cache_dtype, int out_dtype) {
    Plan p{};
    p.NT = (cache_dtype == K3_F16 ? 1 : 2) + (out_dtype == K3_F32);
    p.GT = 4 / p.NT;
    p.T = static_cast<int>(std::max<int64_t>(1, std::min(T, kPassRows / (B * H))));
    p.rows = rows_of(p.T, H);
    p.G = static_cast<int>(cdiv(p.rows.count(), 16));
    p.tiles = static_cast<int>(cdiv(p.G, p.GT));
    p.groups = B * p.G;
    p.ptiles = prefix > 0 ? static_cast<int>(cdiv(p.groups, p.GT)) : 0;
    p.Mrec = 16 * static_cast<int>(std::min<int64_t>(p.GT, prefix > 0 ? p.groups : p.G));
    // every range that is not full, a tile and sequence one at most, and the others: at most 256 a turn, and of a round at least
    const int64_t base = B * p.tiles + p.ptiles;
    const int64_t positions = p.ptiles * std::min(prefix, max_length) + B * p.tiles * std::max<int64_t>(max_length - prefix, 0);
    p.turns = static_cast<int>(std::min<int64_t>(kTurns, std::max<int64_t>(1, positions / (256 * 1024))));
    p.most = static_cast<int>(base + std::min<int64_t>(256 * p.turns, positions / kRound + 1));
    auto up = [](int64_t v) { return (v + 255) & ~int64_t(255); };
    int64_t o = 0;
    p.qop = o, o += up(p.groups * p.NT * kSteps * kFrag);
    p.scales = o, o += up(p.groups * kParts * 16 * 4);
    p.ml = o, o += up(static_cast<int64_t>(p.most) * p.Mrec * 8);
    p.part = o, o += up(static_cast<int64_t>(p.most) * p.Mrec * kLat * (p.NT == 1 ? 2 : 4));
    p.head = o, o += 256;
    p.seq = o, o += up(B * 8);
    p.item = o, o += up(static_cast<int64_t>(p.most) * static_cast<int64_t>(sizeof(Item)));
    p.total = o;
    return p;
}

template <typename QT, bool F16, int NT, int MT>
int launch_qa_of(const QaArgs &a, hipStream_t st) {
    const int bytes = std::max({((a.nope + 31) / 32) * 32 * kWLd, 16 * MT * kFLd * 4, kListLds});
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(qa_kernel<QT, F16, NT, MT>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, 256 * kWLd);
    const int rc = check_hip(attr, "mla paged: query LDS size");
    if (rc) return rc;
    qa_kernel<QT, F16, NT, MT><<<dim3(static_cast<unsigned>(4 * a.H * cdiv(a.M, 16 * MT) + 1)), 256, bytes, st>>>(a);
    return check_hip(hipGetLastError(), "mla paged: query launch");
}
template <typename QT>
int launch_qa(const QaArgs &a, bool f16, int NT, hipStream_t st) {
    if (NT == 3) return a.M > 32 ? launch_qa_of<QT, false, 3, 4>(a, st) : launch_qa_of<QT, false, 3, 1>(a, st);
    if (!f16) return a.M > 32 ? launch_qa_of<QT, false, 2, 4>(a, st) : launch_qa_of<QT, false, 2, 1>(a, st);
    if (NT == 1) return a.M > 32 ? launch_qa_of<QT, true, 1, 4>(a, st) : launch_qa_of<QT, true, 1, 1>(a, st);
    return a.M > 32 ? launch_qa_of<QT, true, 2, 4>(a, st) : launch_qa_of<QT, true, 2, 1>(a, st);
}

template <bool F16, int NT>
int launch_attend(const AttendArgs &a, int most, hipStream_t st) {
    static const hipError_t attr =
        hipFuncSetAttribute(reinterpret_cast<const void *>(attend_kernel<F16, NT>), hipFuncAttributeMaxDynamicSharedMemorySize, attend_lds());
    const int rc = check_hip(attr, "mla paged: attention LDS size");
    if (rc) return rc;
    // (an eighth of both kinds of item to an XCD: one more than an eighth of all at most)
    attend_kernel<F16, NT><<<dim3(static_cast<unsigned>(cdiv(most, 8) * 8 + 8)), 512, attend_lds(), st>>>(a);
    return check_hip(hipGetLastError(), "mla paged: attention launch");
}

template <int TERMS, int PER>
int launch_uv_of(const UvArgs &a, hipStream_t st) {
    constexpr int bytes = TERMS * PER * kCLd + (PER == 1 ? 8 * kLat * 4 : 0);
    static const hipError_t attr =
        hipFuncSetAttribute(reinterpret_cast<const void *>(uv_kernel<TERMS, PER>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    const int rc = check_hip(attr, "mla paged: output LDS size");
    if (rc) return rc;
    uv_kernel<TERMS, PER><<<dim3(static_cast<unsigned>(a.H), static_cast<unsigned>(cdiv(a.M, PER))), 512, bytes, st>>>(a);
    return check_hip(hipGetLastError(), "mla paged: join and W_UV launch");
}
template <int TERMS>
int launch_uv(const UvArgs &a, hipStream_t st) {
    // A block reads its head's W_UV: the fewest queries to a block with which all blocks are on the card at once (of 32 and 16 queries two a CU, of 8
    // one), else 32.
    // Measured, us, 8 / 16 / 32 queries: 32 requests of 64 heads 12.7 / 17.1 / 25.8, 25 of 96 13.4 / 10.2 / 13.4, 64 of 64 13.2 / 9.3 / 12.8, 120 of 64
    // 24.4 / 12.6 / 13.8, 800 of 64 119 / 51.6 / 45.3.  Few queries have waves enough for all a query's records: 6 of 64 heads, some 80 records each,
    // 16.4 for a wave a query, 11.6 for eight.  Whole calls, eight waves a query / a wave (8 queries a block): requests of up to 16,384, 64 heads, 4 of
    // them 32.6 / 45.7, 8 34.0 / 40.3, 12 38.9 / 39.0, 16 42.6 / 40.2; of up to 500 20.3 / 21.1, 23.8 / 22.7, 27.6 / 22.5, 30.1 / 23.7.  With 16 heads
    // eight waves are the shorter at 16 queries too (30.0 / 37.2), with 96 the longer from 6 on (40.1 / 39.6, 27.7 / 24.3).
    if (a.H * cdiv(a.M, 16) > 512) return launch_uv_of<TERMS, 32>(a, st);
    if (a.H * cdiv(a.M, 8) > 256) return launch_uv_of<TERMS, 16>(a, st);
    if (a.M > 8) return launch_uv_of<TERMS, 8>(a, st);
    return launch_uv_of<TERMS, 1>(a, st);
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" int64_t k3_mla_paged_workspace_size(int64_t B, int64_t T, int64_t H, int64_t max_length, int64_t shared, int cache_dtype,
                                               int out_dtype) {
    if (B <= 0 || T <= 0 || H <= 0 || max_length < 0 || shared < 0) return 0;
    return plan_of(B, T, H, max_length, shared, cache_dtype, out_dtype).total;
}

extern "C" int k3_mla_paged_attention(const void *q_nope, int64_t qn_batch, int64_t qn_token, int64_t qn_head, const void *q_rot,
                                      int64_t qr_batch, int64_t qr_token, int64_t qr_head, int q_dtype, const void *w_uk,
                                      const void *w_uv, const void *lat, int64_t lat_page, int64_t lat_row, const void *rot,
                                      int64_t rot_page, int64_t rot_row, int cache_dtype, int64_t pages, int64_t page_size,
                                      const int32_t *table, int64_t table_row, int64_t blocks, const int32_t *prefix,
                                      int64_t prefix_pages, const int32_t *lengths, const int32_t *counts, int64_t max_length, int64_t B,
                                      int64_t T, int64_t H, int64_t kv_lora_rank, int64_t rope_dim, int64_t nope_dim, int64_t v_dim,
                                      float scale, const float *gate, void *out, int out_dtype, void *workspace, int64_t workspace_bytes,
                                      void *stream) {
    if (B == 0 || T == 0) return K3_OK;
    if (!q_nope || !q_rot || !w_uk || !w_uv || !out || !workspace || !lengths || (pages > 0 && (!lat || !rot)) || (blocks > 0 && !table) ||
        (prefix_pages > 0 && !prefix))
        return set_error(K3_ERR_NULL, "mla paged: null pointer");
    if (q_dtype != K3_F32 && q_dtype != K3_BF16) return set_error(K3_ERR_DTYPE, "mla paged: q_dtype %d", q_dtype);
    if (out_dtype != K3_F32 && out_dtype != K3_BF16) return set_error(K3_ERR_DTYPE, "mla paged: out_dtype %d", out_dtype);
    if (cache_dtype != K3_F16 && cache_dtype != K3_BF16) return set_error(K3_ERR_DTYPE, "mla paged: cache dtype %d", cache_dtype);
    if (kv_lora_rank != kLat || rope_dim != kRot)
        return set_error(K3_ERR_SHAPE, "mla paged: kv_lora_rank=%lld rope=%lld; the kernels take 512 and 64", (long long)kv_lora_rank,
                         (long long)rope_dim);
    if (nope_dim <= 0 || nope_dim > 256 || nope_dim % 8 || v_dim <= 0 || v_dim > 1024 || v_dim % 8)
        return set_error(K3_ERR_SHAPE, "mla paged: nope=%lld must be a multiple of 8 up to 256 and v=%lld one up to 1024",
                         (long long)nope_dim, (long long)v_dim);
    if (page_size < kRound || page_size > (1 << 16) || (page_size & (page_size - 1)))
        return set_error(K3_ERR_SHAPE, "mla paged: page_size=%lld must be a power of two, 32 to 65536", (long long)page_size);
    if (B < 0 || B > 65535 || T < 0 || T > (1 << 24) || H <= 0 || H > 4096 || B * H > kPassRows || pages < 0 || pages >= (1ll << 31) || blocks < 0 ||
        prefix_pages < 0 || max_length < 0 || max_length > (1 << 24) || blocks > (1 << 24) || prefix_pages > (1 << 24) || max_length > blocks * page_size)
        return set_error(K3_ERR_SHAPE, "mla paged: B=%lld, T=%lld, H=%lld, %lld pages, max_length=%lld of %lld blocks or prefix of %lld pages out of range",
                         (long long)B, (long long)T, (long long)H, (long long)pages, (long long)max_length, (long long)blocks, (long long)prefix_pages);
    if (B > 1 && table_row < blocks) return set_error(K3_ERR_SHAPE, "mla paged: the table's rows overlap, %lld apart", (long long)table_row);
    if (qn_batch % 4 || qn_token % 4 || qn_head % 4 || qr_batch % 4 || qr_token % 4 || qr_head % 4)
        return set_error(K3_ERR_SHAPE, "mla paged: query strides must be multiples of 4 elements");
    if (lat_row < kLat || rot_row < kRot || lat_row % 8 || rot_row % 8 || lat_page % 8 || rot_page % 8 || lat_row > (1 << 20) || rot_row > (1 << 20))
        return set_error(K3_ERR_SHAPE, "mla paged: cache row pitches too small, too large or not multiples of 16 bytes");
    if (!aligned16(q_nope) || !aligned16(q_rot) || !aligned16(w_uk) || !aligned16(w_uv) || !aligned16(out) || !aligned16(workspace) ||
        !aligned16(lat) || !aligned16(rot) || (gate && !aligned16(gate)))
        return set_error(K3_ERR_ALIGN, "mla paged: queries, weights, cache, output and workspace must be 16-byte aligned");
    const Plan p = plan_of(B, T, H, max_length, prefix_pages * page_size, cache_dtype, out_dtype);
    if (workspace_bytes < p.total)
        return set_error(K3_ERR_WORKSPACE, "mla paged: workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)p.total);
    int shift = 0;
    while ((1ll << shift) < page_size) ++shift;
    auto st = static_cast<hipStream_t>(stream);
    char *ws = static_cast<char *>(workspace);
    const bool f16 = cache_dtype == K3_F16;
    for (int64_t t0 = 0; t0 < T; t0 += p.T) {
        // (the last pass may have fewer queries; it has the others' room)
        const int Tp = static_cast<int>(std::min<int64_t>(p.T, T - t0)), M = static_cast<int>(B * Tp);
        const Rows rows = Tp == p.T ? p.rows : Rows{Tp, static_cast<int>(H), 0};
        const int G = static_cast<int>(cdiv(rows.count(), 16));
        const int tiles = static_cast<int>(cdiv(G, p.GT)), groups = static_cast<int>(B * G);
        const int ptiles = prefix_pages > 0 ? static_cast<int>(cdiv(groups, p.GT)) : 0;
        const Lists lists{lengths, counts, reinterpret_cast<Head *>(ws + p.head), reinterpret_cast<int2 *>(ws + p.seq),
                          reinterpret_cast<Item *>(ws + p.item), static_cast<int>(B), Tp, static_cast<int>(t0), static_cast<int>(T),
                          static_cast<int>(max_length), static_cast<int>(std::min(prefix_pages * page_size, max_length)), tiles, ptiles, p.most, p.turns,
                          ptiles > 0 && G % p.GT == 0};
        const QaArgs qa{q_nope, q_rot, qn_batch, qn_token, qn_head, qr_batch, qr_token, qr_head, static_cast<const uint16_t *>(w_uk),
                        ws + p.qop, reinterpret_cast<float *>(ws + p.scales), static_cast<int>(H), static_cast<int>(nope_dim), M, Tp,
                        static_cast<int>(t0), G, rows, lists};
        int rc = q_dtype == K3_BF16 ? launch_qa<uint16_t>(qa, f16, p.NT, st) : launch_qa<float>(qa, f16, p.NT, st);
        if (rc) return rc;
        AttendArgs a{};
        a.qop = qa.qop, a.scales = qa.scales, a.lat = static_cast<const char *>(lat), a.rot = static_cast<const char *>(rot);
        a.lat_page = 2 * lat_page, a.rot_page = 2 * rot_page;
        a.lat_row = static_cast<uint32_t>(2 * lat_row), a.rot_row = static_cast<uint32_t>(2 * rot_row);
        a.table = table, a.prefix = prefix, a.table_row = table_row, a.pages = static_cast<int>(pages), a.shift = shift;
        a.lists = lists;
        a.part = ws + p.part, a.ml = reinterpret_cast<float2 *>(ws + p.ml);
        a.rows = rows, a.G = G, a.groups = groups, a.Mrec = p.Mrec, a.c = scale * 1.4426950408889634f;
        rc = p.NT == 3   ? launch_attend<false, 3>(a, p.most, st)
             : !f16      ? launch_attend<false, 2>(a, p.most, st)
             : p.NT == 1 ? launch_attend<true, 1>(a, p.most, st)
                         : launch_attend<true, 2>(a, p.most, st);
        if (rc) return rc;
        const UvArgs u{a.part, a.ml, lists.head, lists.seq, static_cast<const uint16_t *>(w_uv), out, gate, static_cast<int>(H), static_cast<int>(v_dim), M, Tp,
                       static_cast<int>(t0), static_cast<int>(T), G, p.GT, tiles, ptiles, p.Mrec, out_dtype == K3_BF16, p.NT == 1, rows};
        rc = u.out_bf16 ? launch_uv<2>(u, st) : launch_uv<3>(u, st);
        if (rc) return rc;
    }
    return K3_OK;
}
