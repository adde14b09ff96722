// Latent (MLA) attention over the 4-bit cache, in the absorbed form: one token or several of each of B sequences.
//
//     qa[t,h]  = q_nope[t,h] W_UK[h]                                              [512]
//     s[t,h,j] = scale (qa[t,h] . lat[j] + q_rot[t,h] . rot[j])                   j < sees(t)
//     p = softmax_j(s);   o[t,h] = W_UV[h] (sum_j p[t,h,j] lat[j]);   weight[j] += sum_{t,h} p[t,h,j]   (if asked for)
//
// Every head of every query of a sequence reads the same 400 bytes of a position, so a sequence is one problem of
// T x H rows against its cache.  Launches:
//   qa       q_nope W_UK on the bf16 matrix cores (fp32 queries as three bf16 terms), rounded into the 6-bit terms
//            that the scaled matrix product takes (mla_q4.h)
//   attend   a block = 16 RG rows x a range of positions, eight waves: the maximum and sum run with the positions
//   uv       the ranges' records joined, the context times W_UV, the output gate
//   weights  (if asked for) p once more from the rows' final maxima and sums, added over the rows
//
// attend, per round of 64 positions: the codes go to LDS as they are, 256 bytes and 16 scale bytes a position, and both products
// take them from there: the score waves (0..3) as operands of the scaled product, the context waves (4..7, 128 columns each)
// transposed, 4 bits at a time (ds_read_b64_tr_b4), decoded in registers to fp16 and multiplied with the positions' scales, which the
// score waves leave in LDS as fp16 (exact, see mla_q4.h).  (Decoding into a value tile in LDS, 1 KB a position written and read, held
// rounds of 32 positions only and took 0.86 us for each at 32 rows, 1.15 at 64.)  One barrier an iteration: round i + 1 is stored, round
// i's scores and the last round's probabilities are formed, the context waves take the products of the round before.  A row's reference
// maximum moves only when a score exceeds it by kSlack (log2), so the accumulators are seldom rescaled.
//
// A position whose scale byte is 255 (NaN) makes its scores NaN by the matrix product itself, so every row that sees it is NaN; its
// scale for the second product is zero, so a row that does not see it (weight zero) stays clean.
#include <algorithm>
#include <type_traits>

#include "mla_q4.h"

namespace k3 {
namespace {

typedef short s4_t __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s4_t *lds_s4;
typedef __attribute__((address_space(3))) i32x2 *lds_i2;

// n / d by a multiplication: ceil(2^32 / d) (0: d is 1) is exact where n d < 2^32, as for the rows, queries and blocks of a pass (a
// division is some 40 dependent instructions, and most kernels here make several before their first load).
inline uint32_t inverse_of(int64_t d) { return d == 1 ? 0u : static_cast<uint32_t>(cdiv(1ll << 32, d)); }
__device__ __forceinline__ int quotient(int n, uint32_t inverse) {
    return inverse ? static_cast<int>(__umulhi(static_cast<uint32_t>(n), inverse)) : n;
}

// The order of a sequence's rows: by query (row = t H + h: the heads of one query are neighbours, few queries fill the tiles)
// or by head (row = h Tp + t, Tp = T rounded up to 16: a tile is 16 queries of one head, so a block of the query and output
// launches, which takes one head's matrix, writes and reads whole tiles).
struct Rows {
    int T, H, Tp;                           // Tp 0: by query
    uint32_t inverse, inverse_t;            // of d = Tp or H, and of T
    __host__ __device__ int count() const { return Tp ? H * Tp : T * H; }
    __device__ int of(int t, int h) const { return Tp ? h * Tp + t : t * H + h; }
    __device__ int major(int row) const { return quotient(row, inverse); }
    __device__ int seq(int m) const { return quotient(m, inverse_t); }      // of query m of all sequences
    __device__ int token(int m) const { return m - seq(m) * T; }
    __device__ int query(int row) const { return Tp ? row - major(row) * Tp : major(row); }       // may be >= T: no row
    // the last query of rows row0 .. row1
    __device__ int last_query(int row0, int row1) const {
        const int last = major(row1);
        if (!Tp) return last;
        return major(row0) != last ? T - 1 : min(row1 - last * Tp, T - 1);
    }
};

// ------------------------------------------------------------------ ranges
// What the blocks of the attention take, a range of positions of a sequence each ("slot", with a record of its own for every row).
// Sequences of one length, or with rows enough for the card: range `slot % NS` of sequence `slot / NS`.  Sequences of lengths of their
// own that are few blocks: a list made on the device, by a block of the query launch, with ranges of one length that fills the card
// with what there is rather than with the capacity.  (32 sequences of up to 8192 positions, 1028 on average: NS ranges of the capacity
// each took 68 us in all, the list 54.)
struct Ranges {
    const int32_t *lengths;     // [B]
    int4 *slot;                 // [slots]: sequence (-1: none), first position, last + 1, the sequence's length
    int2 *seq;                  // [B]: first slot, number of slots; null: no list
    int B, cap, slots, spread, least;   // spread: slots less one a sequence; least: shortest range
};
constexpr int kMaxListed = 512;         // sequences of a list

// by 256 threads
__device__ __forceinline__ void list_ranges(const Ranges &a, int *lds) {
    int *const first = lds, *const len = lds + kMaxListed, *const part = lds + 2 * kMaxListed;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int n[2], own = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {       // sequences 2 tid, 2 tid + 1
        const int b = 2 * tid + u;
        n[u] = b < a.B ? min(max(a.lengths[b], 0), a.cap) : 0;
        len[b] = n[u], own += n[u];
    }
    float total = static_cast<float>(own);      // (the ranges' length need not be exact, but the same everywhere: one thread sets it)
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o);
    if (lane == 0) part[wave] = __float_as_int(total);
    __syncthreads();
    if (tid == 0) {
        float t = 0.f;
        for (int i = 0; i < 4; ++i) t += __int_as_float(part[i]);
        part[4] = max(a.least, (static_cast<int>(t * 1.001f / static_cast<float>(a.spread)) + 64) & ~63);
    }
    __syncthreads();
    const int Ts = part[4];
    int c[2], sum = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) c[u] = (n[u] + Ts - 1) / Ts, sum += c[u];
    int before = sum;                   // inclusive over the wave's threads
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(before, o);
        if (lane >= o) before += x;
    }
    if (lane == 63) part[8 + wave] = before;
    __syncthreads();
    before -= sum;
    for (int i = 0; i < wave; ++i) before += part[8 + i];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int b = 2 * tid + u;
        first[b] = before;
        if (b < a.B) a.seq[b] = make_int2(min(before, a.slots - 1), min(c[u], a.slots - before));
        before += c[u];
    }
    if (tid == 255) part[12] = before;
    __syncthreads();
    const int used = part[12];
    for (int s = tid; s < a.slots; s += 256) {
        int b = 0;                      // the last sequence that starts at or before s (one of several that start there has ranges: the last)
#pragma unroll
        for (int o = kMaxListed / 2; o; o >>= 1)
            if (first[b + o] <= s) b += o;
        const int at = (s - first[b]) * Ts;
        a.slot[s] = s < used ? make_int4(b, at, min(at + Ts, len[b]), len[b]) : make_int4(-1, 0, 0, 0);
    }
}

// ------------------------------------------------------------------ qa
struct QaArgs {
    const void *q_nope, *q_rot;
    int64_t n_b, n_t, n_h, r_b, r_t, r_h;   // strides in elements (batch, query, head)
    const uint16_t *w_uk;                   // [H, nope, 512]
    char *qop;                              // [B][tiles] operand tiles
    int64_t q_seq;                          // bytes of a sequence's tiles
    int H, nope, M, t0;                     // rows.T queries from t0 on; M = B T
    Rows rows;
    Ranges ranges;
};

constexpr int kWLd = 272;                   // LDS bytes per staged weight row (128 columns + 16 bytes)
constexpr int kFLd = 132;                   // floats per staged result row

// three bf16 terms of 8 fp32 values
__device__ __forceinline__ void terms8(const float (&v)[8], u32x4 (&f)[3]) {
    uint32_t t[3][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) split3_near<false>(v[i], t[0][i], t[1][i], t[2][i]);
#pragma unroll
    for (int x = 0; x < 3; ++x)
        f[x] = u32x4{hi16x2(t[x][0], t[x][1]), hi16x2(t[x][2], t[x][3]), hi16x2(t[x][4], t[x][5]), hi16x2(t[x][6], t[x][7])};
}

// 8 query values of a lane: slots 8 q4 .. +8 of a step of 32 hold n = 4 q4 + {0..3} and 16 + 4 q4 + {0..3}, the order in which
// the transposed reads of the weights give theirs
template <typename QT>
struct QueryRaw {
    typedef typename std::conditional<std::is_same<QT, float>::value, f32x4, u32x2>::type V;
    V x[2];
    __device__ __forceinline__ void load(const QT *q, int n, int nope, bool live) {
#pragma unroll
        for (int i = 0; i < 2; ++i) x[i] = live && n + 16 * i < nope ? *reinterpret_cast<const V *>(q + n + 16 * i) : V{};
    }
    __device__ __forceinline__ void terms(u32x4 (&f)[3]) const {
        if constexpr (std::is_same<QT, float>::value) {
            const float v[8] = {x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]};
            terms8(v, f);
        } else {
            f[0] = u32x4{x[0][0], x[0][1], x[1][0], x[1][1]};
        }
    }
};

// grid (H, ceil(M / (16 MT)), 4): queries 16 MT y .. of head x, latent columns 128 z .. +128; z = 4, if there: the list of ranges
// MT 1: few queries, a wave to 32 of the columns; bound by the latency of reading W_UK once (every load in flight at once).
// MT 4: 64 queries to a block's 32 KB of W_UK, a wave to 16 of them, whose bf16 terms it forms once for all columns; bound by the
// 6-bit terms' rounding and by writing them.  (A wave to 32 columns of all 64 formed each query's terms four times: 87 us for
// 1024 fp32 queries of 64 heads, 64 for 512; this: 56 and 44.)
template <typename QT, int NT, int RT, int MT>
__global__ __launch_bounds__(256) void qa_kernel(QaArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float *fs = reinterpret_cast<float *>(lds);                         // [16 MT][kFLd], after the products
    constexpr int kTerms = std::is_same<QT, float>::value ? 3 : 1, kAhead = 4, kTiles = MT == 1 ? 2 : 8;    // column tiles of a wave
    static_assert(MT == 1 || MT == 4, "a wave to 32 columns, or to a tile of queries");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, q4 = lane >> 4;
    const int h = blockIdx.x, m0 = blockIdx.y * 16 * MT, quarter = blockIdx.z;
    if (quarter == 4) {
        if (h == 0 && m0 == 0) list_ranges(a.ranges, reinterpret_cast<int *>(lds));
        return;
    }
    const int steps = (a.nope + 31) >> 5, T = a.rows.T;
    const uint16_t *w = a.w_uk + static_cast<int64_t>(h) * a.nope * kQ4Lat + quarter * 128;
    const int qt = MT == 1 ? 0 : wave, col = MT == 1 ? wave * 32 : 0, mine = m0 + 16 * qt + r16;   // the wave's queries and columns
    const bool live = mine < a.M;
    const int qb = live ? a.rows.seq(mine) : 0, qt0 = live ? a.t0 + mine - qb * T : 0;
    const QT *q = static_cast<const QT *>(a.q_nope) + qb * a.n_b + qt0 * a.n_t + h * a.n_h + 4 * q4;
    QueryRaw<QT> ahead[kAhead];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) ahead[s].load(q, 32 * s, a.nope - 4 * q4, live);
    for (int i0 = 0; i0 < 2 * steps; i0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = (i0 + u) * 256 + tid, n = i >> 4;
            v[u] = n < a.nope ? *reinterpret_cast<const uint4 *>(w + static_cast<int64_t>(n) * kQ4Lat + (i & 15) * 8) : make_uint4(0u, 0u, 0u, 0u);
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
    auto step = [&](int s, const QueryRaw<QT> &raw) __attribute__((always_inline)) {
        const char *wr = lds + (32 * s + 4 * q4 + (r16 >> 2)) * kWLd + (r16 & 3) * 8 + col * 2;
        u32x4 qf[3];
        raw.terms(qf);
#pragma unroll
        for (int j0 = 0; j0 < kTiles; j0 += 2) {
            u32x4 wf[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const s4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(wr + (j0 + j) * 32));
                const s4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(wr + (j0 + j) * 32 + 16 * kWLd));
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
        QueryRaw<QT> raw;
        raw.load(q, 32 * s, a.nope - 4 * q4, live);
        step(s, raw);
    }
    __syncthreads();   // the weights are read
#pragma unroll
    for (int j = 0; j < kTiles; ++j) *reinterpret_cast<f32x4 *>(fs + (16 * qt + r16) * kFLd + col + j * 16 + 4 * q4) = acc[j];
    __syncthreads();
    if (tid < 64 * MT && m0 + (tid >> 2) < a.M) {
        // one group of 32 columns of one query: its terms
        const int i = tid >> 2, g = tid & 3, m = m0 + i, row = a.rows.of(a.rows.token(m), h), at = quarter * 16 + (row & 15);
        char *tile = a.qop + a.rows.seq(m) * a.q_seq + static_cast<int64_t>(row >> 4) * q4_tile_bytes(NT, RT);
        const float *src = fs + i * kFLd + g * 32;
        float v[32];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(src + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[j + k] = x[k], top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
        }
        int byte = static_cast<int>(top >> 23) - 2 + ((top & 0x7fffffu) > 0x700000u ? 1 : 0);   // top / 2^(byte - 127) <= 7.5
        byte = min(max(byte, 1), 253);
        const bool bad = top >= 0x7f800000u;
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            const float s = __uint_as_float(static_cast<uint32_t>(byte) << 23);
            f32x16_t even, odd;
#pragma unroll
            for (int j = 0; j < 16; ++j) even[j] = v[2 * j], odd[j] = v[2 * j + 1];
            const u32x6 code = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, s);   // columns even, odd, even, ..
            if (x + 1 < NT) {
                const f32x32_t back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(code, s);
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] -= back[j];
            }
            char *o = tile + q4_code_at(x, g);
            *reinterpret_cast<u32x4 *>(o + at * 16) = u32x4{code[0], code[1], code[2], code[3]};
            *reinterpret_cast<u32x2 *>(o + 1024 + at * 8) = u32x2{code[4], code[5]};
            // (a NaN or an infinity: the whole product is NaN, by the first term's byte)
            reinterpret_cast<uint8_t *>(tile + q4_scale_at(NT, x))[at * 4 + g] = static_cast<uint8_t>(bad ? 255 : byte);
            byte = max(byte - (x == 0 ? 4 : 5), 1);
        }
    }
    if (quarter != 0) return;
    // rotary columns 8 c .. +8 of a query (one query tile: by the threads that had no group)
    for (int j = MT == 1 ? tid - 64 : tid; j < 128 * MT; j += 256) {
        const int i = j >> 3, m = m0 + i, c = j & 7;
        if (j < 0 || m >= a.M) continue;
        const int b = a.rows.seq(m), t = m - b * T, row = a.rows.of(t, h), at = (c & 3) * 16 + (row & 15);
        char *tile = a.qop + b * a.q_seq + static_cast<int64_t>(row >> 4) * q4_tile_bytes(NT, RT);
        const QT *qr = static_cast<const QT *>(a.q_rot) + b * a.r_b + (a.t0 + t) * a.r_t + h * a.r_h + c * 8;
        u32x4 f[3] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
        if constexpr (std::is_same<QT, float>::value) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(qr), y = *reinterpret_cast<const f32x4 *>(qr + 4);
            const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            terms8(v, f);
        } else {
            const u32x2 x = *reinterpret_cast<const u32x2 *>(qr), y = *reinterpret_cast<const u32x2 *>(qr + 4);
            f[0] = u32x4{x.x, x.y, y.x, y.y};
        }
#pragma unroll
        for (int x = 0; x < RT; ++x) *reinterpret_cast<u32x4 *>(tile + q4_rope_at(NT, x, c >> 2) + at * 16) = f[x];
    }
}

// ------------------------------------------------------------------ attend
struct AttendArgs {
    const char *qop;
    int64_t q_seq;
    const uint8_t *packed, *scales, *rot;
    int64_t p_b, p_t, s_b, s_t, r_b, r_t;       // bytes
    const int32_t *lengths, *counts;            // [B] or null
    int length, cap, count;                     // where those are null
    const int4 *slot;                           // the list of ranges, or null
    float *part;                                // [slots][rows][512]
    float2 *ml;                                 // [slots][rows]
    Rows order;
    int t0, rows, Ts, NS, rblocks, B;           // rows: order.count()
    uint32_t inverse_rblocks, inverse_ns;
    float c;                                    // scale * log2(e)
    int swizzle;
};

constexpr int kRound = 64;                      // positions per round: four tiles of 16
constexpr int kKLd = 272;                       // LDS bytes of a staged row of codes: 256 + 16 scale bytes
constexpr int kRLd = 144;                       // .. of a rotary row: 128 + 16
constexpr int kKBytes = kRound * kKLd, kRBytes = kRound * kRLd, kTBytes = kRound * 32;
constexpr int kCLd = 132;                       // floats of a context row on its way out: 128 + 4

// RG: groups of 16 rows.  1, 2: 4 / RG score waves to a group, which tell each other their tiles' maxima through LDS and a
// barrier, so a round's probabilities are formed one iteration after its scores (kLag 2); 4: a wave to a group, in the same one.
constexpr int attend_lag(int RG) { return RG == 4 ? 1 : 2; }
constexpr int attend_lds(int RG, int RT, int PT) {   // PT fp16 terms of the probabilities (bf16: one more)
    const int slots = attend_lag(RG) + 2;
    return slots * (kKBytes + kTBytes) + 2 * kRBytes + 2 * RG * (PT + 1) * 2048 + RG * RT * 2048;
}

// NT latent and RT rotary terms of the queries, PT fp16 terms of the probabilities
template <int RG, int NT, int RT, int PT>
__global__ __launch_bounds__(512, 1) void attend_kernel(AttendArgs a) {
    constexpr int TG = 4 / RG, NTILE = RG;       // score waves of a row group; tiles of 16 positions per score wave
    constexpr int kLag = attend_lag(RG), kSlots = kLag + 2;
    constexpr int kPLd = (PT + 1) * 2048;        // LDS bytes of a row group's probabilities
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float xm[2][TG][RG * 16];         // tile maxima [parity][score wave of the group][row]
    __shared__ float xf[2][RG * 16];             // rescale factors [parity][row]
    __shared__ float xl[TG][RG * 16];
    __shared__ int wide;                         // a staged scale byte needs bf16's range
    char *const kbuf = lds, *const tbuf = kbuf + kSlots * kKBytes, *const rbuf = tbuf + kSlots * kTBytes;
    char *const pbuf = rbuf + 2 * kRBytes, *const qbuf = pbuf + 2 * RG * kPLd;   // qbuf: the queries' rotary operands
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, q4 = lane >> 4;
    const int nb = gridDim.x;
    const int w = a.swizzle ? (blockIdx.x & 7) * (nb >> 3) + (blockIdx.x >> 3) : blockIdx.x;
    const int slot = quotient(w, a.inverse_rblocks);
    int rb = w - slot * a.rblocks;
    int4 range;                                 // sequence, first position, last + 1, length
    if (a.slot) {
        const int4 r = a.slot[slot];
        range = make_int4(__builtin_amdgcn_readfirstlane(r.x), __builtin_amdgcn_readfirstlane(r.y), __builtin_amdgcn_readfirstlane(r.z),
                          __builtin_amdgcn_readfirstlane(r.w));
        if (range.x < 0) return;
    } else {
        range.x = quotient(slot, a.inverse_ns), range.y = (slot - range.x * a.NS) * a.Ts, range.z = range.y + a.Ts;
        range.w = a.lengths ? min(max(a.lengths[range.x], 0), a.cap) : a.length;
    }
    const int b = range.x, len = range.w;
    // whole blocks of one head: the last queries, which see most, first
    if (a.order.Tp && a.order.Tp % (16 * RG) == 0) rb = rb % a.order.H * (a.order.Tp / (16 * RG)) + (a.order.Tp / (16 * RG) - 1 - rb / a.order.H);
    const int row0 = rb * 16 * RG;
    const int cnt = a.counts ? min(max(a.counts[b], 0), a.count) : a.count;
    // the last query of the block that is there sees most
    const int tlast = min(a.t0 + a.order.last_query(row0, min(row0 + 16 * RG, a.rows) - 1), cnt - 1);
    const int most = tlast >= a.t0 ? q4_sees(tlast, cnt, len) : 0;
    const int t_begin = range.y, t_end = min(most, range.z);
    float2 *ml = a.ml + static_cast<int64_t>(slot) * a.rows;
    if (t_end <= t_begin) {
        if (tid < 16 * RG && row0 + tid < a.rows) ml[row0 + tid] = make_float2(-INFINITY, 0.f);
        return;
    }
    const int n = t_end - t_begin, nr = (n + kRound - 1) / kRound;

    // ---- staging, by the context waves: a thread takes four groups of codes (positions st / 16 and every 16th from there), two
    // 16-byte rotary chunks (st / 8 and 32 more) and four scale bytes (st / 4)
    const uint8_t *const kp = a.packed + b * a.p_b + t_begin * a.p_t, *const sp = a.scales + b * a.s_b + t_begin * a.s_t;
    const uint8_t *const op = a.rot + b * a.r_b + t_begin * a.r_t;
    const int st = tid & 255, srow = st >> 4, sgrp = st & 15, orow = st >> 3, ochunk = st & 7, brow = st >> 2, bquad = st & 3;
    struct Stage {
        u32x4 k[4], o[2];
        uint32_t s;
    };
    // The next round to load: its rows' addresses and the bytes there are from them on (rows past the last are outside and load
    // zeros), moved on by a round's rows.
    struct Next {
        const uint8_t *k, *o, *s;
        int kb, ob, sb;
    } nx;
    const int64_t kstep = kRound * a.p_t, ostep = kRound * a.r_t, sstep = kRound * a.s_t;
    const uint32_t ko = static_cast<uint32_t>(srow) * static_cast<uint32_t>(a.p_t) + sgrp * 16u, k16 = 16u * static_cast<uint32_t>(a.p_t);
    const uint32_t oo = static_cast<uint32_t>(orow) * static_cast<uint32_t>(a.r_t) + ochunk * 16u, o32 = 32u * static_cast<uint32_t>(a.r_t);
    const uint32_t so = static_cast<uint32_t>(brow) * static_cast<uint32_t>(a.s_t) + bquad * 4u;
    auto rewind = [&]() __attribute__((always_inline)) {
        nx = Next{kp, op, sp, static_cast<int>((n - 1) * a.p_t + 256), static_cast<int>((n - 1) * a.r_t + 128), static_cast<int>((n - 1) * a.s_t + 16)};
    };
    auto load = [&](Stage &g) __attribute__((always_inline)) {
        const auto rk = make_rsrc(nx.k, static_cast<uint32_t>(nx.kb)), ro = make_rsrc(nx.o, static_cast<uint32_t>(nx.ob));
#pragma unroll
        for (int u = 0; u < 4; ++u) g.k[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, ko + u * k16, 0, 0));
#pragma unroll
        for (int u = 0; u < 2; ++u) g.o[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(ro, oo + u * o32, 0, 0));
        g.s = buf_load4(make_rsrc(nx.s, static_cast<uint32_t>(nx.sb)), so);
        nx.k += kstep, nx.o += ostep, nx.s += sstep;
        nx.kb = max(nx.kb - static_cast<int>(kstep), 0), nx.ob = max(nx.ob - static_cast<int>(ostep), 0), nx.sb = max(nx.sb - static_cast<int>(sstep), 0);
    };
    auto store = [&](const Stage &g, int rd) __attribute__((always_inline)) {
        char *k = kbuf + rd % kSlots * kKBytes, *o = rbuf + (rd & 1) * kRBytes + orow * kRLd + ochunk * 16;
#pragma unroll
        for (int u = 0; u < 4; ++u) *reinterpret_cast<u32x4 *>(k + (16 * u + srow) * kKLd + sgrp * 16) = g.k[u];
#pragma unroll
        for (int u = 0; u < 2; ++u) *reinterpret_cast<u32x4 *>(o + 32 * u * kRLd) = g.o[u];
        *reinterpret_cast<uint32_t *>(k + brow * kKLd + 256 + bquad * 4) = g.s;
    };
    // Of round rd's scale bytes a second form, by the score waves: 2^(byte - 127) in 16 bits, [group][position], for the context
    // waves (a NaN's is zero).
    auto scales = [&](int rd, auto bf) __attribute__((always_inline)) {
        const uint32_t four = *reinterpret_cast<const uint32_t *>(kbuf + rd % kSlots * kKBytes + brow * kKLd + 256 + bquad * 4);
        char *t = tbuf + rd % kSlots * kTBytes + bquad * 4 * (2 * kRound) + 2 * brow;
        bool out = false;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const uint32_t e = (four >> (8 * x)) & 255u;
            uint32_t h;
            if constexpr (decltype(bf)::value) {
                h = e == 255u ? 0u : e == 0u ? 64u : e << 7;          // bf16; 2^-127 is a subnormal
            } else {
                const bool in = e - kHalfLow <= kHalfHigh - kHalfLow;
                h = in ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(__uint_as_float(e << 23))) : 0u;
                out = out || !(in || e == 255u);
            }
            *reinterpret_cast<uint16_t *>(t + x * (2 * kRound)) = static_cast<uint16_t>(h);
        }
        if (out && rd * kRound + brow < n) wide = 1;
    };
    if (tid == 0) wide = 0;
    // Iterations 0 .. nr - 1 + kLag, a multiple of kAhead (rounds past the last are zeros that no row sees).  A round is loaded kAhead
    // iterations before it is stored (four measured no better than two; 64 rows leave the registers for one).
    constexpr int kAhead = RG == 4 ? 1 : 2;
    const int iters = (nr + kLag + kAhead - 1) / kAhead * kAhead;
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    if (wave < 4) {
        // ================= score waves
        const int rg = wave % RG, tg = wave / RG;
        const char *tile = a.qop + b * a.q_seq + static_cast<int64_t>((row0 >> 4) + rg) * q4_tile_bytes(NT, RT);
        // (the rotary operands first: they go to LDS before the first barrier, which need not wait for the others)
        u32x4 qo[2 * RT];
#pragma unroll
        for (int x = 0; x < 2 * RT; ++x) qo[x] = *reinterpret_cast<const u32x4 *>(tile + q4_rope_at(NT, 0, x) + lane * 16);
        __builtin_amdgcn_sched_barrier(0);
        u32x4 qlo[NT][kQ4Steps];
        u32x2 qhi[NT][kQ4Steps];
        int qs[NT];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            qs[x] = *reinterpret_cast<const int *>(tile + q4_scale_at(NT, x) + lane * 4);
#pragma unroll
            for (int k = 0; k < kQ4Steps; ++k) {
                qlo[x][k] = *reinterpret_cast<const u32x4 *>(tile + q4_code_at(x, k) + lane * 16);
                qhi[x][k] = *reinterpret_cast<const u32x2 *>(tile + q4_code_at(x, k) + 1024 + lane * 8);
            }
        }
        // (the score waves of a row group write the same)
        char *const qr = qbuf + rg * RT * 2048 + lane * 16;
#pragma unroll
        for (int x = 0; x < 2 * RT; ++x) *reinterpret_cast<u32x4 *>(qr + x * 1024) = qo[x];
        const int row = row0 + rg * 16 + r16;
        const int tq = a.order.query(row), sees = row < a.rows && tq < a.order.T ? q4_sees(a.t0 + tq, cnt, len) : 0;
        const int limit = min(sees, t_end) - t_begin;       // positions of this split that the row sees
        float m_ref, l_run, mt[2];
        f32x4 sc[kLag][NTILE];                              // scaled scores of round i (log2 units; hidden: -infinity)

        // round rd's scores; their maximum over the wave's tiles
        auto scores = [&](int rd, f32x4 (&out)[NTILE]) __attribute__((always_inline)) {
            float top = -INFINITY;
            struct Keys {
                u32x4 c[kQ4Steps], o[2];
                int scale;
            } keys[2];                                      // a tile's are read while the one's before are multiplied
            auto read = [&](int u, Keys &t) __attribute__((always_inline)) {
                const int at = (tg * NTILE + u) * 16;
                const char *k = kbuf + rd % kSlots * kKBytes + (at + r16) * kKLd, *o = rbuf + (rd & 1) * kRBytes + (at + r16) * kRLd + q4 * 16;
#pragma unroll
                for (int x = 0; x < 2; ++x) t.o[x] = *reinterpret_cast<const u32x4 *>(o + x * 64);
                t.scale = *reinterpret_cast<const int *>(k + 256 + q4 * 4);
#pragma unroll
                for (int s = 0; s < kQ4Steps; ++s) t.c[s] = *reinterpret_cast<const u32x4 *>(k + q4 * 64 + s * 16);
            };
            read(0, keys[0]);
#pragma unroll
            for (int u = 0; u < NTILE; ++u) {
                const int at = (tg * NTILE + u) * 16;
                const Keys &t = keys[u & 1];
                if (u + 1 < NTILE) read(u + 1, keys[(u + 1) & 1]);
                f32x4 d[4];                                 // the terms in chains of their own
#pragma unroll
                for (int x = 0; x < 4; ++x) d[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int x = RT - 1; x >= 0; --x)
                        d[3] = q4_mfma_bf16(t.o[s], *reinterpret_cast<const u32x4 *>(qr + (2 * x + s) * 1024), d[3]);
#pragma unroll
                for (int x = NT - 1; x >= 0; --x) {
                    f32x4 &c = d[x < 3 ? x : 3];
                    c = q4_mfma<0>(t.c[0], t.scale, qlo[x][0], qhi[x][0], qs[x], c);
                    c = q4_mfma<1>(t.c[1], t.scale, qlo[x][1], qhi[x][1], qs[x], c);
                    c = q4_mfma<2>(t.c[2], t.scale, qlo[x][2], qhi[x][2], qs[x], c);
                    c = q4_mfma<3>(t.c[3], t.scale, qlo[x][3], qhi[x][3], qs[x], c);
                }
                const f32x4 s = d[0] + ((d[3] + d[2]) + d[1]);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    out[u][v] = rd * kRound + at + 4 * q4 + v < limit ? s[v] * a.c : -INFINITY;
                    top = fmaxf(top, out[u][v]);
                }
                if (RG == 4 || NT == 5) __builtin_amdgcn_sched_barrier(0);   // (the next tile's operands are more than the registers hold)
            }
            return q4_rows_max(top);
        };
        // round rd's probabilities, lifted by kLift over the row's reference, with the maximum mt over all of the round's tiles
        auto probs = [&](int rd, const f32x4 (&s)[NTILE], float mt, auto bf) __attribute__((always_inline)) {
            float f = 1.f;
            if (mt > m_ref + kSlack || (m_ref == -INFINITY && mt != -INFINITY)) {
                f = m_ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_ref - mt);
                l_run *= f;
                m_ref = mt;
            }
            const float ref = m_ref == -INFINITY ? 0.f : m_ref - kLift;
            // slot [tile][half][row][8 positions]: what lane (row, tile) of the second product takes in its two steps
            char *p = pbuf + ((rd & 1) * RG + rg) * kPLd + ((q4 >> 1) * 16 + r16) * 16 + (q4 & 1) * 8;
#pragma unroll
            for (int u = 0; u < NTILE; ++u) {
                float e[4];
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    e[v] = __builtin_amdgcn_exp2f(s[u][v] - ref);
                    l_run += e[v];
                }
                char *pu = p + (tg * NTILE + u) * 512;
                if constexpr (!decltype(bf)::value) {
#pragma unroll
                    for (int x = 0; x < PT; ++x) {
                        const uint32_t a0 = q4_pack_f16(e[0], e[1]), a1 = q4_pack_f16(e[2], e[3]);
                        *reinterpret_cast<u32x2 *>(pu + x * 2048) = u32x2{a0, a1};
                        if (x + 1 < PT) {
                            const f16x2 h0 = __builtin_bit_cast(f16x2, a0), h1 = __builtin_bit_cast(f16x2, a1);
                            e[0] -= static_cast<float>(h0[0]), e[1] -= static_cast<float>(h0[1]);
                            e[2] -= static_cast<float>(h1[0]), e[3] -= static_cast<float>(h1[1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < PT + 1; ++x) {
                        const uint32_t a0 = q4_pack_bf16(e[0], e[1]), a1 = q4_pack_bf16(e[2], e[3]);
                        *reinterpret_cast<u32x2 *>(pu + x * 2048) = u32x2{a0, a1};
                        e[0] -= q4_lo(a0), e[1] -= q4_hi(a0), e[2] -= q4_lo(a1), e[3] -= q4_hi(a1);
                    }
                }
            }
            if (tg == 0 && q4 == 0) xf[rd & 1][rg * 16 + r16] = f;
        };
        auto all = [&](auto bf) __attribute__((always_inline)) {
            m_ref = -INFINITY, l_run = 0.f;
            // the context waves' first kLag iterations, before there is a round for them, take zero scales and zero probabilities (a
            // branch around the products would cost a copy of the accumulators)
            for (int i = tid * 16; i < 2 * RG * kPLd; i += 256 * 16) *reinterpret_cast<u32x4 *>(pbuf + i) = u32x4{0u, 0u, 0u, 0u};
            for (int i = tid * 16; i < kLag * kTBytes; i += 256 * 16) *reinterpret_cast<u32x4 *>(tbuf + (kSlots - kLag) * kTBytes + i) = u32x4{0u, 0u, 0u, 0u};
            if (tid < 2 * RG * 16) xf[tid / (RG * 16)][tid % (RG * 16)] = 1.f;
            __syncthreads();        // all this and wide are set; every wave is done with a first pass
            __syncthreads();        // round 0 is staged
            auto part = [&](int i, auto par) __attribute__((always_inline)) {
                constexpr int d = decltype(par)::value;
                if constexpr (kLag == 1) {
                    mt[0] = scores(i, sc[0]);
                    probs(i, sc[0], mt[0], bf);
                } else {
                    mt[d] = scores(i, sc[d]);
                    if (q4 == 0) xm[i & 1][tg][rg * 16 + r16] = mt[d];
                    if (i > 0) {
                        float m = xm[(i - 1) & 1][0][rg * 16 + r16];
#pragma unroll
                        for (int x = 1; x < TG; ++x) m = fmaxf(m, xm[(i - 1) & 1][x][rg * 16 + r16]);
                        probs(i - 1, sc[kLag - 1 - d], m, bf);
                    }
                }
                scales(i, bf);
                __syncthreads();
            };
            if constexpr (kLag == 1) {
                for (int i = 0; i < iters; ++i) part(i, even);
            } else {
                for (int i = 0; i < iters; i += 2) {
                    part(i, even);
                    part(i + 1, odd);
                }
            }
        };
        all(std::false_type{});
        if (__builtin_amdgcn_readfirstlane(wide)) all(std::true_type{});
        const float l = q4_rows_sum(l_run);
        if (q4 == 0) xl[tg][rg * 16 + r16] = l;
        __syncthreads();
        if (tg == 0 && q4 == 0 && row < a.rows) {
            float sum = xl[0][rg * 16 + r16];
#pragma unroll
            for (int x = 1; x < TG; ++x) sum += xl[x][rg * 16 + r16];
            ml[row] = make_float2(m_ref, sum);
        }
    } else {
        // ================= context waves: columns 128 (wave - 4) .. +128
        const int col0 = (wave - 4) * 128;
        f32x4 acc[8][RG];
        auto context = [&](int rd, auto bf, auto stage) __attribute__((always_inline)) {
            constexpr bool kBf = decltype(bf)::value;
            constexpr int N = PT + kBf;
            // lane (column r16, positions 16 q4 .. +16): the codes of a tile of 16 columns, transposed, as they lie in the rows
            const int slot = (rd + kSlots) % kSlots;
            const char *k = kbuf + slot * kKBytes + (16 * q4 + r16) * kKLd + col0 / 2;
            const char *t = tbuf + slot * kTBytes + (col0 / 32) * (2 * kRound) + 32 * q4;
            const char *p = pbuf + (rd & 1) * RG * kPLd + (q4 * 32 + r16) * 16;
            u32x2 code[8];
#pragma unroll
            for (int c = 0; c < 8; ++c)
                code[c] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i2)(k + c * 8)));
            float f[RG];
#pragma unroll
            for (int r = 0; r < RG; ++r) f[r] = xf[rd & 1][r * 16 + r16];
            // 8 of the lane's 16 positions a step: their probabilities, and a scale for every 32 columns.  With up to 32 rows all of them
            // are read before the next round is stored (the stores would hold them up: 19.9 us for 18.6 over 32,768 positions).
            constexpr bool kFirst = RG <= 2;
            u32x4 pf[kFirst ? 2 : 1][RG][N], h[kFirst ? 2 : 1][4];
            auto probabilities = [&](int s) __attribute__((always_inline)) {
#pragma unroll
                for (int r = 0; r < RG; ++r)
#pragma unroll
                    for (int x = 0; x < N; ++x) pf[kFirst ? s : 0][r][x] = *reinterpret_cast<const u32x4 *>(p + r * kPLd + x * 2048 + s * 256);
            };
            auto scale = [&](int s, int g) __attribute__((always_inline)) { h[kFirst ? s : 0][g] = *reinterpret_cast<const u32x4 *>(t + g * (2 * kRound) + s * 16); };
            if (kFirst) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    probabilities(s);
#pragma unroll
                    for (int g = 0; g < 4; ++g) scale(s, g);
                }
            }
            stage();
            bool any = false;
#pragma unroll
            for (int r = 0; r < RG; ++r) any = any || f[r] != 1.f;
            if (__any(any)) {
#pragma unroll
                for (int c = 0; c < 8; ++c)
#pragma unroll
                    for (int r = 0; r < RG; ++r) acc[c][r] *= f[r];
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int b = kFirst ? s : 0;
                if (!kFirst) probabilities(s);
#pragma unroll
                for (int g = 0; g < 4; ++g) {               // 32 columns
                    if (!kFirst) scale(s, g);
#pragma unroll
                    for (int c = 2 * g; c < 2 * g + 2; ++c) {
                        const u32x4 v = kBf ? q4_values_bf16(code[c][s], h[b][g]) : q4_values_f16(code[c][s], h[b][g]);
#pragma unroll
                        for (int x = N - 1; x >= 0; --x)
#pragma unroll
                            for (int r = 0; r < RG; ++r) acc[c][r] = kBf ? q4_mfma_bf16(v, pf[b][r][x], acc[c][r]) : q4_mfma_f16(v, pf[b][r][x], acc[c][r]);
                    }
                    if (RG == 4) __builtin_amdgcn_sched_barrier(0);
                }
            }
        };
        auto all = [&](auto bf) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int r = 0; r < RG; ++r) acc[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
            Stage g[kAhead];
            rewind();
#pragma unroll
            for (int d = 0; d < kAhead; ++d) load(g[d]);
            __syncthreads();
            store(g[0], 0);
            load(g[0]);
            __syncthreads();
            for (int i = 0; i < iters; i += kAhead) {
#pragma unroll
                for (int d = 0; d < kAhead; ++d) {
                    context(i + d - kLag, bf, [&]() __attribute__((always_inline)) {
                        store(g[(d + 1) % kAhead], i + d + 1);
                        load(g[(d + 1) % kAhead]);
                    });
                    __syncthreads();
                }
            }
        };
        all(std::false_type{});
        if (__builtin_amdgcn_readfirstlane(wide)) all(std::true_type{});
        __syncthreads();
        // the records through LDS (the codes are done with), so that a store writes 512 contiguous bytes of two rows: as the
        // accumulators lie, 64 bytes of sixteen rows, the 256 blocks of a short split took 7 us to write them
        float *part = a.part + (static_cast<int64_t>(slot) * a.rows + row0) * kQ4Lat + col0;
        float *const x = reinterpret_cast<float *>(kbuf) + (wave - 4) * 16 * kCLd;
        static_assert(4 * 16 * kCLd * 4 <= kSlots * kKBytes, "the contexts' way out fits the code tiles");
#pragma unroll
        for (int r = 0; r < RG; ++r) {
#pragma unroll
            for (int c = 0; c < 8; ++c) *reinterpret_cast<f32x4 *>(x + r16 * kCLd + c * 16 + 4 * q4) = acc[c][r];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = 2 * i + (lane >> 5);
                const f32x4 v = *reinterpret_cast<const f32x4 *>(x + j * kCLd + (lane & 31) * 4);
                if (row0 + r * 16 + j < a.rows) *reinterpret_cast<f32x4 *>(part + static_cast<int64_t>(r * 16 + j) * kQ4Lat + (lane & 31) * 4) = v;
            }
        }
    }
}

// ------------------------------------------------------------------ uv
struct UvArgs {
    const float *part;
    const float2 *ml;
    const uint16_t *w_uv;    // [H, V, 512]
    void *out;               // [B, Tall, H, V]
    int out_bf16;
    const float *gate;       // [B, Tall, H, V] or null
    float *stats;            // [B][rows]: log2 of what a probability's exponential is divided by; or null
    const int2 *seq;         // the sequences' records, or null: NS each
    const int32_t *lengths, *counts;    // [B] or null: length, and Tall
    Rows order;
    int M, V, rows, NS, Tall, t0, length;
    __device__ __forceinline__ int2 records(int b) const { return seq ? seq[b] : make_int2(b * NS, NS); }  // first, number (at most NS)
};
constexpr int kMaxSplits = 256;

__device__ __forceinline__ void store_out4(const UvArgs &a, int m, int h, int v, f32x4 o) {
    const int b = a.order.seq(m), tq = a.t0 + a.order.token(m);
    const int64_t at = ((static_cast<int64_t>(b) * a.Tall + tq) * a.order.H + h) * a.V + v;
    if (a.gate) {
        const f32x4 g = *reinterpret_cast<const f32x4 *>(a.gate + at);
        // (the gate of a query that sees nothing may be anything: a row of padding's)
        const bool any = q4_sees(tq, a.counts ? min(a.counts[b], a.Tall) : a.Tall, a.lengths ? min(a.lengths[b], a.length) : a.length) > 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = any ? o[i] / (1.0f + expf(-g[i])) : 0.f;
    }
    if (a.out_bf16)
        *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + at) = u32x2{q4_pack_bf16(o[0], o[1]), q4_pack_bf16(o[2], o[3])};
    else
        *reinterpret_cast<f32x4 *>(static_cast<float *>(a.out) + at) = o;
}

// The weights of a row's records, 2^(m_s - M) / L with M = max m_s, L = sum 2^(m_s - M) l_s, by a wave, record 64 u + lane in
// w[u]; a split the row sees nothing of has no record (its sum is exactly 0), and its weight is zero whatever the others are.
__device__ __forceinline__ void record_weights(const UvArgs &a, int b, int row, int2 there, bool stats, float (&w)[kMaxSplits / 64]) {
    const int lane = threadIdx.x & 63;
    const float2 *ml = a.ml + static_cast<int64_t>(there.x) * a.rows + row;
    float2 v[kMaxSplits / 64];
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kMaxSplits / 64; ++u) {
        const int s = lane + 64 * u;
        v[u] = s < there.y ? ml[static_cast<int64_t>(s) * a.rows] : make_float2(-INFINITY, 0.f);
        mx = fmaxf(mx, v[u].x);
    }
    mx = wave_max_all(mx);
    float l = 0.f;
#pragma unroll
    for (int u = 0; u < kMaxSplits / 64; ++u) {
        w[u] = v[u].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(v[u].x - mx);
        l = fmaf(w[u], v[u].y, l);
    }
    l = wave_sum_all(l);
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int u = 0; u < kMaxSplits / 64; ++u) w[u] = v[u].y == 0.f ? 0.f : w[u] * inv;
    // (the sum is lifted by kLift; a row that sees nothing has no probabilities)
    if (stats && a.stats && lane == 0) a.stats[static_cast<int64_t>(b) * a.rows + row] = l == 0.f ? 0.f : mx - kLift + __log2f(l);
}

// Few queries: grid (H, ceil(M / per), Z), WAVES waves, queries per y .. +per (at most 16) of head x, VT tiles of 16 output columns
// (z).  Two waves join a query's records, 256 columns each, four to a lane (with fewer queries than pairs of waves, 2, 4 or 8 pairs
// every 2nd, 4th, 8th record); then a wave multiplies 512 / WAVES columns of all queries with its columns of W_UV (loaded
// first of all), and the waves' products are added in order.  Bound by the latency of the records (NS x 2 KB a query) and of W_UV,
// 128 KB a head.  (A wave that joined its columns of every query, eight records side by side in its lanes, spent more on adding up the
// lanes than on the records: 17 us for 32 queries of 64 heads with 1 to 43 records each, this: 13.)
//   many records: 16 waves have 128 KB of them on the way
//   up to kFewSplits: 8 waves with half of the output columns each (6 records of 96 heads: 6.1 us; 16 waves, all columns: 10.0)
constexpr int kXLd = kQ4Lat + 4, kDLd = 132;        // floats of a context row (512), of a product row (128)
constexpr int kFewSplits = 8;
constexpr int kFewLds = (16 * kXLd + 8 * 16 * kDLd) * 4;

template <int WAVES, int VT>
__global__ __launch_bounds__(64 * WAVES, 1) void uv_few_kernel(UvArgs a, int per) {
    constexpr int kCols = 512 / WAVES, kSteps = kCols / 32, kPairs = WAVES / 2;
    extern __shared__ __attribute__((aligned(16))) float sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, q4 = lane >> 4;
    float *const x = sm, *const d = sm + 16 * kXLd;
    const int h = blockIdx.x, m0 = blockIdx.y * per, col0 = wave * kCols, nv = min(per, a.M - m0);
    const auto rw = make_rsrc(a.w_uv + static_cast<int64_t>(h) * a.V * kQ4Lat, static_cast<uint32_t>(a.V) * (2 * kQ4Lat));
    auto weights_of = [&](int v0, u32x4 (&w)[VT][kSteps]) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < VT; ++t) {
            // (rows past the head's last are outside and load zeros)
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
                w[t][k] = __builtin_bit_cast(u32x4, buf_load16(rw, static_cast<uint32_t>(v0 + t * 16 + r16) * (2 * kQ4Lat) + 2 * (col0 + 8 * q4 + 32 * k)));
        }
    };
    u32x4 w[VT][kSteps];
    const int vz = blockIdx.z * 16 * VT;
    weights_of(vz, w);
    int pairs = 1;                          // of a query
    while (2 * pairs * nv <= kPairs) pairs *= 2;
    const int g = (wave >> 1) & (pairs - 1);
    constexpr int kBatch = 8;
    for (int i = (wave >> 1) / pairs; i < nv; i += kPairs / pairs) {
        const int m = m0 + i, b = a.order.seq(m), row = a.order.of(m - b * a.order.T, h);
        int2 there = a.records(b);
        there.x = __builtin_amdgcn_readfirstlane(there.x), there.y = __builtin_amdgcn_readfirstlane(there.y);
        const int n = there.y;
        const int64_t pitch = static_cast<int64_t>(a.rows) * kQ4Lat;
        const float *src = a.part + there.x * pitch + row * kQ4Lat + (wave & 1) * 256 + lane * 4;
        f32x4 y[kBatch];
        auto load = [&](int k) __attribute__((always_inline)) {     // (written or not: where not, the weight is zero)
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (k + pairs * u >= n) break;
                y[u] = *reinterpret_cast<const f32x4 *>(src + (k + pairs * u) * pitch);
            }
        };
        load(g);
        float f[kMaxSplits / 64];
        record_weights(a, b, row, there, g == 0 && (wave & 1) == 0, f);
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        for (int k = g; k < n; k += pairs * kBatch) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int c = k + pairs * u;
                if (c >= n) break;
                const float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(c < 64 ? f[0] : c < 128 ? f[1] : c < 192 ? f[2] : f[3]), c & 63));
                if (v != 0.f) s += y[u] * v;
            }
            if (k + pairs * kBatch < n) load(k + pairs * kBatch);
        }
        *reinterpret_cast<f32x4 *>(x + (i * pairs + g) * kXLd + (wave & 1) * 256 + lane * 4) = s;
    }
    __syncthreads();
    u32x4 cf[kSteps][3];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        f32x4 u = {0.f, 0.f, 0.f, 0.f}, z = u;
        if (r16 < nv) {
            const float *xr = x + r16 * pairs * kXLd + col0 + 32 * k + 8 * q4;
            for (int c = 0; c < pairs; ++c) u += *reinterpret_cast<const f32x4 *>(xr + c * kXLd), z += *reinterpret_cast<const f32x4 *>(xr + c * kXLd + 4);
        }
        const float v[8] = {u[0], u[1], u[2], u[3], z[0], z[1], z[2], z[3]};
        terms8(v, cf[k]);
    }
    float *const dw = d + ((wave & 7) * 16 + r16) * kDLd + 4 * q4;
    for (int v0 = vz; v0 < a.V; v0 += 16 * VT * gridDim.z) {
        if (v0 != vz) {
            weights_of(v0, w);
            __syncthreads();                // the last products are added up
        }
        f32x4 o[VT];
#pragma unroll
        for (int t = 0; t < VT; ++t) {
            o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 2; k >= 0; --k)
#pragma unroll
                for (int c = 0; c < kSteps; ++c) o[t] = q4_mfma_bf16(w[t][c], cf[c][k], o[t]);
        }
        if (WAVES == 16) {
            if (wave >= 8) {
#pragma unroll
                for (int t = 0; t < VT; ++t) *reinterpret_cast<f32x4 *>(dw + t * 16) = o[t];
            }
            __syncthreads();
            if (wave < 8) {
#pragma unroll
                for (int t = 0; t < VT; ++t) *reinterpret_cast<f32x4 *>(dw + t * 16) = o[t] + *reinterpret_cast<const f32x4 *>(dw + t * 16);
            }
        } else {
#pragma unroll
            for (int t = 0; t < VT; ++t) *reinterpret_cast<f32x4 *>(dw + t * 16) = o[t];
        }
        __syncthreads();
        for (int j = tid; j < 16 * 4 * VT; j += 64 * WAVES) {
            const int i = j / (4 * VT), v = j % (4 * VT) * 4;
            if (i < nv && v0 + v < a.V) {
                f32x4 t = *reinterpret_cast<const f32x4 *>(d + i * kDLd + v);
#pragma unroll
                for (int u = 1; u < 8; ++u) t += *reinterpret_cast<const f32x4 *>(d + (u * 16 + i) * kDLd + v);
                store_out4(a, m0 + i, h, v0 + v, t);
            }
        }
    }
}

// Many queries: grid (H, ceil(M / 64)), four waves, queries 64 y .. +64 of head x, 128 latent columns at a time: a thread joins
// the records of 4 columns of 8 queries and leaves them in LDS as TERMS bf16 terms (two, 2^-17, for a bf16 result); a wave
// takes 32 of 128 output columns for all 64 queries.  Bound by reading the records.  (Not with a list of ranges.)
template <int TERMS>
__global__ __launch_bounds__(256, 2) void uv_many_kernel(UvArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int kLd = 272, kTerm = 64 * kLd;      // bytes: 128 columns + 16
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, q4 = lane >> 4;
    float *const wsp = reinterpret_cast<float *>(lds + TERMS * kTerm);
    const int h = blockIdx.x, m0 = blockIdx.y * 64, nv = min(64, a.M - m0);
    {
        // The records' weights (as record_weights) of all 64 queries at once, four lanes each: a wave a query waited for sixteen loads one
        // after the other, 18 of the launch's 52 us at 1000 queries of 64 heads.
        const int i = tid >> 2, part = tid & 3, m = m0 + min(i, nv - 1), b = a.order.seq(m), row = a.order.of(m - b * a.order.T, h);
        const float2 *ml = a.ml + static_cast<int64_t>(b) * a.NS * a.rows + row;
        float mx = -INFINITY, l = 0.f;
        for (int s = part; s < a.NS; s += 4) mx = fmaxf(mx, ml[static_cast<int64_t>(s) * a.rows].x);
        mx = fmaxf(mx, __shfl_xor(mx, 1));
        mx = fmaxf(mx, __shfl_xor(mx, 2));
        for (int s = part; s < a.NS; s += 4) {
            const float2 v = ml[static_cast<int64_t>(s) * a.rows];
            const float w = v.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(v.x - mx);
            wsp[i * a.NS + s] = w;
            l = fmaf(w, v.y, l);
        }
        l += __shfl_xor(l, 1);
        l += __shfl_xor(l, 2);
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        for (int s = part; s < a.NS; s += 4) wsp[i * a.NS + s] = wsp[i * a.NS + s] == 0.f ? 0.f : wsp[i * a.NS + s] * inv;
        if (a.stats && part == 0 && i < nv) a.stats[static_cast<int64_t>(b) * a.rows + row] = l == 0.f ? 0.f : mx - kLift + __log2f(l);
    }
    __syncthreads();
    const uint32_t pitch = static_cast<uint32_t>(a.rows) * kQ4Lat;
    const auto rw = make_rsrc(a.w_uv + static_cast<int64_t>(h) * a.V * kQ4Lat, static_cast<uint32_t>(a.V) * (2 * kQ4Lat));
    const int c4 = tid & 31, i8 = tid >> 5;
    uint32_t at[8];     // (a pass has fewer than 1.5 x 2^16 rows, and more than one record a row for 2^14 of them or 2^20 positions: 2^30 floats)
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int m = m0 + min(8 * u + i8, nv - 1);
        at[u] = static_cast<uint32_t>(a.order.seq(m) * a.NS) * pitch + static_cast<uint32_t>(a.order.of(a.order.token(m), h) * kQ4Lat + 4 * c4);
    }
    for (int v0 = 0; v0 < a.V; v0 += 128) {
        f32x4 acc[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[t][r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int col0 = 0; col0 < kQ4Lat; col0 += 128) {
            u32x4 w[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int k = 0; k < 4; ++k)         // (rows past the head's last are outside and load zeros)
                    w[t][k] = __builtin_bit_cast(u32x4, buf_load16(rw, static_cast<uint32_t>(v0 + (2 * wave + t) * 16 + r16) * (2 * kQ4Lat) +
                                                                           2 * (col0 + 8 * q4 + 32 * k)));
            }
            f32x4 s[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int k = 0; k < a.NS; ++k) {
                // (in bounds, whether the record was written or not: its weight is zero where it was not)
                f32x4 y[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) y[u] = *reinterpret_cast<const f32x4 *>(a.part + (at[u] + k * pitch + col0));
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int i = 8 * u + i8;
                    const float f = i < nv ? wsp[i * a.NS + k] : 0.f;
                    if (f == 0.f) y[u] = f32x4{0.f, 0.f, 0.f, 0.f};
                    s[u] += f * y[u];
                }
            }
            __syncthreads();    // the last columns' operands are read
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int y = 0; y < TERMS; ++y) {
                    const u32x2 p = {q4_pack_bf16(s[u][0], s[u][1]), q4_pack_bf16(s[u][2], s[u][3])};
                    *reinterpret_cast<u32x2 *>(lds + y * kTerm + (8 * u + i8) * kLd + c4 * 8) = p;
                    s[u] -= f32x4{q4_lo(p.x), q4_hi(p.x), q4_lo(p.y), q4_hi(p.y)};
                }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int y = TERMS - 1; y >= 0; --y)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const u32x4 c = *reinterpret_cast<const u32x4 *>(lds + y * kTerm + (16 * r + r16) * kLd + k * 64 + q4 * 16);
#pragma unroll
                        for (int t = 0; t < 2; ++t) acc[t][r] = q4_mfma_bf16(w[t][k], c, acc[t][r]);
                    }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int i = 16 * r + r16, v = v0 + (2 * wave + t) * 16 + 4 * q4;
                if (i < nv && v < a.V) store_out4(a, m0 + i, h, v, acc[t][r]);
            }
    }
}

// ------------------------------------------------------------------ weights
struct WeightArgs {
    AttendArgs a;
    const float *stats;      // [B][rows]
    float *part;             // [chunks][B][pitch]
    float *weight;           // [B] rows of w_b floats
    int64_t w_b;
    int tiles, chunk, chunks;
    int64_t pitch;           // npos in whole blocks
};
constexpr int kWTiles = 4;   // tiles of 16 positions per wave

// grid (ceil(npos / 512), chunks, B): a wave keeps 64 positions' codes in registers; the block takes the row tiles
// chunk y .. of its sequence one after the other, each staged in LDS for its eight waves while the last one is worked on, and adds
// their probabilities, exp2(c s - log2 of the row's divisor); part[chunk][b][position].  One block a CU: 4000 tiles of 1000 queries of 64 heads
// over as many positions take 100 us, 6000 cycles a tile where its products need 2800 (the rest: exponentials, and the products'
// operands from LDS, 34 KB a wave), and the chunks are uneven there: the first 512 positions are seen by all of their 32 tiles, the others by
// half; one tile over 20,001 positions 9 us, most of it the first loads.
template <int NT, int RT>
__global__ __launch_bounds__(512, 1) void weights_kernel(WeightArgs wa) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int kBytes = q4_tile_bytes(NT, RT), kLoads = (kBytes + 8191) / 8192;
    const AttendArgs &a = wa.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, q4 = lane >> 4;
    // the blocks of one chunk on one XCD (blocks b % 8), so that its L2 reads the tiles once
    const int id = blockIdx.y * gridDim.x + blockIdx.x, turn = id / (8 * gridDim.x), place = id % (8 * gridDim.x);
    const bool whole = 8 * (turn + 1) <= static_cast<int>(gridDim.y);
    const int chunk = whole ? 8 * turn + (place & 7) : blockIdx.y, pos = whole ? place >> 3 : blockIdx.x;
    const int b = blockIdx.z, jb = pos * (8 * 16 * kWTiles), j0 = jb + wave * (16 * kWTiles);
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.cap) : a.length;
    const int cnt = a.counts ? min(max(a.counts[b], 0), a.count) : a.count;
    const int n = min(len - j0, 16 * kWTiles);     // positions there are from j0 on
    f32x4 sum[kWTiles];
#pragma unroll
    for (int u = 0; u < kWTiles; ++u) sum[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int last = min(wa.tiles, (chunk + 1) * wa.chunk);
    // positions that the rows of tile i see
    auto seen = [&](int i) __attribute__((always_inline)) {
        const int t = min(a.t0 + a.order.last_query(16 * i, min(16 * i + 16, a.rows) - 1), cnt - 1);
        return t >= a.t0 ? q4_sees(t, cnt, len) : 0;
    };
    auto next = [&](int i) __attribute__((always_inline)) {   // the first tile from i on that sees any of the block's positions
        while (i < last && seen(i) <= jb) ++i;
        return i;
    };
    struct Stage {          // the next tile, loaded before this one's products and stored after them
        u32x4 q[kLoads];
        float st;
    };
    auto load = [&](int i, Stage &g) __attribute__((always_inline)) {
        i = min(i, wa.tiles - 1);
        g.st = wa.stats[static_cast<int64_t>(b) * a.rows + min(i * 16 + r16, a.rows - 1)];
        const char *tile = a.qop + b * a.q_seq + static_cast<int64_t>(i) * kBytes;
#pragma unroll
        for (int u = 0; u < kLoads; ++u)
            g.q[u] = *reinterpret_cast<const u32x4 *>(tile + min(u * 8192 + tid * 16, kBytes - 16));
    };
    auto store = [&](int buf, const Stage &g) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u)
            if (u * 8192 + tid * 16 < kBytes) *reinterpret_cast<u32x4 *>(lds + buf * kBytes + u * 8192 + tid * 16) = g.q[u];
    };
    Stage g;
    int i = next(chunk * wa.chunk);
    load(i, g);
    // The wave's positions.  Their codes come in as whole rows, sixteen lanes a row, and take their lanes' order through LDS (a row
    // quarter to a lane, they took 9.5 us of a launch's 15 for one tile of queries over 20,001 positions), where the second tile will be.
    u32x4 kc[kWTiles][kQ4Steps], ro[kWTiles][2];
    int ks[kWTiles];
    {
        const int64_t there = max(n, 0), first = n > 0 ? j0 : 0;
        const auto rp = make_rsrc(a.packed + b * a.p_b + first * a.p_t, static_cast<uint32_t>(there ? (there - 1) * a.p_t + 256 : 0));
        const auto rs = make_rsrc(a.scales + b * a.s_b + first * a.s_t, static_cast<uint32_t>(there ? (there - 1) * a.s_t + 16 : 0));
        const auto rr = make_rsrc(a.rot + b * a.r_b + first * a.r_t, static_cast<uint32_t>(there ? (there - 1) * a.r_t + 128 : 0));
        const uint32_t pt = static_cast<uint32_t>(a.p_t), rt = static_cast<uint32_t>(a.r_t), st = static_cast<uint32_t>(a.s_t);
#pragma unroll
        for (int u = 0; u < kWTiles; ++u) {         // (rows past the last are outside and load zeros)
#pragma unroll
            for (int s = 0; s < kQ4Steps; ++s)
                kc[u][s] = __builtin_bit_cast(u32x4, buf_load16(rp, static_cast<uint32_t>(u * 16 + 4 * s + q4) * pt + r16 * 16u));
#pragma unroll
            for (int s = 0; s < 2; ++s)
                ro[u][s] = __builtin_bit_cast(u32x4, buf_load16(rr, static_cast<uint32_t>(u * 16 + r16) * rt + s * 64u + q4 * 16u));
            ks[u] = static_cast<int>(buf_load4(rs, static_cast<uint32_t>(u * 16 + r16) * st + q4 * 4u));
        }
        char *const x = lds + kBytes + wave * (16 * kKLd);
#pragma unroll
        for (int u = 0; u < kWTiles; ++u) {
#pragma unroll
            for (int s = 0; s < kQ4Steps; ++s) *reinterpret_cast<u32x4 *>(x + (4 * s + q4) * kKLd + r16 * 16) = kc[u][s];
#pragma unroll
            for (int s = 0; s < kQ4Steps; ++s) kc[u][s] = *reinterpret_cast<const u32x4 *>(x + r16 * kKLd + q4 * 64 + s * 16);
        }
    }
    store(0, g);
    __builtin_amdgcn_s_waitcnt(0x0f70);     // vmcnt(0): all is here (else every tile's first product would wait for the next tile's loads)
    __syncthreads();
    int buf = 0;
    while (i < last) {
        const float st = g.st;
        const int ahead = next(i + 1);
        if (ahead < last) load(ahead, g);
        const char *tile = lds + buf * kBytes + lane * 16;
        if (n > 0 && seen(i) > j0) {
            const int row = i * 16 + r16, tq = a.order.query(row);
            const int limit = (row < a.rows && tq < a.order.T ? q4_sees(a.t0 + tq, cnt, len) : 0) - j0;
            struct Term {
                u32x4 lo[kQ4Steps];
                u32x2 hi[kQ4Steps];
                int scale;
            } q[2];                         // a term's operands are read while the one's before are multiplied
            auto operands = [&](int x, Term &t) __attribute__((always_inline)) {
                t.scale = *reinterpret_cast<const int *>(tile + q4_scale_at(NT, x) - lane * 12);
#pragma unroll
                for (int s = 0; s < kQ4Steps; ++s) {
                    t.lo[s] = *reinterpret_cast<const u32x4 *>(tile + q4_code_at(x, s));
                    t.hi[s] = *reinterpret_cast<const u32x2 *>(tile + q4_code_at(x, s) + 1024 - lane * 8);
                }
            };
            f32x4 d[kWTiles];               // the smallest terms first
#pragma unroll
            for (int u = 0; u < kWTiles; ++u) d[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            operands(NT - 1, q[(NT - 1) & 1]);
#pragma unroll
            for (int x = RT - 1; x >= 0; --x)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const u32x4 qr = *reinterpret_cast<const u32x4 *>(tile + q4_rope_at(NT, x, s));
#pragma unroll
                    for (int u = 0; u < kWTiles; ++u) d[u] = q4_mfma_bf16(ro[u][s], qr, d[u]);
                }
#pragma unroll
            for (int x = NT - 1; x >= 0; --x) {
                if (x > 0) operands(x - 1, q[(x - 1) & 1]);
                const Term &t = q[x & 1];
#pragma unroll
                for (int u = 0; u < kWTiles; ++u) d[u] = q4_mfma<0>(kc[u][0], ks[u], t.lo[0], t.hi[0], t.scale, d[u]);
#pragma unroll
                for (int u = 0; u < kWTiles; ++u) d[u] = q4_mfma<1>(kc[u][1], ks[u], t.lo[1], t.hi[1], t.scale, d[u]);
#pragma unroll
                for (int u = 0; u < kWTiles; ++u) d[u] = q4_mfma<2>(kc[u][2], ks[u], t.lo[2], t.hi[2], t.scale, d[u]);
#pragma unroll
                for (int u = 0; u < kWTiles; ++u) d[u] = q4_mfma<3>(kc[u][3], ks[u], t.lo[3], t.hi[3], t.scale, d[u]);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int u = 0; u < kWTiles; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(d[u][v], a.c, -st));
                    sum[u][v] += u * 16 + 4 * q4 + v < limit ? p : 0.f;
                }
        }
        if (ahead < last) store(buf ^ 1, g);
        __syncthreads();
        buf ^= 1, i = ahead;
    }
    // over the 16 rows of the tiles (lanes of a DPP row), in a fixed order
    float *out = wa.part + (static_cast<int64_t>(chunk) * a.B + b) * wa.pitch + j0 + 4 * q4;
#pragma unroll
    for (int u = 0; u < kWTiles; ++u) {
#pragma unroll
        for (int v = 0; v < 4; ++v) sum[u][v] = q4_row16_sum(sum[u][v]);
        if (r16 == 0) *reinterpret_cast<f32x4 *>(out + u * 16) = sum[u];
    }
}

// weight[b][j] += the chunks' sums: four threads a position, each every fourth chunk, added in order
__global__ __launch_bounds__(256) void weights_add_kernel(WeightArgs wa) {
    __shared__ float part[4][64];
    const int c = threadIdx.x & 63, g = threadIdx.x >> 6, j = blockIdx.x * 64 + c, b = blockIdx.y;
    const int len = wa.a.lengths ? min(max(wa.a.lengths[b], 0), wa.a.cap) : wa.a.length;
    const float *src = wa.part + b * wa.pitch + j;
    const int64_t pitch = wa.a.B * wa.pitch;
    float s = 0.f;
    if (j < len) {
#pragma unroll 8
        for (int k = g; k < wa.chunks; k += 4) s += src[k * pitch];
    }
    part[g][c] = s;
    __syncthreads();
    if (g == 0 && j < len) wa.weight[b * wa.w_b + j] += (part[0][c] + part[1][c]) + (part[2][c] + part[3][c]);
}

// ------------------------------------------------------------------ host side
struct Plan {
    int NT, RT, PT, RG, tiles, rblocks, Ts, NS, slots, spread, listed, many, chunk, chunks;     // listed: Ts is the shortest range
    Rows order;
    int64_t qop, ml, part, stats, wpart, slot, seq, total;
};

constexpr int64_t kChunkRows = 1 << 16;   // rows (heads x queries, all sequences) of one pass over the queries, before a head's are padded
constexpr int64_t kLongest = 1 << 20;     // positions of a range: byte offsets in it take 32 bits, 2^30 at a pitch of 1 KB
// Queries of a sequence from which rows go by head, by head / by query, us in all, 64 heads: 17 over 64 39.0 / 37.2, 32 over 1024 with
// weights 54.0 / 56.7, 32 over 2048 42.9 / 43.3, 48 57.1 / 59.7.
constexpr int kByHead = 32;

Rows rows_of(int64_t T, int64_t H) {
    const int64_t Tp = T >= kByHead ? cdiv(T, 16) * 16 : 0;
    return Rows{static_cast<int>(T), static_cast<int>(H), static_cast<int>(Tp), inverse_of(Tp ? Tp : H), inverse_of(T)};
}

// What the launches are cut into; a function of its arguments alone.
Plan plan_of(int64_t B, int64_t T, int64_t H, int64_t npos, int q_bf16, int out_bf16, int weights, int varied) {
    Plan p{};
    const bool fine = !out_bf16 || weights;
    p.NT = fine ? 5 : 3, p.RT = q_bf16 ? 1 : fine ? 3 : 2, p.PT = out_bf16 ? 1 : 2;
    p.order = rows_of(std::max<int64_t>(1, std::min(T, kChunkRows / (B * H))), H);
    const int64_t rows = p.order.count();
    // Rows of a block.  A round costs 0.9 us at 16 rows, 1.1 at 32 and 1.8 at 64 (bf16 results; fp32 1.2, 1.6, 2.5), so more rows cost less
    // each; but they fill the card with shorter ranges, and every range begins (two rounds' worth) and leaves records (2 KB a row),
    // and a batch of small blocks is cut into fewer ranges of unequal length.  Measured, us at 16 / 32 / 64 rows and bf16, by the rounds a CU would
    // have with 16 (r; sequences of their own lengths: half the capacity's):
    //   r 6 (5 tokens of 96 heads over 3500) 33.2 / 33.2 / 37.4;  8 (1 of 64 over 32,768) 34.7 / 38.1 / 43.4;  13 (5 of 96 over
    //   7001) 39.1 / 40.7 / 41.1;  16 (1 of 64 over 65,536) 41.7 / 42.2 / 47.1, (2 over 32,768) 41.5 / 40.6 / 43.4;  26 (5 of 96 over
    //   14,000) 52.9 / 47.4 / 48.8;  32 (1 of 64 over 131,072) 58.4 / 53.2 / 56.1;  51 (5 of 96 over 28,000) 80.7 / 64.0 / 63.0
    //   batches of 64 heads: 8 of up to 8192 31.7 / 35.1 / 35.8, 32 of them 49.5 / 41.7 / 44.2, 64 of up to 1024 53.2 / 49.2 / 48.9
    const int64_t r = B * cdiv(rows, 16) * cdiv(npos, kRound) / (varied && B > 1 ? 512 : 256);
    p.RG = rows <= 16 || (B * cdiv(rows, 16) < 128 && r <= 14) ? 1 : rows <= 32 || (B * cdiv(rows, 32) < 128 && r <= 48) ? 2 : 4;
    p.rblocks = static_cast<int>(cdiv(rows, 16 * p.RG));
    p.tiles = p.rblocks * p.RG;
    const int64_t base = B * p.rblocks;
    // One block a CU, and at least two rounds to a block: 4096 positions in ranges of 64 took 29.2 us for 27.0.
    int64_t ns = std::max<int64_t>(1, std::min<int64_t>(kMaxSplits, 256 / base));
    int64_t ts = std::min(kLongest, std::max<int64_t>(2 * kRound, cdiv(cdiv(std::max<int64_t>(npos, 1), ns), kRound) * kRound));
    p.NS = static_cast<int>(cdiv(std::max<int64_t>(npos, 1), ts));
    p.listed = varied && B > 1 && base < 512;
    if (p.listed) {
        // a range that is not full for every sequence, so that many fewer for the rest, but as many as there are sequences at least,
        // and as it takes to hold all of the capacity
        const int64_t spread = std::max({256 / p.rblocks - B, B, cdiv(B * npos, kLongest)});
        ts = std::max<int64_t>(2 * kRound, cdiv(cdiv(npos, kMaxSplits), kRound) * kRound);
        p.NS = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(cdiv(npos, ts), spread + 1)));
        p.spread = static_cast<int>(spread), p.slots = static_cast<int>(spread + B);
    } else {
        p.slots = static_cast<int>(B * p.NS);
    }
    p.Ts = static_cast<int>(ts);
    // uv_many where uv_few's blocks (16 queries of a head) would not all run at once.  Measured, us in all, many / few: 256 queries of 16
    // heads over 1024 (256 blocks) 51.5 / 49.6, 320 (320) 54.7 / 60.2; 64 of 64 over 2048 (256) 61.7 / 58.8, 72 (320) 64.1 / 67.5; 48 of 96
    // (288) 63.2 / 68.5; 600 of 2 over 8000 (76) 73.9 / 55.6; 128 of 64 over 512 (512) 49.0 / 63.2.
    p.many = !p.listed && H * cdiv(B * p.order.T, 16) > 256;
    const int64_t pos_blocks = std::max<int64_t>(1, cdiv(npos, 128 * kWTiles));
    p.chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.tiles, 256 / (pos_blocks * B))));
    p.chunk = static_cast<int>(cdiv(p.tiles, p.chunks));
    p.chunks = static_cast<int>(cdiv(p.tiles, p.chunk));
    auto up = [](int64_t v) { return (v + 255) & ~int64_t(255); };
    int64_t o = 0;
    p.qop = o, o += up(B * p.tiles * q4_tile_bytes(p.NT, p.RT));
    p.ml = o, o += up(p.slots * rows * 8);
    p.part = o, o += up(p.slots * rows * kQ4Lat * 4);
    p.slot = o, o += p.listed ? up(p.slots * 16) : 0;
    p.seq = o, o += p.listed ? up(B * 8) : 0;
    p.stats = o, o += weights ? up(B * rows * 4) : 0;
    p.wpart = o, o += weights ? up(p.chunks * B * pos_blocks * (128 * kWTiles) * 4) : 0;
    p.total = o;
    return p;
}

template <int RG, int NT, int RT, int PT>
int launch_attend(const AttendArgs &a, int slots, hipStream_t st) {
    constexpr int bytes = attend_lds(RG, RT, PT);
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(attend_kernel<RG, NT, RT, PT>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    const int rc = check_hip(attr, "mla q4: attention LDS size");
    if (rc) return rc;
    attend_kernel<RG, NT, RT, PT><<<dim3(static_cast<unsigned>(slots * a.rblocks)), 512, bytes, st>>>(a);
    return check_hip(hipGetLastError(), "mla q4: attention launch");
}

template <int RG>
int launch_attend_of(const AttendArgs &a, const Plan &p, hipStream_t st) {
    if (p.NT == 3) return p.RT == 1 ? launch_attend<RG, 3, 1, 1>(a, p.slots, st) : launch_attend<RG, 3, 2, 1>(a, p.slots, st);
    if (p.PT == 1) return p.RT == 1 ? launch_attend<RG, 5, 1, 1>(a, p.slots, st) : launch_attend<RG, 5, 3, 1>(a, p.slots, st);
    return p.RT == 1 ? launch_attend<RG, 5, 1, 2>(a, p.slots, st) : launch_attend<RG, 5, 3, 2>(a, p.slots, st);
}

template <typename QT, int NT, int RT, int MT>
int launch_qa_of(const QaArgs &a, hipStream_t st) {
    const int bytes = std::max(((a.nope + 31) / 32) * 32 * kWLd, 16 * MT * kFLd * 4);
    static_assert(32 * kWLd >= (2 * kMaxListed + 16) * 4, "the list of ranges fits");
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(qa_kernel<QT, NT, RT, MT>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, 256 * kWLd);
    const int rc = check_hip(attr, "mla q4: query LDS size");
    if (rc) return rc;
    qa_kernel<QT, NT, RT, MT><<<dim3(a.H, static_cast<unsigned>(cdiv(a.M, 16 * MT)), a.ranges.seq ? 5 : 4), 256, bytes, st>>>(a);
    return check_hip(hipGetLastError(), "mla q4: query launch");
}

template <typename QT, int NT, int RT>
int launch_qa(const QaArgs &a, hipStream_t st) {
    // (24 queries of 64 heads 41.5 us in all either way, 64 61.1 / 62.3)
    return a.M > 32 ? launch_qa_of<QT, NT, RT, 4>(a, st) : launch_qa_of<QT, NT, RT, 1>(a, st);
}

template <int WAVES, int VT>
int launch_few(const UvArgs &a, int per, unsigned tiles, hipStream_t st) {
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(uv_few_kernel<WAVES, VT>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, kFewLds);
    const int rc = check_hip(attr, "mla q4: output LDS size");
    if (rc) return rc;
    uv_few_kernel<WAVES, VT><<<dim3(static_cast<unsigned>(a.order.H), tiles, 8 / VT), 64 * WAVES, kFewLds, st>>>(a, per);
    return check_hip(hipGetLastError(), "mla q4: join and W_UV launch");
}

int launch_uv(const UvArgs &a, int many, hipStream_t st) {
    const unsigned H = static_cast<unsigned>(a.order.H);
    if (!many) {
        // The fewest queries to a block with which all blocks run at once (one a CU, for its LDS); then the output columns in as many
        // parts (8 waves hold half of them), which join the same records (1 token of 64 heads with 64 records: 40.7 us in all in one part, 37.7 in two, 37.2 in four;
        // 32 tokens, in one part a block a CU: 42.3, 47.4, 57.6).
        const int least = a.NS <= kFewSplits ? 2 : 1;
        int per = static_cast<int>(std::min<int64_t>(16, a.M));
        while (per > 1 && least * H * cdiv(a.M, per - 1) <= 256) --per;
        const unsigned tiles = static_cast<unsigned>(cdiv(a.M, per)), blocks = H * tiles;
        if (a.NS <= kFewSplits) return blocks <= 64 ? launch_few<8, 2>(a, per, tiles, st) : launch_few<8, 4>(a, per, tiles, st);
        return blocks <= 64 ? launch_few<16, 2>(a, per, tiles, st) : blocks <= 128 ? launch_few<16, 4>(a, per, tiles, st)
                                                                                  : launch_few<16, 8>(a, per, tiles, st);
    }
    static const hipError_t many2 = hipFuncSetAttribute(reinterpret_cast<const void *>(uv_many_kernel<2>),
                                                        hipFuncAttributeMaxDynamicSharedMemorySize, 2 * 64 * 272 + 64 * kMaxSplits * 4);
    static const hipError_t many3 = hipFuncSetAttribute(reinterpret_cast<const void *>(uv_many_kernel<3>),
                                                        hipFuncAttributeMaxDynamicSharedMemorySize, 3 * 64 * 272 + 64 * kMaxSplits * 4);
    const int rc = check_hip(a.out_bf16 ? many2 : many3, "mla q4: output LDS size");
    if (rc) return rc;
    if (a.out_bf16)
        uv_many_kernel<2><<<dim3(H, static_cast<unsigned>(cdiv(a.M, 64))), 256, 2 * 64 * 272 + 64 * a.NS * 4, st>>>(a);
    else
        uv_many_kernel<3><<<dim3(H, static_cast<unsigned>(cdiv(a.M, 64))), 256, 3 * 64 * 272 + 64 * a.NS * 4, st>>>(a);
    return check_hip(hipGetLastError(), "mla q4: join and W_UV launch");
}

template <int RT>
int launch_weights(const WeightArgs &wa, hipStream_t st) {
    constexpr int bytes = q4_tile_bytes(5, RT) + std::max(q4_tile_bytes(5, RT), 8 * 16 * kKLd);     // (the second tile's place also turns the codes)
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(weights_kernel<5, RT>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    int rc = check_hip(attr, "mla q4: weights LDS size");
    if (rc) return rc;
    const unsigned B = static_cast<unsigned>(wa.a.B);
    weights_kernel<5, RT><<<dim3(static_cast<unsigned>(wa.pitch / (128 * kWTiles)), static_cast<unsigned>(wa.chunks), B), 512, bytes, st>>>(wa);
    rc = check_hip(hipGetLastError(), "mla q4: weights launch");
    if (rc) return rc;
    weights_add_kernel<<<dim3(static_cast<unsigned>(wa.pitch / 64), B), 256, 0, st>>>(wa);
    return check_hip(hipGetLastError(), "mla q4: weight sum launch");
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" int64_t k3_mla_q4_workspace_size(int64_t B, int64_t T, int64_t H, int64_t v_dim, int64_t max_length, int q_dtype,
                                            int out_dtype, int weights, int varied) {
    if (B <= 0 || T <= 0 || H <= 0 || v_dim <= 0 || max_length < 0) return 0;
    return plan_of(B, T, H, max_length, q_dtype == K3_BF16, out_dtype == K3_BF16, weights != 0, varied != 0).total;
}

extern "C" int k3_mla_q4_attention(const void *q_nope, int64_t qn_batch, int64_t qn_token, int64_t qn_head, const void *q_rot,
                                   int64_t qr_batch, int64_t qr_token, int64_t qr_head, int q_dtype, const void *w_uk,
                                   const void *w_uv, const void *packed, int64_t p_batch, int64_t p_row, const void *scales,
                                   int64_t s_batch, int64_t s_row, const void *rot, int64_t rot_batch, int64_t rot_row,
                                   const int32_t *lengths, const int32_t *counts, int64_t max_length, int64_t B, int64_t T,
                                   int64_t H, int64_t kv_lora_rank, int64_t rope_dim, int64_t nope_dim, int64_t v_dim, float scale,
                                   const float *gate, void *out, int out_dtype, float *weight, int64_t w_batch, void *workspace,
                                   int64_t workspace_bytes, void *stream) {
    if (B == 0 || T == 0) return K3_OK;
    if (!q_nope || !q_rot || !w_uk || !w_uv || !out || !workspace || (max_length > 0 && (!packed || !scales || !rot)))
        return set_error(K3_ERR_NULL, "mla q4: null pointer");
    if (q_dtype != K3_F32 && q_dtype != K3_BF16) return set_error(K3_ERR_DTYPE, "mla q4: q_dtype %d", q_dtype);
    if (out_dtype != K3_F32 && out_dtype != K3_BF16) return set_error(K3_ERR_DTYPE, "mla q4: out_dtype %d", out_dtype);
    if (kv_lora_rank != kQ4Lat || rope_dim != kQ4Rope)
        return set_error(K3_ERR_SHAPE, "mla q4: kv_lora_rank=%lld rope=%lld; the kernels take 512 and 64", (long long)kv_lora_rank,
                         (long long)rope_dim);
    if (nope_dim <= 0 || nope_dim > 256 || nope_dim % 8 || v_dim <= 0 || v_dim > 1024 || v_dim % 8)
        return set_error(K3_ERR_SHAPE, "mla q4: nope=%lld must be a multiple of 8 up to 256 and v=%lld one up to 1024",
                         (long long)nope_dim, (long long)v_dim);
    if (B < 0 || B > 65535 || T < 0 || T > (1 << 24) || H <= 0 || H > 4096 || B * H > kChunkRows || max_length < 0 || max_length > (1 << 24))
        return set_error(K3_ERR_SHAPE, "mla q4: B=%lld, T=%lld, H=%lld or max_length=%lld out of range", (long long)B, (long long)T,
                         (long long)H, (long long)max_length);
    if (qn_batch % 4 || qn_token % 4 || qn_head % 4 || qr_batch % 4 || qr_token % 4 || qr_head % 4)
        return set_error(K3_ERR_SHAPE, "mla q4: query strides must be multiples of 4 elements");
    if (max_length > 0 && (p_row < 256 || p_row % 16 || p_batch % 16 || s_row < 16 || s_row % 4 || s_batch % 4 || rot_row < kQ4Rope || rot_row % 8 ||
                           rot_batch % 8 || p_row > (1 << 16) || s_row > (1 << 16) || rot_row > (1 << 15)))
        return set_error(K3_ERR_SHAPE, "mla q4: cache row pitches too small, too large or not multiples of 16 bytes (scales: 4)");
    if (weight && !blocks_apart(B, w_batch, 1, max_length, max_length))
        return set_error(K3_ERR_SHAPE, "mla q4: the sequences' weights overlap, %lld apart", (long long)w_batch);
    if (!aligned16(q_nope) || !aligned16(q_rot) || !aligned16(w_uk) || !aligned16(w_uv) || !aligned16(out) || !aligned16(workspace) ||
        !aligned16(packed) || !aligned16(rot) || (reinterpret_cast<uintptr_t>(scales) & 3u) || (gate && !aligned16(gate)))
        return set_error(K3_ERR_ALIGN, "mla q4: queries, weights, cache, output and workspace must be 16-byte (scales 4-byte) aligned");
    const Plan p = plan_of(B, T, H, max_length, q_dtype == K3_BF16, out_dtype == K3_BF16, weight != nullptr, lengths != nullptr);
    if (workspace_bytes < p.total)
        return set_error(K3_ERR_WORKSPACE, "mla q4: workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)p.total);
    // (a range of a list is at most as long as all positions shared out: 1.01 kLongest + 128 positions, 1.02 2^30 bytes at pitches of 1 KB)
    const int64_t longest = p.listed ? std::max<int64_t>(p.Ts, B * max_length / p.spread * 1.01 + 128) : p.Ts;
    if (longest * std::max({p_row, s_row, 2 * rot_row}) >= (1ll << 31))
        return set_error(K3_ERR_SHAPE, "mla q4: a range of %lld positions spans 2 GiB at these row pitches", (long long)longest);
    auto st = static_cast<hipStream_t>(stream);
    char *ws = static_cast<char *>(workspace);
    for (int64_t t0 = 0; t0 < T; t0 += p.order.T) {
        // (the last pass may have fewer queries, so few that its rows go by query; it has the others' room, block height and join)
        Rows order = rows_of(std::min<int64_t>(p.order.T, T - t0), H);
        const int rows = order.count(), M = static_cast<int>(B * order.T);
        const int64_t q_seq = static_cast<int64_t>(p.tiles) * q4_tile_bytes(p.NT, p.RT);
        QaArgs qa{q_nope, q_rot, qn_batch, qn_token, qn_head, qr_batch, qr_token, qr_head, static_cast<const uint16_t *>(w_uk),
                  ws + p.qop, q_seq, static_cast<int>(H), static_cast<int>(nope_dim), M, static_cast<int>(t0), order, {}};
        if (p.listed)
            qa.ranges = Ranges{lengths, reinterpret_cast<int4 *>(ws + p.slot), reinterpret_cast<int2 *>(ws + p.seq), static_cast<int>(B),
                               static_cast<int>(max_length), p.slots, p.spread, p.Ts};
        int rc;
        if (q_dtype == K3_BF16)
            rc = p.NT == 5 ? launch_qa<uint16_t, 5, 1>(qa, st) : launch_qa<uint16_t, 3, 1>(qa, st);
        else
            rc = p.NT == 5 ? launch_qa<float, 5, 3>(qa, st) : launch_qa<float, 3, 2>(qa, st);
        if (rc) return rc;
        AttendArgs a{};
        a.qop = ws + p.qop, a.q_seq = q_seq;
        a.packed = static_cast<const uint8_t *>(packed), a.scales = static_cast<const uint8_t *>(scales);
        a.rot = static_cast<const uint8_t *>(rot);
        a.p_b = p_batch, a.p_t = p_row, a.s_b = s_batch, a.s_t = s_row, a.r_b = 2 * rot_batch, a.r_t = 2 * rot_row;
        a.lengths = lengths, a.counts = counts;
        a.length = static_cast<int>(max_length), a.cap = a.length, a.count = static_cast<int>(T);
        a.slot = qa.ranges.slot;
        a.part = reinterpret_cast<float *>(ws + p.part), a.ml = reinterpret_cast<float2 *>(ws + p.ml);
        a.order = order, a.t0 = static_cast<int>(t0), a.rows = rows, a.Ts = p.Ts, a.NS = p.NS;
        a.inverse_ns = inverse_of(p.NS);
        a.rblocks = static_cast<int>(cdiv(rows, 16 * p.RG)), a.inverse_rblocks = inverse_of(a.rblocks), a.B = static_cast<int>(B), a.c = scale * 1.4426950408889634f;
        // blocks b % 8 run on one XCD: with several ranges its blocks get neighbouring ones (one L2 reads them); with one range the blocks
        // that see most, which come first, are to be spread
        a.swizzle = p.NS > 1 && (p.slots * a.rblocks) % 8 == 0;
        rc = p.RG == 4 ? launch_attend_of<4>(a, p, st) : p.RG == 2 ? launch_attend_of<2>(a, p, st) : launch_attend_of<1>(a, p, st);
        if (rc) return rc;
        UvArgs u{};
        u.part = a.part, u.ml = a.ml, u.w_uv = static_cast<const uint16_t *>(w_uv);
        u.out = out, u.out_bf16 = out_dtype == K3_BF16, u.gate = gate;
        u.stats = weight ? reinterpret_cast<float *>(ws + p.stats) : nullptr;
        u.seq = qa.ranges.seq;
        u.order = order, u.M = M, u.V = static_cast<int>(v_dim), u.rows = rows, u.NS = p.NS;
        u.Tall = static_cast<int>(T), u.t0 = a.t0, u.lengths = lengths, u.counts = counts, u.length = a.length;
        rc = launch_uv(u, p.many, st);
        if (rc) return rc;
        if (weight && max_length > 0) {
            WeightArgs wa{a, u.stats, reinterpret_cast<float *>(ws + p.wpart), weight, w_batch, static_cast<int>(cdiv(rows, 16)), p.chunk,
                          0, cdiv(max_length, 128 * kWTiles) * (128 * kWTiles)};
            wa.chunks = static_cast<int>(cdiv(wa.tiles, wa.chunk));
            rc = p.RT == 1 ? launch_weights<1>(wa, st) : launch_weights<3>(wa, st);
            if (rc) return rc;
        }
    }
    return K3_OK;
}
