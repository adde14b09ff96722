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
//   uv       the ranges' records joined, the context times W_UV
//   out      (few rows) the four column quarters of that product added, and the output gate
//   weights  (if asked for) p once more from the rows' final maxima and sums, added over the rows
//
// attend, per round of 32 positions: a thread stages one group (16 bytes of codes and their scale byte); the codes go to
// LDS as they are, where the score waves (0..3) read them as matrix operands; the same thread decodes its group
// (exactly: E2M1 times a power of two) into the value tile, which the context waves (4..7, 128 columns each) read
// transposed (fp16, see mla_q4.h).  In iteration i the score waves take round i's scores and turn round i - 1's into
// probabilities, and the context waves take round i - 2's products, one barrier per iteration.  A row's reference maximum moves
// only when a score exceeds it by kSlack (log2), so the accumulators are seldom rescaled.
//
// A position whose scale byte is 255 (NaN) makes its scores NaN by the matrix product itself, so every row that sees it is NaN; its
// values are staged as zeros, so a row that does not see it (weight zero) stays clean.
#include <algorithm>
#include <type_traits>

#include "mla_q4.h"

namespace k3 {
namespace {

typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4_t *lds_s4;

// ------------------------------------------------------------------ qa
struct QaArgs {
    const void *q_nope, *q_rot;
    int64_t n_b, n_t, n_h, r_b, r_t, r_h;   // strides in elements (batch, query, head)
    const uint16_t *w_uk;                   // [H, nope, 512]
    char *qop;                              // [B][tiles] operand tiles
    int64_t q_seq;                          // bytes of a sequence's tiles
    int H, nope, T, M, t0;                  // T queries from t0 on; M = B T
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

// grid (H, ceil(M / 16), 4): queries 16 y .. +16 of head x, latent columns 128 z .. +128
template <typename QT, int NT, int RT>
__global__ __launch_bounds__(256) void qa_kernel(QaArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float *fs = reinterpret_cast<float *>(lds);                         // [16][kFLd], after the products
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, q4 = lane >> 4;
    const int h = blockIdx.x, m0 = blockIdx.y * 16, quarter = blockIdx.z;
    const int steps = (a.nope + 31) >> 5;
    const uint16_t *w = a.w_uk + static_cast<int64_t>(h) * a.nope * kQ4Lat + quarter * 128;
    for (int i = tid; i < steps * 32 * 16; i += 256) {
        const int n = i >> 4, c = i & 15;
        const uint4 v = n < a.nope ? *reinterpret_cast<const uint4 *>(w + static_cast<int64_t>(n) * kQ4Lat + c * 8) : make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4 *>(lds + n * kWLd + c * 16) = v;
    }
    // this lane's query values: slots 8 q4 .. +8 of a step hold n = 4 q4 + {0..3} and 16 + 4 q4 + {0..3}, as the
    // transposed reads of the weights give them
    const int m = m0 + r16;
    const bool live = m < a.M;
    const int b = live ? m / a.T : 0, t = live ? a.t0 + m % a.T : 0;
    const QT *q = static_cast<const QT *>(a.q_nope) + b * a.n_b + t * a.n_t + h * a.n_h;
    f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        u32x4 qf[3];
        constexpr int kTerms = std::is_same<QT, float>::value ? 3 : 1;
        if constexpr (kTerms == 3) {
            float v[8];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int n = 32 * s + 16 * x + 4 * q4;
                const float4 g = live && n < a.nope ? *reinterpret_cast<const float4 *>(q + n) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[4 * x] = g.x, v[4 * x + 1] = g.y, v[4 * x + 2] = g.z, v[4 * x + 3] = g.w;
            }
            terms8(v, qf);
        } else {
            uint2 g[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int n = 32 * s + 16 * x + 4 * q4;
                g[x] = live && n < a.nope ? *reinterpret_cast<const uint2 *>(q + n) : make_uint2(0u, 0u);
            }
            qf[0] = u32x4{g[0].x, g[0].y, g[1].x, g[1].y};
        }
        const char *wr = lds + (32 * s + 4 * q4 + (r16 >> 2)) * kWLd + (r16 & 3) * 8 + wave * 64;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const s4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(wr + j * 32));
            const s4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(wr + j * 32 + 16 * kWLd));
            const u32x4 wf = __builtin_bit_cast(u32x4, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int k = kTerms - 1; k >= 0; --k) acc[j] = q4_mfma_bf16(wf, qf[k], acc[j]);
        }
    }
    __syncthreads();   // the weights are read
#pragma unroll
    for (int j = 0; j < 2; ++j) *reinterpret_cast<f32x4 *>(fs + r16 * kFLd + wave * 32 + j * 16 + 4 * q4) = acc[j];
    __syncthreads();
    const int part = tid < 64 ? 0 : 1;
    const int i = part == 0 ? tid >> 2 : (tid - 64) >> 3;       // query of the tile
    if (m0 + i >= a.M || i >= 16) return;
    const int mi = m0 + i, bi = mi / a.T, row = (mi % a.T) * a.H + h;
    char *tile = a.qop + bi * a.q_seq + static_cast<int64_t>(row >> 4) * q4_tile_bytes(NT, RT);
    if (part == 0) {
        // one group of 32 columns: its terms
        const int g = tid & 3, at = quarter * 16 + (row & 15);
        const float *src = fs + i * kFLd + g * 32;
        float v[32];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            v[j] = src[j];
            top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
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
    } else if (quarter == 0) {
        // rotary columns 8 c .. +8 of query i
        const int c = (tid - 64) & 7, at = (c & 3) * 16 + (row & 15);
        const QT *qr = static_cast<const QT *>(a.q_rot) + bi * a.r_b + (a.t0 + mi % a.T) * a.r_t + h * a.r_h + c * 8;
        u32x4 f[3] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
        if constexpr (std::is_same<QT, float>::value) {
            float v[8];
            const float4 x = *reinterpret_cast<const float4 *>(qr), y = *reinterpret_cast<const float4 *>(qr + 4);
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
            terms8(v, f);
        } else {
            const uint2 x = *reinterpret_cast<const uint2 *>(qr), y = *reinterpret_cast<const uint2 *>(qr + 4);
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
    float *part;                                // [B][NS][rows][512]
    float2 *ml;                                 // [B][NS][rows]
    int H, T, t0, rows, Ts, NS, rblocks, B;
    float c;                                    // scale * log2(e)
    int swizzle;
};

constexpr int kRound = 32;                      // positions per round
constexpr int kKLd = 272;                       // LDS bytes of a staged row of codes: 256 + 16 scale bytes
constexpr int kRLd = 144;                       // .. of a rotary row: 128 + 16
constexpr int kVLd = 1056;                      // .. of a value row: 1024 + 32
constexpr int kKBytes = kRound * kKLd, kRBytes = kRound * kRLd, kVBytes = kRound * kVLd;

constexpr int kKSlots = 3;

constexpr int attend_lds(int RG, int RT, int PT) {   // PT fp16 terms of the probabilities (bf16: one more)
    return kKSlots * kKBytes + 2 * kRBytes + 2 * kVBytes + 2 * RG * (PT + 1) * 1024 + RG * RT * 2048;
}

// RG: groups of 16 rows (2: two score waves to a group, one tile of 16 positions each; 4: one, two tiles);
// NT latent and RT rotary terms of the queries, PT fp16 terms of the probabilities
template <int RG, int NT, int RT, int PT>
__global__ __launch_bounds__(512, 1) void attend_kernel(AttendArgs a) {
    constexpr int TG = 4 / RG, NTILE = 2 / TG;   // score waves of a row group; tiles of 16 positions per score wave
    constexpr int kPLd = (PT + 1) * 1024;        // LDS bytes of a row group's probabilities
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float xm[2][TG][RG * 16];         // tile maxima [parity][score wave of the group][row]
    __shared__ float xf[2][RG * 16];             // rescale factors [parity][row]
    __shared__ float xl[TG][RG * 16];
    __shared__ int wide;                         // a staged scale byte needs bf16's range
    char *const kbuf = lds, *const rbuf = lds + kKSlots * kKBytes, *const vbuf = rbuf + 2 * kRBytes, *const pbuf = vbuf + 2 * kVBytes;
    char *const qbuf = pbuf + 2 * RG * kPLd;     // the queries' rotary operands
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, q4 = lane >> 4;
    const int nb = gridDim.x;
    const int w = a.swizzle ? (blockIdx.x & 7) * (nb >> 3) + (blockIdx.x >> 3) : blockIdx.x;
    const int rb = w % a.rblocks, split = (w / a.rblocks) % a.NS, b = w / (a.rblocks * a.NS);
    const int row0 = rb * 16 * RG;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.cap) : a.length;
    const int cnt = a.counts ? min(max(a.counts[b], 0), a.count) : a.count;
    // the last query of the block that is there sees most
    const int tlast = min(a.t0 + (min(row0 + 16 * RG, a.rows) - 1) / a.H, cnt - 1);
    const int most = tlast >= a.t0 + row0 / a.H ? q4_sees(tlast, cnt, len) : 0;
    const int t_begin = split * a.Ts, t_end = min(most, t_begin + a.Ts);
    float2 *ml = a.ml + (static_cast<int64_t>(b) * a.NS + split) * a.rows;
    if (t_end <= t_begin) {
        if (tid < 16 * RG && row0 + tid < a.rows) ml[row0 + tid] = make_float2(-INFINITY, 0.f);
        return;
    }
    const int n = t_end - t_begin, nr = (n + kRound - 1) / kRound;

    // ---- staging, by the context waves: thread = (positions st / 16 and 16 more, group st % 16) and a 16-byte rotary chunk
    const auto rp = make_rsrc(a.packed + b * a.p_b + t_begin * a.p_t, static_cast<uint32_t>((n - 1) * a.p_t + 256));
    const auto rs = make_rsrc(a.scales + b * a.s_b + t_begin * a.s_t, static_cast<uint32_t>((n - 1) * a.s_t + 16));
    const auto rr = make_rsrc(a.rot + b * a.r_b + t_begin * a.r_t, static_cast<uint32_t>((n - 1) * a.r_t + 128));
    const int st = tid & 255, srow = st >> 4, sgrp = st & 15, orow = st >> 3, ochunk = st & 7;
    struct Stage {
        u32x4 k[2], o;
        uint32_t s[2];
    };
    auto load = [&](Stage &g, int rd) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = rd * kRound + 16 * u + srow;
            const bool ok = i < n;
            g.k[u] = __builtin_bit_cast(u32x4, buf_load16(rp, ok ? static_cast<uint32_t>(i) * static_cast<uint32_t>(a.p_t) + sgrp * 16u : kOobOffset));
            g.s[u] = __builtin_amdgcn_raw_buffer_load_b8(rs, ok ? static_cast<uint32_t>(i) * static_cast<uint32_t>(a.s_t) + sgrp : kOobOffset, 0, 0);
        }
        const int j = rd * kRound + orow;
        g.o = __builtin_bit_cast(u32x4, buf_load16(rr, j < n ? static_cast<uint32_t>(j) * static_cast<uint32_t>(a.r_t) + ochunk * 16u : kOobOffset));
    };
    auto store_k = [&](const Stage &g, int rd, bool look) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            char *k = kbuf + (rd % kKSlots) * kKBytes + (16 * u + srow) * kKLd;
            *reinterpret_cast<u32x4 *>(k + sgrp * 16) = g.k[u];
            reinterpret_cast<uint8_t *>(k)[256 + sgrp] = static_cast<uint8_t>(g.s[u]);
            // (a NaN's values are staged as zeros; -0 codes count as values)
            if (look && g.s[u] - kHalfLow > kHalfHigh - kHalfLow && g.s[u] != 255u && (g.k[u].x | g.k[u].y | g.k[u].z | g.k[u].w) != 0u)
                wide = 1;
        }
        *reinterpret_cast<u32x4 *>(rbuf + (rd & 1) * kRBytes + orow * kRLd + ochunk * 16) = g.o;
    };
    // this thread's group (which it staged itself) as fp16 or bf16, 64 bytes; lanes 4..7, 8..11, 12..15 of a 16-lane row
    // start at another 16 bytes, so a store instruction's lanes spread over the banks
    auto store_v = [&](int rd, int u, auto bf) __attribute__((always_inline)) {
        const char *ks = kbuf + (rd % kKSlots) * kKBytes + (16 * u + srow) * kKLd;
        const u32x4 k = *reinterpret_cast<const u32x4 *>(ks + sgrp * 16);
        const uint32_t s = reinterpret_cast<const uint8_t *>(ks)[256 + sgrp];
        char *v = vbuf + (rd & 1) * kVBytes + (16 * u + srow) * kVLd + sgrp * 64;
        const int x = (lane >> 2) & 3;
        const u32x4 y = (x & 1) ? u32x4{k.y, k.x, k.w, k.z} : k;
        u32x4 z = (x & 2) ? u32x4{y.z, y.w, y.x, y.y} : y;
        if (s == 255u) z = u32x4{0u, 0u, 0u, 0u};
        const float f = s == 255u ? 0.f : e8m0_to_f32(s);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x4 o;
            if constexpr (decltype(bf)::value)
                o = u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(z[j], f, 0)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(z[j], f, 1)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(z[j], f, 2)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(z[j], f, 3))};
            else
                o = u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(z[j], f, 0)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(z[j], f, 1)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(z[j], f, 2)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(z[j], f, 3))};
            *reinterpret_cast<u32x4 *>(v + ((j ^ x) << 4)) = o;
        }
    };

    // iterations 0 .. nr + 1, an even number of them (rounds past the last are zeros that no row sees)
    const int iters = (nr + 3) & ~1;
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    if (tid == 0) wide = 0;
    if (wave < 4) {
        // ================= score waves
        const int rg = TG == 1 ? wave : wave % RG, tg = TG == 1 ? 0 : wave / RG;
        const char *tile = a.qop + b * a.q_seq + static_cast<int64_t>((row0 >> 4) + rg) * q4_tile_bytes(NT, RT);
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
        // (the two score waves of a row group write the same)
        char *const qr = qbuf + rg * RT * 2048 + lane * 16;
#pragma unroll
        for (int x = 0; x < 2 * RT; ++x) *reinterpret_cast<u32x4 *>(qr + x * 1024) = *reinterpret_cast<const u32x4 *>(tile + q4_rope_at(NT, 0, x) + lane * 16);
        const int row = row0 + rg * 16 + r16;
        const int sees = row < a.rows ? q4_sees(a.t0 + row / a.H, cnt, len) : 0;
        const int limit = min(sees, t_end) - t_begin;       // positions of this split that the row sees
        float m_ref, l_run, mt[2];
        f32x4 sc[2][NTILE];                                 // scores of round i (parity)

        auto scores = [&](int rd, f32x4 (&out)[NTILE]) __attribute__((always_inline)) {
            f32x4 hr[NTILE];
#pragma unroll
            for (int u = 0; u < NTILE; ++u) hr[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int x = RT - 1; x >= 0; --x) {
                    const u32x4 qv = *reinterpret_cast<const u32x4 *>(qr + (2 * x + s) * 1024);
#pragma unroll
                    for (int u = 0; u < NTILE; ++u) {
                        const char *o = rbuf + (rd & 1) * kRBytes + ((tg * NTILE + u) * 16 + r16) * kRLd + s * 64 + q4 * 16;
                        hr[u] = q4_mfma_bf16(*reinterpret_cast<const u32x4 *>(o), qv, hr[u]);
                    }
                }
#pragma unroll
            for (int u = 0; u < NTILE; ++u) {
                const char *k = kbuf + (rd % kKSlots) * kKBytes + ((tg * NTILE + u) * 16 + r16) * kKLd;
                const int ks = *reinterpret_cast<const int *>(k + 256 + q4 * 4);
                u32x4 kc[kQ4Steps];
#pragma unroll
                for (int s = 0; s < kQ4Steps; ++s) kc[s] = *reinterpret_cast<const u32x4 *>(k + q4 * 64 + s * 16);
                f32x4 hi = {0.f, 0.f, 0.f, 0.f}, lo = hi;
#pragma unroll
                for (int x = NT - 1; x >= 0; --x) {
                    f32x4 &d = x < 2 ? hi : lo;
                    d = q4_mfma<0>(kc[0], ks, qlo[x][0], qhi[x][0], qs[x], d);
                    d = q4_mfma<1>(kc[1], ks, qlo[x][1], qhi[x][1], qs[x], d);
                    d = q4_mfma<2>(kc[2], ks, qlo[x][2], qhi[x][2], qs[x], d);
                    d = q4_mfma<3>(kc[3], ks, qlo[x][3], qhi[x][3], qs[x], d);
                }
                out[u] = hi + (lo + hr[u]);
                __builtin_amdgcn_sched_barrier(0);   // (hoisting the next tile's operands costs the registers of a query term)
            }
        };
        // scores -> scaled (log2 units), hidden positions -infinity; the tile maxima are published
        auto publish = [&](int rd, f32x4 (&s)[NTILE]) __attribute__((always_inline)) {
            float mt = -INFINITY;
#pragma unroll
            for (int u = 0; u < NTILE; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const int j = rd * kRound + (tg * NTILE + u) * 16 + 4 * q4 + v;
                    s[u][v] = j < limit ? s[u][v] * a.c : -INFINITY;
                    mt = fmaxf(mt, s[u][v]);
                }
            mt = q4_rows_max(mt);
            if (TG > 1 && q4 == 0) xm[rd & 1][tg][rg * 16 + r16] = mt;
            return mt;
        };
        auto probs = [&](int rd, const f32x4 (&s)[NTILE], float mt, auto bf) __attribute__((always_inline)) {
            if constexpr (TG > 1) mt = fmaxf(xm[rd & 1][0][rg * 16 + r16], xm[rd & 1][TG - 1][rg * 16 + r16]);
            float f = 1.f;
            if (mt > m_ref + kSlack || m_ref == -INFINITY) {
                f = m_ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_ref - mt);
                if (mt == -INFINITY) f = 1.f;
                l_run *= f;
                m_ref = mt;
            }
            const float ref = m_ref == -INFINITY ? 0.f : m_ref - kLift;
            char *p = pbuf + ((rd & 1) * RG + rg) * kPLd + lane * 16;
#pragma unroll
            for (int u = 0; u < NTILE; ++u) {
                float e[4];
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    e[v] = __builtin_amdgcn_exp2f(s[u][v] - ref);
                    l_run += e[v];
                }
                char *pu = p + (tg * NTILE + u) * 8;
                if constexpr (!decltype(bf)::value) {
#pragma unroll
                    for (int x = 0; x < PT; ++x) {
                        const uint32_t a0 = q4_pack_f16(e[0], e[1]), a1 = q4_pack_f16(e[2], e[3]);
                        *reinterpret_cast<u32x2 *>(pu + x * 1024) = u32x2{a0, a1};
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
                        *reinterpret_cast<u32x2 *>(pu + x * 1024) = u32x2{a0, a1};
                        e[0] -= q4_lo(a0), e[1] -= q4_hi(a0), e[2] -= q4_lo(a1), e[3] -= q4_hi(a1);
                    }
                }
            }
            if (tg == 0 && q4 == 0) xf[rd & 1][rg * 16 + r16] = f;
        };

        auto all = [&](auto bf) __attribute__((always_inline)) {
            m_ref = -INFINITY, l_run = 0.f;
            __syncthreads();   // wide is clear
            __syncthreads();   // round 0 is staged
            auto part = [&](int i, auto par) __attribute__((always_inline)) {
                constexpr int d = decltype(par)::value;
                scores(i, sc[d]);
                probs(i - 1, sc[1 - d], mt[1 - d], bf);
                mt[d] = publish(i, sc[d]);
                __syncthreads();
            };
            scores(0, sc[0]);
            mt[0] = publish(0, sc[0]);
            __syncthreads();
            part(1, odd);
            for (int i = 2; i < iters; i += 2) {
                part(i, even);
                part(i + 1, odd);
            }
        };
        all(std::false_type{});
        if (__builtin_amdgcn_readfirstlane(wide)) all(std::true_type{});
        const float l = q4_rows_sum(l_run);
        if (TG > 1 && q4 == 0) xl[tg][rg * 16 + r16] = l;
        __syncthreads();
        if (tg == 0 && q4 == 0 && row < a.rows) ml[row] = make_float2(m_ref, TG > 1 ? xl[0][rg * 16 + r16] + xl[TG - 1][rg * 16 + r16] : l);
    } else {
        // ================= context waves: columns 128 (wave - 4) .. +128
        const int col0 = (wave - 4) * 128;
        f32x4 acc[8][RG];
        auto context = [&](int rd, auto bf) __attribute__((always_inline)) {
            constexpr bool kBf = decltype(bf)::value;
            constexpr int N = PT + kBf;
            const char *p = pbuf + (rd & 1) * RG * kPLd + lane * 16;
            const char *v = vbuf + (rd & 1) * kVBytes + (4 * q4 + (r16 >> 2)) * kVLd + (col0 + (r16 & 3) * 4) * 2;
            float f[RG];
            bool any = false;
#pragma unroll
            for (int r = 0; r < RG; ++r) {
                f[r] = xf[rd & 1][r * 16 + r16];
                any = any || f[r] != 1.f;
            }
            if (__any(any)) {
#pragma unroll
                for (int c = 0; c < 8; ++c)
#pragma unroll
                    for (int r = 0; r < RG; ++r) acc[c][r] *= f[r];
            }
            u32x4 pf[RG][N];
#pragma unroll
            for (int r = 0; r < RG; ++r)
#pragma unroll
                for (int x = 0; x < N; ++x) pf[r][x] = *reinterpret_cast<const u32x4 *>(p + r * kPLd + x * 1024);
            // the columns' operands are read two tiles ahead; nothing moves across a tile (that costs registers)
            auto column = [&](int c) __attribute__((always_inline)) {
                const s4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(v + c * 32));
                const s4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(v + c * 32 + 16 * kVLd));
                return __builtin_bit_cast(u32x4, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            u32x4 vf[2] = {column(0), column(1)};
#pragma unroll
            for (int c = 0; c < 8; ++c) {
#pragma unroll
                for (int t = N - 1; t >= 0; --t)
#pragma unroll
                    for (int r = 0; r < RG; ++r)
                        acc[c][r] = kBf ? q4_mfma_bf16(vf[c & 1], pf[r][t], acc[c][r]) : q4_mfma_f16(vf[c & 1], pf[r][t], acc[c][r]);
                if (c + 2 < 8) vf[c & 1] = column(c + 2);
                // the next round's values are decoded while the matrix cores work on this one's
                if (c == 1 || c == 4) store_v(rd + 1, c / 4, bf);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto all = [&](auto bf) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int r = 0; r < RG; ++r) acc[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
            constexpr bool kLook = !decltype(bf)::value;
            Stage g[2];
            load(g[0], 0);
            load(g[1], 1);
            __syncthreads();
            store_k(g[0], 0, kLook);
            load(g[0], 2);
            __syncthreads();
            // store round i + 1's codes (loaded two iterations before), load round i + 3, decode round i - 1, take round
            // i - 2's products
            auto stage = [&](int i, auto par) __attribute__((always_inline)) {
                constexpr int d = decltype(par)::value;
                store_k(g[1 - d], i + 1, kLook);
                load(g[1 - d], i + 3);
            };
            stage(0, even);
            __syncthreads();
            stage(1, odd);
            store_v(0, 0, bf);
            store_v(0, 1, bf);
            __syncthreads();
            for (int i = 2; i < iters; i += 2) {
                stage(i, even);
                context(i - 2, bf);
                __syncthreads();
                stage(i + 1, odd);
                context(i - 1, bf);
                __syncthreads();
            }
        };
        all(std::false_type{});
        if (__builtin_amdgcn_readfirstlane(wide)) all(std::true_type{});
        __syncthreads();
        float *part = a.part + ((static_cast<int64_t>(b) * a.NS + split) * a.rows + row0) * kQ4Lat + col0 + 4 * q4;
#pragma unroll
        for (int r = 0; r < RG; ++r) {
            if (row0 + r * 16 + r16 >= a.rows) continue;
#pragma unroll
            for (int c = 0; c < 8; ++c)
                *reinterpret_cast<f32x4 *>(part + static_cast<int64_t>(r * 16 + r16) * kQ4Lat + c * 16) = acc[c][r];
        }
    }
}

// ------------------------------------------------------------------ uv
struct UvArgs {
    const float *part;
    const float2 *ml;
    const uint16_t *w_uv;    // [H, V, 512]
    float *opart;            // [4][M][H][V], or null: out
    void *out;               // [B, Tall, H, V]
    int out_bf16;
    const float *gate;       // [B, Tall, H, V] or null
    float2 *stats;           // [B][rows]: maximum less kLift, 1 / sum (which is lifted); or null
    int H, T, M, V, rows, NS, Tall, t0;
};
constexpr int kMaxSplits = 256;

__device__ __forceinline__ void store_out4(void *out, int bf16, const float *gate, int64_t at, f32x4 v) {
    if (gate) {
        const f32x4 g = *reinterpret_cast<const f32x4 *>(gate + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = v[i] / (1.0f + expf(-g[i]));
    }
    if (bf16)
        *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(out) + at) = u32x2{q4_pack_bf16(v[0], v[1]), q4_pack_bf16(v[2], v[3])};
    else
        *reinterpret_cast<f32x4 *>(static_cast<float *>(out) + at) = v;
}

// grid (H, ceil(M / 16), 512 / CP): queries 16 y .. +16 of head x over the latent columns CP z .. +CP
//   join    ctx = sum_s 2^(m_s - M) ctx_s / L, the splits in a fixed order (few queries: eight groups of splits, added
//           in group order)
//   W_UV    fp32 contexts as three bf16 terms
template <int CP>
__global__ __launch_bounds__(256) void uv_kernel(UvArgs a) {
    constexpr int kLd = CP + 4;
    extern __shared__ __attribute__((aligned(16))) float sm[];
    float *const ctx = sm, *const wsp = sm + 16 * kLd, *const red = wsp + 16 * a.NS;   // red: 8 x CP, few queries
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, q4 = lane >> 4;
    const int h = blockIdx.x, m0 = blockIdx.y * 16, col0 = blockIdx.z * CP;
    const int nv = min(16, a.M - m0);
    for (int i = wave; i < nv; i += 4) {
        const int m = m0 + i, b = m / a.T, row = (m % a.T) * a.H + h;
        const float2 *ml = a.ml + static_cast<int64_t>(b) * a.NS * a.rows + row;
        float2 v[kMaxSplits / 64];
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < kMaxSplits / 64; ++u) {
            const int s = lane + 64 * u;
            v[u] = s < a.NS ? ml[static_cast<int64_t>(s) * a.rows] : make_float2(-INFINITY, 0.f);
            mx = fmaxf(mx, v[u].x);
        }
        mx = wave_max_all(mx);
        float l = 0.f, e[kMaxSplits / 64];
#pragma unroll
        for (int u = 0; u < kMaxSplits / 64; ++u) {
            // (a split the row sees nothing of has no record: its weight is zero, whatever the maximum is)
            e[u] = v[u].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(v[u].x - mx);
            l = fmaf(e[u], v[u].y == 0.f ? 0.f : v[u].y, l);
        }
        l = wave_sum_all(l);
        const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
        for (int u = 0; u < kMaxSplits / 64; ++u) {
            const int s = lane + 64 * u;
            if (s < a.NS) wsp[i * a.NS + s] = v[u].y == 0.f ? 0.f : e[u] * inv;
        }
        if (a.stats && blockIdx.z == 0 && lane == 0) a.stats[static_cast<int64_t>(b) * a.rows + row] = make_float2(mx - kLift, inv);
    }
    __syncthreads();
    constexpr int kC4 = CP / 4, kG = 256 / kC4;     // threads across the columns; groups of threads
    const int c4 = tid % kC4, gr = tid / kC4;
    int np = 1;                                     // groups that take different queries
    while (np < nv && np < kG) np *= 2;
    const int sg = gr / np, ns = kG / np;
    for (int i0 = 0; i0 < nv; i0 += np) {
        const int i = i0 + gr % np;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        if (i < nv) {
            const int m = m0 + i, b = m / a.T, row = (m % a.T) * a.H + h;
            const float *src = a.part + (static_cast<int64_t>(b) * a.NS * a.rows + row) * kQ4Lat + col0 + 4 * c4;
            for (int j = sg; j < a.NS; j += 4 * ns) {
                f32x4 x[4];
                float wgt[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int k = j + u * ns;
                    wgt[u] = k < a.NS ? wsp[i * a.NS + k] : 0.f;
                    x[u] = wgt[u] != 0.f ? *reinterpret_cast<const f32x4 *>(src + static_cast<int64_t>(k) * a.rows * kQ4Lat)
                                         : f32x4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) s += x[u] * wgt[u];
            }
        }
        if (ns == 1) {
            if (i < nv) *reinterpret_cast<f32x4 *>(ctx + i * kLd + 4 * c4) = s;
        } else {
            *reinterpret_cast<f32x4 *>(red + gr * CP + 4 * c4) = s;
            __syncthreads();
            if (gr < np && i0 + gr < nv) {
                f32x4 t = *reinterpret_cast<const f32x4 *>(red + gr * CP + 4 * c4);
                for (int k = 1; k < ns; ++k) t += *reinterpret_cast<const f32x4 *>(red + (k * np + gr) * CP + 4 * c4);
                *reinterpret_cast<f32x4 *>(ctx + (i0 + gr) * kLd + 4 * c4) = t;
            }
            __syncthreads();
        }
    }
    for (int i = tid; i < (16 - nv) * CP; i += 256) ctx[(nv + i / CP) * kLd + i % CP] = 0.f;   // queries past the last
    __syncthreads();
    u32x4 cf[CP / 32][3];
#pragma unroll
    for (int k = 0; k < CP / 32; ++k) {
        const f32x4 x = *reinterpret_cast<const f32x4 *>(ctx + r16 * kLd + k * 32 + 8 * q4);
        const f32x4 y = *reinterpret_cast<const f32x4 *>(ctx + r16 * kLd + k * 32 + 8 * q4 + 4);
        const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        terms8(v, cf[k]);
    }
    const int m = m0 + r16;
    const int64_t at = m < a.M ? ((static_cast<int64_t>(m / a.T) * a.Tall + a.t0 + m % a.T) * a.H + h) * a.V : 0;
    for (int vt = wave; vt * 16 < a.V; vt += 4) {
        const int v = vt * 16 + r16;
        const uint16_t *wr = a.w_uv + (static_cast<int64_t>(h) * a.V + v) * kQ4Lat + col0 + 8 * q4;
        f32x4 d = {0.f, 0.f, 0.f, 0.f}, dl = d;
#pragma unroll
        for (int k = 0; k < CP / 32; ++k) {
            const u32x4 wf = v < a.V ? *reinterpret_cast<const u32x4 *>(wr + k * 32) : u32x4{0u, 0u, 0u, 0u};
            dl = q4_mfma_bf16(wf, cf[k][2], dl);
            dl = q4_mfma_bf16(wf, cf[k][1], dl);
            d = q4_mfma_bf16(wf, cf[k][0], d);
        }
        d += dl;
        if (m >= a.M || vt * 16 + 4 * q4 >= a.V) continue;
        if (a.opart)
            *reinterpret_cast<f32x4 *>(a.opart + ((static_cast<int64_t>(blockIdx.z) * a.M + m) * a.H + h) * a.V + vt * 16 + 4 * q4) = d;
        else
            store_out4(a.out, a.out_bf16, a.gate, at + vt * 16 + 4 * q4, d);
    }
}

// o = the four column quarters' products in order (then the output gate); four values a thread
__global__ __launch_bounds__(256) void out_kernel(UvArgs a) {
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
    const int64_t hv = static_cast<int64_t>(a.H) * a.V, n = a.M * hv;
    if (i >= n) return;
    f32x4 o = *reinterpret_cast<const f32x4 *>(a.opart + i);
#pragma unroll
    for (int q = 1; q < 4; ++q) o += *reinterpret_cast<const f32x4 *>(a.opart + q * n + i);
    const int64_t m = i / hv;
    store_out4(a.out, a.out_bf16, a.gate, ((m / a.T) * a.Tall + a.t0 + m % a.T) * hv + i % hv, o);
}

// ------------------------------------------------------------------ weights
struct WeightArgs {
    AttendArgs a;
    const float2 *stats;     // [B][rows]
    float *part;             // [chunks][B][npos]
    float *weight;           // [B] rows of w_b floats
    int64_t w_b;
    int tiles, chunk, chunks, npos;
};
constexpr int kWTiles = 4;   // tiles of 16 positions per wave

// grid (ceil(npos / 512), chunks, B): a wave keeps 64 positions' codes in registers and takes the row tiles
// chunk y .. of its sequence, adding their probabilities; part[chunk][b][position]
template <int NT, int RT>
__global__ __launch_bounds__(512, 1) void weights_kernel(WeightArgs wa) {
    const AttendArgs &a = wa.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q4 = lane >> 4;
    const int b = blockIdx.z, j0 = (blockIdx.x * 8 + wave) * (16 * kWTiles);
    if (j0 >= wa.npos) return;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.cap) : a.length;
    const int cnt = a.counts ? min(max(a.counts[b], 0), a.count) : a.count;
    const int n = len - j0;                        // positions there are from j0 on
    f32x4 sum[kWTiles];
#pragma unroll
    for (int u = 0; u < kWTiles; ++u) sum[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int first = blockIdx.y * wa.chunk, last = min(wa.tiles, first + wa.chunk);
    if (n > 0) {
        const auto rp = make_rsrc(a.packed + b * a.p_b + j0 * a.p_t, static_cast<uint32_t>(min(n - 1, 16 * kWTiles - 1) * a.p_t + 256));
        const auto rs = make_rsrc(a.scales + b * a.s_b + j0 * a.s_t, static_cast<uint32_t>(min(n - 1, 16 * kWTiles - 1) * a.s_t + 16));
        const auto rr = make_rsrc(a.rot + b * a.r_b + j0 * a.r_t, static_cast<uint32_t>(min(n - 1, 16 * kWTiles - 1) * a.r_t + 128));
        u32x4 kc[kWTiles][kQ4Steps], ro[kWTiles][2];
        int ks[kWTiles];
#pragma unroll
        for (int u = 0; u < kWTiles; ++u) {
            const int j = u * 16 + r16;
            const bool ok = j < n;
#pragma unroll
            for (int s = 0; s < kQ4Steps; ++s)
                kc[u][s] = __builtin_bit_cast(u32x4, buf_load16(rp, ok ? static_cast<uint32_t>(j) * static_cast<uint32_t>(a.p_t) + q4 * 64u + s * 16u : kOobOffset));
#pragma unroll
            for (int s = 0; s < 2; ++s)
                ro[u][s] = __builtin_bit_cast(u32x4, buf_load16(rr, ok ? static_cast<uint32_t>(j) * static_cast<uint32_t>(a.r_t) + s * 64u + q4 * 16u : kOobOffset));
            uint32_t k4 = 0;
#pragma unroll
            for (int s = 0; s < kQ4Steps; ++s)
                k4 |= static_cast<uint32_t>(__builtin_amdgcn_raw_buffer_load_b8(
                          rs, ok ? static_cast<uint32_t>(j) * static_cast<uint32_t>(a.s_t) + q4 * 4u + s : kOobOffset, 0, 0)) << (8 * s);
            ks[u] = static_cast<int>(k4);
        }
        for (int i = first; i < last; ++i) {
            const int tlast = min(a.t0 + (min(i * 16 + 16, a.rows) - 1) / a.H, cnt - 1);
            if (q4_sees(tlast, cnt, len) <= j0) continue;    // (tlast < t0: no query of the tile is there, and its rows see nothing)
            const int row = i * 16 + r16;
            const int limit = (row < a.rows ? q4_sees(a.t0 + row / a.H, cnt, len) : 0) - j0;
            const float2 st = row < a.rows ? wa.stats[static_cast<int64_t>(b) * a.rows + row] : make_float2(0.f, 0.f);
            const char *tile = a.qop + b * a.q_seq + static_cast<int64_t>(i) * q4_tile_bytes(NT, RT);
            f32x4 hi[kWTiles], lo[kWTiles];
#pragma unroll
            for (int u = 0; u < kWTiles; ++u) hi[u] = lo[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = RT - 1; x >= 0; --x)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const u32x4 qr = *reinterpret_cast<const u32x4 *>(tile + q4_rope_at(NT, x, s) + lane * 16);
#pragma unroll
                    for (int u = 0; u < kWTiles; ++u) lo[u] = q4_mfma_bf16(ro[u][s], qr, lo[u]);
                }
#pragma unroll
            for (int x = NT - 1; x >= 0; --x) {
                const int qs = *reinterpret_cast<const int *>(tile + q4_scale_at(NT, x) + lane * 4);
                u32x4 qlo[kQ4Steps];
                u32x2 qhi[kQ4Steps];
#pragma unroll
                for (int s = 0; s < kQ4Steps; ++s) {
                    qlo[s] = *reinterpret_cast<const u32x4 *>(tile + q4_code_at(x, s) + lane * 16);
                    qhi[s] = *reinterpret_cast<const u32x2 *>(tile + q4_code_at(x, s) + 1024 + lane * 8);
                }
#pragma unroll
                for (int u = 0; u < kWTiles; ++u) {
                    f32x4 &d = x < 2 ? hi[u] : lo[u];
                    d = q4_mfma<0>(kc[u][0], ks[u], qlo[0], qhi[0], qs, d);
                    d = q4_mfma<1>(kc[u][1], ks[u], qlo[1], qhi[1], qs, d);
                    d = q4_mfma<2>(kc[u][2], ks[u], qlo[2], qhi[2], qs, d);
                    d = q4_mfma<3>(kc[u][3], ks[u], qlo[3], qhi[3], qs, d);
                }
            }
#pragma unroll
            for (int u = 0; u < kWTiles; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float p = __builtin_amdgcn_exp2f((hi[u][v] + lo[u][v]) * a.c - st.x) * st.y;
                    sum[u][v] += u * 16 + 4 * q4 + v < limit ? p : 0.f;
                }
        }
    }
    // over the 16 rows of the tiles (lanes of a DPP row), in a fixed order
    float *out = wa.part + (static_cast<int64_t>(blockIdx.y) * a.B + b) * wa.npos + j0;
#pragma unroll
    for (int u = 0; u < kWTiles; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            float p = sum[u][v];
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) p += __shfl_xor(p, o);
            const int j = u * 16 + 4 * q4 + v;
            if (r16 == 0 && j0 + j < wa.npos) out[j] = p;
        }
}

// weight[b][j] += the chunks' sums in order
__global__ __launch_bounds__(256) void weights_add_kernel(WeightArgs wa) {
    const int j = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
    if (j >= wa.npos) return;
    const int len = wa.a.lengths ? min(max(wa.a.lengths[b], 0), wa.a.cap) : wa.a.length;
    if (j >= len) return;
    float s = 0.f;
    for (int k = 0; k < wa.chunks; ++k) s += wa.part[(static_cast<int64_t>(k) * wa.a.B + b) * wa.npos + j];
    wa.weight[b * wa.w_b + j] += s;
}

// ------------------------------------------------------------------ host side
struct Plan {
    int NT, RT, PT, RG, T, rows, tiles, rblocks, Ts, NS, uv_quarters, chunk, chunks;
    int64_t qop, ml, part, stats, opart, wpart, total;
};

constexpr int64_t kChunkRows = 1 << 16;   // rows (heads x queries, all sequences) of one pass over the queries

// What the launches are cut into; a function of its arguments alone.
Plan plan_of(int64_t B, int64_t T, int64_t H, int64_t V, int64_t npos, int q_bf16, int out_bf16, int weights, int varied) {
    Plan p{};
    const bool fine = !out_bf16 || weights;
    p.NT = fine ? 5 : 3, p.RT = q_bf16 ? 1 : fine ? 3 : 2, p.PT = out_bf16 ? 1 : 2;
    p.T = static_cast<int>(std::max<int64_t>(1, std::min(T, kChunkRows / (B * H))));
    p.rows = static_cast<int>(p.T * H);
    p.RG = p.rows > 64 ? 4 : 2;
    p.rblocks = static_cast<int>(cdiv(p.rows, 16 * p.RG));
    p.tiles = p.rblocks * p.RG;
    const int64_t base = B * p.rblocks;
    // one block a CU; sequences of their own lengths: four, so the longest one's blocks are not what all wait for
    int64_t ns = std::max<int64_t>(1, std::min<int64_t>(kMaxSplits, (varied && B > 1 ? 1024 : 256) / base));
    int64_t ts = cdiv(cdiv(std::max<int64_t>(npos, 1), ns), kRound) * kRound;
    p.Ts = static_cast<int>(ts);
    p.NS = static_cast<int>(cdiv(std::max<int64_t>(npos, 1), ts));
    const int64_t M = B * p.T;
    p.uv_quarters = H * cdiv(M, 16) < 512;
    const int64_t pos_blocks = std::max<int64_t>(1, cdiv(npos, 128 * kWTiles));
    p.chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.tiles, 512 / (pos_blocks * B))));
    p.chunk = static_cast<int>(cdiv(p.tiles, p.chunks));
    p.chunks = static_cast<int>(cdiv(p.tiles, p.chunk));
    auto up = [](int64_t v) { return (v + 255) & ~int64_t(255); };
    int64_t o = 0;
    p.qop = o, o += up(B * p.tiles * q4_tile_bytes(p.NT, p.RT));
    p.ml = o, o += up(B * p.NS * p.rows * 8);
    p.part = o, o += up(B * p.NS * p.rows * kQ4Lat * 4);
    p.stats = o, o += weights ? up(B * p.rows * 8) : 0;
    p.opart = o, o += p.uv_quarters ? up(4 * M * H * V * 4) : 0;
    p.wpart = o, o += weights ? up(static_cast<int64_t>(p.chunks) * B * npos * 4) : 0;
    p.total = o;
    return p;
}

template <int RG, int NT, int RT, int PT>
int launch_attend(const AttendArgs &a, hipStream_t st) {
    constexpr int bytes = attend_lds(RG, RT, PT);
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(attend_kernel<RG, NT, RT, PT>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    const int rc = check_hip(attr, "mla q4: attention LDS size");
    if (rc) return rc;
    attend_kernel<RG, NT, RT, PT><<<dim3(static_cast<unsigned>(a.B * a.NS * a.rblocks)), 512, bytes, st>>>(a);
    return check_hip(hipGetLastError(), "mla q4: attention launch");
}

template <int RG>
int launch_attend_of(const AttendArgs &a, const Plan &p, hipStream_t st) {
    if (p.NT == 3) return p.RT == 1 ? launch_attend<RG, 3, 1, 1>(a, st) : launch_attend<RG, 3, 2, 1>(a, st);
    if (p.PT == 1) return p.RT == 1 ? launch_attend<RG, 5, 1, 1>(a, st) : launch_attend<RG, 5, 3, 1>(a, st);
    return p.RT == 1 ? launch_attend<RG, 5, 1, 2>(a, st) : launch_attend<RG, 5, 3, 2>(a, st);
}

template <typename QT, int NT, int RT>
int launch_qa(const QaArgs &a, hipStream_t st) {
    const int bytes = std::max(((a.nope + 31) / 32) * 32 * kWLd, 16 * kFLd * 4);
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(qa_kernel<QT, NT, RT>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, 256 * kWLd);
    const int rc = check_hip(attr, "mla q4: query LDS size");
    if (rc) return rc;
    qa_kernel<QT, NT, RT><<<dim3(a.H, static_cast<unsigned>(cdiv(a.M, 16)), 4), 256, bytes, st>>>(a);
    return check_hip(hipGetLastError(), "mla q4: query launch");
}

template <int CP>
int launch_uv(const UvArgs &a, hipStream_t st) {
    const int bytes = (16 * (CP + 4) + 16 * a.NS + 8 * CP) * 4;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(uv_kernel<CP>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, (24 * (CP + 4) + 16 * kMaxSplits) * 4);
    const int rc = check_hip(attr, "mla q4: output LDS size");
    if (rc) return rc;
    uv_kernel<CP><<<dim3(a.H, static_cast<unsigned>(cdiv(a.M, 16)), kQ4Lat / CP), 256, bytes, st>>>(a);
    return check_hip(hipGetLastError(), "mla q4: join and W_UV launch");
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" int64_t k3_mla_q4_workspace_size(int64_t B, int64_t T, int64_t H, int64_t v_dim, int64_t max_length, int q_dtype,
                                            int out_dtype, int weights, int varied) {
    if (B <= 0 || T <= 0 || H <= 0 || v_dim <= 0 || max_length < 0) return 0;
    return plan_of(B, T, H, v_dim, max_length, q_dtype == K3_BF16, out_dtype == K3_BF16, weights != 0, varied != 0).total;
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
    if (max_length > 0 && (p_row < 256 || p_row % 16 || p_batch % 16 || s_row < 16 || rot_row < kQ4Rope || rot_row % 8 ||
                           rot_batch % 8 || p_row > (1 << 16) || s_row > (1 << 16) || rot_row > (1 << 15)))
        return set_error(K3_ERR_SHAPE, "mla q4: cache row pitches too small, too large or not multiples of 16 bytes");
    if (!aligned16(q_nope) || !aligned16(q_rot) || !aligned16(w_uk) || !aligned16(w_uv) || !aligned16(out) || !aligned16(workspace) ||
        !aligned16(packed) || !aligned16(rot) || (gate && !aligned16(gate)))
        return set_error(K3_ERR_ALIGN, "mla q4: queries, weights, cache, output and workspace must be 16-byte aligned");
    const Plan p = plan_of(B, T, H, v_dim, max_length, q_dtype == K3_BF16, out_dtype == K3_BF16, weight != nullptr, lengths != nullptr);
    if (workspace_bytes < p.total)
        return set_error(K3_ERR_WORKSPACE, "mla q4: workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)p.total);
    if (static_cast<int64_t>(p.Ts) * std::max(p_row, 2 * rot_row) >= (1ll << 31))
        return set_error(K3_ERR_SHAPE, "mla q4: a split of %d positions spans 2 GiB", p.Ts);
    auto st = static_cast<hipStream_t>(stream);
    char *ws = static_cast<char *>(workspace);
    for (int64_t t0 = 0; t0 < T; t0 += p.T) {
        const int Tc = static_cast<int>(std::min<int64_t>(p.T, T - t0));
        const int rows = static_cast<int>(Tc * H), rblocks = static_cast<int>(cdiv(rows, 16 * p.RG));
        const int64_t q_seq = static_cast<int64_t>(p.tiles) * q4_tile_bytes(p.NT, p.RT);
        QaArgs qa{q_nope, q_rot, qn_batch, qn_token, qn_head, qr_batch, qr_token, qr_head, static_cast<const uint16_t *>(w_uk),
                  ws + p.qop, q_seq, static_cast<int>(H), static_cast<int>(nope_dim), Tc, static_cast<int>(B * Tc), static_cast<int>(t0)};
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
        a.part = reinterpret_cast<float *>(ws + p.part), a.ml = reinterpret_cast<float2 *>(ws + p.ml);
        a.H = static_cast<int>(H), a.T = Tc, a.t0 = static_cast<int>(t0), a.rows = rows, a.Ts = p.Ts, a.NS = p.NS, a.rblocks = rblocks;
        a.B = static_cast<int>(B), a.c = scale * 1.4426950408889634f;
        a.swizzle = (a.B * a.NS * rblocks) % 8 == 0;
        rc = p.RG == 4 ? launch_attend_of<4>(a, p, st) : launch_attend_of<2>(a, p, st);
        if (rc) return rc;
        UvArgs u{};
        u.part = a.part, u.ml = a.ml, u.w_uv = static_cast<const uint16_t *>(w_uv);
        u.opart = p.uv_quarters ? reinterpret_cast<float *>(ws + p.opart) : nullptr;
        u.out = out, u.out_bf16 = out_dtype == K3_BF16, u.gate = gate;
        u.stats = weight ? reinterpret_cast<float2 *>(ws + p.stats) : nullptr;
        u.H = a.H, u.T = Tc, u.M = static_cast<int>(B * Tc), u.V = static_cast<int>(v_dim), u.rows = rows, u.NS = p.NS;
        u.Tall = static_cast<int>(T), u.t0 = a.t0;
        rc = p.uv_quarters ? launch_uv<128>(u, st) : launch_uv<512>(u, st);
        if (rc) return rc;
        if (p.uv_quarters) {
            out_kernel<<<dim3(static_cast<unsigned>(cdiv(static_cast<int64_t>(u.M) * H * v_dim, 1024))), 256, 0, st>>>(u);
            rc = check_hip(hipGetLastError(), "mla q4: output launch");
            if (rc) return rc;
        }
        if (weight && max_length > 0) {
            WeightArgs wa{a, u.stats, reinterpret_cast<float *>(ws + p.wpart), weight, w_batch, static_cast<int>(cdiv(rows, 16)), p.chunk,
                          0, static_cast<int>(max_length)};
            wa.chunks = static_cast<int>(cdiv(wa.tiles, wa.chunk));
            const dim3 grid(static_cast<unsigned>(cdiv(max_length, 128 * kWTiles)), static_cast<unsigned>(wa.chunks), static_cast<unsigned>(B));
            if (p.RT == 1)
                weights_kernel<5, 1><<<grid, 512, 0, st>>>(wa);
            else
                weights_kernel<5, 3><<<grid, 512, 0, st>>>(wa);
            rc = check_hip(hipGetLastError(), "mla q4: weights launch");
            if (rc) return rc;
            weights_add_kernel<<<dim3(static_cast<unsigned>(cdiv(max_length, 256)), static_cast<unsigned>(B)), 256, 0, st>>>(wa);
            rc = check_hip(hipGetLastError(), "mla q4: weight sum launch");
            if (rc) return rc;
        }
    }
    return K3_OK;
}
