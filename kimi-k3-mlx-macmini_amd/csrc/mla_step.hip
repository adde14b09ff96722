// One decode token through a whole MLA layer at batch 1: the projections on either side
// of the absorbed attention core, the latent-cache append and the output gate.
//
// Reference: MLAAttention.__call__ (air_llm/models/kimi_k3/attention_mla.py:168-216):
//   q   = rmsnorm(x @ q_a.T, q_a_layernorm) @ q_b.T                  -> [H, nope + rope]
//   ckv = x @ kv_a.T;  c_new = rmsnorm(ckv[:r], kv_a_layernorm);  r_new = ckv[r:]
//   cache.append(c_new, r_new)                                      (attention_mla.py:89-108)
//   o   = absorbed attention core over the cache                     (attention_mla.py:193-212)
//   o   = o * sigmoid(x @ g_proj.T)  (mla_use_output_gate);  out = o @ o_proj.T
//
// Seven stream-ordered launches, no host synchronisation:
//   S1  rows of q_a, kv_a and g_proj against x (one grid, three block ranges);
//   S2  rows of q_b against the normalised q_a output (every block normalises the 1536-wide
//       vector itself, so no launch is spent on it), and one block that normalises the kv
//       latent and writes the new cache row (bf16) at position pos;
//   core  the absorbed core of k3_mla_decode_absorbed (four launches) over the pos + 1
//       cache rows, its last launch multiplying o by sigmoid(gate) as it writes it;
//   S3  rows of o_proj against the gated o.
// The row launches are the dense row kernels of dense_rows.h.
//
// Over the 4-bit cache (k3_mla_step_decode_q4) S2 leaves the cache row to a launch of its own, which normalises the latent and rounds
// it into its codes, and the core is k3_mla_q4_attention's for one query.
#include <algorithm>

#include "dense_rows.h"

namespace k3 {
namespace {

size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

struct StepWs {
    size_t qa, ckv, gl, q, o, core, total;
};

StepWs step_ws_layout(int64_t ql, int64_t H, int64_t nope, int64_t rope, int64_t v, int64_t r, int64_t core) {
    StepWs L{};
    size_t off = 0;
    L.qa = off, off += up256(ql * 4);
    L.ckv = off, off += up256((r + rope) * 4);
    L.gl = off, off += up256(H * v * 4);
    L.q = off, off += up256(H * (nope + rope) * 4);
    L.o = off, off += up256(H * v * 4);
    L.core = off, off += static_cast<size_t>(core);
    L.total = off;
    return L;
}

// the layer's operands, as both forms of the step take them
struct StepArgs {
    const void *x;
    int x_dtype;
    const void *q_a;
    const float *q_a_norm;
    const void *q_b, *kv_a;
    const float *kv_a_norm;
    const void *g_proj, *o_proj;
    int64_t cache_rows, pos;
    float eps;
    void *out;
    int out_dtype;
    int64_t hidden, ql, H, nope, rope, v, r;
    void *workspace;
};

int check_step(const StepArgs &a) {
    if (!a.x || !a.q_a || !a.q_a_norm || !a.q_b || !a.kv_a || !a.kv_a_norm || !a.o_proj || !a.out || !a.workspace)
        return set_error(K3_ERR_NULL, "mla step: null pointer");
    if (a.x_dtype != K3_F32 && a.x_dtype != K3_BF16) return set_error(K3_ERR_DTYPE, "mla step: x_dtype %d", a.x_dtype);
    if (a.out_dtype != K3_F32 && a.out_dtype != K3_BF16) return set_error(K3_ERR_DTYPE, "mla step: out_dtype %d", a.out_dtype);
    const int64_t qhd = a.nope + a.rope, hv = a.H * a.v;
    if (a.hidden <= 0 || a.hidden % 8 || a.ql <= 0 || a.ql % 8 || hv <= 0 || hv % 8 || a.hidden > kMaxWidth || a.ql > kMaxWidth ||
        hv > kMaxWidth || a.r % 4 || a.rope % 4)
        return set_error(K3_ERR_SHAPE, "mla step: hidden, q_lora_rank and heads*v must be multiples of 8, <= %d",
                         kMaxWidth);
    if (a.pos < 0 || a.pos >= a.cache_rows)
        return set_error(K3_ERR_SHAPE, "mla step: position %lld outside the cache's %lld rows", (long long)a.pos,
                         (long long)a.cache_rows);
    if (!aligned16(a.x) || !aligned16(a.q_a) || !aligned16(a.q_b) || !aligned16(a.kv_a) || !aligned16(a.o_proj) ||
        (a.g_proj && !aligned16(a.g_proj)) || !aligned16(a.q_a_norm) || !aligned16(a.kv_a_norm) || !aligned16(a.workspace))
        return set_error(K3_ERR_ALIGN, "mla step: vectors, weights and workspace must be 16-byte aligned");
    if (a.H * qhd * a.ql * 2 >= (1ll << 31) || a.hidden * hv * 2 >= (1ll << 31) || a.ql * a.hidden * 2 >= (1ll << 31))
        return set_error(K3_ERR_SHAPE, "mla step: a weight matrix exceeds 2 GiB");
    return K3_OK;
}

// S1 and S2: q, the gate's logits and the latent before its norm, in the workspace; lat_row, rot_row: the bf16 cache row to
// write, or null
int step_front(const StepArgs &s, const StepWs &L, uint16_t *lat_row, uint16_t *rot_row, hipStream_t st) {
    char *ws = static_cast<char *>(s.workspace);
    float *qa = reinterpret_cast<float *>(ws + L.qa), *ckv = reinterpret_cast<float *>(ws + L.ckv);
    // S1: q_a, kv_a, g_proj rows against x
    RowsArgs a{};
    a.x = s.x;
    a.x_bf16 = s.x_dtype == K3_BF16;
    a.K = static_cast<int>(s.hidden);
    a.w[0] = static_cast<const uint16_t *>(s.q_a), a.N[0] = static_cast<int>(s.ql), a.y[0] = qa;
    a.w[1] = static_cast<const uint16_t *>(s.kv_a), a.N[1] = static_cast<int>(s.r + s.rope), a.y[1] = ckv;
    a.w[2] = static_cast<const uint16_t *>(s.g_proj), a.N[2] = s.g_proj ? static_cast<int>(s.H * s.v) : 0;
    a.y[2] = reinterpret_cast<float *>(ws + L.gl);
    const int rc = launch_rows<kModeX>(a, st);
    if (rc) return rc;
    // S2: q_b rows against the normalised q_a output; the cache row
    RowsArgs b{};
    b.src = qa, b.nw = s.q_a_norm, b.eps = s.eps, b.K = static_cast<int>(s.ql);
    b.w[0] = static_cast<const uint16_t *>(s.q_b), b.N[0] = static_cast<int>(s.H * (s.nope + s.rope));
    b.y[0] = reinterpret_cast<float *>(ws + L.q);
    b.ckv = ckv, b.kvw = s.kv_a_norm;
    b.lat_row = lat_row, b.rot_row = rot_row;
    b.r = static_cast<int>(s.r), b.rope = static_cast<int>(s.rope), b.append = lat_row != nullptr;
    return launch_rows<kModeNorm>(b, st);
}

// S3: o_proj rows against the gated o
int step_back(const StepArgs &s, const StepWs &L, hipStream_t st) {
    RowsArgs c{};
    c.o = reinterpret_cast<float *>(static_cast<char *>(s.workspace) + L.o), c.gl = nullptr, c.K = static_cast<int>(s.H * s.v);
    c.w[0] = static_cast<const uint16_t *>(s.o_proj), c.N[0] = static_cast<int>(s.hidden);
    c.out = s.out, c.out_bf16 = s.out_dtype == K3_BF16;
    return launch_rows<kModeGate>(c, st);
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" int64_t k3_mla_step_workspace_size(int64_t hidden, int64_t q_lora_rank, int64_t heads, int64_t nope_dim,
                                              int64_t rope_dim, int64_t v_dim, int64_t kv_lora_rank, int64_t T) {
    (void)hidden;
    return static_cast<int64_t>(
        step_ws_layout(q_lora_rank, heads, nope_dim, rope_dim, v_dim, kv_lora_rank, k3_mla_workspace_size(heads, T)).total);
}

extern "C" int k3_mla_step_decode(const void *x, int x_dtype, const void *q_a, const float *q_a_norm, const void *q_b,
                                  const void *kv_a, const float *kv_a_norm, const void *w_uk, const void *w_uv,
                                  const void *g_proj, const void *o_proj, void *lat, int64_t ld_lat, void *rot,
                                  int64_t ld_rot, int64_t cache_rows, int64_t pos, float eps, float scale, void *out,
                                  int out_dtype,
                                  int64_t hidden, int64_t q_lora_rank, int64_t heads, int64_t nope_dim,
                                  int64_t rope_dim, int64_t v_dim, int64_t kv_lora_rank, void *workspace,
                                  int64_t workspace_bytes, void *stream) {
    const StepArgs s{x,      x_dtype,     q_a,   q_a_norm, q_b,      kv_a,     kv_a_norm, g_proj,       o_proj,   cache_rows, pos, eps, out, out_dtype,
                     hidden, q_lora_rank, heads, nope_dim, rope_dim, v_dim,    kv_lora_rank, workspace};
    if (!w_uk || !w_uv || !lat || !rot) return set_error(K3_ERR_NULL, "mla step: null pointer");
    int rc = check_step(s);
    if (rc) return rc;
    const int64_t T = pos + 1, qhd = nope_dim + rope_dim;
    const StepWs L = step_ws_layout(q_lora_rank, heads, nope_dim, rope_dim, v_dim, kv_lora_rank, k3_mla_workspace_size(heads, T));
    if (workspace_bytes < static_cast<int64_t>(L.total))
        return set_error(K3_ERR_WORKSPACE, "mla step: workspace %lld < %zu bytes", (long long)workspace_bytes, L.total);
    char *ws = static_cast<char *>(workspace);
    const float *q = reinterpret_cast<float *>(ws + L.q);
    auto st = static_cast<hipStream_t>(stream);
    rc = step_front(s, L, static_cast<uint16_t *>(lat) + pos * ld_lat, static_cast<uint16_t *>(rot) + pos * ld_rot, st);
    if (rc) return rc;
    // core over the pos + 1 cache rows
    rc = mla_decode_core(q, q + nope_dim, qhd, qhd, K3_F32, w_uk, w_uv, lat, ld_lat, rot, ld_rot, T, heads,
                         kv_lora_rank, rope_dim, nope_dim, v_dim, scale, ws + L.o, K3_F32, v_dim,
                         g_proj ? reinterpret_cast<float *>(ws + L.gl) : nullptr,
                         ws + L.core, workspace_bytes - static_cast<int64_t>(L.core), stream);
    return rc ? rc : step_back(s, L, st);
}

extern "C" int64_t k3_mla_step_q4_workspace_size(int64_t q_lora_rank, int64_t heads, int64_t nope_dim, int64_t rope_dim, int64_t v_dim,
                                                 int64_t kv_lora_rank, int64_t T, int weights) {
    return static_cast<int64_t>(step_ws_layout(q_lora_rank, heads, nope_dim, rope_dim, v_dim, kv_lora_rank,
                                               k3_mla_q4_workspace_size(1, 1, heads, v_dim, T, K3_F32, K3_F32, weights, 0))
                                    .total);
}

extern "C" int k3_mla_step_decode_q4(const void *x, int x_dtype, const void *q_a, const float *q_a_norm, const void *q_b,
                                     const void *kv_a, const float *kv_a_norm, const void *w_uk, const void *w_uv,
                                     const void *g_proj, const void *o_proj, void *packed, int64_t p_row, void *scales, int64_t s_row,
                                     void *rot, int64_t rot_row, float *weight, int64_t cache_rows, int64_t pos, float eps, float scale,
                                     void *out, int out_dtype, int64_t hidden, int64_t q_lora_rank, int64_t heads, int64_t nope_dim,
                                     int64_t rope_dim, int64_t v_dim, int64_t kv_lora_rank, void *workspace, int64_t workspace_bytes,
                                     void *stream) {
    const StepArgs s{x,      x_dtype,     q_a,   q_a_norm, q_b,      kv_a,     kv_a_norm, g_proj,       o_proj,   cache_rows, pos, eps, out, out_dtype,
                     hidden, q_lora_rank, heads, nope_dim, rope_dim, v_dim,    kv_lora_rank, workspace};
    if (!w_uk || !w_uv || !packed || !scales || !rot) return set_error(K3_ERR_NULL, "mla step: null pointer");
    int rc = check_step(s);
    if (rc) return rc;
    // (what the core would refuse, before the cache row is written)
    if (kv_lora_rank != 512 || rope_dim != 64 || nope_dim % 8 || nope_dim <= 0 || nope_dim > 256 || v_dim % 8 || v_dim > 1024 ||
        heads > 4096 || cache_rows > (1 << 24))
        return set_error(K3_ERR_SHAPE, "mla step: the 4-bit cache takes kv_lora_rank 512, rope 64, nope up to 256, v up to 1024");
    // (pitches up to 1 KB: then no range of positions that the core takes spans 2 GiB, which it would refuse)
    if (p_row < 256 || p_row % 16 || p_row > 1024 || s_row < 16 || s_row % 4 || s_row > 1024 || rot_row < 64 || rot_row % 8 || rot_row > 512)
        return set_error(K3_ERR_SHAPE, "mla step: cache row pitches too small, too large or not multiples of 16 bytes");
    if (!aligned16(packed) || !aligned16(rot) || (reinterpret_cast<uintptr_t>(scales) & 3u) || !aligned16(w_uk) || !aligned16(w_uv))
        return set_error(K3_ERR_ALIGN, "mla step: cache and weights must be 16-byte (scales 4-byte) aligned");
    const int64_t T = pos + 1, qhd = nope_dim + rope_dim;
    const StepWs L = step_ws_layout(q_lora_rank, heads, nope_dim, rope_dim, v_dim, kv_lora_rank,
                                    k3_mla_q4_workspace_size(1, 1, heads, v_dim, T, K3_F32, K3_F32, weight != nullptr, 0));
    if (workspace_bytes < static_cast<int64_t>(L.total))
        return set_error(K3_ERR_WORKSPACE, "mla step: workspace %lld < %zu bytes", (long long)workspace_bytes, L.total);
    char *ws = static_cast<char *>(workspace);
    const float *q = reinterpret_cast<float *>(ws + L.q), *ckv = reinterpret_cast<float *>(ws + L.ckv);
    auto st = static_cast<hipStream_t>(stream);
    rc = step_front(s, L, nullptr, nullptr, st);
    if (rc) return rc;
    rc = mla_q4_append(ckv, 0, 0, K3_F32, ckv + kv_lora_rank, 0, 0, K3_F32, kv_a_norm, eps, packed, 0, p_row, scales, 0, s_row, rot, 0,
                       rot_row, nullptr, pos, nullptr, weight, 0, 1, 1, cache_rows, st);
    if (rc) return rc;
    rc = k3_mla_q4_attention(q, 0, 0, qhd, q + nope_dim, 0, 0, qhd, K3_F32, w_uk, w_uv, packed, 0, p_row, scales, 0, s_row, rot, 0, rot_row,
                             nullptr, nullptr, T, 1, 1, heads, kv_lora_rank, rope_dim, nope_dim, v_dim, scale,
                             g_proj ? reinterpret_cast<float *>(ws + L.gl) : nullptr, ws + L.o, K3_F32, weight, 0, ws + L.core,
                             workspace_bytes - static_cast<int64_t>(L.core), stream);
    return rc ? rc : step_back(s, L, st);
}
