"""The MLA layer over the 4-bit cache (cfg.mla_cache_bits = 4): prompts, decode steps, batches, growth and eviction, each
output against the layer in 64 bits over the codes that the cache holds.

What the layer computes around the core are fp32 sums of at most 1024 products (bf16 weights enter exactly, fp32 vectors
to 2^-24), three of them one after the other; the errors of a vector's entries are independent, so normwise each leaves about
sqrt(1024) 2^-24 = 2e-6, and the core's own (2^-22 a query, probability and value sum) is below that: 1e-5.
A probability's relative error is that of its score, at most the score's size (< 8 here) times that: 2^-13."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

import _q4_oracle as oracle

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TOL, WEIGHT_TOL = 1e-5, 2.0 ** -13
HID, QL, NOPE, ROPE, V = 256, 384, 128, 64, 128


def _layer(heads, seed=1, mats=BF16, kv_b=BF16, gate=True, **kw):
    from k3hip.mla import MLAAttention
    g = torch.Generator().manual_seed(seed)
    lin = lambda o, i, dt: (torch.randn(o, i, generator=g) * i ** -0.5).to(BF16).to(dt).cuda()  # noqa: E731
    gain = lambda n: (1 + 0.1 * torch.randn(n, generator=g)).cuda()  # noqa: E731
    w = {"q_a_proj.weight": lin(QL, HID, mats), "q_a_layernorm.weight": gain(QL), "q_b_proj.weight": lin(heads * 192, QL, mats),
         "kv_a_proj_with_mqa.weight": lin(576, HID, mats), "kv_a_layernorm.weight": gain(512),
         "kv_b_proj.weight": lin(heads * 256, 512, kv_b), "g_proj.weight": lin(heads * V, HID, mats),
         "o_proj.weight": lin(HID, heads * V, mats)}
    cfg = SimpleNamespace(hidden_size=HID, num_attention_heads=heads, q_lora_rank=QL, kv_lora_rank=512, qk_nope_head_dim=NOPE,
                          qk_rope_head_dim=ROPE, v_head_dim=V, q_head_dim=192, rms_norm_eps=1e-5, mla_use_output_gate=gate,
                          mla_cache_bits=4, **kw)
    return MLAAttention(cfg, w), w


def _x(seed, *s, dtype=F32):
    return torch.randn(*s, HID, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _norm(x, gain):
    return gain.double() * x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)


def _want(w, heads, x, cache, gate=True):
    """The outputs of the tokens x [B, T, HID], the last T of the cache, and the attention they gave: float64."""
    d = {k: v.double() for k, v in w.items()}
    x = x.double()
    B, T, _ = x.shape
    n = cache.length
    q = (_norm(x @ d["q_a_proj.weight"].T, w["q_a_layernorm.weight"]) @ d["q_b_proj.weight"].T).reshape(B, T, heads, 192)
    kb = d["kv_b_proj.weight"].reshape(heads, 256, 512)
    out, mass = [], []
    for b in range(B):
        lat, rot = oracle.values(cache.packed[b, :n], cache.scales[b, :n]), cache.rot[b, :n].double()
        qa = torch.einsum("thd,hdr->htr", q[b, ..., :NOPE].cpu(), kb[:, :NOPE].cpu()).to(x.device)
        s = (qa @ lat.T + q[b, ..., NOPE:].transpose(0, 1) @ rot.T) * 192 ** -0.5
        hidden = torch.arange(n, device=x.device)[None] > torch.arange(n - T, n, device=x.device)[:, None]
        p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
        o = torch.einsum("htr,hvr->thv", (p @ lat).cpu(), kb[:, NOPE:].cpu()).to(x.device).reshape(T, heads * V)
        if gate:
            o = o * torch.sigmoid(x[b] @ d["g_proj.weight"].T)
        out.append(o @ d["o_proj.weight"].T)
        mass.append(p.sum((0, 1)))
    return torch.stack(out), torch.stack(mass)


def _close(got, want):
    rel = float((got.double() - want).norm() / want.norm())
    assert got.shape == want.shape and rel <= TOL, rel


def _stored(w, x, cache, at):
    """The positions at .. of the cache hold the tokens' latents to half a step of their group's scale (a whole one from
    6 to 7 times it, where the codes end)."""
    d = x.double() @ w["kv_a_proj_with_mqa.weight"].double().T
    c, n = _norm(d[..., :512], w["kv_a_layernorm.weight"]), at + x.shape[1]
    unit = (2.0 ** (cache.scales[:, at:n].double() - 127)).repeat_interleave(32, -1)
    lat, rot = cache.view()
    assert lat.shape == (x.shape[0], cache.length, 512) and lat.dtype == F32
    assert torch.equal(lat.double(), oracle.values(cache.packed[:, :cache.length], cache.scales[:, :cache.length]))
    assert bool(((lat[:, at:n].double() - c).abs() <= unit * (1 + 1e-4)).all())
    assert bool(((rot[:, at:n].double() - d[..., 512:]).abs() <= 2.0 ** -8 * d[..., 512:].abs() + 1e-4).all())


@pytest.mark.parametrize("mats,heads,gate,dtype", [(BF16, 16, True, F32), (BF16, 4, False, BF16), (F32, 8, True, F32)])
def test_prompt_decode_evict_decode(mats, heads, gate, dtype):
    """One sequence: a prompt up to just below the first capacity, single tokens past it, a few tokens at once, a cut, single
    tokens again; outputs and summed weights at every call."""
    layer, w = _layer(heads, mats=mats, gate=gate, mla_cache_weights=True)
    assert layer.fused_step == (mats == BF16)
    x = _x(7, 1, 252, dtype=dtype)
    out, cache = layer(x)
    want, mass = _want(w, heads, x, cache, gate)
    _close(out, want)
    _stored(w, x, cache, 0)
    total = mass
    for i, T in enumerate((1, 1, 1, 1, 1, 1, 3, 1)):
        x = _x(20 + i, 1, T, dtype=dtype)
        before = cache.length
        out, same = layer(x, cache)
        assert same is cache and cache.length == before + T
        want, mass = _want(w, heads, x, cache, gate)
        _close(out, want)
        _stored(w, x, cache, before)
        total = torch.nn.functional.pad(total, (0, T)) + mass
        assert bool(((cache.weight[:, :cache.length].double() - total).abs() <= WEIGHT_TOL * total).all())
    assert cache.capacity == 512 and not cache.weight[:, cache.length:].any()
    n, old = cache.length, [t.clone() for t in cache.buffers()]
    index = cache.evict(100, sink=4, recent=32)
    assert index[0].tolist() == oracle.evict(old[3][0, :n].tolist(), n, 100, 4, 32)
    assert cache.length == 100 and cache.capacity == 512
    for a, b in zip(cache.buffers(), old):
        assert torch.equal(a[0, :100], b[0, index[0].long()]) and not a[:, 100:].any()
    total = total[:, index[0].long()]
    for i in range(3):
        x = _x(40 + i, 1, 1, dtype=dtype)
        out, _ = layer(x, cache)
        want, mass = _want(w, heads, x, cache, gate)
        _close(out, want)
        total = torch.nn.functional.pad(total, (0, 1)) + mass
        assert bool(((cache.weight[:, :cache.length].double() - total).abs() <= WEIGHT_TOL * total).all())


def test_first_token_makes_the_cache():
    for kw in ({}, {"mla_cache_weights": True}):
        layer, w = _layer(4, **kw)
        x = _x(3, 1, 1)
        out, cache = layer(x)
        assert cache.length == 1 and cache.capacity == 256 and (cache.weight is not None) == bool(kw)
        _close(out, _want(w, 4, x, cache)[0])
        if kw:
            assert abs(float(cache.weight[0, 0]) - 4) < 1e-5


def test_batch():
    """Three sequences at once, a prompt and then single tokens, by the same calls."""
    layer, w = _layer(8, seed=5, mla_cache_weights=True)
    cache = None
    total = torch.zeros(3, 0, device="cuda", dtype=F64)
    for i, T in enumerate((40, 1, 1, 5, 1)):
        x = _x(60 + i, 3, T)
        out, cache = layer(x, cache)
        want, mass = _want(w, 8, x, cache)
        _close(out, want)
        total = torch.nn.functional.pad(total, (0, T)) + mass
        assert bool(((cache.weight[:, :cache.length].double() - total).abs() <= WEIGHT_TOL * total).all())
    index = cache.evict(20, 2, 8)
    assert index.shape == (3, 20) and cache.length == 20
    x = _x(90, 3, 1)
    out, _ = layer(x, cache)
    _close(out, _want(w, 8, x, cache)[0])


def test_shortened_cache_takes_new_tokens():
    """A caller that takes positions back (drafts that were not accepted): the next ones overwrite them and start without weight."""
    layer, w = _layer(8, mla_cache_weights=True)
    _, cache = layer(_x(1, 1, 20))
    kept = cache.weight.clone()
    layer(_x(2, 1, 4), cache)
    cache.length = 20
    cache.weight[:, :20] = kept[:, :20]
    for T in (1, 2):
        x = _x(3 + T, 1, T)
        out, _ = layer(x, cache)
        want, mass = _want(w, 8, x, cache)
        _close(out, want)
        n = cache.length
        assert bool(((cache.weight[:, n - T:n].double() - mass[:, n - T:]).abs() <= WEIGHT_TOL * mass[:, n - T:]).all())


def test_masked_form_over_the_decoded_latents():
    """fp32 kv_b takes the tensor form; its sums are library products in fp32."""
    layer, w = _layer(4, mats=F32, kv_b=F32)
    x = _x(1, 1, 30)
    out, cache = layer(x)
    _close(out, _want(w, 4, x, cache)[0])
    out, _ = layer(_x(2, 1, 1), cache)
    _close(out, _want(w, 4, _x(2, 1, 1), cache)[0])


@pytest.mark.parametrize("T", [1, 3])
def test_refusals_leave_the_cache(T):
    layer, w = _layer(4)
    _, cache = layer(_x(3, 1, 10))
    before = [t.clone() for t in cache.buffers()]
    with pytest.raises(ValueError, match="no gradient"):
        layer(_x(4, 1, T).requires_grad_(), cache)
    layer, w = _layer(4, kv_b=F32, mats=F32)
    cache.weight = torch.zeros(1, cache.capacity, device="cuda")
    with pytest.raises(ValueError, match="no attention weights"):
        layer(_x(4, 1, T), cache)
    assert cache.length == 10 and all(torch.equal(a, b) for a, b in zip(cache.buffers(), before))


def test_a_misaligned_buffer_leaves_the_cache_at_its_length():
    """Scale rows at an odd address: the append writes them, the attention refuses them, and a sound buffer goes on from there."""
    layer, w = _layer(4)
    _, cache = layer(_x(3, 1, 10))
    scales = cache.scales
    cache.scales = torch.zeros(1, 256, 17, dtype=torch.uint8, device="cuda")[..., 1:]
    before = [t[:, :10].clone() for t in cache.buffers()]
    for _ in range(2):
        with pytest.raises(ValueError):
            layer(_x(4, 1, 3), cache)
        assert cache.length == 10 and all(torch.equal(a[:, :10], b) for a, b in zip(cache.buffers(), before))
    cache.scales = scales
    out, _ = layer(_x(4, 1, 3), cache)
    assert cache.length == 13
    _close(out, _want(w, 4, _x(4, 1, 3), cache)[0])


def test_another_batch_is_refused():
    layer, w = _layer(4)
    _, cache = layer(_x(3, 2, 10))
    for T in (1, 2):
        with pytest.raises(ValueError):
            layer(_x(4, 1, T), cache)
    assert cache.length == 10


def test_a_callers_cache_and_layers_without_the_option():
    """The cache decides: a 4-bit one runs in a layer made without the option, and a bf16 one in a layer made with it."""
    from k3hip.mla import new_cache
    from k3hip.mla_q4 import new_cache_q4
    layer, w = _layer(8)
    layer.cfg.mla_cache_bits = None
    plain = type(layer)(layer.cfg, w)
    cache, x = new_cache_q4(1, 50), _x(1, 1, 40)
    out, same = plain(x, cache)
    assert same is cache and cache.length == 40
    _close(out, _want(w, 8, x, cache)[0])
    out, _ = plain(_x(2, 1, 1), cache)
    _close(out, _want(w, 8, _x(2, 1, 1), cache)[0])
    a, b = new_cache(1, 512, 64, 50), new_cache(1, 512, 64, 50)
    for t in (x, _x(2, 1, 1)):
        y, _ = layer(t, a)
        z, _ = plain(t, b)
        assert torch.equal(y, z)


def test_step_equals_the_calls_it_is_made_of():
    """The one-call decode step against projections, append and attention called one by one, on a cache with strided rows."""
    from k3hip.mla_q4 import MLACacheQ4
    layer, w = _layer(16, mla_cache_weights=True)
    _, cache = layer(_x(1, 1, 130))
    wide = [torch.zeros(1, 256, 2 * t.shape[2], dtype=t.dtype, device="cuda")[..., :t.shape[2]] for t in (cache.packed, cache.scales, cache.rot)]
    for a, b in zip(wide, (cache.packed, cache.scales, cache.rot)):
        a.copy_(b)
    strided = MLACacheQ4(*wide, cache.length, cache.weight.clone())
    layer.fused_step, x = True, _x(2, 1, 1)
    a, _ = layer(x, strided)
    b, _ = layer(x, cache)
    assert torch.equal(a, b) and all(torch.equal(s, t) for s, t in zip(strided.buffers(), cache.buffers()))
    cache.length -= 1
    layer.fused_step = False
    c, _ = layer(x, cache)
    assert float((b - c).norm() / b.norm()) <= 2 * TOL


@pytest.mark.parametrize("mats", [BF16, F32])
def test_fp32_kv_b_is_not_rounded_for_one_token(mats):
    """kv_b with values between bf16's (which are up to 2^-9 apart from them): a prompt, one token and a few, all by the masked
    form, whatever the projections' dtype."""
    layer, w = _layer(4, mats=mats, kv_b=F32)
    w = {**w, "kv_b_proj.weight": w["kv_b_proj.weight"] * (1 + 2.0 ** -9)}
    layer = type(layer)(layer.cfg, w)
    assert layer.fused_step == (mats == BF16)
    cache = None
    for i, T in enumerate((20, 1, 1, 3)):
        x = _x(70 + i, 1, T)
        out, cache = layer(x, cache)
        _close(out, _want(w, 4, x, cache)[0])
