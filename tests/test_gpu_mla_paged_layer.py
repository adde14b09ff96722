"""The MLA layer over the paged cache: prompts, decode steps, drafts taken back, a common prefix, requests that end and begin, each request's output
against the layer over a cache of its own (tests/test_gpu_mla.py checks that one) and against 64 bits.

What the layer computes around the core are fp32 sums of at most 1024 products, three of them one after the other, whose errors are independent:
sqrt(1024) 2^-24 = 2e-6 each, normwise.  The core, fp32 result: fp16 pages hold latents and rotary values to 2^-11, bf16 pages to 2^-8, and each position's
rounding is its own; a result is a mean of positions and its scores (of size 8 at most) take 2^-11 x 8 / sqrt(576) of it, so what a page's type makes of
a result is below 4 roundings: 4 x 2^-11 and 4 x 2^-8 against unrounded caches.  Over the pages' own values: 2^-22 x 8."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16, F32, F64, I32 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.int32
HID, QL, V = 256, 384, 128


def _layer(heads, gate=True, seed=1):
    from k3hip.mla import MLAAttention
    g = torch.Generator().manual_seed(seed)
    lin = lambda o, i: (torch.randn(o, i, generator=g) * i ** -0.5).to(BF16).cuda()  # noqa: E731
    gain = lambda n: (1 + 0.1 * torch.randn(n, generator=g)).cuda()  # noqa: E731
    w = {"q_a_proj.weight": lin(QL, HID), "q_a_layernorm.weight": gain(QL), "q_b_proj.weight": lin(heads * 192, QL),
         "kv_a_proj_with_mqa.weight": lin(576, HID), "kv_a_layernorm.weight": gain(512), "kv_b_proj.weight": lin(heads * 256, 512),
         "g_proj.weight": lin(heads * V, HID), "o_proj.weight": lin(HID, heads * V)}
    cfg = SimpleNamespace(hidden_size=HID, num_attention_heads=heads, q_lora_rank=QL, kv_lora_rank=512, qk_nope_head_dim=128,
                          qk_rope_head_dim=64, v_head_dim=V, q_head_dim=192, rms_norm_eps=1e-5, mla_use_output_gate=gate)
    return MLAAttention(cfg, w), w


def _norm(x, gain):
    return gain.double() * x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)


def _want(w, heads, x, lat, rot, gate):
    """The outputs of tokens x [T, HID], the last T of lat [n, 512] and rot [n, 64]: float64."""
    d = {k: v.double() for k, v in w.items()}
    x, lat, rot = x.double(), lat.double(), rot.double()
    T, n = len(x), len(lat)
    q = (_norm(x @ d["q_a_proj.weight"].T, w["q_a_layernorm.weight"]) @ d["q_b_proj.weight"].T).reshape(T, heads, 192).transpose(0, 1)
    kb = d["kv_b_proj.weight"].reshape(heads, 256, 512)
    s = (torch.matmul(torch.matmul(q[..., :128], kb[:, :128]), lat.T) + torch.matmul(q[..., 128:], rot.T)) * 192 ** -0.5
    hidden = torch.arange(n, device=x.device)[None] > torch.arange(n - T, n, device=x.device)[:, None]
    p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
    o = torch.matmul(torch.matmul(p, lat), kb[:, 128:].transpose(1, 2)).transpose(0, 1).reshape(T, heads * V)
    if gate:
        o = o * torch.sigmoid(x @ d["g_proj.weight"].T)
    return o @ d["o_proj.weight"].T


def _rel(got, want):
    return float((got.double() - want).norm() / want.norm())


def _rows(cache, b):
    t = cache.pages
    n, page = int(t.lengths[b]), t.page_size
    rows = t.table[b, :-(-n // page)].long()
    return cache.latent[rows].reshape(-1, 512)[:n], cache.rot[rows].reshape(-1, 64)[:n]


@pytest.mark.parametrize("dtype,x_dtype,heads,gate", [(F16, F32, 4, True), (F16, BF16, 24, False), (BF16, F32, 16, True), (BF16, BF16, 3, True)])
def test_a_batch_of_requests(dtype, x_dtype, heads, gate):
    from k3hip.mla import new_cache
    from k3hip.mla_paged import new_cache_paged
    from k3hip.pages import PageTable
    layer, w = _layer(heads, gate)
    g = torch.Generator().manual_seed(heads)
    prompts = [70, 1, 130]
    x = torch.randn(3, 130, HID, generator=g).to(x_dtype).cuda()
    t = PageTable(3, 512, 20, page_size=64)
    cache = new_cache_paged(t, dtype)
    own = [new_cache(1, 512, 64, 1, dtype=F32) for _ in range(3)]
    page_tol = 4 * (2.0 ** -11 if dtype == F16 else 2.0 ** -8)

    def step(x, counts):
        t.extend(torch.tensor(counts, dtype=I32, device="cuda"), tokens=x.shape[1])
        out, same = layer(x, cache)
        assert same is cache and out.dtype == F32
        for b, n in enumerate(counts):
            if n == 0:
                assert not bool(out[b].any())
                continue
            alone, own[b] = layer(x[b:b + 1, :n], own[b])
            want = _want(w, heads, x[b, :n], *_rows(cache, b), gate)
            assert _rel(out[b, :n], want) < 2e-5
            assert _rel(out[b, :n], alone[0].double()) < page_tol
            assert not bool(out[b, n:].any())

    step(x, prompts)
    for i in range(3):                                      # decode, one request resting
        step(torch.randn(3, 1, HID, generator=g).to(x_dtype).cuda(), [1, 1, 1] if i != 1 else [1, 0, 1])
    drafts = torch.randn(3, 4, HID, generator=g).to(x_dtype).cuda()
    step(drafts, [4, 2, 3])
    # some drafts are rejected: their positions go, the next tokens take their places
    kept = t.lengths - torch.tensor([2, 0, 3], dtype=I32, device="cuda")
    t.truncate(kept)
    for b, n in enumerate(kept.tolist()):
        own[b].length = n
    step(torch.randn(3, 1, HID, generator=g).to(x_dtype).cuda(), [1, 1, 1])
    # the first ends, another takes its place
    t.release(torch.tensor([True, False, False], device="cuda"))
    own[0] = new_cache(1, 512, 64, 1, dtype=F32)
    step(torch.randn(3, 50, HID, generator=g).to(x_dtype).cuda(), [50, 1, 1])


def test_a_common_prefix_and_two_layers():
    """Requests behind one system prompt give what they give with prompts of their own, in layers that share the tables."""
    from k3hip.mla_paged import new_cache_paged
    from k3hip.pages import PageTable
    layers = [_layer(16, True, seed)[0] for seed in (1, 2)]
    g = torch.Generator().manual_seed(8)
    system, B = torch.randn(1, 128, HID, generator=g).cuda(), 6
    turns = [torch.randn(B, n, HID, generator=g).cuda() for n in (9, 1, 1)]

    def run(x, caches):
        for layer, c in zip(layers, caches):
            x = layer(x, c)[0]
        return x

    apart = PageTable(B, 512, 40, page_size=64)
    own = [new_cache_paged(apart) for _ in layers]
    apart.extend(128)
    run(system.expand(B, -1, -1).contiguous(), own)
    t = PageTable(B, 512, 40, page_size=64)
    caches = [new_cache_paged(t) for _ in layers]
    t.extend(torch.tensor([0, 128, 0, 0, 0, 0], dtype=I32, device="cuda"), tokens=128)
    x = torch.zeros(B, 128, HID, device="cuda")
    x[1] = system[0]
    run(x, caches)
    used = int(t.used)
    t.share(128, source=1)
    for x in turns:
        apart.extend(x.shape[1]), t.extend(x.shape[1])
        a, b = run(x, own), run(x, caches)
        # (the same values in other places, summed in another order: fp32)
        assert _rel(b, a.double()) < 1e-5
    assert used == 2 and int(t.used) == 2 + B and int(apart.used) == 3 * B
    t.release(torch.ones(B, dtype=torch.bool, device="cuda"))
    assert int(t.used) == 2 and t.lengths.tolist() == [128] * B
    t.extend(9)
    apart.truncate(torch.full((B,), 128, dtype=I32, device="cuda")), apart.extend(9)
    assert _rel(run(turns[0], caches), run(turns[0], own).double()) < 1e-5


def test_a_request_without_pages_gives_zeros():
    from k3hip.mla_paged import new_cache_paged
    from k3hip.pages import PageTable
    layer, _ = _layer(4)
    t = PageTable(3, 128, 2, page_size=32)
    cache = new_cache_paged(t)
    t.extend(20)
    assert t.counts.tolist() == [20, 20, 0]
    out, _ = layer(torch.randn(3, 20, HID).cuda(), cache)
    assert bool(torch.isfinite(out).all()) and bool(out[:2].any()) and not bool(out[2].any())
