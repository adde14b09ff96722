"""Calls of the 4-bit cache that would write where they must not, refused before anything is launched, and calls that are not to be
refused (no GPU)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from test_mla_q4_host import BF16, U8, _cache, _launches


# ------------------------------------------------------------------------------- sequences that share memory
def _append(cache, **kw):
    from k3hip.mla_q4 import mla_q4_append
    B = cache[0].shape[0]
    mla_q4_append(torch.zeros(B, 1, 512), torch.zeros(B, 1, 64), *cache, **kw)


def _attend(cache, **kw):
    from k3hip.mla_q4 import mla_q4_attention
    B = cache[0].shape[0]
    w = torch.zeros(4, 128, 512, dtype=BF16)
    return mla_q4_attention(torch.zeros(B, 1, 4, 128), torch.zeros(B, 1, 4, 64), w, w, *cache, 0.1, **kw)


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("share", [
    lambda t: t[:1].expand(2, -1, -1),                                                                      # one buffer for both
    lambda t: t.as_strided(t.shape, (t.shape[2] * (t.shape[1] - 1), t.shape[2], 1)),                        # the last row is the next one's first
    lambda t: t.as_strided(t.shape, (t.shape[2] // 2, 2 * t.shape[2], 1)),                                  # rows that overlap side by side
])
def test_append_refuses_sequences_that_share_rows(monkeypatch, which, share):
    calls = _launches(monkeypatch)
    cache = list(_cache())
    cache[which] = share(cache[which])
    with pytest.raises(ValueError, match="overlap"):
        _append(cache)
    assert not calls
    _attend(cache)                          # reading them is in order
    assert len(calls) == 1


@pytest.mark.parametrize("weight", [torch.zeros(8).expand(2, 8), torch.zeros(15).as_strided((2, 8), (7, 1))])
def test_summed_weights_of_sequences_that_share_memory(monkeypatch, weight):
    calls = _launches(monkeypatch)
    for f in (_append, _attend):
        with pytest.raises(ValueError, match="overlap"):
            f(_cache(), weight=weight)
    assert not calls
    from k3hip.evict import cache_evict
    cache_evict(weight, [], 4)              # which reads them
    assert len(calls) == 1


@pytest.mark.parametrize("B,cap", [(1, 8), (2, 8), (3, 1), (2, 0)])
def test_sequences_that_lie_apart_pass(monkeypatch, B, cap):
    calls = _launches(monkeypatch)
    for cache in (_cache(B, cap), tuple(t.transpose(0, 1) for t in _cache(cap, B)),       # batch first, position first
                  tuple(torch.cat((t, t), 2)[..., :t.shape[2]] for t in _cache(B, cap))):
        _append(cache, start=0 if cap else torch.zeros(B, dtype=torch.int32), weight=torch.zeros(B, cap + 3)[:, :cap])
    assert len(calls) == (3 if cap else 0)


def test_entry_points_refuse_sequences_that_share_memory():
    from k3hip import _lib
    lib = _lib.lib()
    p, n = ctypes.c_void_p(4096), None
    app = [p, 1536, 512, 0, p, 192, 64, 0, p, 2048, 256, p, 128, 16, p, 512, 64, n, 0, n, p, 8, 2, 3, 8, 512, 64, n]
    att = [p, 1536, 512, 128, p, 768, 256, 64, 0, p, p, p, 2048, 256, p, 128, 16, p, 512, 64, n, n, 8, 2, 3, 4, 512, 64, 128, 96,
           0.1, n, p, 0, p, 8, p, 0, n]
    longs, ptrs = (ctypes.c_int64 * 2), (ctypes.c_void_p * 2)
    one, big = longs(64, 16), longs(512, 128)
    ev = [p, 8, n, 8, 2, 4, 1, 2, p, p, 2, ptrs(4096, 8192), big, one, ptrs(16384, 32768), big, one, one, 4, n]
    for call, base, at in (
            (lib.k3_mla_q4_append, app, {9: 2044}), (lib.k3_mla_q4_append, app, {9: 0}), (lib.k3_mla_q4_append, app, {9: -2048}),
            (lib.k3_mla_q4_append, app, {12: 127}), (lib.k3_mla_q4_append, app, {15: 511}), (lib.k3_mla_q4_append, app, {21: 7}),
            (lib.k3_mla_q4_append, app, {21: 0}), (lib.k3_mla_q4_attention, att, {35: 7}), (lib.k3_mla_q4_attention, att, {35: 0}),
            (lib.k3_cache_evict, ev, {15: longs(512, 63)}), (lib.k3_cache_evict, ev, {15: longs(0, 128)})):
        args = list(base)
        for i, v in at.items():
            args[i] = v
        assert call(*args) == _lib.K3_ERR_SHAPE and b"overlap" in lib.k3_last_error(), (call.__name__, at)


# ------------------------------------------------------------------------------- buffers of an autograd graph
def test_buffers_that_are_written_carry_no_gradient(monkeypatch):
    """As torch refuses to write into a leaf; under no_grad it is in order, as there."""
    from k3hip.mla_q4 import new_cache_q4
    calls = _launches(monkeypatch)
    weight, rot = torch.zeros(2, 8, requires_grad=True), _cache()[2].requires_grad_()
    for f in (lambda: _append(_cache(), weight=weight), lambda: _attend(_cache(), weight=weight),
              lambda: _append(_cache()[:2] + (rot,)), lambda: _attend(_cache()[:2] + (rot,))):
        with pytest.raises(ValueError, match="no gradient"):
            f()
        assert not calls
        with torch.no_grad():
            f()
        assert len(calls) == 1
        calls.clear()
    for name in ("weight", "rot"):          # the one-call decode step asks for the pitches before it launches anything
        cache = new_cache_q4(1, 1, True, "cpu")
        getattr(cache, name).requires_grad_()
        with pytest.raises(ValueError, match="no gradient"):
            cache.row_pitches()
        with torch.no_grad():
            assert cache.row_pitches() == (256, 16, 64)


# ------------------------------------------------------------------------------- fp32 kv_b
def test_one_token_with_fp32_kv_b_stays_on_the_masked_form(monkeypatch):
    """The one-call step takes W_UK and W_UV in bf16; fp32 ones are not rounded to it because a call has one token."""
    from k3hip.mla_q4 import MLACacheQ4, new_cache_q4
    from test_mla_q4_host import _cfg, _layer
    calls = _launches(monkeypatch)
    monkeypatch.setattr(MLACacheQ4, "view", lambda c: (torch.zeros(1, c.length, 512), c.rot[:, :c.length]))
    layer, x = _layer(_cfg()), torch.zeros(1, 1, 64)
    layer.fused_step = True
    layer.kv_b = layer.kv_b.float()
    cache = new_cache_q4(1, 1, device="cpu")
    layer(x, cache)
    assert [name for name, _ in calls] == ["k3_mla_q4_append"] and cache.length == 1
    with pytest.raises(ValueError, match="bf16 kv_b"):
        layer.decode_step(x, cache)
    assert len(calls) == 1 and cache.length == 1


# ------------------------------------------------------------------------------- large batches
@pytest.mark.parametrize("lengths", [None, 5, torch.arange(700, dtype=torch.int32) % 9])
def test_a_batch_past_65536_rows_goes_out_in_parts(monkeypatch, lengths):
    """700 sequences of 96 heads: two calls, each with its own part of everything that is per sequence."""
    from k3hip.mla_q4 import mla_q4_attention
    calls = _launches(monkeypatch)
    B, H, cap = 700, 96, 8
    q, w = torch.zeros(1, 1, 1, 192).expand(B, 1, H, 192), torch.zeros(H, 128, 512, dtype=BF16)
    cache, weight, gate = _cache(B, cap), torch.zeros(B, cap + 2)[:, :cap], torch.zeros(B, 1, H * 128)
    counts = torch.ones(B, dtype=torch.int32)
    o = mla_q4_attention(q[..., :128], q[..., 128:], w, w, *cache, 0.1, lengths=lengths, counts=counts, weight=weight, gate=gate)
    assert o.shape == (B, 1, H, 128) and len(calls) == 2
    first = 0
    for (name, a), n in zip(calls, (682, 18)):
        assert name == "k3_mla_q4_attention" and a[23] == n and a[25] == H
        for i, t in ((11, cache[0]), (14, cache[1]), (17, cache[2]), (21, counts), (31, gate), (34, weight)):
            assert a[i] == t[first].data_ptr(), i
        assert a[35] == cap + 2 and a[22] == (lengths if isinstance(lengths, int) else cap)
        assert a[20] == (lengths[first].data_ptr() if isinstance(lengths, torch.Tensor) else 0)
        first += n


@pytest.mark.parametrize("B,H,parts", [(65536, 1, [65535, 1]), (65535, 1, [65535]), (16, 4096, [16]), (17, 4096, [16, 1])])
def test_parts_keep_within_what_one_call_takes(monkeypatch, B, H, parts):
    from k3hip.mla_q4 import mla_q4_attention
    calls = _launches(monkeypatch)
    q, w = torch.zeros(1, 1, 1, 72).expand(B, 1, H, 72), torch.zeros(1, 8, 1).to(BF16).expand(H, 8, 512)
    mla_q4_attention(q[..., :8], q[..., 8:], w, w, *(t.expand(B, -1, -1) for t in _cache(1, 2)), 0.1)
    assert [a[23] for _, a in calls] == parts


def test_layer_takes_a_batch_past_65536_rows(monkeypatch):
    from types import SimpleNamespace

    from k3hip.mla import MLAAttention
    from test_mla_q4_host import _cfg
    calls = _launches(monkeypatch)
    z = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
    layer = MLAAttention(SimpleNamespace(**{**vars(_cfg()), "num_attention_heads": 96}), {
        "q_a_proj.weight": z(64, 64), "q_a_layernorm.weight": z(64), "q_b_proj.weight": z(96 * 192, 64), "kv_a_proj_with_mqa.weight": z(576, 64),
        "kv_a_layernorm.weight": z(512), "kv_b_proj.weight": z(96 * 256, 512), "o_proj.weight": z(64, 96 * 128)})
    out, cache = layer(torch.zeros(700, 1, 64))
    assert out.shape == (700, 1, 64) and cache.length == 1
    assert [name for name, _ in calls] == ["k3_mla_q4_append"] + ["k3_mla_q4_attention"] * 2


# ------------------------------------------------------------------------------- a refusal after the append
@pytest.mark.parametrize("B,T", [(1, 3), (2, 1)])
def test_layer_takes_back_positions_that_are_not_attended_to(monkeypatch, B, T):
    """Append takes buffers that attention refuses (a misaligned view, say): then the cache is as long as it was."""
    from k3hip import _lib
    from k3hip.mla_q4 import new_cache_q4
    from test_mla_q4_host import _cfg, _layer
    calls = _launches(monkeypatch)
    layer, cache, x = _layer(_cfg()), new_cache_q4(B, 1, device="cpu"), torch.zeros(B, T, 64)
    layer(x, cache)

    def refuse(name, *a):
        calls.append((name, a))
        if name == "k3_mla_q4_attention":
            raise ValueError("must be 16-byte (scales 4-byte) aligned")
    monkeypatch.setattr(_lib, "call", refuse)
    for _ in range(2):
        with pytest.raises(ValueError, match="aligned"):
            layer(x, cache)
        assert cache.length == T and calls[-2][0] == "k3_mla_q4_append" and calls[-2][1][18] == T


# ------------------------------------------------------------------------------- scratch of captured calls
def test_a_captured_call_takes_no_kept_workspace(monkeypatch):
    """Not even one that its stream has: another graph captured there would have the same."""
    from k3hip import _torch as T
    from k3hip import _workspace
    from k3hip.mla_q4 import new_cache_q4
    from test_mla_q4_host import _cfg, _layer
    calls, kept = _launches(monkeypatch), []
    monkeypatch.setattr(_workspace, "get", lambda d, n, tag="": kept.append(tag) or torch.empty(n, dtype=U8))
    layer, cache, x = _layer(_cfg()), new_cache_q4(1, 4, device="cpu"), torch.zeros(1, 1, 64)
    layer._mats = {k: m for k, m in (("q_a", layer.q_a), ("q_b", layer.q_b), ("kv_a", layer.kv_a), ("g", None), ("o", layer.o_w))}
    layer._q_an32, layer._kv_an32 = layer.q_an.float(), layer.kv_an.float()
    for captured, want in ((False, ["mla_q4", "mla_step"]), (True, [])):
        monkeypatch.setattr(T, "capturing", lambda: captured, raising=False)
        _attend(_cache(), lengths=torch.ones(2, dtype=torch.int32))
        layer.decode_step(x, cache)
        assert kept == want
        kept.clear()
    assert [name for name, _ in calls] == ["k3_mla_q4_attention", "k3_mla_step_decode_q4"] * 2
