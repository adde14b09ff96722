"""What the 4-bit cache's calls refuse before anything is launched (no GPU: the check for device tensors comes after the
shapes', and the C entry points check on the host)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import _q4_oracle as oracle

BF16, U8 = torch.bfloat16, torch.uint8


def _cache(B=2, cap=8):
    return torch.zeros(B, cap, 256, dtype=U8), torch.zeros(B, cap, 16, dtype=U8), torch.zeros(B, cap, 64, dtype=BF16)


def _launches(monkeypatch):
    """The Python layer without a GPU: device checks pass, launches are recorded."""
    import contextlib

    from k3hip import _lib, _workspace
    from k3hip import _torch as T
    calls = []
    monkeypatch.setattr(T, "require_device", lambda *ts: None)
    monkeypatch.setattr(T, "stream", lambda t: 0)
    monkeypatch.setattr(T, "current", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(_workspace, "get", lambda d, n, tag="": torch.empty(n, dtype=U8))
    monkeypatch.setattr(_lib, "call", lambda name, *a: calls.append((name, a)))
    return calls


# ------------------------------------------------------------------------------- append
@pytest.mark.parametrize("c,r,start,error", [
    ((2, 3, 511), (2, 3, 64), 0, ValueError), ((2, 3, 512), (2, 3, 63), 0, ValueError), ((2, 3, 512), (2, 4, 64), 0, ValueError),
    ((1, 3, 512), (1, 3, 64), 0, ValueError), ((3, 512), (3, 64), 0, ValueError), ((2, 3, 512), (2, 3, 64), 6, ValueError),
    ((2, 3, 512), (2, 3, 64), -1, ValueError), ((2, 9, 512), (2, 9, 64), 0, ValueError),
])
def test_append_refuses(monkeypatch, c, r, start, error):
    from k3hip.mla_q4 import mla_q4_append
    calls = _launches(monkeypatch)
    with pytest.raises(error):
        mla_q4_append(torch.zeros(*c), torch.zeros(*r), *_cache(), start=start)
    assert not calls


@pytest.mark.parametrize("which,change", [
    (0, lambda t: t.to(torch.int8)), (1, lambda t: t.float()), (2, lambda t: t.float()), (0, lambda t: t[..., :128]),
    (1, lambda t: t[:, :5]), (2, lambda t: t[:1]), (0, lambda t: t[0]), (0, lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)),
])
def test_both_refuse_buffers_of_another_form(monkeypatch, which, change):
    from k3hip.mla_q4 import mla_q4_append, mla_q4_attention
    calls = _launches(monkeypatch)
    cache = list(_cache())
    cache[which] = change(cache[which])
    with pytest.raises((ValueError, TypeError)):
        mla_q4_append(torch.zeros(2, 1, 512), torch.zeros(2, 1, 64), *cache)
    with pytest.raises((ValueError, TypeError)):
        mla_q4_attention(torch.zeros(2, 1, 4, 128), torch.zeros(2, 1, 4, 64), torch.zeros(4, 128, 512, dtype=BF16),
                         torch.zeros(4, 128, 512, dtype=BF16), *cache, 0.1)
    assert not calls


@pytest.mark.parametrize("bad", [torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32)])
def test_lengths_of_another_form(monkeypatch, bad):
    from k3hip.evict import cache_evict
    from k3hip.mla_q4 import mla_q4_append, mla_q4_attention
    calls = _launches(monkeypatch)
    q = (torch.zeros(2, 1, 4, 128), torch.zeros(2, 1, 4, 64), torch.zeros(4, 128, 512, dtype=BF16), torch.zeros(4, 128, 512, dtype=BF16))
    for f in (lambda: mla_q4_append(torch.zeros(2, 1, 512), torch.zeros(2, 1, 64), *_cache(), start=bad),
              lambda: mla_q4_append(torch.zeros(2, 1, 512), torch.zeros(2, 1, 64), *_cache(), counts=bad),
              lambda: mla_q4_attention(*q, *_cache(), 0.1, lengths=bad), lambda: mla_q4_attention(*q, *_cache(), 0.1, counts=bad),
              lambda: cache_evict(torch.zeros(2, 8), [], 4, lengths=bad)):
        with pytest.raises((ValueError, TypeError)):
            f()
    assert not calls


# ------------------------------------------------------------------------------- attention
def _attend(**kw):
    from k3hip.mla_q4 import mla_q4_attention
    a = {"q_nope": torch.zeros(2, 3, 4, 128), "q_rot": torch.zeros(2, 3, 4, 64), "wk": torch.zeros(4, 128, 512, dtype=BF16),
         "wv": torch.zeros(4, 96, 512, dtype=BF16)}
    a.update({k: kw.pop(k) for k in list(kw) if k in a})
    return mla_q4_attention(*a.values(), *_cache(), 0.1, **kw)


@pytest.mark.parametrize("kw,error", [
    ({"q_nope": torch.zeros(2, 3, 4, 120)}, ValueError), ({"q_rot": torch.zeros(2, 3, 4, 32)}, ValueError),
    ({"q_rot": torch.zeros(2, 2, 4, 64)}, ValueError), ({"q_nope": torch.zeros(3, 4, 128)}, ValueError),
    ({"wk": torch.zeros(4, 128, 512)}, TypeError), ({"wv": torch.zeros(3, 96, 512, dtype=BF16)}, ValueError),
    ({"wv": torch.zeros(4, 96, 256, dtype=BF16)}, ValueError), ({"lengths": 9}, ValueError), ({"lengths": -1}, ValueError),
    ({"weight": torch.zeros(2, 8, dtype=BF16)}, TypeError), ({"weight": torch.zeros(2, 7)}, ValueError),
    ({"weight": torch.zeros(8, 2).t()}, ValueError), ({"gate": torch.zeros(2, 3, 4 * 95)}, ValueError),
    ({"gate": torch.zeros(3, 2, 4 * 96)}, ValueError), ({"out_dtype": torch.float16}, TypeError),
    ({"q_nope": torch.zeros(2, 3, 4, 128, requires_grad=True)}, ValueError), ({"q_nope": torch.zeros(2, 3, 4, 128, dtype=torch.float16),
                                                                              "out_dtype": torch.int32}, TypeError),
])
def test_attention_refuses(monkeypatch, kw, error):
    calls = _launches(monkeypatch)
    with pytest.raises(error):
        _attend(**kw)
    assert not calls


def test_attention_passes_views_and_copies_what_it_cannot_read(monkeypatch):
    calls = _launches(monkeypatch)
    q = torch.zeros(2, 3, 4, 192)
    _attend(q_nope=q[..., :128], q_rot=q[..., 128:])
    (name, a), = calls
    assert name == "k3_mla_q4_attention" and a[:4] == (q.data_ptr(), 2304, 768, 192) and a[4] == q.data_ptr() + 512
    odd = torch.zeros(2, 3, 4, 193)
    _attend(q_nope=odd[..., :128], q_rot=odd[..., 128:192])
    assert calls[1][1][1:4] == (1536, 512, 128) and calls[1][1][5:8] == (768, 256, 64)


def test_entry_points_check_their_arguments():
    """Every refusal of the C entry points comes from the host, before a launch."""
    from k3hip import _lib
    lib = _lib.lib()
    p, n = ctypes.c_void_p(4096), None
    app = [p, 1536, 512, 0, p, 192, 64, 0, p, 2048, 256, p, 128, 16, p, 512, 64, n, 0, n, n, 0, 2, 3, 8, 512, 64, n]

    def append(**at):
        args = list(app)
        for k, v in at.items():
            args[int(k[1:])] = v
        return lib.k3_mla_q4_append(*args)
    assert append(_0=n) == _lib.K3_ERR_NULL and append(_8=n) == _lib.K3_ERR_NULL
    assert append(_3=5) == _lib.K3_ERR_DTYPE and append(_7=2) == _lib.K3_ERR_DTYPE
    assert append(_18=6) == _lib.K3_ERR_SHAPE and b"do not fit" in lib.k3_last_error()
    for at in ({"_25": 256}, {"_26": 32}, {"_22": -1}, {"_22": 70000}, {"_2": 510}, {"_10": 255}, {"_13": 15}, {"_16": 63}, {"_24": 2}):
        assert append(**at) == _lib.K3_ERR_SHAPE, at
    assert append(_0=ctypes.c_void_p(4104)) == _lib.K3_ERR_ALIGN and append(_8=ctypes.c_void_p(4097)) == _lib.K3_ERR_ALIGN
    assert append(_23=0) == _lib.K3_OK and append(_22=0) == _lib.K3_OK

    size = lib.k3_mla_q4_workspace_size(2, 3, 4, 96, 8, 0, 0, 1, 0)
    assert size > 0 and lib.k3_mla_q4_workspace_size(0, 3, 4, 96, 8, 0, 0, 1, 0) == 0
    att = [p, 1536, 512, 128, p, 768, 256, 64, 0, p, p, p, 2048, 256, p, 128, 16, p, 512, 64, n, n, 8, 2, 3, 4, 512, 64, 128, 96,
           0.1, n, p, 0, p, 8, p, size, n]

    def attend(**at):
        args = list(att)
        for k, v in at.items():
            args[int(k[1:])] = v
        return lib.k3_mla_q4_attention(*args)
    for i in (0, 4, 9, 10, 11, 14, 17, 32, 36):
        assert attend(**{f"_{i}": n}) == _lib.K3_ERR_NULL, i
    assert attend(_8=4) == _lib.K3_ERR_DTYPE and attend(_33=9) == _lib.K3_ERR_DTYPE
    for at in ({"_26": 256}, {"_27": 32}, {"_28": 120 + 4}, {"_28": 264}, {"_28": 0}, {"_29": 1032}, {"_29": 92}, {"_25": 0}, {"_25": 5000},
               {"_23": 40000}, {"_22": -1}, {"_22": (1 << 24) + 1}, {"_1": 1538}, {"_7": 63}, {"_13": 248}, {"_13": 264}, {"_16": 8}, {"_16": 18}, {"_15": 130},
               {"_19": 60}, {"_24": 1 << 25}):
        assert attend(**at) == _lib.K3_ERR_SHAPE, at
    for i in (0, 4, 9, 10, 11, 17, 32, 36):
        assert attend(**{f"_{i}": ctypes.c_void_p(4104)}) == _lib.K3_ERR_ALIGN, i
    assert attend(_14=ctypes.c_void_p(4098)) == _lib.K3_ERR_ALIGN
    assert attend(_37=size - 1) == _lib.K3_ERR_WORKSPACE
    assert attend(_23=0) == _lib.K3_OK and attend(_24=0) == _lib.K3_OK


# ------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("kw", [
    {"keep": -1}, {"sink": -1}, {"recent": -1}, {"sink": 3, "recent": 2}, {"capacity": 3}, {"lengths": 9}, {"lengths": -2},
    {"weight": torch.zeros(8)}, {"buffers": [torch.zeros(2, 7, 4)]}, {"buffers": [torch.zeros(2, 8)] * 9},
    {"buffers": [torch.zeros(8)]}, {"buffers": [torch.zeros(2, 8, 3, requires_grad=True)]},
])
def test_evict_refuses(monkeypatch, kw):
    from k3hip.evict import cache_evict
    calls = _launches(monkeypatch)
    a = {"weight": torch.zeros(2, 8), "buffers": [torch.zeros(2, 8, 4)], "keep": 4}
    a.update(kw)
    with pytest.raises(ValueError):
        cache_evict(**a)
    with pytest.raises(TypeError):
        cache_evict(torch.zeros(2, 8, dtype=torch.float64), [], 4)
    assert not calls


def test_evict_entry_point_checks_its_arguments():
    from k3hip import _lib
    lib = _lib.lib()
    p, n = ctypes.c_void_p(4096), None
    longs, ptrs = (ctypes.c_int64 * 2), (ctypes.c_void_p * 2)
    one, big = longs(64, 16), longs(512, 128)
    base = [p, 8, n, 8, 2, 4, 1, 2, p, p, 2, ptrs(4096, 8192), big, one, ptrs(16384, 32768), big, one, one, 4, n]

    def evict(**at):
        args = list(base)
        for k, v in at.items():
            args[int(k[1:])] = v
        return lib.k3_cache_evict(*args)
    for i in (0, 8, 9, 11, 12, 13, 14, 15, 16, 17):
        assert evict(**{f"_{i}": n}) == _lib.K3_ERR_NULL, i
    for at in ({"_4": -1}, {"_4": 70000}, {"_3": -1}, {"_5": 2}, {"_6": -1}, {"_7": -1}, {"_10": 9}, {"_18": 3}, {"_13": longs(63, 16)},
               {"_16": longs(64, 15)}, {"_17": longs(-1, 4)}, {"_11": ptrs(4096, 0)}, {"_14": ptrs(0, 4096)}):
        assert evict(**at) == _lib.K3_ERR_SHAPE, at
    assert evict(_4=0) == _lib.K3_OK


# ------------------------------------------------------------------------------- the oracle itself
def test_oracle_rounds_to_the_nearest_value():
    g = torch.Generator().manual_seed(0)
    for _ in range(40):
        x = (torch.randn(32, generator=g, dtype=torch.float64) * 3).float().double().tolist()
        codes, byte = oracle.round_group(x)
        s = 2.0 ** (byte - 127)
        top = max(map(abs, x)) / s
        assert 3.5 < top <= 7
        for v, c in zip(x, codes):
            got = oracle.E2M1[c & 7] * s
            assert all(abs(abs(v) - got) <= abs(abs(v) - e * s) for e in oracle.E2M1)
    assert oracle.round_group([7.0] * 32)[1] == 127 and oracle.round_group([7.01] * 32)[1] == 128
    assert oracle.round_group([2.5, 3.5, 5.0, 0.25, 0.75, 6.0] + [0.0] * 26)[0][:6] == [4, 6, 6, 0, 2, 7]


def test_oracle_evicts():
    assert oracle.evict([5, 1, 3, 3, 3, 2, 9], 7, 5, 1, 1) == [0, 2, 3, 4, 6]
    assert oracle.evict([5, 1, 3, 3, 3, 2, 9], 7, 4, 0, 2) == [0, 2, 5, 6]
    assert oracle.evict([1.0, float("nan"), -1.0], 3, 2, 0, 0) == [0, 2]
    assert oracle.evict([1.0, 2.0], 2, 3, 0, 0) == [0, 1]


# ------------------------------------------------------------------------------- the cache and the layer
def _cfg(**kw):
    from types import SimpleNamespace
    return SimpleNamespace(**{**dict(hidden_size=64, num_attention_heads=2, q_lora_rank=64, kv_lora_rank=512, qk_nope_head_dim=128,
                                     qk_rope_head_dim=64, v_head_dim=128, q_head_dim=192, rms_norm_eps=1e-5, mla_cache_bits=4), **kw})


def _layer(cfg):
    from k3hip.mla import MLAAttention
    z = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
    klr, rope = cfg.kv_lora_rank, cfg.qk_rope_head_dim
    v = cfg.v_head_dim
    return MLAAttention(cfg, {"q_a_proj.weight": z(64, 64), "q_a_layernorm.weight": z(64), "q_b_proj.weight": z(2 * cfg.q_head_dim, 64),
                              "kv_a_proj_with_mqa.weight": z(klr + rope, 64), "kv_a_layernorm.weight": z(klr),
                              "kv_b_proj.weight": z(2 * (cfg.qk_nope_head_dim + v), klr), "o_proj.weight": z(64, 2 * v)})


@pytest.mark.parametrize("kw", [{"mla_cache_bits": 8}, {"mla_cache_bits": 3}, {"mla_cache_group_size": 64}, {"kv_lora_rank": 256},
                                {"qk_rope_head_dim": 32}, {"qk_nope_head_dim": 264, "q_head_dim": 328}, {"v_head_dim": 1032}])
def test_layer_refuses_other_quantised_caches(kw):
    with pytest.raises(ValueError):
        _layer(_cfg(**kw))
    if "mla_cache_bits" not in kw:
        _layer(_cfg(**{**kw, "mla_cache_bits": None}))


@pytest.mark.parametrize("bits", [None, 0, 16])
def test_layer_without_the_option_keeps_its_cache(bits):
    layer = _layer(_cfg(mla_cache_bits=bits))
    assert layer.cache_bits != 4 and layer.cache_dtype == BF16


@pytest.mark.parametrize("weights", [False, True])
def test_cache_grows_by_doubling(weights):
    from k3hip.mla_q4 import new_cache_q4
    cache = new_cache_q4(2, 1, weights, "cpu")
    assert cache.capacity == 256 and cache.bytes_per_token() == 400 and cache.nbytes_used() == 0
    for x in cache.buffers():
        x.copy_(torch.randint(1, 100, x.shape).to(x.dtype))
    before = [x.clone() for x in cache.buffers()]
    cache.length = 250
    assert cache.reserve(6).capacity == 256 and cache.packed is not None
    cache.reserve(7)
    assert cache.capacity == 512 and cache.length == 250 and cache.nbytes_used() == 2 * 250 * 400
    for x, y in zip(cache.buffers(), before):
        assert torch.equal(x[:, :250], y[:, :250]) and not x[:, 250:].any() and x.dtype == y.dtype
    cache.length = 512
    assert cache.reserve(1000).capacity == 1536
    assert (cache.weight is not None) == weights


def test_cache_without_weights_cannot_evict():
    from k3hip.mla_q4 import new_cache_q4
    with pytest.raises(ValueError, match="no attention weights"):
        new_cache_q4(1, 1, device="cpu").evict(4)


@pytest.mark.parametrize("change", [
    lambda c: setattr(c, "rot", c.rot.float()), lambda c: setattr(c, "packed", c.packed[:, :100]),
    lambda c: setattr(c, "scales", c.scales[..., :8]), lambda c: setattr(c, "weight", torch.zeros(1, 255)),
    lambda c: setattr(c, "weight", torch.zeros(1, 256, dtype=torch.float64)),
])
def test_step_refuses_buffers_of_another_form(change):
    from k3hip.mla_q4 import new_cache_q4
    cache = new_cache_q4(1, 1, True, "cpu")
    assert cache.row_pitches() == (256, 16, 64)
    change(cache)
    with pytest.raises((ValueError, TypeError)):
        cache.row_pitches()
    with pytest.raises(ValueError, match="2 sequences"):
        new_cache_q4(2, 1, device="cpu").row_pitches()


def test_append_refuses_gradients(monkeypatch):
    from k3hip.mla_q4 import mla_q4_append
    calls = _launches(monkeypatch)
    with pytest.raises(ValueError, match="no gradient"):
        mla_q4_append(torch.zeros(2, 1, 512, requires_grad=True), torch.zeros(2, 1, 64), *_cache())
    with torch.no_grad():
        mla_q4_append(torch.zeros(2, 1, 512, requires_grad=True), torch.zeros(2, 1, 64), *_cache())
    assert len(calls) == 1


def test_cache_passes_its_buffers_and_length(monkeypatch):
    from k3hip.mla_q4 import new_cache_q4
    calls = _launches(monkeypatch)
    cache = new_cache_q4(1, 1, True, "cpu")
    cache.append(torch.zeros(1, 300, 512), torch.zeros(1, 300, 64))
    cache.attend(torch.zeros(1, 2, 4, 128), torch.zeros(1, 2, 4, 64), torch.zeros(4, 128, 512, dtype=BF16), torch.zeros(4, 128, 512, dtype=BF16),
                 0.1)
    cache.evict(40, 4, 20)
    assert cache.length == 40 and cache.capacity == 512
    (a, append), (b, attend), (c, evict) = calls
    assert (a, b, c) == ("k3_mla_q4_append", "k3_mla_q4_attention", "k3_cache_evict")
    assert append[18] == 0 and append[20] != 0 and append[23:25] == (300, 512) and attend[22] == 300 and evict[3:8] == (300, 1, 40, 4, 20)


def test_step_entry_point_checks_its_arguments():
    from k3hip import _lib
    lib = _lib.lib()
    p, n = ctypes.c_void_p(4096), None
    size = lib.k3_mla_step_q4_workspace_size(64, 2, 128, 64, 128, 512, 6, 1)
    assert size > lib.k3_mla_step_q4_workspace_size(64, 2, 128, 64, 128, 512, 6, 0) > 0
    args = [p, 0, p, p, p, p, p, p, p, n, p, p, 256, p, 16, p, 64, p, 8, 5, 1e-5, 0.1, p, 0, 64, 64, 2, 128, 64, 128, 512, p, size, n]

    def step(**at):
        a = list(args)
        for k, v in at.items():
            a[int(k[1:])] = v
        return lib.k3_mla_step_decode_q4(*a)
    for i in (0, 2, 3, 4, 5, 6, 7, 8, 10, 11, 13, 15, 22, 31):
        assert step(**{f"_{i}": n}) == _lib.K3_ERR_NULL, i
    assert step(_1=3) == _lib.K3_ERR_DTYPE and step(_23=3) == _lib.K3_ERR_DTYPE
    for at in ({"_12": 255}, {"_12": 264}, {"_14": 15}, {"_14": 18}, {"_12": 1040}, {"_14": 1028}, {"_16": 520}, {"_16": 63}, {"_16": 68}, {"_18": 5}, {"_19": -1}, {"_19": 8}, {"_24": 60}, {"_25": 0},
               {"_27": 264}, {"_28": 32}, {"_29": 1032}, {"_30": 256}, {"_18": (1 << 24) + 1}):
        assert step(**at) == _lib.K3_ERR_SHAPE, at
    for i in (0, 2, 3, 4, 5, 6, 7, 8, 10, 11, 15, 31):
        assert step(**{f"_{i}": ctypes.c_void_p(4104)}) == _lib.K3_ERR_ALIGN, i
    assert step(_13=ctypes.c_void_p(4097)) == _lib.K3_ERR_ALIGN
    assert step(_32=size - 1) == _lib.K3_ERR_WORKSPACE
