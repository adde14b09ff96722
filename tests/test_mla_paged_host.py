"""The paged cache's calls without a GPU: what is refused before anything is launched, what the wrappers pass on, the tables' class over the
definition of its one launch."""
from __future__ import annotations

import ctypes

import pytest
import torch

import _paged_oracle as oracle
from test_mla_q4_host import _launches

BF16, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


def _whole(*s):
    return torch.zeros(s, dtype=I32)


# ------------------------------------------------------------------------------- tables
def _tables(**kw):
    from k3hip.pages import page_tables
    args = dict(table=_whole(3, 4), lengths=_whole(3), target=_whole(3), free=_whole(9), used=_whole(1), page_size=32, tokens=2)
    args.update(kw)
    return page_tables(**args)


@pytest.mark.parametrize("kw,error", [
    (dict(table=torch.zeros(3, 4)), TypeError), (dict(table=_whole(12)), ValueError), (dict(table=_whole(4, 3).t()), ValueError),
    (dict(table=_whole(1, 4).expand(3, 4)), ValueError), (dict(table=_whole(20).as_strided((3, 4), (3, 1))), ValueError),
    (dict(lengths=_whole(2)), ValueError), (dict(lengths=torch.zeros(3, dtype=torch.int64)), TypeError), (dict(target=_whole(4)), ValueError),
    (dict(target=_whole(6)[::2]), ValueError), (dict(free=_whole(3, 3)), ValueError), (dict(free=torch.zeros(9)), TypeError),
    (dict(used=_whole(2)), ValueError), (dict(shared=_whole(2)), ValueError), (dict(page_size=0), ValueError), (dict(page_size=48), ValueError),
    (dict(page_size=1 << 17), ValueError), (dict(tokens=-1), ValueError),
])
def test_tables_refuse(monkeypatch, kw, error):
    calls = _launches(monkeypatch)
    with pytest.raises(error):
        _tables(**kw)
    assert not calls


def test_tables_pass_on(monkeypatch):
    calls = _launches(monkeypatch)
    n, u, slots = _tables()
    assert n.shape == (3,) and u.shape == (1,) and slots.shape == (3, 2) and calls[0][0] == "k3_page_tables"
    wide = _whole(3, 9)[:, 2:6]
    _tables(table=wide, tokens=0)
    assert calls[1][1][1:3] == (9, 4)
    lengths, used = _whole(3), _whole(1)
    n, u, _ = _tables(lengths=lengths, used=used, inplace=True)
    assert n is lengths and u is used
    assert _tables(table=_whole(0, 4), lengths=_whole(0), target=_whole(0))[2].shape == (0, 2) and len(calls) == 3


def test_entry_points_refuse():
    from k3hip import _lib
    lib = _lib.lib()
    p, n = ctypes.c_void_p(4096), None
    tab = [p, 4, 4, p, p, n, p, 9, p, 32, 3, 2, p, p, p, p, 1 << 20, n]
    app = [p, 1024, 512, 0, p, 128, 64, 0, n, 1e-5, p, p, 32 * 512, 512, p, 32 * 64, 64, 2, 5, 32, 2, 2, 512, 64, n]
    att = [p, 1536, 512, 128, p, 768, 256, 64, 0, p, p, p, 32 * 512, 512, p, 32 * 64, 64, 2, 5, 32, p, 4, 4, n, 0, p, n, 128, 2, 3, 4, 512, 64,
           128, 96, 0.1, n, p, 0, p, 1 << 30, n]
    S, D, A, W, N = _lib.K3_ERR_SHAPE, _lib.K3_ERR_DTYPE, _lib.K3_ERR_ALIGN, _lib.K3_ERR_WORKSPACE, _lib.K3_ERR_NULL
    odd = ctypes.c_void_p(4100)
    for call, base, at, want in (
            (lib.k3_page_tables, tab, {1: 3}, S), (lib.k3_page_tables, tab, {9: 24}, S), (lib.k3_page_tables, tab, {9: 0}, S),
            (lib.k3_page_tables, tab, {2: 1 << 27, 1: 1 << 27}, S), (lib.k3_page_tables, tab, {10: 70000}, S), (lib.k3_page_tables, tab, {11: -1}, S),
            (lib.k3_page_tables, tab, {16: 8}, W), (lib.k3_page_tables, tab, {0: n}, N), (lib.k3_page_tables, tab, {14: n}, N),
            (lib.k3_page_tables, tab, {15: ctypes.c_void_p(4098)}, A),
            (lib.k3_mla_paged_append, app, {3: 2}, D), (lib.k3_mla_paged_append, app, {17: 0}, D), (lib.k3_mla_paged_append, app, {22: 256}, S),
            (lib.k3_mla_paged_append, app, {2: 514}, S), (lib.k3_mla_paged_append, app, {13: 504}, S), (lib.k3_mla_paged_append, app, {12: 512}, S),
            (lib.k3_mla_paged_append, app, {15: 0}, S), (lib.k3_mla_paged_append, app, {19: 33}, S), (lib.k3_mla_paged_append, app, {0: odd}, A),
            (lib.k3_mla_paged_append, app, {11: odd}, A), (lib.k3_mla_paged_append, app, {10: n}, N),
            (lib.k3_mla_paged_attention, att, {8: 2}, D), (lib.k3_mla_paged_attention, att, {17: 0}, D), (lib.k3_mla_paged_attention, att, {38: 2}, D),
            (lib.k3_mla_paged_attention, att, {31: 256}, S), (lib.k3_mla_paged_attention, att, {33: 132}, S), (lib.k3_mla_paged_attention, att, {34: 1032}, S),
            (lib.k3_mla_paged_attention, att, {19: 16}, S), (lib.k3_mla_paged_attention, att, {19: 96}, S), (lib.k3_mla_paged_attention, att, {27: 129}, S),
            (lib.k3_mla_paged_attention, att, {21: 3}, S), (lib.k3_mla_paged_attention, att, {30: 5000}, S), (lib.k3_mla_paged_attention, att, {3: 126}, S),
            (lib.k3_mla_paged_attention, att, {13: 516}, S), (lib.k3_mla_paged_attention, att, {15: 2044}, S), (lib.k3_mla_paged_attention, att, {16: 56}, S),
            (lib.k3_mla_paged_attention, att, {28: 40000}, S), (lib.k3_mla_paged_attention, att, {0: odd}, A), (lib.k3_mla_paged_attention, att, {14: odd}, A),
            (lib.k3_mla_paged_attention, att, {40: 100}, W), (lib.k3_mla_paged_attention, att, {25: n}, N), (lib.k3_mla_paged_attention, att, {24: 2}, N)):
        args = list(base)
        for i, v in at.items():
            args[i] = v
        assert call(*args) == want, (call.__name__, at, lib.k3_last_error())
    # nothing to do is no error, whatever the rest is
    for call, base, i in ((lib.k3_page_tables, tab, 10), (lib.k3_mla_paged_append, app, 20), (lib.k3_mla_paged_append, app, 21),
                          (lib.k3_mla_paged_append, app, 18), (lib.k3_mla_paged_attention, att, 28), (lib.k3_mla_paged_attention, att, 29)):
        args = list(base)
        args[i] = 0
        assert call(*args) == _lib.K3_OK


# ------------------------------------------------------------------------------- append
def _append(**kw):
    from k3hip.mla_paged import mla_paged_append
    args = dict(c_new=torch.zeros(2, 3, 512), r_new=torch.zeros(2, 3, 64), slots=_whole(2, 3), lat=torch.zeros(4, 32, 512, dtype=F16),
                rot=torch.zeros(4, 32, 64, dtype=F16))
    args.update(kw)
    return mla_paged_append(**args)


@pytest.mark.parametrize("kw,error", [
    (dict(c_new=torch.zeros(2, 3, 511)), ValueError), (dict(c_new=torch.zeros(2, 2, 512)), ValueError), (dict(r_new=torch.zeros(2, 3, 63)), ValueError),
    (dict(c_new=torch.zeros(6, 512), r_new=torch.zeros(6, 64)), ValueError), (dict(c_new=torch.zeros(2, 3, 512, dtype=F16)), TypeError),
    (dict(slots=_whole(2, 4)), ValueError), (dict(slots=_whole(3, 2).t()), ValueError), (dict(slots=torch.zeros(2, 3, dtype=torch.int64)), TypeError),
    (dict(lat=torch.zeros(4, 32, 512)), TypeError), (dict(lat=torch.zeros(4, 32, 512, dtype=BF16)), TypeError),
    (dict(rot=torch.zeros(4, 16, 64, dtype=F16)), ValueError), (dict(lat=torch.zeros(128, 512, dtype=F16)), ValueError),
    (dict(lat=torch.zeros(1, 32, 512, dtype=F16).expand(4, 32, 512)), ValueError), (dict(rot=torch.zeros(4, 1, 64, dtype=F16).expand(4, 32, 64)), ValueError),
    (dict(lat=torch.zeros(4, 24, 512, dtype=F16), rot=torch.zeros(4, 24, 64, dtype=F16)), ValueError), (dict(norm=torch.ones(64)), ValueError),
    (dict(c_new=torch.zeros(2, 3, 512, requires_grad=True)), ValueError), (dict(lat=torch.zeros(4, 32, 512, dtype=F16, requires_grad=True)), ValueError),
    (dict(norm=torch.ones(512, requires_grad=True)), ValueError),
])
def test_append_refuses(monkeypatch, kw, error):
    calls = _launches(monkeypatch)
    with pytest.raises(error):
        _append(**kw)
    assert not calls


def test_append_passes_on(monkeypatch):
    calls = _launches(monkeypatch)
    both = torch.zeros(4, 32, 576, dtype=F16)
    _append(lat=both[..., :512], rot=both[..., 512:], norm=torch.ones(512, dtype=BF16))
    assert calls[0][1][12:14] == (32 * 576, 576)
    # one token of one request out of a wider row: pitches that are never used are not looked at
    row = torch.zeros(1, 1, 580, dtype=BF16)
    _append(c_new=row[..., :512], r_new=row[..., 512:576], slots=_whole(1, 1))
    assert calls[1][1][1:3] == (0, 0)
    _append(c_new=torch.zeros(2, 0, 512), r_new=torch.zeros(2, 0, 64), slots=_whole(2, 0))
    _append(lat=torch.zeros(0, 32, 512, dtype=F16), rot=torch.zeros(0, 32, 64, dtype=F16))
    assert len(calls) == 2


# ------------------------------------------------------------------------------- attention
def _attend(**kw):
    from k3hip.mla_paged import mla_paged_attention
    w = torch.zeros(4, 128, 512, dtype=BF16)
    args = dict(q_nope=torch.zeros(2, 3, 4, 128), q_rot=torch.zeros(2, 3, 4, 64), wk=w, wv=w, lat=torch.zeros(5, 32, 512, dtype=F16),
                rot=torch.zeros(5, 32, 64, dtype=F16), table=_whole(2, 4), lengths=_whole(2), scale=0.1)
    args.update(kw)
    return mla_paged_attention(**args)


@pytest.mark.parametrize("kw,error", [
    (dict(q_nope=torch.zeros(2, 3, 4, 96)), ValueError), (dict(q_rot=torch.zeros(2, 3, 4, 32)), ValueError), (dict(q_rot=torch.zeros(2, 3, 5, 64)), ValueError),
    (dict(q_nope=torch.zeros(2, 4, 128), q_rot=torch.zeros(2, 4, 64)), ValueError), (dict(wk=torch.zeros(4, 128, 512)), TypeError),
    (dict(wv=torch.zeros(5, 128, 512, dtype=BF16)), ValueError), (dict(wv=torch.zeros(4, 128, 256, dtype=BF16)), ValueError),
    (dict(lat=torch.zeros(5, 32, 512)), TypeError), (dict(lat=torch.zeros(5, 32, 512, dtype=BF16)), TypeError), (dict(rot=torch.zeros(6, 32, 64, dtype=F16)), ValueError),
    (dict(lat=torch.zeros(5, 16, 512, dtype=F16), rot=torch.zeros(5, 16, 64, dtype=F16)), ValueError),
    (dict(lat=torch.zeros(5, 48, 512, dtype=F16), rot=torch.zeros(5, 48, 64, dtype=F16)), ValueError),
    (dict(lat=torch.zeros(5, 32, 516, dtype=F16)[..., :512]), ValueError), (dict(rot=torch.zeros(5, 32, 66, dtype=F16)[..., :64]), ValueError),
    (dict(table=_whole(3, 4)), ValueError), (dict(table=torch.zeros(2, 4, dtype=torch.int64)), TypeError), (dict(table=_whole(4, 2).t()), ValueError),
    (dict(lengths=None), ValueError), (dict(lengths=_whole(3)), ValueError), (dict(lengths=torch.zeros(2)), TypeError), (dict(counts=_whole(1)), ValueError),
    (dict(prefix=torch.zeros(2)), TypeError), (dict(prefix=_whole(1, 2)), ValueError), (dict(prefix=_whole(4)[::2]), ValueError),
    (dict(max_length=129), ValueError), (dict(max_length=-1), ValueError), (dict(gate=torch.zeros(2, 3, 4 * 64)), ValueError),
    (dict(gate=torch.zeros(3, 2, 512)), ValueError), (dict(out_dtype=F16), TypeError), (dict(q_nope=torch.zeros(2, 3, 4, 128, requires_grad=True)), ValueError),
    (dict(wk=torch.zeros(4, 128, 512, dtype=BF16, requires_grad=True)), ValueError),
])
def test_attention_refuses(monkeypatch, kw, error):
    calls = _launches(monkeypatch)
    with pytest.raises(error):
        _attend(**kw)
    assert not calls


def test_attention_passes_on(monkeypatch):
    calls = _launches(monkeypatch)
    assert _attend().shape == (2, 3, 4, 128) and calls[0][1][27] == 128
    _attend(max_length=70, prefix=_whole(2))
    assert calls[1][1][24] == 2 and calls[1][1][27] == 70
    assert _attend(q_nope=torch.zeros(2, 0, 4, 128), q_rot=torch.zeros(2, 0, 4, 64)).shape == (2, 0, 4, 128) and len(calls) == 2
    # a batch of more than 65,536 rows in parts
    B = 100
    w = torch.zeros(1000, 8, 512, dtype=BF16)
    _attend(q_nope=torch.zeros(B, 1, 1000, 8), q_rot=torch.zeros(B, 1, 1000, 64), wk=w, wv=w, table=_whole(B, 1), lengths=_whole(B), counts=_whole(B),
            gate=torch.zeros(B, 1, 8000))
    assert [c[1][28] for c in calls[2:]] == [65, 35]


# ------------------------------------------------------------------------------- the tables' class
@pytest.fixture
def on_cpu(monkeypatch):
    """page_tables by its definition."""
    from k3hip import pages

    def plain(table, lengths, target, free, used, page_size, tokens=0, shared=None, inplace=False):
        assert inplace
        t, f, n, u, s = oracle.tables(table.tolist(), lengths.tolist(), target.tolist(), free.tolist(), int(used), page_size, tokens,
                                      None if shared is None else shared.tolist())
        for to, x in ((table, t), (free, f), (lengths, n), (used, [u])):
            to.copy_(torch.tensor(x, dtype=I32).view(to.shape))
        return lengths, used, torch.tensor(s, dtype=I32).view(len(n), tokens)

    monkeypatch.setattr(pages, "page_tables", plain)
    return pages


def _held(t):
    """Pages by request, without the common prefix; all of them different, and none of them free."""
    n = 0 if t.prefix is None else len(t.prefix)
    rows = [r[n:-(-k // t.page_size)] for r, k in zip(t.table.tolist(), t.lengths.tolist())]
    flat = [p for r in rows for p in r] + ([] if t.prefix is None else t.prefix.tolist()) + t.free.tolist()[int(t.used):]
    assert len(flat) == len(set(flat)) and set(flat) <= set(range(t.pages))
    return rows


def test_page_table_of_a_batch(on_cpu):
    t = on_cpu.PageTable(4, 256, 12, page_size=32, device="cpu")
    assert t.capacity == 256 and t.batch == 4
    slots = t.extend(torch.tensor([40, 0, 33, 32], dtype=I32), tokens=40)
    assert t.lengths.tolist() == [40, 0, 33, 32] == t.counts.tolist() and int((slots >= 0).sum()) == 105
    assert [len(r) for r in _held(t)] == [2, 0, 2, 1]
    t.extend(1)
    assert t.lengths.tolist() == [41, 1, 34, 33] and [len(r) for r in _held(t)] == [2, 1, 2, 2]
    # drafts taken back
    t.truncate(torch.tensor([41, 1, 34, 32], dtype=I32))
    assert t.lengths.tolist() == [41, 1, 34, 32] and t.counts.tolist() == [0] * 4 and [len(r) for r in _held(t)] == [2, 1, 2, 1]
    # more than there is: the first that does not fit, and every later one that needs pages, gets none
    t.extend(torch.tensor([60, 200, 1, 0], dtype=I32), tokens=200)
    assert t.counts.tolist() == [60, 0, 1, 0] and t.lengths.tolist() == [101, 1, 35, 32]
    t.release(torch.tensor([True, False, False, True]))
    assert t.lengths.tolist() == [0, 1, 35, 0] and [len(r) for r in _held(t)] == [0, 1, 2, 0] and int(t.used) == 3


def test_page_table_with_a_common_prefix(on_cpu):
    t = on_cpu.PageTable(3, 256, 12, page_size=32, device="cpu")
    t.extend(torch.tensor([0, 70, 0], dtype=I32), tokens=70)
    for length, source in ((40, 1), (0, 1), (96, 1), (64, 0), (64, 3), (512, 1)):
        with pytest.raises(ValueError):
            t.share(length, source)
    t.share(64, source=1)
    assert t.lengths.tolist() == [64, 70, 64] and t.prefix.tolist() == t.table[1, :2].tolist()
    with pytest.raises(ValueError, match="already"):
        t.share(32, 1)
    t.extend(5)
    assert t.lengths.tolist() == [69, 75, 69] and [len(r) for r in _held(t)] == [1, 1, 1]
    # what ends gives back its own pages, and its place begins with the prefix again
    t.release(torch.tensor([True, True, False]))
    assert t.lengths.tolist() == [64, 64, 69] and [len(r) for r in _held(t)] == [0, 0, 1] and int(t.used) == 3
    t.truncate(torch.zeros(3, dtype=I32))
    assert t.lengths.tolist() == [64] * 3 and int(t.used) == 2
    t.extend(1)
    assert t.table[:, :2].tolist() == [t.prefix.tolist()] * 3 and t.lengths.tolist() == [65] * 3
    _held(t)


@pytest.mark.parametrize("call,first", [
    (lambda t: t.extend(torch.tensor([-10, -200, 0], dtype=I32), tokens=1), 65), (lambda t: t.resize(torch.tensor([0, -3, 69], dtype=I32)), 64),
])
def test_no_request_goes_below_a_common_prefix(on_cpu, call, first):
    t = on_cpu.PageTable(3, 256, 12, page_size=32, device="cpu")
    t.extend(torch.tensor([70, 0, 0], dtype=I32), tokens=70)
    t.share(64)
    t.extend(5)
    call(t)
    assert t.lengths.tolist() == [first, 64, 69] and t.counts.tolist() == [0] * 3
    t.extend(40)
    # the rows still begin with the prefix, and what follows is nobody else's
    assert t.table[:, :2].tolist() == [t.prefix.tolist()] * 3
    _held(t)


def test_share_wants_the_others_empty(on_cpu):
    t = on_cpu.PageTable(2, 64, 4, page_size=32, device="cpu")
    t.extend(32)
    with pytest.raises(ValueError, match="hold nothing"):
        t.share(32)


@pytest.mark.parametrize("call", [
    lambda t: t.extend(torch.zeros(2, dtype=I32)), lambda t: t.extend(torch.zeros(3, dtype=I32), tokens=1), lambda t: t.truncate(torch.zeros(3, dtype=I32)),
    lambda t: t.resize(torch.zeros(3, dtype=I32)), lambda t: t.resize(torch.zeros(2)), lambda t: t.release(torch.zeros(3, dtype=torch.bool)), lambda t: t.release(torch.zeros(2, dtype=I32)),
])
def test_page_table_refuses(on_cpu, call):
    with pytest.raises((ValueError, TypeError)):
        call(on_cpu.PageTable(2, 64, 4, page_size=32, device="cpu"))


def test_cache_refuses(on_cpu):
    from k3hip.mla_paged import new_cache_paged
    t = on_cpu.PageTable(2, 64, 4, page_size=32, device="cpu")
    with pytest.raises(TypeError):
        new_cache_paged(t, dtype=F32)
    with pytest.raises(ValueError):
        new_cache_paged(on_cpu.PageTable(2, 64, 4, page_size=16, device="cpu"))
    cache = new_cache_paged(t, BF16)
    assert cache.latent.shape == (4, 32, 512) and cache.latent.dtype == BF16 and cache.bytes_per_token() == 1152
    with pytest.raises(ValueError, match="extend"):
        cache.append(torch.zeros(2, 1, 512), torch.zeros(2, 1, 64))


def test_layer_refuses_what_the_pages_do_not_take(on_cpu):
    from types import SimpleNamespace

    from k3hip.mla import MLAAttention
    from k3hip.mla_paged import new_cache_paged

    def layer(kv_b=BF16, **kw):
        cfg = dict(num_attention_heads=2, q_lora_rank=16, kv_lora_rank=512, qk_nope_head_dim=8, qk_rope_head_dim=64, v_head_dim=8, q_head_dim=72,
                   rms_norm_eps=1e-5)
        cfg = SimpleNamespace(**{**cfg, **kw})
        z = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
        w = {"q_a_proj.weight": z(16, 32), "q_a_layernorm.weight": z(16), "q_b_proj.weight": z(144, 16), "kv_a_proj_with_mqa.weight": z(576, 32),
             "kv_a_layernorm.weight": z(512), "kv_b_proj.weight": torch.zeros(2 * (cfg.qk_nope_head_dim + 8), 512, dtype=kv_b), "o_proj.weight": z(32, 16)}
        return MLAAttention(cfg, w), w

    t = on_cpu.PageTable(2, 64, 4, page_size=32, device="cpu")
    t.extend(1)
    cache = new_cache_paged(t)
    x = torch.zeros(2, 1, 32)
    with pytest.raises(ValueError, match="bf16 kv_b"):
        layer(kv_b=F32)[0](x, cache)
    with pytest.raises(ValueError, match="paged cache takes"):
        layer(qk_nope_head_dim=12, q_head_dim=76)[0](x, cache)
    with pytest.raises(ValueError, match="extend"):
        layer()[0](torch.zeros(2, 2, 32), cache)
    with pytest.raises(ValueError, match="extend"):
        layer()[0](torch.zeros(1, 1, 32), cache)
    with pytest.raises(ValueError, match="gradient"):
        layer()[0](x.requires_grad_(), cache)
