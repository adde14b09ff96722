"""The paged cache on the device where its calls have an edge: counts above the slots, requests below their shared pages, padding that is not
finite, batches and passes that are cut."""
from __future__ import annotations

import pytest
import torch

from test_gpu_mla_paged_layer import HID, _layer

pytestmark = pytest.mark.gpu
BF16, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


def _whole(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def test_counts_above_the_slots_are_cut():
    """A step of three tokens a request, five asked for: what the layer answers is what it answers when three are."""
    from k3hip.mla_paged import new_cache_paged
    from k3hip.pages import PageTable
    layer, _ = _layer(4)
    x = torch.randn(3, 40, HID, generator=torch.Generator().manual_seed(2)).cuda()
    outs = []
    for asked in ([5, 2, 0], [3, 2, 0]):
        t = PageTable(3, 128, 12, page_size=32)
        cache = new_cache_paged(t)
        t.extend(_whole([40, 31, 7]), tokens=40)
        layer(x, cache)
        t.extend(_whole(asked), tokens=3)
        assert t.counts.tolist() == [3, 2, 0] and t.lengths.tolist() == [43, 33, 7]
        outs.append(layer(x[:, :3], cache)[0])
    assert bool((outs[0] == outs[1]).all()) and bool(outs[0][0].any()) and not bool(outs[0][2].any())


# ------------------------------------------------------------------------------- pages that a request shares
def _account(table, lengths, shared, free, used, page, common):
    """Every page is common, in one request's row behind its shared ones, or free; none is in two of these, none in none."""
    held = [p for row, n, s in zip(table.tolist(), lengths.tolist(), shared.tolist()) for p in row[max(s, 0):-(-n // page)]]
    flat = held + list(common) + free.tolist()[int(used):]
    assert sorted(flat) == list(range(len(free))), (held, flat)


@pytest.mark.parametrize("tokens", [0, 5000])         # (one launch, two)
def test_a_request_below_its_shared_pages_loses_none(tokens):
    from k3hip.pages import page_tables
    page = 32
    table, free, used = _whole([[0, 1, -1, -1]]), _whole([0, 1, 2, 3, 4, 5]), _whole([2])
    lengths, shared = _whole([64]), _whole([2])
    for target, held, its in ((0, 0, 2), (96, 96, 0), (0, 0, 0), (128, 128, 0), (128, 128, 0), (40, 40, 0), (0, 0, 0), (96, 96, 0)):
        page_tables(table, lengths, _whole([target]), free, used, page, tokens=tokens, shared=shared, inplace=True)
        assert lengths.tolist() == [held] and shared.tolist() == [its], target
        _account(table, lengths, shared, free, used, page, (0, 1))
    # one that comes below some of them only; one that gets no page keeps its account
    table, free, used = _whole([[0, 1, 2, 3, -1, -1], [0, 1, 2, -1, -1, -1]]), _whole(list(range(8))), _whole([4])
    lengths, shared = _whole([128, 0]), _whole([3, 3])
    for target, held, its in (([40, 0], [40, 0], [3, 3]), ([65, 192], [65, 0], [2, 3]), ([160, 0], [160, 0], [2, 3]), ([0, 1], [0, 1], [2, 0])):
        page_tables(table, lengths, _whole(target), free, used, page, tokens=tokens, shared=shared, inplace=True)
        assert lengths.tolist() == held and shared.tolist() == its, target
        _account(table, lengths, shared, free, used, page, (0, 1, 2))


@pytest.mark.parametrize("B,page,tokens", [(6, 32, 3), (300, 16, 1), (2500, 8, 2)])
def test_no_page_is_lost_on_the_way(B, page, tokens):
    """Requests that begin with common pages, below them and above them again, in any order."""
    import random

    from k3hip.pages import page_tables
    rng = random.Random(B)
    width, common = 7, [5, 0, 3]
    pool = 3 + 4 * B
    rest = [p for p in range(pool) if p not in common]
    rng.shuffle(rest)
    table = _whole([common + [-1] * (width - 3) for _ in range(B)])
    free, used = _whole(common + rest), _whole([3])
    lengths, shared = torch.full((B,), 3 * page, dtype=I32, device="cuda"), torch.full((B,), 3, dtype=I32, device="cuda")
    for step in range(25):
        now = lengths.tolist()
        to = [rng.choice([0, n, n + 1, n - page, n + page, rng.randint(0, width * page)]) for n in now]
        page_tables(table, lengths, _whole(to), free, used, page, tokens=tokens, shared=shared, inplace=True)
        _account(table, lengths, shared, free, used, page, common)
    assert min(shared.tolist()) == 0


# ------------------------------------------------------------------------------- rows of no query
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("B,T,H", [(3, 2, 8), (5, 4, 16), (6, 40, 24), (9, 80, 32)])       # (one to 32 queries a block of the last launch)
def test_a_gate_that_is_no_number_leaves_zeros_where_nothing_is_seen(B, T, H, out):
    import _paged_oracle as oracle
    from k3hip.mla_paged import mla_paged_attention
    g = torch.Generator().manual_seed(B)
    case = oracle.make(g, B, T, H, [T + 30 + 7 * b for b in range(B)], page=32, x=F32)
    counts = _whole([T // 2] + [T] * (B - 1))
    case["lengths"][1] = 0
    case["table"][2] = -1                                           # (no page of it is in the pool)
    gate = torch.randn(B, T, H * 128, generator=g).cuda()
    clean = mla_paged_attention(**case, counts=counts, gate=gate, out_dtype=out)
    nothing = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    nothing[0, T // 2:] = nothing[1] = nothing[2] = True
    for value in (float("nan"), float("-inf"), float("inf")):
        bad = torch.where(nothing[..., None], torch.full_like(gate, value), gate)
        got = mla_paged_attention(**case, counts=counts, gate=bad, out_dtype=out)
        assert not bool(got[nothing].any()) and bool((got == clean).all()) and bool(got[~nothing].any())


@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("heads,T", [(4, 3), (16, 40)])
def test_padding_that_is_no_number_stays_out_of_a_step(heads, T, gate):
    """Rows past a request's tokens hold whatever the caller's buffer does: their outputs are zeros, the others' and the cache as with zeros there."""
    from k3hip.mla_paged import new_cache_paged
    from k3hip.pages import PageTable
    layer, _ = _layer(heads, gate)
    x = torch.randn(3, T, HID, generator=torch.Generator().manual_seed(2)).cuda()
    counts = [T, 1, 0]
    outs, pools = [], []
    for padding in (0.0, float("nan"), float("inf")):
        t = PageTable(3, 128, 12, page_size=32)
        cache = new_cache_paged(t)
        t.extend(_whole(counts), tokens=T)
        x = x.clone()
        for b, n in enumerate(counts):
            x[b, n:] = padding
        outs.append(layer(x, cache)[0])
        pools.append(torch.cat((cache.latent, cache.rot), -1))
    for out, pool in zip(outs, pools):
        assert not bool(out[1, 1:].any()) and not bool(out[2].any()) and bool((out == outs[0]).all()) and bool((pool == pools[0]).all())


# ------------------------------------------------------------------------------- more than a launch's row of blocks
def test_append_of_more_tokens_than_a_row_of_blocks():
    """2^26 tokens are 2^32 threads; most slots are outside the pool, so only a few of them are written."""
    from k3hip.mla_paged import mla_paged_append
    M = (1 << 26) + 5
    row = torch.randn(2, 1, 576, generator=torch.Generator().manual_seed(1)).cuda()
    c, r = row[:1, :, :512].expand(1, M, 512), row[:1, :, 512:].expand(1, M, 64)        # (one row, M times)
    slots = torch.full((1, M), -1, dtype=I32, device="cuda")
    written = {0: 3, 7: 40, (1 << 26) - 1: 31, 1 << 26: 0, M - 1: 63}
    for m, s in written.items():
        slots[0, m] = s
    lat, rot = torch.zeros(2, 32, 512, dtype=F16, device="cuda"), torch.zeros(2, 32, 64, dtype=F16, device="cuda")
    mla_paged_append(c, r, slots, lat, rot)
    want = torch.zeros(64, 576, dtype=F16, device="cuda")
    want[list(written.values())] = row[0].to(F16)
    assert bool((torch.cat((lat, rot), -1).view(64, 576) == want).all())


# ------------------------------------------------------------------------------- batches and queries in parts
def _sampled(case, got, which, out, **kw):
    import _paged_oracle as oracle
    from test_gpu_mla_paged import _check
    for b in which:
        part = {k: v[b:b + 1] if k in ("q_nope", "q_rot", "table", "lengths") else v for k, v in case.items()}
        _check(got[b:b + 1], *oracle.attention(**part, out_dtype=out, **{k: v[b:b + 1] for k, v in kw.items()}), label=b)


@pytest.mark.parametrize("H,pages,out", [(60, F16, BF16), (16, F16, BF16), (32, F16, F32), (40, BF16, BF16), (16, BF16, F32), (24, F16, F32)])
def test_more_than_1024_sequences_behind_a_prefix(H, pages, out):
    """(whose ranges' length is not searched for), one of them long; groups that fill whole tiles and groups that do not."""
    import _paged_oracle as oracle
    from k3hip.mla_paged import mla_paged_attention
    B = 1030
    lens = [96 + b % 70 for b in range(B)]
    lens[3], lens[700], lens[1029] = 96 + 3000, 20, 0
    case = oracle.make(torch.Generator().manual_seed(H), B, 1, H, lens, page=32, pages_dtype=pages, x=BF16, prefix=96)
    got = mla_paged_attention(**case, out_dtype=out)
    _sampled(case, got, (0, 3, 4, 256, 700, 1028), out)
    assert not bool(got[1029].any())


@pytest.mark.parametrize("pages,out", [(F16, BF16), (F16, F32), (BF16, BF16), (BF16, F32)])
def test_passes_with_counts_gate_and_prefix(pages, out):
    """86,400 rows: 227 queries of each, then 73 (of requests that have 300, 228, 150 and none)."""
    import _paged_oracle as oracle
    from k3hip.mla_paged import mla_paged_attention
    B, T, H = 4, 300, 72
    g = torch.Generator().manual_seed(5)
    case = oracle.make(g, B, T, H, [128 + 320, 228, 128 + 190, 128 + 64], page=64, pages_dtype=pages, x=F32, prefix=128)
    counts, gate = _whole([999, 228, 150, 0]), 2 * torch.randn(B, T, H * 128, generator=g).cuda()
    gate[1, 228:] = gate[2, 150:] = gate[3] = float("nan")
    got = mla_paged_attention(**case, counts=counts, gate=gate, out_dtype=out)
    _sampled(case, got, range(3), out, counts=counts, gate=gate.nan_to_num())
    assert not bool(got[1, 228:].any()) and not bool(got[2, 150:].any()) and not bool(got[3].any())


@pytest.mark.parametrize("pages", [F16, BF16])
def test_counts_and_gate_at_an_fp32_result(pages):
    """What the layer calls: fp32 queries and results, counts and a gate; few queries and many, behind a prefix and without."""
    import _paged_oracle as oracle
    from k3hip.mla_paged import mla_paged_attention
    for T, H, prefix, lens in ((1, 96, 0, [1, 700, 0]), (5, 12, 64, [90, 70, 69]), (40, 16, 0, [64, 40, 300])):
        g = torch.Generator().manual_seed(T)
        case = oracle.make(g, 3, T, H, lens, page=32, pages_dtype=pages, x=F32, prefix=prefix)
        counts, gate = _whole([1, T, T // 2]), 2 * torch.randn(3, T, H * 128, generator=g).cuda()
        _sampled(case, mla_paged_attention(**case, counts=counts, gate=gate), range(3), F32, counts=counts, gate=gate)


@pytest.mark.parametrize("dtype,x_dtype", [(F16, F32), (F16, BF16), (BF16, F32), (BF16, BF16)])
def test_a_batch_of_one_place(dtype, x_dtype):
    """One request, one token a step (tolerances: tests/test_gpu_mla_paged_layer.py)."""
    from k3hip.mla import new_cache
    from k3hip.mla_paged import new_cache_paged
    from k3hip.pages import PageTable
    from test_gpu_mla_paged_layer import _rel, _rows, _want
    layer, w = _layer(16)
    g = torch.Generator().manual_seed(3)
    t, own = PageTable(1, 256, 8, page_size=32), new_cache(1, 512, 64, 1, dtype=F32)
    cache = new_cache_paged(t, dtype)
    for T in (1, 1, 70, 1, 1):
        x = torch.randn(1, T, HID, generator=g).to(x_dtype).cuda()
        t.extend(T)
        out = layer(x, cache)[0]
        alone, own = layer(x, own)
        assert out.shape == (1, T, HID) and out.dtype == F32
        assert _rel(out[0], _want(w, 16, x[0], *_rows(cache, 0), True)) < 2e-5
        assert _rel(out[0], alone[0].double()) < 4 * (2.0 ** -11 if dtype == F16 else 2.0 ** -8)
