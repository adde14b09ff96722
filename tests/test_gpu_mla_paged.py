"""The paged latent cache on the device: tables, append, attention against their definitions (tests/_paged_oracle.py)."""
from __future__ import annotations

import math
import random

import pytest
import torch

import _paged_oracle as oracle

pytestmark = pytest.mark.gpu
BF16, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _check(out, want, bound, label=""):
    got = out.double()
    assert bool(torch.isfinite(got).all()), label
    over = (got - want).abs() - bound
    assert float(over.max()) <= 0, (label, float(over.max()), float(((got - want).abs() / bound.clamp(min=1e-30)).max()))


# ------------------------------------------------------------------------------- tables
def _tables_case(rng, B, width, page, tokens, pool_slack, ended=0.3, shared=False):
    most = width * page
    lengths = [rng.randint(0, most) for _ in range(B)]
    target = [0 if rng.random() < ended else min(most + rng.choice([0, 0, 0, 1]), n + rng.randint(0, max(1, tokens) + page)) for n in lengths]
    have = [-(-n // page) for n in lengths]
    pool = sum(have) + max(0, sum(-(-t // page) for t in target) - sum(have)) + pool_slack
    pool = max(pool, sum(have), 1)
    order = list(range(pool))
    rng.shuffle(order)
    it = iter(order)
    table = [[next(it) for _ in range(h)] + [-7] * (width - h) for h in have]
    return table, lengths, target, order, sum(have), [rng.randint(0, 2) for _ in range(B)] if shared else None


@pytest.mark.parametrize("B,width,page,tokens,slack,shared", [
    (1, 1, 1, 1, 0, False), (1, 4, 64, 0, 3, False), (3, 5, 32, 1, -4, False), (64, 16, 64, 1, 9, True), (33, 9, 16, 7, -30, True),
    (2049, 3, 8, 1, 5, False), (5, 40, 32, 1300, 11, False), (17, 2, 128, 300, -5, True), (4000, 2, 2, 3, -100, True),
])
def test_page_tables_match_the_definition(B, width, page, tokens, slack, shared):
    from k3hip.pages import page_tables
    for seed in range(3):
        table, lengths, target, free, used, sh = _tables_case(random.Random(seed * 100 + B), B, width, page, tokens, slack, shared=shared)
        whole = lambda x: torch.tensor(x, dtype=I32, device="cuda")  # noqa: E731
        t, f = whole(table), whole(free)
        args = (whole(lengths), whole(target), f, whole([used]), page)
        new, taken, slots = page_tables(t, *args, tokens=tokens, shared=whole(sh) if sh else None)
        w_table, w_free, w_lengths, w_used, w_slots = oracle.tables(table, lengths, target, free, used, page, tokens, sh)
        assert t.tolist() == w_table and f.tolist() == w_free and new.tolist() == w_lengths and taken.tolist() == [w_used]
        assert slots.tolist() == w_slots
        assert args[0].tolist() == lengths and args[3].tolist() == [used]
        # the same call again answers the same (what it gave is not read as what was held)
        again = page_tables(t, *args, tokens=tokens, shared=whole(sh) if sh else None)
        assert t.tolist() == w_table and f.tolist() == w_free and again[0].tolist() == w_lengths and again[2].tolist() == w_slots


def test_page_tables_in_place_and_odd_values():
    from k3hip.pages import page_tables
    whole = lambda x: torch.tensor(x, dtype=I32, device="cuda")  # noqa: E731
    table, free = [[3, 4, -1], [5, -1, -1], [6, 7, 8]], [3, 4, 5, 6, 7, 8, 0, 1, 2]
    lengths, target = [70, -5, 10 ** 9], [-3, 65, 96]       # a negative length is none, one past the table is cut; a negative target is 0
    t, f, n, u = whole(table), whole(free), whole(lengths), whole([6])
    new, used, slots = page_tables(t, n, whole(target), f, u, 32, tokens=2, inplace=True)
    assert new is n and used is u
    want = oracle.tables(table, lengths, target, free, 6, 32, 2)
    assert (t.tolist(), f.tolist(), n.tolist(), u.tolist()[0], slots.tolist()) == want
    # a list whose count of taken entries is out of range
    for wrong in (-4, 99):
        t, f = whole(table), whole(free)
        new, used, slots = page_tables(t, whole([70, 32, 96]), whole([0, 64, 0]), f, whole([wrong]), 32, tokens=1)
        want = oracle.tables(table, [70, 32, 96], [0, 64, 0], free, wrong, 32, 1)
        assert (t.tolist(), f.tolist(), new.tolist(), used.tolist()[0], slots.tolist()) == want


# ------------------------------------------------------------------------------- append
@pytest.mark.parametrize("pages", [F16, BF16])
@pytest.mark.parametrize("x", [F32, BF16])
@pytest.mark.parametrize("B,T,page,norm", [(1, 1, 1, True), (5, 1, 64, False), (3, 37, 32, True), (2, 130, 16, False)])
def test_append(B, T, page, norm, x, pages):
    from k3hip.mla_paged import mla_paged_append
    g = _gen(B * T)
    total = -(-B * T // page) + 2
    rows = torch.randperm(total * page, generator=g)[:B * T].to(I32).view(B, T)
    rows[0, T // 2] = -1
    if T > 2:
        rows[-1, -1] = total * page          # past the pool
    ckv = (3 * torch.randn(B, T, 580, generator=g)).to(x).cuda()
    c, r = ckv[..., :512], ckv[..., 512:576]
    w = torch.rand(512, generator=g).cuda() + 0.5 if norm else None
    store = torch.full((total, page, 584), 7.0, dtype=pages, device="cuda")
    lat, rot = store[..., :512], store[..., 512:576]
    mla_paged_append(c, r, rows.cuda(), lat, rot, norm=w, eps=1e-5)
    want = torch.full((total * page, 576), 7.0, dtype=torch.float64)
    cd, rd = c.cpu().double(), r.cpu().double()
    if norm:
        cd = w.cpu().double() * cd / (cd.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    ok = (rows >= 0) & (rows < total * page)
    want[rows[ok].long()] = torch.cat((cd, rd), -1)[ok]
    got = torch.cat((lat, rot), -1).reshape(-1, 576).cpu().double()
    # one rounding of the type, and of fp32's sum of 512 squares (2^-24 x 512 / 2 at most) and three products; below 2^-14 fp16's
    # values are 2^-24 apart whatever their size, so a rounding is off by up to 2^-25 there
    least = 2.0 ** -25 if pages == F16 else 0.0
    assert bool(((got - want).abs() <= want.abs() * (oracle.HALF_STEP[pages] + 2.0 ** -15) + least).all())
    assert bool((store[..., 576:] == 7.0).all())
    exact = want.float().to(pages).double()
    if not norm:
        assert bool((got == exact).all())    # (the one rounding there is)


def test_append_of_what_fp16_does_not_hold():
    from k3hip.mla_paged import mla_paged_append
    c = torch.zeros(1, 1, 512, device="cuda")
    c[0, 0, :4] = torch.tensor([65519.9, 65520.0, -1e9, math.nan])
    lat, rot = torch.zeros(1, 32, 512, dtype=F16, device="cuda"), torch.zeros(1, 32, 64, dtype=F16, device="cuda")
    mla_paged_append(c, torch.full((1, 1, 64), 2.0 ** -24, device="cuda"), torch.tensor([[5]], dtype=I32, device="cuda"), lat, rot)
    assert lat[0, 5, :3].tolist() == [65504.0, math.inf, -math.inf] and bool(lat[0, 5, 3].isnan())
    assert bool((rot[0, 5] == 2.0 ** -24).all()) and float(lat[0, 4].abs().sum() + lat[0, 6].abs().sum()) == 0


# ------------------------------------------------------------------------------- attention
def _run(case, **kw):
    from k3hip.mla_paged import mla_paged_attention
    return mla_paged_attention(**{k: v for k, v in case.items()}, **kw)


FORMS = [(F16, BF16, BF16), (F16, F32, F32), (BF16, BF16, BF16), (BF16, F32, F32), (F16, F32, BF16), (F16, BF16, F32)]
FORMS_PO = [(F16, BF16), (F16, F32), (BF16, BF16), (BF16, F32)]      # pages, result: one, two, two and three terms


@pytest.mark.parametrize("pages,x,out", FORMS)
@pytest.mark.parametrize("T,H,lens,prefix,page", [
    (1, 64, [1], 0, 64), (1, 16, [31, 32, 33], 0, 32), (1, 96, [700, 0, 65], 0, 64), (1, 8, [200] * 9, 0, 64), (3, 20, [130, 3, 2], 0, 64),
    (1, 64, [300, 257, 256, 0, 100], 256, 64), (2, 12, [64, 65, 66, 190, 1], 64, 32), (40, 16, [40, 100], 0, 128), (17, 5, [145, 141], 128, 32),
    (1, 1, [1000], 0, 32), (1, 128, [2500, 2049], 2048, 1024), (32, 3, [32, 100], 0, 32), (79, 5, [200, 150, 80], 64, 64), (64, 16, [64, 129], 0, 64),
])
def test_attention(T, H, lens, prefix, page, pages, x, out):
    case = oracle.make(_gen(T * H + len(lens)), len(lens), T, H, lens, page=page, pages_dtype=pages, x=x, prefix=prefix)
    want, bound = oracle.attention(**case, out_dtype=out)
    _check(_run(case, out_dtype=out), want, bound)


@pytest.mark.parametrize("nope,v", [(8, 8), (64, 72), (256, 520), (192, 1024), (120, 136)])
def test_attention_of_other_head_sizes(nope, v):
    for out in (BF16, F32):
        case = oracle.make(_gen(nope), 2, 2, 4, [77, 40], nope=nope, v=v, x=out)
        want, bound = oracle.attention(**case, out_dtype=out)
        _check(_run(case, out_dtype=out), want, bound)


@pytest.mark.parametrize("pages,out", [(F16, BF16), (F16, F32), (BF16, BF16)])
def test_attention_with_counts_and_gate(pages, out):
    case = oracle.make(_gen(5), 4, 5, 12, [90, 7, 5, 66], pages_dtype=pages, x=F32, prefix=0)
    counts = torch.tensor([3, 5, 0, 99], dtype=I32, device="cuda")
    gate = torch.randn(4, 5, 12 * 128, generator=_gen(6)).cuda() * 2
    want, bound = oracle.attention(**case, counts=counts, gate=gate, out_dtype=out)
    got = _run(case, counts=counts, gate=gate, out_dtype=out)
    _check(got, want, bound)
    assert not bool(got[2].any()) and not bool(got[0, 3:].any())


@pytest.mark.parametrize("pages,out", [(F16, BF16), (BF16, F32)])
def test_attention_over_ranges_of_more_than_64_rounds(pages, out):
    # so many requests that a block takes all 4416 positions of the prefix, 138 rounds
    case = oracle.make(_gen(9), 150, 1, 64, [4416 + b % 3 for b in range(150)], pages_dtype=pages, prefix=4416)
    got = _run(case, out_dtype=out)
    for b in (0, 1, 77, 149):
        one = {k: v[b:b + 1] if k in ("q_nope", "q_rot", "table", "lengths") else v for k, v in case.items()}
        _check(got[b:b + 1], *oracle.attention(**one, out_dtype=out))
    # a page of the prefix that is none: its positions count as not there
    case["prefix"][40] = case["lat"].shape[0]
    got = _run(case, out_dtype=out)
    one = {k: v[5:6] if k in ("q_nope", "q_rot", "table", "lengths") else v for k, v in case.items()}
    _check(got[5:6], *oracle.attention(**one, out_dtype=out))


# ------------------------------------------------------------------------------- what is masked, what is infinite
@pytest.mark.parametrize("pages,out", [(F16, BF16), (F16, F32), (BF16, F32)])
def test_what_is_masked_does_not_matter(pages, out):
    # drafts: the first query does not see the last position, whatever it holds; a short request beside longer ones in the same tiles
    case = oracle.make(_gen(3), 3, 4, 16, [100, 67, 66], pages_dtype=pages, prefix=64)
    clean = _run(case, out_dtype=out)
    _check(clean, *oracle.attention(**case, out_dtype=out))
    for value in (math.nan, math.inf, -math.inf):
        lat, rot = case["lat"].clone(), case["rot"].clone()
        last = int(case["lengths"][0]) - 1
        lat[case["table"][0, last // 64].long(), last % 64, ::7] = value
        rot[case["table"][0, last // 64].long(), last % 64] = value
        got = _run({**case, "lat": lat, "rot": rot}, out_dtype=out)
        assert bool(got[0, 3].isnan().all()) and bool((got[0, :3] == clean[0, :3]).all()) and bool((got[1:] == clean[1:]).all())
    # a position of the common prefix: every query that sees it, and none that does not (the third request, cut to 20)
    case["lengths"][2] = 20
    clean = _run(case, out_dtype=out)
    lat = case["lat"].clone()
    lat[case["prefix"][0].long(), 40, 5] = math.inf
    got = _run({**case, "lat": lat}, out_dtype=out)
    assert bool(got[:2].isnan().all()) and bool((got[2] == clean[2]).all())


@pytest.mark.parametrize("out", [BF16, F32])
def test_a_query_that_is_not_finite_is_alone(out):
    case = oracle.make(_gen(4), 2, 2, 20, [90, 40], x=F32)
    clean = _run(case, out_dtype=out)
    q = case["q_nope"].clone()
    q[0, 1, 3, 17], q[1, 0, 0, 0] = math.nan, math.inf
    got = _run({**case, "q_nope": q}, out_dtype=out)
    assert bool(got[0, 1, 3].isnan().all()) and bool(got[1, 0, 0].isnan().all())
    got[0, 1, 3], got[1, 0, 0] = clean[0, 1, 3], clean[1, 0, 0]
    assert bool((got == clean).all())


def test_queries_that_see_nothing_are_zero():
    case = oracle.make(_gen(5), 4, 3, 8, [40, 5, 2, 64])
    case["lengths"][0] = 0
    case["lengths"][3] = -9
    got = _run(case, counts=torch.tensor([3, 3, 3, 3], dtype=I32, device="cuda"))
    assert not bool(got[0].any()) and not bool(got[3].any()) and not bool(got[2, 0].any()) and bool(got[2, 1:].all())
    none = _run(case, counts=torch.zeros(4, dtype=I32, device="cuda"))
    assert not bool(none.any())
    empty = {**case, "table": case["table"][:, :0].contiguous()}
    assert not bool(_run(empty).any())


@pytest.mark.parametrize("pages,out", [(F16, BF16), (F16, F32), (BF16, BF16)])
def test_pages_outside_the_pool_count_as_not_there(pages, out):
    case = oracle.make(_gen(6), 3, 1, 16, [200, 130, 64], pages_dtype=pages)
    for b, k, p in ((0, 0, -1), (0, 2, case["lat"].shape[0]), (1, 1, -2 ** 31), (2, 0, 2 ** 31 - 1)):
        case["table"][b, k] = p
    want, bound = oracle.attention(**case, out_dtype=out)
    got = _run(case, out_dtype=out)
    _check(got, want, bound)
    assert not bool(got[2].any())


@pytest.mark.parametrize("pages,out", FORMS_PO)
def test_ranges_without_a_page_beside_scores_far_below_zero(pages, out):
    # whole ranges lie on pages outside the pool (the first, the last, some between); the scores of the others are about -300
    case = oracle.make(_gen(16), 2, 1, 16, [640, 300], pages_dtype=pages, x=F32)
    case["rot"] = case["rot"].clone()
    case["rot"][..., 0] = -300.0
    case["q_rot"] = case["q_rot"].clone()
    case["q_rot"][..., 0] = 192 ** 0.5
    for b, k in ((0, 0), (0, 3), (0, 4), (0, 9), (1, 1)):
        case["table"][b, k] = -1
    want, bound = oracle.attention(**case, out_dtype=out)
    assert float(want.abs().mean()) > 1e-2
    _check(_run(case, out_dtype=out), want, bound)


# ------------------------------------------------------------------------------- sizes of the values
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("size", [1e-30, 1e-4, 1e25])
def test_queries_of_any_size(size, out):
    # the scale takes the size back, so scores are as ever
    case = oracle.make(_gen(7), 2, 1, 16, [150, 33], x=F32)
    case["q_nope"], case["q_rot"], case["scale"] = case["q_nope"] * size, case["q_rot"] * size, case["scale"] / size
    want, bound = oracle.attention(**case, out_dtype=out)
    _check(_run(case, out_dtype=out), want, bound)


@pytest.mark.parametrize("pages,out", FORMS_PO)
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -12, 2.0 ** 11])
def test_latents_of_any_size(size, pages, out):
    # (2^-20: fp16's last bits, below its smallest normal value)
    case = oracle.make(_gen(17), 2, 1, 16, [150, 33], pages_dtype=pages, x=F32)
    case["lat"] = (case["lat"].float() * size).clamp(-6e4, 6e4).to(pages)
    case["q_nope"] = case["q_nope"] * min(1.0, 1 / size)
    want, bound = oracle.attention(**case, out_dtype=out)
    _check(_run(case, out_dtype=out), want, bound)


def test_parts_of_a_query_of_unequal_size():
    # no rotary part, or one that is 2^20 times the rest: each has its scale
    case = oracle.make(_gen(8), 2, 1, 16, [150, 33], x=F32)
    for nope, rot in ((1.0, 0.0), (0.0, 1.0), (2.0 ** -20, 1.0), (1.0, 2.0 ** -20)):
        c = {**case, "q_nope": case["q_nope"] * nope, "q_rot": case["q_rot"] * rot}
        for out in (BF16, F32):
            want, bound = oracle.attention(**c, out_dtype=out)
            # (a part below 2^-38 of the row's largest is not there: here 2^-20 of it stays, with 2^-18 of its own accuracy)
            _check(_run(c, out_dtype=out), want, bound)


@pytest.mark.parametrize("pages,out", FORMS_PO)
def test_scores_that_keep_growing(pages, out):
    # every round exceeds all before it by far, in either half of it, so the reference moves again and again; and the other way round
    case = oracle.make(_gen(9), 2, 1, 20, [640, 639], pages_dtype=pages, x=F32)
    ramp = torch.linspace(0, 400, 640, device="cuda")
    for order in (ramp, ramp.flip(0), ramp.roll(17)):
        rot = case["rot"].clone()
        for b in range(2):
            pos = torch.arange(int(case["lengths"][b]), device="cuda")
            rot[case["table"][b, pos // 64].long(), pos % 64, 0] = order[pos].to(pages)
        q_rot = case["q_rot"].clone()
        q_rot[..., 0] = 192 ** 0.5
        c = {**case, "rot": rot, "q_rot": q_rot}
        want, bound = oracle.attention(**c, out_dtype=out)
        _check(_run(c, out_dtype=out), want, bound)


# ------------------------------------------------------------------------------- layouts
def test_layouts_and_strides():
    case = oracle.make(_gen(10), 3, 2, 12, [100, 31, 65], x=F32)
    want = _run(case)
    P = case["lat"].shape[0]
    both = torch.cat((case["lat"], case["rot"], case["rot"]), -1)                # one pool of wider rows
    wide = torch.full((3, 9), 77, dtype=I32, device="cuda")
    wide[:, 3:3 + case["table"].shape[1]] = case["table"]
    across = torch.stack((case["lat"], case["lat"]), 1)[:, 1]                    # pages further apart
    q = torch.cat((case["q_nope"], case["q_rot"]), -1)
    for c in (dict(lat=both[..., :512], rot=both[..., 512:576]), dict(table=wide[:, 3:3 + case["table"].shape[1]]), dict(lat=across),
              dict(q_nope=case["q_nope"].transpose(1, 2).contiguous().transpose(1, 2)),
              dict(q_nope=torch.cat((q[..., :1], q[..., :128]), -1)[..., 1:], q_rot=q.flip(-1).flip(-1)[..., 128:]),
              dict(wk=case["wk"].transpose(0, 1).contiguous().transpose(0, 1)), dict(max_length=int(case["lengths"].max()))):
        assert bool((_run({**case, **c}) == want).all()), list(c)
    assert P == across.shape[0]
    # a first half of the queries that is cut from a larger batch
    part = {**case, **{k: case[k][1:] for k in ("q_nope", "q_rot", "table", "lengths")}}
    _check(_run(part), *oracle.attention(**part))


@pytest.mark.parametrize("T,out", [(1, BF16), (20, BF16), (3, F32)])
def test_bf16_queries_whose_rows_lie_8_bytes_off(T, out):
    # (pitches of 196 and more elements: read as they are, every second row off a multiple of 16 bytes)
    case = oracle.make(_gen(18), 3, T, 12, [100, 31, 65], nope=136)
    q = torch.cat((case["q_nope"], case["q_rot"], case["q_rot"][..., :4]), -1)
    wide = {**case, "q_nope": q[..., :136], "q_rot": torch.cat((case["q_rot"], case["q_rot"][..., :4]), -1)[..., :64]}
    assert q.stride(2) % 8 == 4
    assert bool((_run(wide, out_dtype=out) == _run({**case, "q_nope": case["q_nope"].contiguous(), "q_rot": case["q_rot"].contiguous()}, out_dtype=out)).all())


def test_max_length_cuts():
    case = oracle.make(_gen(11), 2, 1, 8, [100, 50])
    cut = {**case, "lengths": case["lengths"].clamp(max=70)}
    assert bool((_run(case, max_length=70) == _run(cut)).all())
    long = {**case, "lengths": torch.tensor([10 ** 9, 50], dtype=I32, device="cuda"), "table": case["table"][:, :1].contiguous()}
    assert bool((_run(long) == _run({**long, "lengths": torch.tensor([64, 50], dtype=I32, device="cuda")})).all())


def test_a_pool_of_more_than_4_gib():
    # the pages in use lie behind 2^31 and 2^32 bytes
    pages = (1 << 32) // (64 * 1024) + 40
    case = oracle.make(_gen(12), 2, 1, 16, [130, 64], spare=0)
    lat = torch.empty(pages, 64, 512, dtype=F16, device="cuda")
    rot = torch.empty(pages, 64, 64, dtype=F16, device="cuda")
    n = case["lat"].shape[0]
    to = torch.tensor([pages - 1, (1 << 31) // (64 * 1024) + 1, pages - 20, 7, pages - 3][:n], device="cuda")
    lat[to], rot[to] = case["lat"], case["rot"]
    moved = {**case, "lat": lat, "rot": rot, "table": torch.where(case["table"] >= 0, to[case["table"].clamp(min=0).long()].to(I32), case["table"])}
    assert bool((_run(moved) == _run(case)).all())
    from k3hip.mla_paged import mla_paged_append
    slot = torch.tensor([[(pages - 1) * 64 + 63]], dtype=I32, device="cuda")
    mla_paged_append(torch.full((1, 1, 512), 3.0, device="cuda"), torch.full((1, 1, 64), 4.0, device="cuda"), slot, lat, rot)
    assert bool((lat[-1, 63] == 3).all()) and bool((rot[-1, 63] == 4).all()) and bool((lat[-1, 62] == case["lat"][0, 62]).all())


# ------------------------------------------------------------------------------- many
def _sampled(case, got, which, out, **kw):
    for b in which:
        one = {k: v[b:b + 1] if k in ("q_nope", "q_rot", "table", "lengths") else v for k, v in case.items()}
        _check(got[b:b + 1], *oracle.attention(**one, out_dtype=out, **kw), label=b)


@pytest.mark.parametrize("B,H,T,out", [(1100, 64, 1, BF16), (1500, 8, 1, F32), (40, 64, 33, BF16), (3, 96, 300, BF16), (2, 64, 70, F32)])
def test_many_rows(B, H, T, out):
    # batches in parts, more sequences than the list's lengths are searched for, queries in passes (and a last pass of few)
    g = _gen(B)
    lens = [int(n) for n in torch.randint(0, 3 * T + 90, (B,), generator=g)]
    lens[0], lens[-1] = 3 * T + 90, 1
    case = oracle.make(g, B, T, H, lens, page=32)
    got = _run(case, out_dtype=out)
    _sampled(case, got, {0, 1, B // 2, B - 1}, out)


def test_many_rows_behind_a_prefix():
    g = _gen(2)
    case = oracle.make(g, 700, 1, 24, [96 + b % 70 for b in range(700)], page=32, prefix=96)
    case["lengths"][5] = 0
    for out in (BF16, F32):
        got = _run(case, out_dtype=out)
        _sampled(case, got, (0, 5, 6, 350, 699), out)


def test_the_same_bits_every_time():
    for out in (BF16, F32):
        case = oracle.make(_gen(14), 24, 2, 16, [600 + 40 * b for b in range(24)], prefix=512)
        first = _run(case, out_dtype=out)
        for _ in range(3):
            assert bool((_run(case, out_dtype=out) == first).all())


# ------------------------------------------------------------------------------- streams and graphs
def test_another_stream():
    case = oracle.make(_gen(15), 8, 1, 16, [500 + b for b in range(8)])
    want = _run(case)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [_run(case) for _ in range(3)]
    assert all(bool((_run(case) == want).all()) for _ in range(3))
    side.synchronize()
    assert all(bool((g == want).all()) for g in got)


def test_a_captured_step_follows_the_lengths():
    """Tables, append and attention of a step in one graph, replayed while requests grow, with eager work between."""
    from k3hip.mla_paged import new_cache_paged
    from k3hip.pages import PageTable
    g = _gen(16)
    H, B = 16, 5
    case = oracle.make(g, B, 1, H, [1] * B, x=F32)
    start = torch.tensor([0, 63, 64, 100, 31], dtype=I32, device="cuda")

    def fresh():
        t = PageTable(B, 512, 30, page_size=64)
        c = new_cache_paged(t, F16)
        t.extend(start, tokens=100)
        data = torch.Generator().manual_seed(3)
        c.append(torch.randn(B, 100, 512, generator=data).cuda(), torch.randn(B, 100, 64, generator=data).cuda())
        return t, c

    def step(t, c, new, q):
        t.extend(1)
        c.append(new[..., :512], new[..., 512:], norm=torch.ones(512, device="cuda"))
        return c.attend(q[..., :128], q[..., 128:], case["wk"], case["wv"], 192 ** -0.5)

    news = [torch.randn(B, 1, 576, generator=g).cuda() for _ in range(7)]
    qs = [torch.randn(B, 1, H, 192, generator=g).cuda() for _ in range(7)]
    t, c = fresh()
    eager = [step(t, c, n, q).clone() for n, q in zip(news, qs)]
    lengths = t.lengths.clone()

    t2, c2 = fresh()
    new, q = news[0].clone(), qs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                       # (a warm-up on tables of its own)
        step(*fresh(), new, q)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t2.extend(1)
        c2.append(new[..., :512], new[..., 512:], norm=torch.ones(512, device="cuda"))
        out = c2.attend(q[..., :128], q[..., 128:], case["wk"], case["wv"], 192 ** -0.5)
    for i in range(7):
        new.copy_(news[i]), q.copy_(qs[i])
        graph.replay()
        other = _run(case)                              # (eager work on the same stream, with a workspace of its own)
        torch.cuda.synchronize()
        assert bool((out == eager[i]).all()), i
        assert bool(torch.isfinite(other).all())
    assert bool((t2.lengths == lengths).all()) and bool((t2.table == t.table).all())


def test_two_captured_calls_have_scratch_of_their_own():
    a = oracle.make(_gen(17), 6, 1, 16, [900 + b for b in range(6)])
    b = oracle.make(_gen(18), 6, 1, 16, [100 + 80 * b for b in range(6)])
    want = _run(a), _run(b)
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = _run(c)
        graphs.append(g), outs.append(o)
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(bool((o == w).all()) for o, w in zip(outs, want))
        for o in outs:
            o.zero_()
