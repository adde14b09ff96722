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
