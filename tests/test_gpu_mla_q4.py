"""The 4-bit latent cache on the GPU against its definition in 64 bits: writing, attention of one token and of several,
the summed weights, eviction, and the four together."""
from __future__ import annotations

import math

import pytest
import torch

import _q4_oracle as oracle

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
SCALE = 192 ** -0.5


def _rand(seed, *s, std=1.0, dtype=F32):
    return (torch.randn(*s, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _cache(B, cap, fill=0):
    mk = lambda w, dt: torch.full((B, cap, w), fill, dtype=dt, device="cuda")  # noqa: E731
    return mk(256, torch.uint8), mk(16, torch.uint8), mk(64, BF16)


def _ints(v):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------- writing
def _hard_rows():
    """Groups whose rounding goes by the details: ties, the step to the next scale, zeros, the ends of the range, NaN."""
    rows = []
    base = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -6.0]
    for top in (4.0, 6.0, 6.999, 7.0, 7.0001, 7.9):
        for e in (-100, -3, 0, 5, 100):
            rows.append([v * 2.0 ** e for v in base + [top] + [0.0] * 15])
    rows.append([0.0] * 32)
    rows.append([-0.0] * 32)
    rows.append([3.0e38] + [1e38] * 31)
    rows.append([2.0 ** -125] + [2.0 ** -126] * 31)
    rows.append([math.nan] + [1.0] * 31)
    rows.append([1.0] * 31 + [math.inf])
    rows.append([1.0] * 31 + [-math.inf])
    return rows


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_rounds_every_group_by_the_rule(dtype):
    from k3hip.mla_q4 import mla_q4_append
    groups = _hard_rows()
    x = _rand(1, 16, 512)
    flat = x.view(-1, 32)
    flat[:len(groups)] = torch.tensor(groups, dtype=torch.float64).to(F32)
    x = x.to(dtype)
    packed, scales, rot = _cache(1, 16)
    r = _rand(2, 1, 16, 64)
    mla_q4_append(x.view(1, 16, 512).cuda(), r.cuda(), packed, scales, rot)
    codes = torch.stack((packed & 15, packed >> 4), -1).reshape(-1, 32).cpu()
    for i, g in enumerate(x.view(-1, 32).to(torch.float64).tolist()):
        want, byte = oracle.round_group(g)
        assert int(scales.view(-1)[i]) == byte, (i, g)
        if byte != 255:
            got = [oracle.E2M1[c & 7] * (-1 if c & 8 else 1) for c in codes[i].tolist()]
            assert got == [oracle.E2M1[c & 7] * (-1 if c & 8 else 1) for c in want], (i, g)
    assert torch.equal(rot[0].cpu(), r[0].to(BF16))


@pytest.mark.parametrize("B,T,cap,start,counts", [
    (1, 1, 1, 0, None), (1, 1, 256, 255, None), (3, 5, 16, 7, None), (2, 67, 300, [0, 233], None),
    (4, 9, 40, [0, 31, 3, 40], [9, 9, 0, 5]), (2, 4, 8, [-2, 6], None), (3, 1, 4, [1, 2, 3], [1, 0, 7]),
])
def test_append_writes_only_its_positions(B, T, cap, start, counts):
    from k3hip.mla_q4 import mla_q4_append
    from k3hip.mxfp4 import decode_mxfp4
    both = _rand(3, B, T, 576)                       # latents and rotary rows as views of one projection
    c, r = both.cuda()[..., :512], both.cuda()[..., 512:]
    packed, scales, rot = _cache(B, cap, 7)
    mla_q4_append(c, r, packed, scales, rot, start=start if isinstance(start, int) else _ints(start), counts=_ints(counts))
    values = decode_mxfp4(packed.view(-1, 256), scales.view(-1, 16)).view(B, cap, 512).cpu()
    for b in range(B):
        s0 = start if isinstance(start, int) else start[b]
        n = T if counts is None else min(counts[b], T)
        new = {s0 + i: i for i in range(n) if 0 <= s0 + i < cap}
        for j in range(cap):
            if j in new:
                x = both[b, new[j]]
                want = []
                for g in x[:512].view(16, 32).to(torch.float64).tolist():
                    code, byte = oracle.round_group(g)
                    want += [oracle.E2M1[k & 7] * (-1.0 if k & 8 else 1.0) * 2.0 ** (byte - 127) for k in code]
                assert torch.equal(values[b, j].double(), torch.tensor(want, dtype=torch.float64))
                assert torch.equal(rot[b, j].cpu(), x[512:].to(BF16))
            else:
                assert bool((packed[b, j] == 7).all()) and bool((scales[b, j] == 7).all()) and bool((rot[b, j] == 7).all())


def test_append_zeroes_the_weight_of_what_it_writes():
    from k3hip.mla_q4 import mla_q4_append
    B, T, cap = 4, 3, 10
    w = torch.ones(B, 2 * cap, device="cuda")[:, 3:3 + cap]
    mla_q4_append(_rand(1, B, T, 512).cuda(), _rand(2, B, T, 64).cuda(), *_cache(B, cap), start=_ints([0, 8, -1, 4]), counts=_ints([3, 3, 3, 1]),
                  weight=w)
    zero = [(w[b] == 0).nonzero().flatten().tolist() for b in range(B)]
    assert zero == [[0, 1, 2], [8, 9], [0, 1], [4]] and int((w == 1).sum()) == B * cap - 8


def test_append_nothing():
    from k3hip.mla_q4 import mla_q4_append
    packed, scales, rot = _cache(2, 4, 3)
    mla_q4_append(torch.zeros(2, 0, 512, device="cuda"), torch.zeros(2, 0, 64, device="cuda"), packed, scales, rot, start=4)
    assert bool((packed == 3).all())


# ------------------------------------------------------------------------------- attention
def _problem(B, T, H, cap, seed, nope=128, v=128, x=F32, std=2.0):
    q = _rand(seed, B, T, H, nope + 64, std=std, dtype=x).cuda()
    wk, wv = _rand(seed + 1, H, nope, 512, std=512 ** -0.5, dtype=BF16).cuda(), _rand(seed + 2, H, v, 512, std=512 ** -0.5, dtype=BF16).cuda()
    return (q[..., :nope], q[..., nope:], wk, wv, *oracle.random_cache(B, cap, seed + 3, "cuda"))


def _check(args, lengths=None, counts=None, weight=False, out=F32, scale=SCALE):
    """One call against the oracle; returns what the call gave."""
    from k3hip.mla_q4 import mla_q4_attention
    B, T = args[0].shape[:2]
    cap = args[4].shape[1]
    w0 = _rand(99, B, cap).abs().cuda()
    w = w0.clone() if weight else None
    o = mla_q4_attention(*args, scale, lengths=lengths if lengths is None or isinstance(lengths, int) else _ints(lengths),
                         counts=_ints(counts), weight=w, out_dtype=out)
    n = [cap] * B if lengths is None else [lengths] * B if isinstance(lengths, int) else [min(max(x, 0), cap) for x in lengths]
    c = [T] * B if counts is None else [min(max(x, 0), T) for x in counts]
    fine = out == F32 or weight
    want, tol, mass, mass_tol = oracle.attention(*args, scale, n, c, fine, out == F32, torch.finfo(out).eps / 2)
    assert o.shape == want.shape and o.dtype == out
    assert bool(((o.double() - want).abs() <= tol).all()), float(((o.double() - want).abs() / tol).max())
    if weight:
        # (the last addition rounds to the sum's precision)
        got, tol = w.double() - w0.double(), mass_tol + 2.0 ** -24 * (w0.double() + mass)
        assert bool(((got - mass).abs() <= tol).all()), float(((got - mass).abs() / tol.clamp(min=1e-300)).max())
        for b in range(B):
            assert torch.equal(w[b, n[b]:], w0[b, n[b]:])
    return o, w


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("x", [F32, BF16])
@pytest.mark.parametrize("H,n", [(1, 1), (16, 31), (17, 32), (33, 33), (64, 1), (64, 64), (64, 65), (96, 257), (5, 1000), (128, 511)])
def test_one_token(H, n, x, out):
    _check(_problem(1, 1, H, n, 10 + H + n, x=x), out=out)


@pytest.mark.parametrize("out,weight", [(F32, False), (BF16, False), (BF16, True), (F32, True)])
@pytest.mark.parametrize("T,H,n", [(2, 64, 2), (3, 96, 100), (7, 5, 333), (17, 16, 40), (33, 8, 129), (65, 64, 65), (5, 33, 700)])
def test_several_tokens(T, H, n, out, weight):
    _check(_problem(1, T, H, n, 20 + T + H, x=BF16 if T % 2 else F32), out=out, weight=weight)


@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("T,lengths,counts", [
    (1, [0, 1, 40, 33, 2], None), (1, [40, 0, 7, 40, 40], [1, 1, 0, 1, 1]), (4, [4, 40, 2, 0, 39], None),
    (6, [40, 6, 9, 3, 0], [6, 2, 0, 6, 1]), (3, [99, -4, 40, 20, 1], [9, 1, -1, 3, 2]),
])
def test_sequences_of_unequal_length(T, lengths, counts, weight):
    """Empty sequences, queries that see nothing, lengths and counts out of range (held to it)."""
    o, _ = _check(_problem(5, T, 24, 40, 30), lengths, counts, weight)
    for b in range(5):
        n, c = min(max(lengths[b], 0), 40), T if counts is None else min(max(counts[b], 0), T)
        for t in range(T):
            if t >= c or n - c + t + 1 <= 0:
                assert bool((o[b, t] == 0).all())


def _lengths(kind, B, cap):
    g = torch.Generator().manual_seed(B)
    if kind == "one long":
        return [cap if b == B // 2 else b % 4 for b in range(B)]
    if kind == "none":
        return [0] * B
    if kind == "full":
        return [cap] * B
    return [int(cap ** float(torch.rand(1, generator=g))) if b % 7 else 0 for b in range(B)]


@pytest.mark.parametrize("kind", ["one long", "none", "full", "spread"])
@pytest.mark.parametrize("B,T,H,cap,out", [(2, 1, 64, 1500, F32), (32, 1, 64, 700, BF16), (33, 2, 16, 900, F32), (130, 1, 3, 300, BF16),
                                           (511, 1, 2, 70, F32), (3, 40, 8, 260, F32), (600, 1, 2, 50, F32), (16, 33, 64, 60, BF16)])
def test_batches_of_unequal_length(kind, B, T, H, cap, out):
    """Batches that share the card out over the positions there are: one long sequence among empty ones, nothing, all of
    the capacity, lengths of every size; as many sequences as such a batch may have, and batches with rows enough without it."""
    _check(_problem(B, T, H, cap, 170), _lengths(kind, B, cap), out=out, weight=H == 16)


@pytest.mark.parametrize("nope,v", [(8, 8), (40, 24), (128, 64), (192, 128), (256, 256), (64, 1024)])
def test_head_widths(nope, v):
    _check(_problem(2, 2, 6, 50, 40, nope, v), weight=True)


def test_capacity_zero_and_no_queries():
    from k3hip.mla_q4 import mla_q4_attention
    args = _problem(2, 3, 4, 0, 50)
    w = torch.zeros(2, 0, device="cuda")
    assert bool((mla_q4_attention(*args, SCALE, weight=w) == 0).all())
    args = _problem(2, 0, 4, 10, 50)
    assert mla_q4_attention(*args, SCALE).shape == (2, 0, 4, 128)
    args = _problem(2, 3, 4, 10, 50)
    assert bool((mla_q4_attention(*args, SCALE, lengths=0) == 0).all())


def test_strided_operands():
    """Cache buffers that are views of larger ones, queries of another order, weights of a larger tensor."""
    B, T, H, n = 2, 3, 10, 45
    q_nope, q_rot, wk, wv, packed, scales, rot = _problem(B, T, H, n, 60)
    big = [torch.full((B, n + 20, 2, w), 255, dtype=d, device="cuda") for w, d in ((256, torch.uint8), (16, torch.uint8), (64, BF16))]
    views = []
    for x, src in zip(big, (packed, scales, rot)):
        x[:, 5:5 + n, 1] = src
        views.append(x[:, 5:5 + n, 1])
    q = torch.empty(H, B, T, 200, device="cuda")
    qn, qr = q[..., 4:132].permute(1, 2, 0, 3), q[..., 136:].permute(1, 2, 0, 3)
    qn.copy_(q_nope), qr.copy_(q_rot)
    _check((qn, qr, wk, wv, *views), weight=True)
    odd = torch.empty(B, T, H, 129 + 65, device="cuda")         # rows of an odd pitch: copied
    qn, qr = odd[..., 1:129], odd[..., 130:]
    qn.copy_(q_nope), qr.copy_(q_rot)
    _check((qn, qr, wk, wv, *views))


@pytest.mark.parametrize("n,lengths", [(70, [70, 33]), (64, [64, 1])])
def test_what_is_hidden_does_not_matter(n, lengths):
    """NaN scale bytes, infinite rotary values and any codes behind a sequence's end, and in positions
    that only the later queries see."""
    args = list(_problem(2, 4, 12, n, 70))
    clean, w = _check(tuple(args), lengths, weight=True)
    packed, scales, rot = (t.clone() for t in args[4:])
    for b, m in enumerate(lengths):
        packed[b, m:], scales[b, m:], rot[b, m:] = 0x77, 255, math.inf
    from k3hip.mla_q4 import mla_q4_attention
    o = mla_q4_attention(*args[:4], packed, scales, rot, SCALE, lengths=_ints(lengths))
    assert torch.equal(o, clean)
    # the newest position of sequence 0 is NaN: its last query alone sees it
    scales[0, lengths[0] - 1, 3] = 255
    weight = torch.zeros(2, n, device="cuda")
    o = mla_q4_attention(*args[:4], packed, scales, rot, SCALE, lengths=_ints(lengths), weight=weight)
    assert torch.equal(o[0, :3], clean[0, :3]) and torch.equal(o[1], clean[1])
    assert bool(o[0, 3].isnan().all())
    assert bool(weight[0, :lengths[0]].isnan().all()) and not bool(weight[1].isnan().any())
    rot[0, lengths[0] - 1] = math.nan
    scales[0, lengths[0] - 1] = 120
    o = mla_q4_attention(*args[:4], packed, scales, rot, SCALE, lengths=_ints(lengths))
    assert torch.equal(o[0, :3], clean[0, :3]) and bool(o[0, 3].isnan().all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(bad):
    from k3hip.mla_q4 import mla_q4_attention
    args = list(_problem(1, 2, 20, 90, 80))
    clean = mla_q4_attention(*args, SCALE)
    args[0] = args[0].clone()
    args[0][0, 1, 7, 5] = bad
    o = mla_q4_attention(*args, SCALE)
    assert bool(o[0, 1, 7].isnan().all())
    o[0, 1, 7] = clean[0, 1, 7]
    assert torch.equal(o, clean)


@pytest.mark.parametrize("std", [1e-12, 1e-3, 30.0, 300.0])
def test_queries_of_any_size(std):
    """From all weights alike to one position taking all."""
    args = _problem(1, 3, 9, 300, 90, std=std)
    if std > 100:      # scores of hundreds: the bound of the oracle grows with them
        from k3hip.mla_q4 import mla_q4_attention
        want, tol, _, _ = oracle.attention(*args, SCALE, [300], [3], True, True, 2.0 ** -24)
        o = mla_q4_attention(*args, SCALE)
        assert bool(((o.double() - want).abs() <= tol).all())
    else:
        _check(args, weight=True)


@pytest.mark.parametrize("byte", [2, 30, 102, 106, 108, 136, 138, 142, 200, 225])
def test_cache_values_of_any_size(byte):
    """Latents far from one: the scale bytes' exponent goes through the products as it is (225: values of 2^100, with
    queries small enough for finite scores)."""
    q_nope, q_rot, wk, wv, packed, scales, rot = _problem(1, 2, 8, 60, 100)
    scales = scales - 126 + byte if byte > 4 else torch.full_like(scales, 2)
    q = q_nope * 2.0 ** -(byte - 126) if byte > 126 else q_nope
    _check((q, q_rot, wk, wv, packed, scales, rot))


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("H", [20, 80])
@pytest.mark.parametrize("at,byte", [(0, 90), (33, 150), (64, 60), (127, 103), (100, 141)])
def test_a_single_group_past_half_precision(at, byte, H, out):
    """One group of one position whose values fp16 does not hold, early or late in the sequence; the query is small there, so the
    scores stay finite."""
    q_nope, q_rot, wk, wv, packed, scales, rot = _problem(1, 2, H, 128, 105, x=out)
    scales[0, at, 5] = byte
    wk = wk.clone()
    if byte > 127:
        wk[:, :, 160:192] *= 2.0 ** (126 - byte)
    _check((q_nope, q_rot, wk, wv, packed, scales, rot), out=out)
    _check((q_nope, q_rot, wk, wv, packed, scales, rot), [at], out=out)     # behind the end: no reason to care


def test_growing_scores_move_the_reference():
    """Scores that rise by hundreds along the sequence, so every round's maximum is a new one."""
    q_nope, q_rot, wk, wv, packed, scales, rot = _problem(1, 2, 40, 320, 110)
    rot.zero_()
    rot[0, :, 0] = torch.arange(320, device="cuda").to(BF16)
    q_rot = torch.zeros_like(q_rot)
    q_rot[..., 0] = 100.0
    _check((q_nope, q_rot, wk, wv, packed, scales, rot), weight=True)
    q_rot[..., 0] = -100.0
    _check((q_nope, q_rot, wk, wv, packed, scales, rot), weight=True)


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("T,H,n", [(129, 64, 4096), (1, 16, 700)])
@pytest.mark.parametrize("k", [10, 20, 28, 33, 36])
def test_a_long_flat_tail_beside_one_large_position(k, T, H, n, out):
    """Position 0 has 2^k times the weight of any other and no values, so the output is the tail's alone: 129 queries run over all
    positions as one range.  Bounds, u = 2^-24: scores of up to 25 (72 u of them, twice, for a probability and the divisor: 2^-12), the sums
    (v / 8 + 300) u < 2^-14, W_UV 66 u, the rotary query's terms 2^-25 of a score (bf16: 2^-17, twice: 2^-11.3), a probability's 2^-22
    (bf16: 2^-11): 2^-11 in all, for bf16 2^-10 more and the output's rounding; and, whatever a probability's size, fp16's half step, 2^-35 of the largest, for each position."""
    from k3hip.mla_q4 import mla_q4_attention
    wk, wv = (t.cuda() for t in (_rand(420, H, 128, 512, std=512 ** -0.5, dtype=BF16), _rand(421, H, 128, 512, std=512 ** -0.5, dtype=BF16)))
    packed, scales, rot = _cache(1, n)
    packed[0, 1:], rot[0, 0, 0] = 0x22, 1.0                    # the tail's values are all 1
    scales.fill_(127)
    q_nope, q_rot = torch.zeros(1, T, H, 128, device="cuda"), torch.zeros(1, T, H, 64, device="cuda")
    q_rot[..., 0] = k * math.log(2) / SCALE
    weight = torch.zeros(1, n, device="cuda")
    o = mla_q4_attention(q_nope, q_rot, wk, wv, packed, scales, rot, SCALE, out_dtype=out)
    mla_q4_attention(q_nope, q_rot, wk, wv, packed, scales, rot, SCALE, out_dtype=out, weight=weight)
    tail = (n - T + torch.arange(T, device="cuda")).double()   # positions of it that query t sees
    p = 1 / (2.0 ** k + tail)
    rows, mags = wv.double().sum(2), wv.double().abs().sum(2)  # [H, v]
    want = (p * tail)[:, None, None] * rows
    tol = 2.0 ** -11 * (p * tail)[:, None, None] * mags + (tail * 2.0 ** -35 * 2.0 ** k * p)[:, None, None] * mags
    if out == BF16:
        tol += 2.0 ** -10 * (p * tail)[:, None, None] * mags + 2.0 ** -8 * want.abs()
    assert bool(((o[0].double() - want).abs() <= tol).all()), float(((o[0].double() - want).abs() / tol).max())
    # the summed weights count every position, however small
    got, one = weight[0, 1:n - T + 1].double(), H * float(p.sum())
    assert bool(((got - one).abs() <= 2.0 ** -11 * one).all())


@pytest.mark.parametrize("T,H,n,out", [(1, 64, 20000, F32), (1, 64, 20000, BF16), (4, 96, 6000, BF16), (128, 16, 1024, F32)])
def test_long_caches(T, H, n, out):
    args = _problem(1, T, H, n, 120)
    if T > 16:      # some of the queries: each one's bound is formed by itself
        from k3hip.mla_q4 import mla_q4_attention
        o = mla_q4_attention(*args, SCALE, out_dtype=out)
        for t in (0, 1, T // 2, T - 1):
            part = (args[0][:, t:t + 1], args[1][:, t:t + 1], *args[2:])
            want, tol, _, _ = oracle.attention(*part, SCALE, [n - T + 1 + t], [1], True, out == F32, torch.finfo(out).eps / 2)
            assert bool(((o[:, t:t + 1].double() - want).abs() <= tol).all())
        return
    _check(args, out=out, weight=T == 1)


def test_a_cache_past_four_gigabytes():
    """2^24 positions: byte offsets of the codes pass 2^32.  All positions are zero but a few, most of them at the
    far end, so the sums are known."""
    from k3hip.mla_q4 import mla_q4_attention
    n, H = 1 << 24, 4
    packed, scales, rot = _cache(1, n)
    scales.fill_(127)
    q_nope, q_rot, wk, wv, p, s, r = _problem(1, 1, H, 8, 130, std=8.0)
    at = [5, n // 2 + 1, n - 40, n - 33, n - 32, n - 3, n - 2, n - 1]
    packed[0, at], scales[0, at], rot[0, at] = p[0], s[0], r[0]
    weight = torch.zeros(1, n, device="cuda")
    o = mla_q4_attention(q_nope, q_rot, wk, wv, packed, scales, rot, SCALE, weight=weight)
    qa = torch.einsum("hn,hnr->hr", q_nope[0, 0].double(), wk.double())
    lat, rows = oracle.values(p[0], s[0]), r[0].double()
    z = (qa @ lat.T + q_rot[0, 0].double() @ rows.T) * SCALE
    m = z.amax(1, keepdim=True).clamp(min=0)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True) + (n - len(at)) * torch.exp(-m)
    want = torch.einsum("hr,hvr->hv", (e / total) @ lat, wv.double())
    # Relative error of a probability: twice a score's (of its magnitudes 2^-18, the terms and the summation: see the oracle), and
    # that of the normaliser, whose longest run is a lane's 8 a round over a range of 2^16 positions, 2^14 additions: 2^-10
    mags = (qa.abs() @ lat.abs().T + q_rot[0, 0].double().abs() @ rows.abs().T).amax(1, keepdim=True) * SCALE
    rel = 2 * 2.0 ** -18 * mags + 2.0 ** -10
    mag = torch.einsum("hr,hvr->hv", (e / total) @ lat.abs(), wv.double().abs())
    assert bool(((o[0, 0].double() - want).abs() <= rel * mag).all())
    got = weight[0, at].double()
    assert bool(((got - (e / total).sum(0)).abs() <= (rel * e / total).sum(0)).all())
    assert abs(float(weight.double().sum()) - H) < float(rel.max()) * H


@pytest.mark.parametrize("B,T", [(1, 80), (2, 64)])
def test_many_queries_past_eight_million_positions(B, T):
    """Rows enough to fill the card with one range a sequence, which would span 2 GiB of codes: cut into ranges that do not, for all
    sequences and in the list of unequal ones.  All positions are zero but a few at the ends and at 2^20, so the sums are known."""
    from k3hip.mla_q4 import mla_q4_attention
    n, H = (1 << 23) + 5000, 128
    packed, scales, rot = _cache(B, n)
    scales.fill_(127)
    q_nope, q_rot, wk, wv, p, s, r = _problem(B, T, H, 8, 410, std=8.0)
    at = torch.tensor([0, (1 << 20) - 1, 1 << 20, n // 2, n - 2 * T, n - 40, n - 2, n - 1], device="cuda")
    packed[0, at], scales[0, at], rot[0, at] = p[0], s[0], r[0]
    o = mla_q4_attention(q_nope, q_rot, wk, wv, packed, scales, rot, SCALE, lengths=None if B == 1 else _ints([n, 3]))
    qa = torch.matmul(q_nope[0].transpose(0, 1).double(), wk.double())                          # [H, T, 512]
    lat, rows = oracle.values(p[0], s[0]), r[0].double()
    qr = q_rot[0].transpose(0, 1).double()
    sees = n - T + 1 + torch.arange(T, device="cuda")
    z = (torch.matmul(qa, lat.T.contiguous()) + torch.matmul(qr, rows.T.contiguous())) * SCALE  # [H, T, 8]
    z = z.masked_fill(at >= sees[:, None], -math.inf)
    m = z.amax(-1, keepdim=True).clamp(min=0)
    e = torch.exp(z - m)
    zeros = (sees - (at < sees[:, None]).sum(1))[:, None]
    prob = e / (e.sum(-1, keepdim=True) + zeros * torch.exp(-m))
    want = torch.matmul(torch.matmul(prob, lat), wv.double().transpose(1, 2).contiguous())
    # a probability: as over 2^24 positions, a lane's longest run being 16 a round over a range of 2^20: 2^18 additions, 2^-6
    mags = (torch.matmul(qa.abs(), lat.abs().T.contiguous()) + torch.matmul(qr.abs(), rows.abs().T.contiguous())).amax(-1, keepdim=True) * SCALE
    rel = 2 * 2.0 ** -18 * mags + 2.0 ** -6
    mag = torch.matmul(torch.matmul(prob, lat.abs()), wv.double().abs().transpose(1, 2).contiguous())
    assert bool(((o[0].transpose(0, 1).double() - want).abs() <= rel * mag).all())
    assert float(mag.mean()) > 1e-3 and not o[1:].any()


def test_prompt_in_several_passes(monkeypatch):
    """More rows than one pass over the queries takes (65,536): the same as its parts."""
    from k3hip.mla_q4 import mla_q4_attention
    T, H, n = 1100, 64, 1100
    args = _problem(1, T, H, n, 140, x=BF16)
    weight = torch.zeros(1, n, device="cuda")
    o = mla_q4_attention(*args, SCALE, weight=weight, out_dtype=BF16)
    for t in (0, 1023, 1024, 1099):
        part = (args[0][:, t:t + 1], args[1][:, t:t + 1], *args[2:])
        want, tol, _, _ = oracle.attention(*part, SCALE, [t + 1], [1], True, False, 2.0 ** -8)
        assert bool(((o[:, t:t + 1].double() - want).abs() <= tol).all())
    half = torch.zeros(1, n, device="cuda")
    mla_q4_attention(args[0][:, :600], args[1][:, :600], *args[2:], SCALE, lengths=600, weight=half)
    mla_q4_attention(args[0][:, 600:], args[1][:, 600:], *args[2:], SCALE, weight=half)
    assert bool(((weight - half).abs() <= 2 ** -16 * weight).all())
    assert abs(float(weight.double().sum()) - T * H) < 2 ** -16 * T * H


@pytest.mark.parametrize("out", [F32, BF16])
def test_a_last_pass_of_few_queries(out):
    """1024 queries of 64 heads and 5 more, whose rows go by query where the others' go by head: outputs under a gate on both sides
    of the boundary, and the weights of both passes together."""
    from k3hip.mla_q4 import mla_q4_attention
    T, H = 1029, 64
    args = _problem(1, T, H, T, 430, x=BF16)
    gate = _rand(434, 1, T, H * 128).cuda()
    weight = torch.zeros(1, T, device="cuda")
    o = mla_q4_attention(*args, SCALE, weight=weight, gate=gate, out_dtype=out)
    for t in (0, 1022, 1023, 1024, 1025, 1028):
        part = (args[0][:, t:t + 1], args[1][:, t:t + 1], *args[2:])
        want, tol, _, _ = oracle.attention(*part, SCALE, [t + 1], [1], True, out == F32, torch.finfo(out).eps / 2)
        open_by = torch.sigmoid(gate[0, t].double()).view(1, 1, H, 128)      # (in fp32 to 2^-21)
        assert bool(((o[:, t:t + 1].double() - want * open_by).abs() <= tol * open_by + 2.0 ** -21 * want.abs()).all())
    parts = torch.zeros(1, T, device="cuda")
    mla_q4_attention(args[0][:, :1000], args[1][:, :1000], *args[2:], SCALE, lengths=1000, weight=parts)
    mla_q4_attention(args[0][:, 1000:], args[1][:, 1000:], *args[2:], SCALE, weight=parts)
    assert bool(((weight - parts).abs() <= 2 ** -16 * parts).all())
    assert abs(float(weight.double().sum()) - T * H) < 2 ** -16 * T * H


def test_several_passes_of_several_sequences():
    """Three sequences of 346 queries of 64 heads, 341 and 5 a pass, with lengths and counts of their own."""
    from k3hip.mla_q4 import mla_q4_attention
    B, T, H, cap = 3, 346, 64, 400
    args, lengths, counts = _problem(B, T, H, cap, 440), [400, 346, 150], [346, 344, 345]
    weight = torch.zeros(B, cap, device="cuda")
    o = mla_q4_attention(*args, SCALE, lengths=_ints(lengths), counts=_ints(counts), weight=weight)
    for b in range(B):
        one = [t[b:b + 1] for t in (args[0], args[1], *args[4:])]
        for t in (0, 194, 195, 196, 340, 341, 343, 344, 345):
            sees = max(0, lengths[b] - counts[b] + t + 1) if t < counts[b] else 0
            if sees == 0:
                assert not o[b, t].any()
                continue
            part = (one[0][:, t:t + 1], one[1][:, t:t + 1], *args[2:4], *one[2:])
            want, tol, _, _ = oracle.attention(*part, SCALE, [sees], [1], True, True, 2.0 ** -24)
            assert bool(((o[b:b + 1, t:t + 1].double() - want).abs() <= tol).all()), (b, t)
        alone, n = torch.zeros(1, cap, device="cuda"), counts[b]
        mla_q4_attention(one[0][:, :n], one[1][:, :n], *args[2:4], *one[2:], SCALE, lengths=lengths[b], weight=alone)
        assert bool(((weight[b:b + 1] - alone).abs() <= 2 ** -16 * alone).all()) and not weight[b, lengths[b]:].any()


def test_a_batch_past_65536_rows():
    """900 sequences of 80 heads, 72,000 rows, in two launches of the kernels; a gate, lengths of every size."""
    from k3hip.mla_q4 import mla_q4_attention
    B, H, cap = 900, 80, 24
    args, lengths = _problem(B, 1, H, cap, 400, v=32), [b % (cap + 1) for b in range(B)]
    o, _ = _check(args, lengths, weight=True)
    gate = _rand(401, B, 1, H * 32).cuda()
    gated = mla_q4_attention(*args, SCALE, lengths=_ints(lengths), weight=torch.zeros(B, cap, device="cuda"), gate=gate)
    want = o.double() * torch.sigmoid(gate.double()).view_as(o)
    assert bool(((gated.double() - want).abs() <= 2 ** -21 * want.abs()).all())


def test_repeated_calls_give_the_same_bits():
    from k3hip.mla_q4 import mla_q4_attention
    args = _problem(3, 2, 48, 900, 150)
    runs = []
    for _ in range(3):
        w = torch.zeros(3, 900, device="cuda")
        runs.append((mla_q4_attention(*args, SCALE, lengths=_ints([900, 17, 512]), weight=w), w))
    for o, w in runs[1:]:
        assert torch.equal(o, runs[0][0]) and torch.equal(w, runs[0][1])


def test_output_gate():
    from k3hip.mla_q4 import mla_q4_attention
    args = _problem(2, 2, 8, 50, 160)
    gate = _rand(161, 2, 2, 8 * 128).cuda()
    plain, gated = mla_q4_attention(*args, SCALE), mla_q4_attention(*args, SCALE, gate=gate)
    want = plain.double() * torch.sigmoid(gate.double()).view_as(plain)
    assert bool(((gated.double() - want).abs() <= 2 ** -21 * want.abs()).all())


# ------------------------------------------------------------------------------- streams, graphs, threads
def test_captured_batch_replays_with_other_lengths():
    """The sharing out is made anew from the lengths at every replay."""
    from k3hip.mla_q4 import mla_q4_attention
    B, cap = 20, 900
    args, n = _problem(B, 1, 64, cap, 190), _ints(_lengths("spread", B, cap))
    mla_q4_attention(*args, SCALE, lengths=n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = mla_q4_attention(*args, SCALE, lengths=n)
    for kind in ("full", "one long", "none", "spread", "full"):
        n.copy_(_ints(_lengths(kind, B, cap)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, mla_q4_attention(*args, SCALE, lengths=n)), kind


def test_another_stream():
    from k3hip.mla_q4 import mla_q4_attention
    args = _problem(1, 2, 32, 400, 170)
    want = mla_q4_attention(*args, SCALE)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = mla_q4_attention(*args, SCALE)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)


def _step(q, x, c, r, cache, lengths, weight, wk, wv):
    """One decode step as a serving program makes it: append, attend, count."""
    from k3hip.mla_q4 import mla_q4_append, mla_q4_attention
    mla_q4_append(c, r, *cache, start=lengths)
    lengths += 1
    return mla_q4_attention(q[..., :128], q[..., 128:], wk, wv, *cache, SCALE, lengths=lengths, weight=weight)


def test_captured_steps_replay():
    """Append, attention with weights and the length counter in one graph, replayed with new inputs between eager
    work; every replay against the eager steps."""
    B, H, cap = 3, 16, 64
    wk, wv = _rand(1, H, 128, 512, std=0.05, dtype=BF16).cuda(), _rand(2, H, 128, 512, std=0.05, dtype=BF16).cuda()
    steps = [(_rand(10 + i, B, 1, H, 192).cuda(), _rand(30 + i, B, 1, 512).cuda(), _rand(50 + i, B, 1, 64).cuda()) for i in range(6)]
    eager = []
    cache, n, w = _cache(B, cap), _ints([0, 5, 20]), torch.zeros(B, cap, device="cuda")
    for q, c, r in steps:
        eager.append((_step(q, None, c, r, cache, n, w, wk, wv).clone(), w.clone()))
    q, c, r = (t.clone() for t in steps[0])
    gcache, gn, gw = _cache(B, cap), _ints([0, 5, 20]), torch.zeros(B, cap, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):          # a warm-up on copies
        _step(q, None, c, r, tuple(t.clone() for t in gcache), gn.clone(), gw.clone(), wk, wv)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(q, None, c, r, gcache, gn, gw, wk, wv)
    for i, step in enumerate(steps):
        for dst, src in zip((q, c, r), step):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i][0]) and torch.equal(gw, eager[i][1])
        _step(*([steps[0][0], None] + list(steps[0][1:])), _cache(B, cap), _ints([1, 1, 1]), None, wk, wv)   # eager work between


def test_two_captured_graphs_do_not_share_scratch():
    from k3hip.mla_q4 import mla_q4_attention
    a, b = _problem(1, 1, 64, 700, 180), _problem(1, 1, 64, 700, 190)
    want = [mla_q4_attention(*x, SCALE) for x in (a, b)]
    graphs, outs = [], []
    for x in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mla_q4_attention(*x, SCALE))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, y in zip(outs, want):
            assert torch.equal(o, y)


def test_graphs_captured_on_a_stream_in_use_replay_side_by_side():
    """A stream with a workspace of its own from eager calls, and two graphs captured on it, batches of other sizes whose lists of
    ranges do not fit each other: replayed at once on two streams, beside eager calls on the first."""
    from k3hip.mla_q4 import mla_q4_attention
    a, b = _problem(20, 1, 64, 900, 450), _problem(3, 2, 32, 500, 460)
    calls = [(a, _ints(_lengths("spread", 20, 900))), (b, _ints([500, 0, 77]))]
    want = [mla_q4_attention(*x, SCALE, lengths=n) for x, n in calls]
    stream, graphs, outs = torch.cuda.Stream(), [], []
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for x, n in calls:
            mla_q4_attention(*x, SCALE, lengths=n)
    torch.cuda.synchronize()
    for x, n in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(mla_q4_attention(*x, SCALE, lengths=n))
        graphs.append(g)
    others = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, others):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(stream):
            eager = [mla_q4_attention(*x, SCALE, lengths=n) for x, n in calls]
        torch.cuda.synchronize()
        for o, e, y in zip(outs, eager, want):
            assert torch.equal(o, y) and torch.equal(e, y)


def test_two_threads_on_one_stream():
    import threading

    from k3hip.mla_q4 import mla_q4_attention
    args = [_problem(1, 1, 32, 600, 200), _problem(2, 3, 32, 300, 210)]
    want = [mla_q4_attention(*a, SCALE) for a in args]
    wrong = []

    def work(i):
        for _ in range(20):
            if not torch.equal(mla_q4_attention(*args[i], SCALE), want[i]):
                wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ------------------------------------------------------------------------------- eviction
def _weights(B, n, kind, seed):
    w = torch.exp(2.5 * _rand(seed, B, n))
    if kind == "ties":
        w = w.round()
    elif kind == "one value":
        w = torch.full((B, n), 0.5)
    elif kind == "any":
        w = _rand(seed, B, n)
        for i, v in enumerate((math.nan, math.inf, -math.inf, -0.0, 0.0, 1e-42, -1e-42, 3e38)):
            w[:, i::17] = v
    return w


@pytest.mark.parametrize("kind", ["spread", "ties", "one value", "any"])
@pytest.mark.parametrize("B,n,keep,sink,recent,lengths", [
    (1, 1, 1, 0, 0, None), (1, 2, 1, 0, 1, None), (1, 100, 0, 0, 0, None), (1, 1025, 512, 4, 64, None),
    (1, 5000, 4999, 10, 30, None), (3, 700, 128, 4, 124, [700, 130, 128]), (4, 300, 50, 3, 20, [0, 1, 49, 300]),
    (2, 40, 64, 4, 8, None), (2, 2049, 1, 0, 0, [2049, 999]), (1, 66000, 7001, 4, 100, None),
])
def test_evict(B, n, keep, sink, recent, lengths, kind):
    from k3hip.evict import cache_evict
    w = _weights(B, n, kind, n + keep)
    packed, scales, rot = oracle.random_cache(B, n, 7)
    odd = _rand(8, B, n, 3, 5).to(torch.float16)                 # rows of 30 bytes
    bufs = [packed, scales, rot, w, odd]
    new, index, kept = cache_evict(w.cuda(), [b.cuda() for b in bufs], keep, lengths=_ints(lengths), sink=sink, recent=recent,
                                   capacity=keep + 3)
    for b in range(B):
        m = n if lengths is None else lengths[b]
        want = oracle.evict(w[b, :m].tolist(), m, keep, sink, recent)
        assert int(kept[b]) == len(want)
        assert index[b].tolist() == want + [-1] * (keep - len(want))
        for x, y in zip(new, bufs):
            assert x.shape == (B, keep + 3, *y.shape[2:])
            bits = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
            assert torch.equal(bits(x[b, :len(want)].cpu()), bits(y[b][want]))
            assert bool((bits(x[b, len(want):].cpu()) == 0).all())


def test_evict_whole_chunks_above_and_at_the_threshold():
    """Neighbourhoods of 32,768 positions that stay as a whole, that are all alike, and that go as a whole."""
    from k3hip.evict import cache_evict
    n, keep = 140000, 70000
    w = torch.cat([torch.full((40000,), 3.0), torch.full((70000,), 2.0), torch.full((30000,), 1.0)])[None]
    (x,), index, kept = cache_evict(w.cuda(), [torch.arange(n, device="cuda")[None, :, None].contiguous()], keep)
    want = torch.arange(keep)
    assert int(kept) == keep and torch.equal(index[0].cpu().long(), want) and torch.equal(x[0, :, 0].cpu(), want)
    w = w.flip(1)
    _, index, _ = cache_evict(w.cuda(), [], keep, sink=5, recent=100)
    # the last 40,000 hold the 100 recent; 5 first; the rest are the first ones of weight 2 (from 30,000 on)
    want = torch.cat([torch.arange(5), torch.arange(30000, 30000 + keep - 40000 - 5), torch.arange(100000, n)])
    assert torch.equal(index[0].cpu().long(), want)


def test_evict_strided_buffers_and_the_bf16_cache():
    from k3hip.evict import cache_evict
    from k3hip.mla import MLACache
    B, n, keep = 2, 90, 31
    cache = MLACache(_rand(1, B, 128, 512, dtype=BF16).cuda(), _rand(2, B, 128, 64, dtype=BF16).cuda(), n)
    big = _weights(B, 3 * n, "spread", 3).cuda()
    w = big[:, ::3]                                              # copied
    lat, rot = cache.view()                                      # rows of a larger buffer
    (a, c), index, kept = cache_evict(w, [lat, rot], keep, sink=2, recent=5)
    for b in range(B):
        want = oracle.evict(w[b].tolist(), n, keep, 2, 5)
        assert index[b].tolist() == want and torch.equal(a[b], lat[b, want]) and torch.equal(c[b], rot[b, want])


def test_evict_captured():
    from k3hip.evict import cache_evict
    w, x = _weights(2, 500, "spread", 5).cuda(), _rand(6, 2, 500, 64).cuda()
    n = _ints([500, 300])
    cache_evict(w, [x], 100, lengths=n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (y,), index, kept = cache_evict(w, [x], 100, lengths=n, sink=4, recent=10)
    for i in range(4):
        w.copy_(_weights(2, 500, "ties", 20 + i))
        n.copy_(_ints([500 - 7 * i, 90 + 20 * i]))
        graph.replay()
        torch.cuda.synchronize()
        (y2,), index2, kept2 = cache_evict(w, [x], 100, lengths=n, sink=4, recent=10)
        assert torch.equal(index, index2) and torch.equal(kept, kept2) and torch.equal(y, y2)
        assert index[0].tolist() == oracle.evict(w[0].tolist(), 500 - 7 * i, 100, 4, 10)


# ------------------------------------------------------------------------------- together
def test_a_conversation_that_is_cut_short():
    """A prompt is written and attended to with its weights summed, the cache is cut, and decoding goes on over what is
    left: every step's attention against the same positions in 64 bits."""
    from k3hip.evict import cache_evict
    from k3hip.mla_q4 import mla_q4_append, mla_q4_attention
    B, T, H, keep, cap = 2, 48, 16, 20, 64
    args = _problem(B, T, H, 1, 300)
    wk, wv = args[2], args[3]
    c, r = _rand(301, B, T, 512).cuda(), _rand(302, B, T, 64).cuda()
    cache, weight = _cache(B, cap), torch.zeros(B, cap, device="cuda")
    lengths = _ints([T, 37])
    mla_q4_append(c, r, *cache, start=0, counts=lengths)
    mla_q4_attention(args[0], args[1], wk, wv, *cache, SCALE, lengths=lengths, counts=lengths, weight=weight)
    _, _, mass, tol = oracle.attention(args[0], args[1], wk, wv, *cache, SCALE, [T, 37], [T, 37], True, True, 0.0)
    assert bool(((weight.double() - mass).abs() <= tol + 2.0 ** -24 * mass).all())
    before = [t.clone() for t in cache]
    (*cache, weight), index, lengths = cache_evict(weight, [*cache, weight], keep, lengths=lengths, sink=2, recent=6, capacity=cap)
    for b in range(B):
        kept = index[b].long()
        for x, y in zip(cache, before):
            assert torch.equal(x[b, :keep], y[b, kept])
    for i in range(5):
        q = _rand(310 + i, B, 1, H, 192, std=2.0).cuda()
        mla_q4_append(_rand(320 + i, B, 1, 512).cuda(), _rand(330 + i, B, 1, 64).cuda(), *cache, start=lengths)
        lengths = lengths + 1
        o = mla_q4_attention(q[..., :128], q[..., 128:], wk, wv, *cache, SCALE, lengths=lengths, weight=weight)
        n = [keep + i + 1] * B
        assert lengths.tolist() == n
        want, tol, _, _ = oracle.attention(q[..., :128], q[..., 128:], wk, wv, *cache, SCALE, n, [1] * B, True, True, 2.0 ** -24)
        assert bool(((o.double() - want).abs() <= tol).all())
