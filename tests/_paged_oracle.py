"""The paged latent cache restated: tables one request after the other, attention in 64 bits, and what the kernels may be off by."""
from __future__ import annotations

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def tables(table, lengths, target, free, used, page, tokens, shared=None):
    """page_tables on Python lists -> (table, free, lengths, used, slots); the inputs are left alone."""
    table, free, lengths = [list(r) for r in table], list(free), list(lengths)
    width, pool = len(table[0]) if table else 0, len(free)
    used = min(max(used, 0), pool)
    pages = lambda n: -(-n // page)  # noqa: E731
    lengths = [min(max(n, 0), width * page) for n in lengths]
    target = [max(t, 0) for t in target]
    target = [n if t > width * page else t for n, t in zip(lengths, target)]
    back = []
    for b, (n, to) in enumerate(zip(lengths, target)):
        if pages(to) < pages(n):
            back += table[b][max(pages(to), shared[b] if shared else 0):pages(n)]
    base = max(used - len(back), 0)
    back = back[:used - base]
    free[base:used] = back
    used, dry, slots = base, False, []
    for b, (n, to) in enumerate(zip(lengths, target)):
        more = pages(to) - pages(n)
        dry = dry or (more > 0 and more > pool - used)
        if more > 0 and dry:
            to = n
        elif more > 0:
            table[b][pages(n):pages(to)] = free[used:used + more]
            used += more
        new = [table[b][i // page] * page + i % page for i in range(n, min(to, n + tokens))]
        slots.append(new + [-1] * (tokens - len(new)))
        lengths[b] = to
    return table, free, lengths, used, slots


def attention(q_nope, q_rot, wk, wv, lat, rot, table, lengths, scale, counts=None, prefix=None, gate=None, out_dtype=torch.float32):
    """-> (o, bound) float64 [B, T, H, v]: the definition, and how far a result may be off, both by element.

    The bound counts, with u a type's half step: the result's own rounding; six standard deviations of a score's error, whose terms
    (one for each column: u of the query terms times the product, independent) add as a root of squares, and of the probabilities'
    roundings, which add so over the positions; 2^-19 of the sum of magnitudes for the fp32 sums (576 and more products, 2^-24 each, and the
    context's terms before W_UV, 2^-16 at a bf16 result).  At a bf16 result over fp16 pages the contexts of ranges are fp16, over their sums: every
    column of range i off by 2^-11 |c_i| at most, independently, weighed with the range's share w_i; sum_i w_i |c_i| is at most sum_j p_j |lat_j|, so
    six deviations are 6 2^-11 of the root of the squares of W_UV times that.  Below 2^-14 fp16's values are 2^-24 apart whatever their size, so
    a column of a range is off by 2^-25 at least there, as the pages' own values are: 6 2^-25 of the root of the squares of W_UV."""
    f64 = torch.float64
    B, T, H, nope = q_nope.shape
    V, page, pool = wv.shape[1], lat.shape[1], lat.shape[0]
    fine = out_dtype == torch.float32
    u_q = (2.0 ** -24 if fine else 2.0 ** -16) if lat.dtype == torch.bfloat16 else 2.0 ** -22 if fine else 2.0 ** -11
    o, bound = (torch.zeros(B, T, H, V, dtype=f64, device=lat.device) for _ in range(2))
    n_prefix = 0 if prefix is None else len(prefix)
    for b in range(B):
        n, cnt = int(lengths[b]), T if counts is None else min(max(int(counts[b]), 0), T)
        n = min(max(n, 0), table.shape[1] * page)
        rows = table[b].clone().to(torch.int64)
        if n_prefix:
            rows[:n_prefix] = prefix[:len(rows)]
        there = ((rows >= 0) & (rows < pool)).repeat_interleave(page)[:n]
        rows = rows.clamp(0, max(pool - 1, 0))
        L = lat[rows].reshape(-1, 512)[:n].to(f64)
        R = rot[rows].reshape(-1, 64)[:n].to(f64)
        for t in range(cnt):
            see = torch.arange(n, device=lat.device) < n - cnt + t + 1
            see = see & there
            if not bool(see.any()):
                continue
            Ls, Rs = L[see], R[see]
            qa = torch.einsum("hd,hdr->hr", q_nope[b, t].to(f64), wk.to(f64))
            qr = q_rot[b, t].to(f64)
            s = (qa @ Ls.t() + qr @ Rs.t()) * scale
            p = torch.softmax(s, -1)
            v = torch.einsum("jr,hvr->hjv", Ls, wv.to(f64))
            out = torch.einsum("hj,hjv->hv", p, v)
            sigma = u_q * abs(scale) * ((qa.square() @ Ls.square().t() + qr.square() @ Rs.square().t()).sqrt())      # [H, j]
            spread = torch.einsum("hj,hjv->hv", p * sigma, v.abs()) + (p * sigma).sum(-1, keepdim=True) * out.abs()
            weight = u_q * torch.einsum("hj,hjv->hv", p.square(), v.square()).sqrt()
            sums = torch.einsum("hj,hjr,hvr->hv", p, Ls.abs().expand(H, -1, -1), wv.to(f64).abs())
            if not fine and lat.dtype == torch.float16:
                weight = weight + u_q * torch.einsum("hr,hvr->hv", (p @ Ls.abs()).square(), wv.to(f64).square()).sqrt()
                weight = weight + 2.0 ** -25 * wv.to(f64).square().sum(-1).sqrt()
            bound[b, t] = 6 * (spread + weight) + sums * (2.0 ** -19 if fine else 2.0 ** -15)
            if gate is not None:
                g = torch.sigmoid(gate[b, t].to(f64).reshape(H, V))
                out, bound[b, t] = out * g, bound[b, t] * g
            o[b, t] = out
            bound[b, t] += HALF_STEP[out_dtype] * out.abs()
    return o, bound


def make(gen, B, T, H, lens, page=64, pages_dtype=torch.float16, x=torch.bfloat16, nope=128, v=128, prefix=0, spare=3, device="cuda"):
    """Queries, weights, pool and tables of sequences of these lengths (a prefix of whole pages counted in): pages in any order, what is not
    held full of NaNs."""
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    n_prefix, width = prefix // page, max(1, max(-(-int(k) // page) for k in lens))
    held = [max(0, -(-int(k) // page) - n_prefix) for k in lens]
    total = n_prefix + sum(held) + spare
    order = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = n_prefix
    for b, k in enumerate(held):
        table[b, :min(n_prefix, width)] = order[:min(n_prefix, width)]
        table[b, n_prefix:n_prefix + k] = order[at:at + k]
        at += k
    lat = n(total, page, 512) * torch.exp(0.5 * n(512))
    lat = (lat * torch.rsqrt(lat.square().mean(-1, keepdim=True) + 1e-5)).to(pages_dtype)
    rot = n(total, page, 64).to(pages_dtype)
    lat[order[at:].long()] = math.nan
    rot[order[at:].long()] = math.nan
    for b, k in enumerate(lens):        # behind the last position
        last, left = divmod(int(k), page)
        if left and (int(k) > prefix):
            lat[table[b, last].long(), left:] = math.nan
            rot[table[b, last].long(), left:] = math.inf
    q = (2.0 * n(B, T, H, nope + 64)).to(x)
    wk, wv = (n(H, nope, 512) * 512 ** -0.5).to(torch.bfloat16), (n(H, v, 512) * 512 ** -0.5).to(torch.bfloat16)
    d = lambda t: t.to(device)  # noqa: E731
    q = d(q)
    return dict(q_nope=q[..., :nope], q_rot=q[..., nope:], wk=d(wk), wv=d(wv), lat=d(lat), rot=d(rot), table=d(table),
                lengths=torch.tensor([int(k) for k in lens], dtype=torch.int32, device=device), scale=(nope + 64) ** -0.5,
                prefix=d(order[:n_prefix].contiguous()) if n_prefix else None)
