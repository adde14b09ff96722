"""What the paged latent cache is measured on: its tables, writing it, attending over it.

The cache of a batch of requests lies in pages of ``page`` positions that belong to no request for good;
a cached position is 512 latent numbers and 64 rotary numbers in fp16 or bf16.  Three kinds of call:

* ``tables``  requests change length: pages are taken from the list of free ones or given back, and every
              new token gets the row ("slot") that it is written to;
* ``append``  new latents are RMS-normed and written, with their rotary rows, to the slots;
* ``attend``  one or more tokens of every request over the pages (the absorbed latent attention); where the
              requests share a prefix, its pages are common to all.

Values: latents as an RMS norm leaves them, with channels of unequal size; weights of variance
1 / fan_in; queries that make scores of deviation about 2, so a few positions get most of the
weight and the rest little, as trained attention does.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
R, ROPE, NOPE, V = 512, 64, 128, 128
SCALE, EPS = (NOPE + ROPE) ** -0.5, 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp16": torch.float16}
MAX_PAIRS = 1 << 28       # heads x queries x positions of an attend case, over all sequences
MAX_CACHED = 1 << 19      # positions of their own, over all sequences


# ------------------------------------------------------------------------------- the cases
def _attend(name, batch, tokens, prefix, length, heads, pages, x, out, ragged=True, page=64) -> dict:
    return {"name": name, "kind": "attend", "batch": batch, "tokens": tokens, "prefix": prefix, "length": length, "heads": heads,
            "pages": pages, "x": x, "out": out, "ragged": ragged, "page": page}


def listed() -> list[dict]:
    return [
        # A decode step of 64 requests: one token each, a page for those whose last one is full, some have ended.
        {"name": "tables_decode", "kind": "tables", "batch": 64, "tokens": 1, "length": 32768, "page": 64, "ended": 0.05, "tight": False},
        # Prompts come in while others end: a row for every prompt token.
        {"name": "tables_prompts", "kind": "tables", "batch": 48, "tokens": 8192, "length": 8192, "page": 64, "ended": 0.3, "tight": True},
        # The latents of a decode step, as the projection leaves them.
        {"name": "append_decode", "kind": "append", "batch": 64, "tokens": 1, "pages": "fp16", "x": "fp32", "ragged": False, "norm": True, "page": 64},
        # Eight prompts of unequal length, padded to one tensor.
        {"name": "append_prompts", "kind": "append", "batch": 8, "tokens": 4096, "pages": "bf16", "x": "fp32", "ragged": True, "norm": True, "page": 64},
        # One request early in a conversation: launches and the weights are all there is.
        _attend("attend_short", 1, 1, 0, 17, 96, "fp16", "bf16", "bf16", False),
        # A decode step of 32 requests of unequal length that share nothing.
        _attend("attend_batch", 32, 1, 0, 8192, 64, "fp16", "bf16", "bf16"),
        # The same at full accuracy, few and long ones.
        _attend("attend_batch_fp32", 6, 1, 0, 16384, 64, "fp16", "fp32", "fp32"),
        # bf16 pages, as the cache of one sequence is held; an odd batch and 96 heads.
        _attend("attend_batch_bf16", 25, 1, 1024, 3001, 96, "bf16", "bf16", "bf16"),
        # A decode step of 64 requests behind one system prompt.
        _attend("attend_prefix", 64, 1, 8192, 1024, 64, "fp16", "bf16", "bf16"),
        # Three drafted tokens and the last one of each request are verified together.
        _attend("attend_drafts", 16, 4, 4096, 2048, 64, "fp16", "fp32", "fp32"),
        # The rest of four prompts over a prefix that is cached.
        _attend("attend_prompts", 4, 200, 2048, 333, 64, "fp16", "bf16", "bf16"),
        # Many short requests about one long document: the largest.
        _attend("attend_document", 120, 1, 32768, 300, 64, "fp16", "bf16", "bf16"),
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    """One more case of these ranges."""
    kind = rng.choice(["tables", "append", "attend", "attend", "attend", "attend"])
    page = rng.choice([32, 64, 64, 128])
    if kind == "tables":
        tokens = rng.choice([1, _log(rng, 1, 16), _log(rng, 17, 8192)])
        batch = min(_log(rng, 1, 512), 1 << 19 if tokens == 1 else max(1, (48 * 8192) // tokens))
        return {"kind": kind, "batch": batch, "tokens": tokens, "length": max(tokens, _log(rng, 64, 32768)), "page": page,
                "ended": rng.choice([0.0, rng.uniform(0, 0.5)]), "tight": rng.random() < 0.4}
    pages = rng.choice(["fp16", "fp16", "bf16"])
    if kind == "append":
        batch = _log(rng, 1, 256)
        tokens = rng.choice([1, _log(rng, 1, max(1, 32768 // batch))])
        return {"kind": kind, "batch": batch, "tokens": tokens, "pages": pages, "x": rng.choice(["bf16", "fp32"]),
                "ragged": rng.random() < 0.5, "norm": rng.random() < 0.7, "page": page}
    heads = rng.choice([8, 16, 24, 32, 48, 64, 64, 96])
    tokens = rng.choice([1, 1, 1, _log(rng, 2, 8), _log(rng, 9, 256)])
    batch = _log(rng, 1, 128 if tokens == 1 else max(1, 256 // tokens))
    most = MAX_PAIRS // (heads * tokens * batch)
    prefix = rng.choice([0, _log(rng, page, min(32768, max(page, most // 2))) // page * page])
    length = max(tokens, _log(rng, 1, max(1, min(32768, most - prefix, MAX_CACHED // batch))))
    return {"kind": kind, "batch": batch, "tokens": tokens, "prefix": prefix, "length": length, "heads": heads, "pages": pages,
            "x": rng.choice(["bf16", "fp32"]), "out": rng.choice(["bf16", "fp32"]), "ragged": batch > 1 and rng.random() < 0.8, "page": page}


# ------------------------------------------------------------------------------- the inputs
class _Rand:
    def __init__(self, seed: int):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def n(self, *s, std: float = 1.0):
        return torch.randn(*s, device=DEV, generator=self.g) * std

    def u(self, *s):
        return torch.rand(*s, device=DEV, generator=self.g)

    def order(self, n: int):
        return torch.randperm(n, device=DEV, generator=self.g).to(torch.int32)

    def latents(self, *s):
        """RMS-normed rows whose channels differ in size by a factor of a few."""
        x = self.n(*s, R) * torch.exp(0.5 * self.n(R))
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)

    def lengths(self, batch: int, most: int, least: int):
        """Sequence lengths over the range's logarithm, the longest one among them."""
        n = torch.exp(math.log(least) + self.u(batch) * (math.log(most) - math.log(least))).round().to(torch.int32)
        n[-1] = most
        return n.clamp(least, most)


def _up(n, page: int):
    return (n + page - 1) // page


def prepare(case: dict, seed: int) -> dict:
    rand, batch, page, tokens = _Rand(seed), case["batch"], case["page"], case["tokens"]
    s = {"case": case}
    if case["kind"] == "tables":
        return {**s, **_prepare_tables(case, rand)}
    if case["kind"] == "append":
        dt, pdt = DTYPES[case["x"]], DTYPES[case["pages"]]
        width = _up(tokens, page) + 1
        counts = torch.full((batch,), tokens, dtype=torch.int32, device=DEV)
        if case["ragged"]:
            counts = rand.lengths(batch, tokens, max(1, tokens // 8))
        start = (rand.u(batch, 1) * page).to(torch.int32)               # a request's first new row lies anywhere in a page
        table = rand.order(batch * width + 3)[:batch * width].view(batch, width)
        at = start + torch.arange(tokens, device=DEV, dtype=torch.int32)
        slots = table.gather(1, (at // page).to(torch.int64)) * page + at % page
        s["slots"] = torch.where(torch.arange(tokens, device=DEV) < counts.unsqueeze(1), slots, -1).to(torch.int32)
        s["lat"] = rand.latents(batch * width + 3, page).to(pdt)         # what earlier requests left
        s["rot"] = rand.n(batch * width + 3, page, ROPE).to(pdt)
        ckv = rand.n(batch, tokens, R + ROPE, std=1.5).to(dt)            # the projection's output: latents, then the rotary part
        s["c"], s["r"] = ckv[..., :R], ckv[..., R:]
        s["norm"] = torch.exp(0.5 * rand.n(R)) if case["norm"] else None
        return s
    H, dt, pdt, n_prefix = case["heads"], DTYPES[case["x"]], DTYPES[case["pages"]], case["prefix"] // page
    mine = rand.lengths(batch, case["length"], tokens) if case["ragged"] else torch.full((batch,), case["length"], dtype=torch.int32, device=DEV)
    s["lengths"] = mine + case["prefix"]
    if case["ragged"] and batch > 3:
        s["lengths"][batch // 2] = 0                                      # a place of the batch that holds no request
    width = _up(case["length"], page)
    order = rand.order(n_prefix + batch * width)
    s["prefix"] = order[:n_prefix].contiguous() if n_prefix else None
    s["table"] = torch.cat((order[:n_prefix].expand(batch, n_prefix), order[n_prefix:].view(batch, width)), 1).contiguous()
    s["lat"], s["rot"] = rand.latents(len(order), page).to(pdt), rand.n(len(order), page, ROPE).to(pdt)
    s["wk"] = rand.n(H, NOPE, R, std=R ** -0.5).to(torch.bfloat16)
    s["wv"] = rand.n(H, V, R, std=R ** -0.5).to(torch.bfloat16)
    q = rand.n(batch, tokens, H, NOPE + ROPE, std=2.0).to(dt)
    s["q_nope"], s["q_rot"] = q[..., :NOPE], q[..., NOPE:]
    return s


def _prepare_tables(case: dict, rand: _Rand) -> dict:
    batch, page, tokens, most = case["batch"], case["page"], case["tokens"], case["length"]
    width = _up(most, page)
    if tokens <= 16:        # requests under way take the next tokens
        lengths = rand.lengths(batch, most, 1)
        target = (lengths + 1 + (rand.u(batch) * tokens).to(torch.int32)).clamp(max=most)
    else:                   # prompts begin
        lengths = torch.zeros(batch, dtype=torch.int32, device=DEV)
        target = rand.lengths(batch, tokens, max(1, tokens // 8))
    ended = rand.u(batch) < case["ended"]
    lengths = torch.where(ended & (lengths == 0), (1 + rand.u(batch) * (most - 1)).to(torch.int32), lengths)
    target = torch.where(ended, 0, target).to(torch.int32)
    have, want = _up(lengths, page), _up(target, page)
    taken = int(have.sum())
    more = int((want - have).clamp(min=0).sum()) - int((have - want).clamp(min=0).sum())
    order = rand.order(batch * width + 32)
    left = max(0, more * 2 // 3) if case["tight"] else max(0, more) + 17      # pages that nobody holds
    table = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
    held = torch.arange(width, device=DEV) < have.unsqueeze(1)
    table[held] = order[:taken]
    return {"table": table, "lengths": lengths.contiguous(), "target": target.contiguous(), "free": order.contiguous(),
            "used": torch.full((1,), len(order) - left, dtype=torch.int32, device=DEV)}


# ------------------------------------------------------------------------------- the plain forms
def _plain_tables(s: dict):
    c, table, free, used = s["case"], s["table"], s["free"], s["used"]
    page, width = c["page"], table.shape[1]
    have, want = _up(s["lengths"], page), _up(s["target"], page)
    k = torch.arange(width, device=DEV)
    gives = (k >= want.unsqueeze(1)) & (k < have.unsqueeze(1))
    back = table[gives]                                                   # in the batch's order
    base = used.to(torch.int64) - back.shape[0]
    free[base + torch.arange(back.shape[0], device=DEV)] = back
    need = (want - have).clamp(min=0)
    after = torch.cumsum(need, 0)
    granted = (need == 0) | (after <= free.shape[0] - base)
    takes = (k >= have.unsqueeze(1)) & (k < want.unsqueeze(1)) & granted.unsqueeze(1)
    at = base + (after - need).unsqueeze(1) + k - have.unsqueeze(1)
    table[takes] = free[at[takes]]
    lengths = torch.where(granted, s["target"], s["lengths"])
    new_used = (base + torch.where(granted, need, torch.zeros_like(need)).sum()).to(torch.int32)
    i = torch.arange(c["tokens"], device=DEV, dtype=torch.int32)
    pos = s["lengths"].unsqueeze(1) + i
    there = pos < lengths.unsqueeze(1)
    rows = table.gather(1, (pos // page).clamp(max=width - 1).to(torch.int64)) * page + pos % page
    return table, free, lengths, new_used, torch.where(there, rows, -torch.ones_like(rows))


def _plain_append(s: dict):
    c, slots = s["c"].to(torch.float32), s["slots"]
    if s["norm"] is not None:
        c = s["norm"] * (c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS))
    new = slots >= 0
    at = slots[new].to(torch.int64)
    s["lat"].view(-1, R)[at] = c[new].to(s["lat"].dtype)
    s["rot"].view(-1, ROPE)[at] = s["r"][new].to(s["rot"].dtype)
    return s["lat"], s["rot"]


def _plain_attend(s: dict):
    c, f32 = s["case"], torch.float32
    batch, tokens, heads = s["q_nope"].shape[:3]
    P, n_prefix = c["prefix"], c["prefix"] // c["page"]
    rows = s["table"][:, n_prefix:].to(torch.int64)
    lat, rot = s["lat"][rows].reshape(batch, -1, R).to(f32), s["rot"][rows].reshape(batch, -1, ROPE).to(f32)
    q = s["q_nope"].to(f32).permute(2, 0, 1, 3).reshape(heads, batch * tokens, NOPE)
    qa = torch.matmul(q, s["wk"].to(f32)).reshape(heads, batch, tokens, R).permute(1, 2, 0, 3).reshape(batch, tokens * heads, R)
    qr = s["q_rot"].to(f32).reshape(batch, tokens * heads, ROPE)
    scores = torch.matmul(qa, lat.transpose(1, 2)) + torch.matmul(qr, rot.transpose(1, 2))
    if P:
        plat, prot = s["lat"][s["prefix"].to(torch.int64)].reshape(P, R).to(f32), s["rot"][s["prefix"].to(torch.int64)].reshape(P, ROPE).to(f32)
        scores = torch.cat((torch.matmul(qa, plat.t()) + torch.matmul(qr, prot.t()), scores), -1)
    sees = s["lengths"].unsqueeze(1) - tokens + 1 + torch.arange(tokens, device=DEV)          # [batch, tokens]
    seen = (torch.arange(scores.shape[-1], device=DEV) < sees.unsqueeze(-1)).unsqueeze(2)     # [batch, tokens, 1, positions]
    scores = (scores * SCALE).reshape(batch, tokens, heads, -1).masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    p = (p / p.sum(-1, keepdim=True).clamp(min=1e-38)).reshape(batch, tokens * heads, -1)
    ctx = torch.matmul(p[..., P:], lat)
    if P:
        ctx = ctx + torch.matmul(p[..., :P], plat)
    o = torch.matmul(ctx.reshape(batch * tokens, heads, R).transpose(0, 1), s["wv"].to(f32).transpose(1, 2))
    return o.transpose(0, 1).reshape(batch, tokens, heads, V).to(DTYPES[c["out"]])


# ------------------------------------------------------------------------------- one pass
_modules = None


def _package():
    global _modules
    if _modules is None:
        at = str(Path(__file__).resolve().parent.parent / "kimi-k3-mlx-macmini_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        from k3hip import mla_paged, pages
        _modules = mla_paged, pages
    return _modules


def run(s: dict):
    c = s["case"]
    if not own:
        return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend}[c["kind"]](s)
    mla_paged, pages = _package()
    if c["kind"] == "tables":
        lengths, used, slots = pages.page_tables(s["table"], s["lengths"], s["target"], s["free"], s["used"], c["page"], tokens=c["tokens"])
        return s["table"], s["free"], lengths, used, slots
    if c["kind"] == "append":
        mla_paged.mla_paged_append(s["c"], s["r"], s["slots"], s["lat"], s["rot"], norm=s["norm"], eps=EPS)
        return s["lat"], s["rot"]
    return mla_paged.mla_paged_attention(s["q_nope"], s["q_rot"], s["wk"], s["wv"], s["lat"], s["rot"], s["table"], s["lengths"], SCALE,
                                         prefix=s["prefix"], out_dtype=DTYPES[c["out"]])


# ------------------------------------------------------------------------------- what a pass cannot do without
def _share(least: float, most: float) -> float:
    """The mean of lengths spread over a range's logarithm, over the longest."""
    return (1 - least / most) / math.log(most / least) if most > least else 1.0


def work(case: dict) -> dict:
    batch, tokens = case["batch"], case["tokens"]
    if case["kind"] == "tables":
        moved = batch * ((tokens * _share(max(1, tokens // 8), tokens) if tokens > 16 else (tokens + 1) / 2) + case["ended"] * case["length"] / 3)
        return {"bytes": int(4 * (3 * batch + batch * tokens + 2 * moved / case["page"])), "flops": 0}
    row = 2 * (R + ROPE)
    size = 2 if case["x"] == "bf16" else 4
    if case["kind"] == "append":
        n = batch * tokens * (_share(max(1, tokens // 8), tokens) if case["ragged"] else 1.0)
        return {"bytes": int(n * (size * (R + ROPE) + row) + 4 * batch * tokens), "flops": int(n * 4 * R)}
    heads, there = case["heads"], batch - (1 if case["ragged"] and batch > 3 else 0)
    mine = there * case["length"] * (_share(tokens, case["length"]) if case["ragged"] else 1.0)
    cached = case["prefix"] + mine
    pairs = heads * tokens * max(0.0, there * case["prefix"] + mine - there * (tokens - 1) / 2)
    queries = there * tokens * heads
    # scores and contexts in the latent columns, with every query taken there and back, or in the heads' own with every
    # position taken there: what is less
    absorbed = 2 * pairs * (2 * R + ROPE) + 2 * queries * R * (NOPE + V)
    expanded = 2 * pairs * (NOPE + ROPE + V) + 2 * cached * heads * R * (NOPE + V)
    out = 2 if case["out"] == "bf16" else 4
    nbytes = cached * (row + 4 / case["page"]) + 2 * heads * R * (NOPE + V) + queries * size * (NOPE + ROPE) + batch * tokens * heads * out * V
    return {"bytes": int(nbytes), "flops": int(min(absorbed, expanded))}


# ------------------------------------------------------------------------------- the results in 64 bits
def _exact_tables(s: dict):
    """One request after the other, as the definition says it."""
    page, tokens = s["case"]["page"], s["case"]["tokens"]
    table, free, used = s["table"].tolist(), s["free"].tolist(), int(s["used"])
    lengths, target = s["lengths"].tolist(), s["target"].tolist()
    pages = lambda n: -(-n // page)  # noqa: E731
    back = [p for row, n, to in zip(table, lengths, target) for p in row[pages(to):pages(n)]]
    used -= len(back)
    free[used:used + len(back)] = back
    dry, slots = False, []
    for b, (n, to) in enumerate(zip(lengths, target)):
        more = pages(to) - pages(n)
        dry = dry or (more > 0 and more > len(free) - used)
        if more > 0 and dry:
            to = lengths[b]
        elif more > 0:
            table[b][pages(n):pages(to)] = free[used:used + more]
            used += more
        slots.append([table[b][i // page] * page + i % page for i in range(n, min(to, n + tokens))])
        slots[b] += [-1] * (tokens - len(slots[b]))
        lengths[b] = to
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return whole(table), whole(free), whole(lengths), whole([used]), whole(slots)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["kind"] == "tables":
        return _exact_tables(s)
    if case["kind"] == "append":
        lat, rot = s["lat"].to(f64).view(-1, R), s["rot"].to(f64).view(-1, ROPE)
        for b in range(case["batch"]):
            at = s["slots"][b][s["slots"][b] >= 0].to(torch.int64)
            c, r = s["c"][b, :len(at)].to(f64), s["r"][b, :len(at)].to(f64)
            lat[at] = c if s["norm"] is None else s["norm"].to(f64) * c / (c.square().sum(1, keepdim=True) / R + EPS).sqrt()
            rot[at] = r
        return lat.view(s["lat"].shape), rot.view(s["rot"].shape)
    heads, tokens, page = case["heads"], case["tokens"], case["page"]
    wk, wv = s["wk"].to(f64), s["wv"].to(f64)
    out = torch.zeros(case["batch"], tokens, heads, V, dtype=f64, device=DEV)
    lengths = s["lengths"].tolist()

    def positions(pages):
        pages = pages.to(torch.int64)
        return s["lat"][pages].reshape(-1, R).to(f64), s["rot"][pages].reshape(-1, ROPE).to(f64)

    first = case["prefix"] // page
    common = positions(s["prefix"]) if first else None
    expanded = [(common[0] @ wk[h].t(), common[0] @ wv[h].t()) for h in range(heads)] if first else None
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        lat, rot = positions(s["table"][b, first:])
        hidden = torch.arange(case["prefix"] + len(lat), device=DEV) > (torch.arange(tokens, device=DEV) + n - tokens).unsqueeze(1)
        keys, values = torch.einsum("jr,hdr->hjd", lat, wk), torch.einsum("jr,hdr->hjd", lat, wv)
        for h in range(heads):        # every head on keys and values of its own
            qn, qr = s["q_nope"][b, :, h].to(f64), s["q_rot"][b, :, h].to(f64)
            z = qn @ keys[h].t() + qr @ rot.t()
            if first:
                z = torch.cat((qn @ expanded[h][0].t() + qr @ common[1].t(), z), 1)
            p = torch.softmax((z * SCALE).masked_fill(hidden, -math.inf), -1)
            out[b, :, h] = p[:, case["prefix"]:] @ values[h]
            if first:
                out[b, :, h] += p[:, :case["prefix"]] @ expanded[h][1]
    return out
