"""What the 4-bit latent cache is measured on: writing it, attending over it, shortening it.

A cached position is 512 latent numbers as MXFP4 (256 bytes of E2M1 codes, 16 E8M0 scale bytes,
one per 32 numbers) and 64 rotary numbers in bf16.  Three kinds of call:

* ``append``  new latents are rounded to the format and written at each sequence's end;
* ``attend``  queries of one or more tokens over the cache (the absorbed latent attention), with
              or without the sum of the attention weights that every position received;
* ``evict``   the positions with the largest sums stay, in order, the others go.

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
R, ROPE, NOPE, V, GROUP = 512, 64, 128, 128, 32
SCALE = (NOPE + ROPE) ** -0.5
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
MAX_PAIRS = 1 << 27       # heads x queries x positions of the largest attend case, over all sequences


# ------------------------------------------------------------------------------- the cases
def listed() -> list[dict]:
    return [
        # A decode step writes one token: the smallest call, once per layer and step.
        {"name": "append_one_token", "kind": "append", "batch": 1, "tokens": 1, "past": 4095, "ragged": False, "x": "fp32"},
        # Four prompts of unequal length, padded to one tensor, go into their caches.
        {"name": "append_prompts", "kind": "append", "batch": 4, "tokens": 8192, "past": 0, "ragged": True, "x": "bf16"},
        # One token early in a conversation: launches and the weights are all there is.
        {"name": "attend_short", "kind": "attend", "batch": 1, "tokens": 1, "length": 17, "heads": 96, "ragged": False,
         "weight": False, "x": "bf16", "out": "bf16"},
        # One token late in a long conversation.
        {"name": "attend_long", "kind": "attend", "batch": 1, "tokens": 1, "length": 32768, "heads": 64, "ragged": False,
         "weight": False, "x": "fp32", "out": "fp32"},
        # The same while the weights are summed for a later eviction.
        {"name": "attend_long_weights", "kind": "attend", "batch": 1, "tokens": 1, "length": 20001, "heads": 64,
         "ragged": False, "weight": True, "x": "bf16", "out": "bf16"},
        # A decode step of 32 sequences of unequal length.
        {"name": "attend_batch", "kind": "attend", "batch": 32, "tokens": 1, "length": 8192, "heads": 64, "ragged": True,
         "weight": False, "x": "bf16", "out": "bf16"},
        # Four drafted tokens and the last one are verified together.
        {"name": "attend_drafts", "kind": "attend", "batch": 1, "tokens": 5, "length": 7001, "heads": 96, "ragged": False,
         "weight": False, "x": "bf16", "out": "bf16"},
        # A chunk of a long prompt over what the earlier chunks left.
        {"name": "attend_chunk", "kind": "attend", "batch": 1, "tokens": 512, "length": 4096, "heads": 64, "ragged": False,
         "weight": False, "x": "fp32", "out": "fp32"},
        # A prompt whose weights are summed; a length that fills no tile evenly.
        {"name": "attend_prompt_weights", "kind": "attend", "batch": 1, "tokens": 1000, "length": 1000, "heads": 64,
         "ragged": False, "weight": True, "x": "bf16", "out": "bf16"},
        # Half of a short cache goes.
        {"name": "evict_short", "kind": "evict", "batch": 1, "length": 1025, "keep": 512, "sink": 4, "recent": 64, "ragged": False},
        # A long conversation is cut to a quarter.
        {"name": "evict_long", "kind": "evict", "batch": 1, "length": 32768, "keep": 8192, "sink": 4, "recent": 1024,
         "ragged": False},
        # A batch of sequences of unequal length, some of them already short enough.
        {"name": "evict_batch", "kind": "evict", "batch": 16, "length": 16384, "keep": 4097, "sink": 4, "recent": 512,
         "ragged": True},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    """One more case of these ranges."""
    kind = rng.choice(["append", "attend", "attend", "attend", "evict"])
    if kind == "append":
        batch = rng.choice([1, _log(rng, 1, 16)])
        tokens = rng.choice([1, _log(rng, 1, 32768 // batch)])
        return {"kind": kind, "batch": batch, "tokens": tokens, "past": rng.choice([0, _log(rng, 1, 8192)]),
                "ragged": rng.random() < 0.5, "x": rng.choice(["bf16", "fp32"])}
    if kind == "attend":
        heads = rng.choice([8, 16, 24, 32, 48, 64, 96])
        tokens = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 1024)])
        batch = rng.choice([1, 1, _log(rng, 1, 32)]) if tokens <= 16 else 1
        most = min(32768, MAX_PAIRS // (heads * tokens * batch), 262144 // batch)
        return {"kind": kind, "batch": batch, "tokens": tokens, "length": max(tokens, _log(rng, 1, most)), "heads": heads,
                "ragged": batch > 1 and rng.random() < 0.7, "weight": rng.random() < 0.35, "x": rng.choice(["bf16", "fp32"]),
                "out": rng.choice(["bf16", "fp32"])}
    batch = rng.choice([1, _log(rng, 1, 16)])
    length = _log(rng, 64, 262144 // batch if batch > 1 else 65536)
    keep = max(2, min(length, int(length * rng.uniform(0.1, 0.9)), 65536 // batch))
    return {"kind": kind, "batch": batch, "length": length, "keep": keep, "sink": rng.choice([0, min(4, keep // 4)]),
            "recent": rng.randint(0, keep // 2), "ragged": batch > 1 and rng.random() < 0.7}


# ------------------------------------------------------------------------------- the inputs
class _Rand:
    def __init__(self, seed: int):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def n(self, *s, std: float = 1.0):
        return torch.randn(*s, device=DEV, generator=self.g) * std

    def u(self, *s):
        return torch.rand(*s, device=DEV, generator=self.g)

    def latents(self, *s):
        """RMS-normed rows whose channels differ in size by a factor of a few."""
        x = self.n(*s, R) * torch.exp(0.5 * self.n(R))
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5)

    def lengths(self, batch: int, most: int, least: int):
        """Sequence lengths over the range's logarithm, the longest one among them."""
        n = torch.exp(math.log(least) + self.u(batch) * (math.log(most) - math.log(least))).round().to(torch.int32)
        n[-1] = most
        return n.clamp(least, most)


def _lengths(rand: _Rand, case: dict, least: int):
    if case["ragged"]:
        return rand.lengths(case["batch"], case["length"], least)
    return torch.full((case["batch"],), case["length"], dtype=torch.int32, device=DEV)


def prepare(case: dict, seed: int) -> dict:
    rand, batch = _Rand(seed), case["batch"]
    s = {"case": case}
    if case["kind"] == "append":
        dt, tokens = DTYPES[case["x"]], case["tokens"]
        cap = -(-(case["past"] + tokens) // 256) * 256
        s["c"], s["r"] = rand.latents(batch, tokens).to(dt), rand.n(batch, tokens, ROPE).to(dt)
        s["packed"] = torch.zeros(batch, cap, R // 2, dtype=torch.uint8, device=DEV)
        s["scales"] = torch.zeros(batch, cap, R // GROUP, dtype=torch.uint8, device=DEV)
        s["rot"] = torch.zeros(batch, cap, ROPE, dtype=torch.bfloat16, device=DEV)
        s["start"] = torch.full((batch,), case["past"], dtype=torch.int32, device=DEV)
        s["counts"] = torch.full((batch,), tokens, dtype=torch.int32, device=DEV)
        if case["ragged"]:
            s["counts"] = rand.lengths(batch, tokens, max(1, tokens // 8))
            s["start"] = (rand.u(batch) * (case["past"] + 1)).to(torch.int32).clamp(max=case["past"])
        return s
    length = case["length"]
    s["lengths"] = _lengths(rand, case, case["tokens"] if case["kind"] == "attend" else max(1, length // 16))
    s["packed"], s["scales"] = _quantise(rand.latents(batch, length))
    s["rot"] = rand.n(batch, length, ROPE).to(torch.bfloat16)
    if case["kind"] == "attend":
        H, dt = case["heads"], DTYPES[case["x"]]
        s["wk"] = rand.n(H, NOPE, R, std=R ** -0.5).to(torch.bfloat16)
        s["wv"] = rand.n(H, V, R, std=R ** -0.5).to(torch.bfloat16)
        q = rand.n(batch, case["tokens"], H, NOPE + ROPE, std=2.0).to(dt)
        s["q_nope"], s["q_rot"] = q[..., :NOPE], q[..., NOPE:]
        # what earlier steps left: of the size that this one adds
        s["weight"] = torch.exp(rand.n(batch, length)) * (H * case["tokens"] / length) if case["weight"] else None
        return s
    # sums of attention weights: spread over decades, some positions alike, the newest not yet seen
    s["weight"] = torch.exp(2.5 * rand.n(batch, length))
    s["weight"] = torch.where(rand.u(batch, length) < 0.1, s["weight"].round(), s["weight"])
    s["weight"][:, -max(1, length // 64):] = 0.0
    return s


# ------------------------------------------------------------------------------- the plain forms
def _power(e: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """2 ** e of whole numbers, from its bits (exact whatever the device's pow does)."""
    if dtype == torch.float64:
        return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)
    return ((e.to(torch.int32) + 127).clamp(min=0) << 23).view(torch.float32)


def _quantise(x: torch.Tensor):
    """fp32 [..., 512] -> (codes [..., 256], scale bytes [..., 16]): the scale is the power of two that puts
    the group's largest magnitude at 4 to 7 (above 7 the next one), codes round to nearest, ties to even."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    top = g.abs().amax(-1)
    e = torch.frexp(torch.where(top > 0, top, torch.ones_like(top)))[1] - 3
    e = e.clamp(-125, 125)
    e = (e + (top > 7 * _power(e))).clamp(max=125)
    byte = torch.where(top > 0, e + 127, torch.full_like(e, 2))
    y = g * _power(127 - byte).unsqueeze(-1)
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + 8 * (y < 0)).to(torch.uint8).reshape(*x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _values(packed: torch.Tensor, scales: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """What the codes and scale bytes stand for."""
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=dtype, device=packed.device)
    code = torch.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], -1, GROUP)
    return (lut[code.to(torch.int32)] * _power(scales.to(torch.int32) - 127, dtype).unsqueeze(-1)).reshape(*packed.shape[:-1], -1)


def _plain_append(s: dict):
    c, tokens, cap = s["c"].to(torch.float32), s["c"].shape[1], s["packed"].shape[1]
    codes, scales = _quantise(c)
    i = torch.arange(tokens, device=DEV)
    new = (i < s["counts"].unsqueeze(1)) & (s["start"].unsqueeze(1) + i < cap)
    b, t = new.nonzero(as_tuple=True)
    at = s["start"][b] + t
    s["packed"][b, at], s["scales"][b, at], s["rot"][b, at] = codes[b, t], scales[b, t], s["r"][b, t].to(torch.bfloat16)
    return _values(s["packed"], s["scales"]), s["rot"]


def _plain_attend(s: dict):
    c = s["case"]
    batch, tokens, heads = s["q_nope"].shape[:3]
    cap = s["packed"].shape[1]
    lat, rot = _values(s["packed"], s["scales"]), s["rot"].to(torch.float32)
    wk, wv = s["wk"].to(torch.float32), s["wv"].to(torch.float32)
    q = s["q_nope"].to(torch.float32).permute(2, 0, 1, 3).reshape(heads, batch * tokens, NOPE)
    qa = torch.matmul(q, wk).reshape(heads, batch, tokens, R).permute(1, 2, 0, 3).reshape(batch, tokens * heads, R)
    qr = s["q_rot"].to(torch.float32).reshape(batch, tokens * heads, ROPE)
    scores = (torch.matmul(qa, lat.transpose(1, 2)) + torch.matmul(qr, rot.transpose(1, 2))) * SCALE
    sees = s["lengths"].unsqueeze(1) - tokens + 1 + torch.arange(tokens, device=DEV)          # [batch, tokens]
    seen = (torch.arange(cap, device=DEV) < sees.unsqueeze(-1)).unsqueeze(2)                  # [batch, tokens, 1, cap]
    scores = scores.reshape(batch, tokens, heads, cap).masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    ctx = torch.matmul(p.reshape(batch, tokens * heads, cap), lat).reshape(batch * tokens, heads, R)
    o = torch.matmul(ctx.transpose(0, 1), wv.transpose(1, 2)).transpose(0, 1).reshape(batch, tokens, heads, V)
    o = o.to(DTYPES[c["out"]])
    return o if s["weight"] is None else (o, s["weight"] + p.sum((1, 2)))


def _plain_evict(s: dict):
    c, w, n = s["case"], s["weight"], s["lengths"].unsqueeze(1)
    keep, i = c["keep"], torch.arange(s["weight"].shape[1], device=DEV)
    order = torch.sort(torch.where(w.isnan(), torch.full_like(w, -math.inf), w), dim=1, descending=True, stable=True)[1]
    tier = (i < n).to(torch.int32) + ((i < n) & ((i < c["sink"]) | (i >= n - c["recent"])))   # 2: stays, 1: by weight, 0: not there
    order = order.gather(1, torch.sort(tier.gather(1, order), dim=1, descending=True, stable=True)[1])[:, :keep]
    last = w.shape[1]
    index = torch.where(tier.gather(1, order) > 0, order, torch.full_like(order, last)).sort(1)[0]
    there = index < last
    at = index.clamp(max=last - 1)
    out = [torch.where(there.unsqueeze(-1), x.gather(1, at.unsqueeze(-1).expand(-1, -1, x.shape[2])), torch.zeros_like(x[:1, :1]))
           for x in (s["packed"], s["scales"], s["rot"])]
    return (*out, torch.where(there, w.gather(1, at), torch.zeros_like(w[:, :1])),
            torch.where(there, index, -torch.ones_like(index)).to(torch.int32), there.sum(1).to(torch.int32))


# ------------------------------------------------------------------------------- one pass
def _package():
    at = str(Path(__file__).resolve().parent.parent / "kimi-k3-mlx-macmini_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from k3hip import evict, mla_q4, mxfp4
    return mla_q4, evict, mxfp4


def run(s: dict):
    c = s["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[c["kind"]](s)
    mla_q4, evict, mxfp4 = _package()
    if c["kind"] == "append":
        mla_q4.mla_q4_append(s["c"], s["r"], s["packed"], s["scales"], s["rot"], start=s["start"], counts=s["counts"])
        batch, cap, half = s["packed"].shape
        lat = mxfp4.decode_mxfp4(s["packed"].view(batch * cap, half), s["scales"].view(batch * cap, R // GROUP))
        return lat.view(batch, cap, R), s["rot"]
    if c["kind"] == "attend":
        weight = None if s["weight"] is None else s["weight"].clone()
        o = mla_q4.mla_q4_attention(s["q_nope"], s["q_rot"], s["wk"], s["wv"], s["packed"], s["scales"], s["rot"], SCALE,
                                    lengths=s["lengths"], weight=weight, out_dtype=DTYPES[c["out"]])
        return o if weight is None else (o, weight)
    (packed, scales, rot, weight), index, lengths = evict.cache_evict(
        s["weight"], [s["packed"], s["scales"], s["rot"], s["weight"]], c["keep"], lengths=s["lengths"], sink=c["sink"],
        recent=c["recent"])
    return packed, scales, rot, weight, index, lengths


# ------------------------------------------------------------------------------- what a pass cannot do without
def work(case: dict) -> dict:
    batch, row = case["batch"], R // 2 + R // GROUP + 2 * ROPE
    share = 0.36 if case["ragged"] else 1.0        # mean of lengths spread over the logarithm of the range, about
    size = 2 if case.get("x") == "bf16" else 4
    if case["kind"] == "append":
        n = batch * case["tokens"] * (0.42 if case["ragged"] else 1.0)
        return {"bytes": int(n * (size * (R + ROPE) + row)), "flops": int(n * 3 * R)}
    if case["kind"] == "evict":
        rows = batch * min(case["keep"], case["length"])
        return {"bytes": int(4 * batch * case["length"] * share + rows * (2 * (row + 4) + 4)), "flops": 0}
    tokens, heads = case["tokens"], case["heads"]
    if case["ragged"]:
        share = (1 - tokens / case["length"]) / max(1e-9, math.log(case["length"] / tokens)) if case["length"] > tokens else 1.0
    cached = batch * case["length"] * share
    pairs = heads * tokens * max(0.0, cached - batch * (tokens - 1) / 2)
    queries = batch * tokens * heads
    # scores and contexts in the latent columns, with every query taken there and back, or in the heads' own with every
    # position taken there: what is less
    absorbed = 2 * pairs * (2 * R + ROPE) + 2 * queries * R * (NOPE + V)
    expanded = 2 * pairs * (NOPE + ROPE + V) + 2 * cached * heads * R * (NOPE + V)
    out = 2 if case["out"] == "bf16" else 4
    nbytes = cached * row + 2 * heads * R * (NOPE + V) + queries * (size * (NOPE + ROPE) + out * V)
    return {"bytes": int(nbytes + (8 * cached if case["weight"] else 0)), "flops": int(min(absorbed, expanded))}


# ------------------------------------------------------------------------------- the results in 64 bits
def _exact_round(x: torch.Tensor) -> torch.Tensor:
    """float64 rows -> what the 4-bit format makes of them: every group on the grid of its power of two."""
    g = x.reshape(-1, GROUP)
    top = g.abs().max(1, keepdim=True)[0]
    unit = _power(torch.frexp(torch.where(top > 0, top, torch.ones_like(top)))[1] - 3, torch.float64)
    unit = torch.where(top > 7 * unit, 2 * unit, unit).clamp(2.0 ** -125, 2.0 ** 125)
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    y = (g / unit).abs().clamp(max=6.0)
    lo = torch.searchsorted(grid, y, right=True).sub(1).clamp(0, 6)
    below, above = y - grid[lo], grid[lo + 1] - y
    up = (above < below) | ((above == below) & (lo % 2 == 1))       # ties to the even code
    return (torch.sign(g) * grid[lo + up.to(lo.dtype)] * unit).reshape(x.shape)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "append":
        lat = torch.zeros(*s["packed"].shape[:2], R, dtype=torch.float64, device=DEV)
        rot = torch.zeros(*s["rot"].shape, dtype=torch.float64, device=DEV)
        for b in range(case["batch"]):
            at, n = int(s["start"][b]), int(s["counts"][b])
            lat[b, at:at + n] = _exact_round(s["c"][b, :n].to(torch.float64))
            rot[b, at:at + n] = s["r"][b, :n].to(torch.float64)
        return lat, rot
    if case["kind"] == "evict":
        rot = torch.zeros(case["batch"], case["keep"], ROPE, dtype=torch.float64, device=DEV)
        weight = torch.zeros(case["batch"], case["keep"], dtype=torch.float64, device=DEV)
        for b in range(case["batch"]):
            n = int(s["lengths"][b])
            w = s["weight"][b, :n].tolist()
            must = set(range(min(case["sink"], n))) | set(range(max(0, n - case["recent"]), n))
            rest = sorted((j for j in range(n) if j not in must), key=lambda j: (-w[j], j))
            kept = torch.tensor(sorted(list(must) + rest[:max(0, min(case["keep"], n) - len(must))]), device=DEV)
            rot[b, :len(kept)] = s["rot"][b, kept].to(torch.float64)
            weight[b, :len(kept)] = s["weight"][b, kept].to(torch.float64)
        return None, None, rot, weight, None, None
    f64 = torch.float64
    heads, tokens = case["heads"], case["tokens"]
    wk, wv = s["wk"].to(f64), s["wv"].to(f64)
    out = torch.zeros(case["batch"], tokens, heads, V, dtype=f64, device=DEV)
    weight = None if s["weight"] is None else s["weight"].to(f64)
    for b in range(case["batch"]):
        n = int(s["lengths"][b])
        lat, rot = _values(s["packed"][b, :n], s["scales"][b, :n], f64), s["rot"][b, :n].to(f64)
        hidden = torch.arange(n, device=DEV) > (torch.arange(tokens, device=DEV) + n - tokens).unsqueeze(1)   # [tokens, n]
        for h in range(heads):        # every head on keys and values of its own
            keys, values = lat @ wk[h].t(), lat @ wv[h].t()
            z = (s["q_nope"][b, :, h].to(f64) @ keys.t() + s["q_rot"][b, :, h].to(f64) @ rot.t()) * SCALE
            p = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
            out[b, :, h] = p @ values
            if weight is not None:
                weight[b, :n] += p.sum(0)
    return out if weight is None else (out, weight)
