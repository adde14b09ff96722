"""The 4-bit latent cache in 64 bits: the rounding, the attention and the eviction, from their definitions,
and how far arithmetic of the kernels' kind may be from them."""
from __future__ import annotations

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
F64 = torch.float64


def round_group(x):
    """32 Python floats -> (codes, scale byte): one group by the rule, in exact arithmetic."""
    import math
    if any(math.isnan(v) or math.isinf(v) for v in x):
        return [0] * 32, 255
    top = max(abs(v) for v in x)
    if top == 0:
        return [0] * 32, 127
    e = math.frexp(top)[1] - 3                     # floor(log2 top) - 2
    if top > 7.0 * 2.0 ** e:
        e += 1
    e = min(max(e, -125), 125)
    codes = []
    for v in x:
        y = min(abs(v) / 2.0 ** e, 6.0)
        best = min(range(8), key=lambda c: (abs(y - E2M1[c]), c % 2))       # nearest, ties to the even code
        codes.append(best + (8 if v < 0 else 0))
    return codes, e + 127


def values(packed, scales, dtype=F64):
    """[..., 256] codes and [..., 16] bytes -> [..., 512]; byte 255 gives NaN."""
    lut = torch.tensor(E2M1 + [-v for v in E2M1], dtype=dtype, device=packed.device)
    code = torch.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], 16, 32).long()
    s = ((scales.long() + 896) << 52).view(F64).to(dtype)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return (lut[code] * s.unsqueeze(-1)).reshape(*packed.shape[:-1], 512)


def random_cache(B, n, seed, device="cpu", std=1.0):
    """Codes over the whole alphabet, scales that give values of about `std`."""
    g = torch.Generator().manual_seed(seed)
    import math
    mid = 127 + round(math.log2(std / 2.93))
    packed = torch.randint(0, 256, (B, n, 256), generator=g, dtype=torch.int32).to(torch.uint8)
    scales = torch.randint(mid - 2, mid + 3, (B, n, 16), generator=g, dtype=torch.int32).to(torch.uint8)
    rot = torch.randn(B, n, 64, generator=g).to(torch.bfloat16)
    return packed.to(device), scales.to(device), rot.to(device)


def attention(q_nope, q_rot, wk, wv, packed, scales, rot, scale, lengths, counts, fine_q, fine_p, out_eps):
    """-> (o, bound on |error of o|, weight sums, bound on theirs), float64.  lengths, counts: lists.

    The bounds, u = 2^-24 (half a step of fp32):
    * qa: fp32 sums of nope products, the fp32 query split exactly: (nope + 4) u of sum |q W|; its terms leave at most 2^-22 (fine, five terms) or
      2^-12 (three) of a unit that is at most the group's largest / 3.75;
    * a score: that, times |lat|; its sum of at most 26 matrix instructions in a row and four joins, each
      rounding once and adding its products exactly to 2u: 64 u of the sum of magnitudes; the rotary query's two terms leave 2^-17 (fine: 2^-25);
      the scaling to log2 units and the subtraction of the maximum: 4 u of |s| and of the maximum;
    * a probability: the score errors of itself and of the normaliser (2 E), exp2 2 u, its terms 2^-11 (one fp16) or 2^-22 (fine, two), a rescale per round;
    * sums over n positions: n / 32 rounds of up to 3 products, the joins of splits: (n / 8 + 300) u;
    * W_UV: three terms, 512 products: 64 u and 2^-24; then the rounding of the output, out_eps.
    """
    u = 2.0 ** -24
    B, T, H, nope = q_nope.shape
    dev = q_nope.device
    o = torch.zeros(B, T, H, wv.shape[1], dtype=F64, device=dev)
    tol = torch.zeros_like(o)
    mass = torch.zeros(B, packed.shape[1], dtype=F64, device=dev)
    mass_tol = torch.zeros_like(mass)
    wk64, wv64 = wk.to(F64), wv.to(F64)
    for b in range(B):
        n, c = lengths[b], counts[b]
        lat, r = values(packed[b], scales[b]), rot[b].to(F64)
        for t in range(c):
            v = n - c + t + 1
            if v <= 0:
                continue
            L, R = lat[:v], r[:v]
            q, qr = q_nope[b, t].to(F64), q_rot[b, t].to(F64)                       # [H, .]
            qa = torch.einsum("hn,hnr->hr", q, wk64)
            s = (qa @ L.T + qr @ R.T) * scale                                       # [H, v]
            top = qa.abs().reshape(H, 16, 32).amax(2, keepdim=True).expand(H, 16, 32).reshape(H, 512)
            left = torch.einsum("hn,hnr->hr", q.abs(), wk64.abs()) * (nope + 4) * u + top * (2.0 ** -22 if fine_q else 2.0 ** -12) / 3.75
            left_r = qr.abs() * (2.0 ** -25 if fine_q else 2.0 ** -17)
            E = (left @ L.abs().T + left_r @ R.abs().T + 64 * u * (qa.abs() @ L.abs().T + qr.abs() @ R.abs().T)) * abs(scale)
            E = (E + 4 * u * (s.abs() + s.abs().amax(1, keepdim=True))).amax(1, keepdim=True)
            p = torch.softmax(s, -1)
            rel_p = torch.expm1(2 * E) + 4 * u + (2.0 ** -22 if fine_p else 2.0 ** -11) + v / 16 * u
            ctx, mag = p @ L, p @ L.abs()
            e_ctx = mag * (rel_p + (v / 8 + 300) * u)
            o[b, t] = torch.einsum("hr,hvr->hv", ctx, wv64)
            tol[b, t] = torch.einsum("hr,hvr->hv", e_ctx + 66 * u * mag, wv64.abs()) + out_eps * o[b, t].abs() + 1e-30
            mass[b, :v] += p.sum(0)
            mass_tol[b, :v] += (p * (torch.expm1(2 * E) + (v / 8 + 300) * u)).sum(0)
    mass_tol += mass * (T * H / 16 + 64) * u
    return o, tol, mass, mass_tol


def evict(weight, n, keep, sink, recent):
    """The kept positions of one sequence (weight: a list of floats), ascending."""
    if n <= keep:
        return list(range(n))
    middle = range(sink, n - recent)
    key = lambda j: (1, 0.0, j) if weight[j] != weight[j] else (0, -weight[j], j)  # noqa: E731
    best = sorted(middle, key=key)[:keep - sink - recent]
    return list(range(sink)) + sorted(best) + list(range(n - recent, n))
