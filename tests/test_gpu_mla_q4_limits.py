"""The 4-bit cache on the device where its calls have an edge: more tokens than a row of blocks, gates that are no numbers."""
from __future__ import annotations

import pytest
import torch

from test_gpu_mla_q4 import SCALE, _cache, _ints, _rand

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def test_append_of_more_tokens_than_a_row_of_blocks():
    """2^26 tokens are 2^32 threads; all but the last five lie before the cache, so they are left out."""
    from k3hip.mla_q4 import mla_q4_append
    M = (1 << 26) + 5
    row = _rand(1, 1, 1, 576).cuda()
    packed, scales, rot = _cache(1, 8)
    mla_q4_append(row[..., :512].expand(1, M, 512), row[..., 512:].expand(1, M, 64), packed, scales, rot, start=_ints([-(1 << 26)]))
    want = _cache(1, 8)
    mla_q4_append(row[..., :512].expand(1, 5, 512), row[..., 512:].expand(1, 5, 64), *want)
    assert all(bool((a == b).all()) for a, b in zip((packed, scales, rot), want)) and bool(rot[0, :5].any()) and not bool(rot[0, 5:].any())


@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("B,T,H,weight", [(4, 2, 8, False), (4, 5, 16, True), (6, 40, 24, False), (9, 80, 32, True)])
def test_a_gate_that_is_no_number_leaves_zeros_where_nothing_is_seen(B, T, H, weight, out):
    import _q4_oracle as oracle
    from k3hip.mla_q4 import mla_q4_attention
    cap = T + 60
    cache = oracle.random_cache(B, cap, 3, "cuda")
    q = _rand(4, B, T, H, 192).cuda()
    wk, wv = (_rand(s, H, 128, 512, std=512 ** -0.5, dtype=BF16).cuda() for s in (5, 6))
    lengths, counts = [T + 30 + b for b in range(B)], [T] * B
    lengths[1], counts[0], lengths[2], counts[3] = 0, T // 2, T - 1, 2 * T        # (the third's first query sees nothing, the fourth has T)
    gate = _rand(7, B, T, H * 128).cuda()
    nothing = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    nothing[0, T // 2:] = nothing[1] = nothing[2, 0] = True

    def run(gate):
        w = torch.zeros(B, cap, device="cuda") if weight else None
        return mla_q4_attention(q[..., :128], q[..., 128:], wk, wv, *cache, SCALE, lengths=_ints(lengths), counts=_ints(counts), weight=w, gate=gate, out_dtype=out), w

    clean, w0 = run(gate)
    assert bool(clean[~nothing].view(int((~nothing).sum()), -1).any(-1).all())
    for value in (float("nan"), float("-inf"), float("inf")):
        got, w = run(torch.where(nothing[..., None], torch.full_like(gate, value), gate))
        assert not bool(got[nothing].any()) and bool((got == clean).all())
        assert w is None or bool((w == w0).all())
    # one length for all, no counts
    both = mla_q4_attention(q[..., :128], q[..., 128:], wk, wv, *cache, SCALE, lengths=T - 1, gate=torch.where(torch.arange(T, device="cuda")[None, :, None] == 0, float("nan"), gate), out_dtype=out)
    assert not bool(both[:, 0].any()) and bool(torch.isfinite(both).all()) and (T == 1 or bool(both[:, 1:].any()))
