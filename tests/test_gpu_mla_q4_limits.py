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
