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
