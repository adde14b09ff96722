"""What a batch's tables may be asked for: more tokens than there are slots, numbers that do not fit 32 bits, tokens given back by a number.  The
tables' class over the definition of its one launch, without a GPU."""
from __future__ import annotations

import pytest
import torch

from test_mla_paged_host import _held, on_cpu  # noqa: F401

I32 = torch.int32


def _counts(*n):
    return torch.tensor(n, dtype=I32)


def test_no_request_gets_more_tokens_than_slots(on_cpu):
    t = on_cpu.PageTable(3, 256, 12, page_size=32, device="cpu")
    slots = t.extend(_counts(5, 2, 3), tokens=3)
    assert t.lengths.tolist() == t.counts.tolist() == [3, 2, 3] == (slots >= 0).sum(1).tolist()
    slots = t.extend(_counts(100, -1, 0), tokens=2)
    assert t.lengths.tolist() == [5, 1, 3] and t.counts.tolist() == [2, 0, 0] == (slots >= 0).sum(1).tolist()
    assert [len(r) for r in _held(t)] == [1, 1, 1]
    with pytest.raises(ValueError, match="tokens"):
        t.extend(4, tokens=2)
    assert t.lengths.tolist() == [5, 1, 3]
    assert t.extend(2, tokens=4).shape == (3, 4) and t.counts.tolist() == [2, 2, 2]


def test_a_number_below_zero_gives_tokens_back(on_cpu):
    t = on_cpu.PageTable(2, 256, 12, page_size=32, device="cpu")
    t.extend(_counts(70, 3), tokens=70)
    assert t.extend(-5).shape == (2, 0)
    assert t.lengths.tolist() == [65, 0] and t.counts.tolist() == [0, 0] and [len(r) for r in _held(t)] == [3, 0]
    assert t.extend(-2, tokens=1).tolist() == [[-1], [-1]] and t.lengths.tolist() == [63, 0] and [len(r) for r in _held(t)] == [2, 0]
    assert t.extend(0).shape == (2, 0)


@pytest.mark.parametrize("most", [2 ** 31 - 1, 2 ** 31 - 256])
def test_lengths_do_not_wrap(on_cpu, monkeypatch, most):
    """``lengths + counts`` is int32: past 2^31 it would be below zero, and the request would give all its pages back."""
    t = on_cpu.PageTable(2, 256, 12, page_size=32, device="cpu")
    t.extend(_counts(70, 3), tokens=70)
    seen = []
    monkeypatch.setattr(t, "resize", lambda target, tokens: seen.append(target.tolist()))
    for counts in (_counts(most, 0), _counts(0, most), most):
        with pytest.raises(ValueError, match="tokens"):
            t.extend(counts, tokens=most)
    assert not seen
    t.extend(_counts(most, -2 ** 31), tokens=2 ** 31 - 257)
    t.extend(2 ** 31 - 257)
    assert seen == [[70 + 2 ** 31 - 257, 3 - 2 ** 31], [70 + 2 ** 31 - 257, 3 + 2 ** 31 - 257]]


def test_a_large_batch_without_heads_is_refused_as_a_small_one_is(monkeypatch):
    import test_mla_paged_host as host
    calls = host._launches(monkeypatch)
    w = torch.zeros(0, 128, 512, dtype=torch.bfloat16)
    for B in (2, 70000):
        host._attend(q_nope=torch.zeros(B, 1, 0, 128), q_rot=torch.zeros(B, 1, 0, 64), wk=w, wv=w, table=torch.zeros(B, 1, dtype=I32),
                     lengths=torch.zeros(B, dtype=I32))
    assert [c[1][28] for c in calls] == [2, 65535, 4465] and {c[1][30] for c in calls} == {0}       # (the entry point refuses 0 heads)


def test_the_one_call_step_refuses_a_paged_cache(on_cpu):
    from types import SimpleNamespace

    from k3hip.mla import MLAAttention
    from k3hip.mla_paged import new_cache_paged
    cfg = SimpleNamespace(num_attention_heads=2, q_lora_rank=16, kv_lora_rank=512, qk_nope_head_dim=8, qk_rope_head_dim=64, v_head_dim=8, q_head_dim=72,
                          rms_norm_eps=1e-5)
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    layer = MLAAttention(cfg, {"q_a_proj.weight": z(16, 32), "q_a_layernorm.weight": z(16), "q_b_proj.weight": z(144, 16), "o_proj.weight": z(32, 16),
                               "kv_a_proj_with_mqa.weight": z(576, 32), "kv_a_layernorm.weight": z(512), "kv_b_proj.weight": z(32, 512)})
    t = on_cpu.PageTable(1, 64, 4, page_size=32, device="cpu")
    t.extend(1)
    with pytest.raises(ValueError, match="paged"):
        layer.decode_step(torch.zeros(1, 1, 32), new_cache_paged(t))
