"""The plan object of packed attention, without a GPU."""

import torch


class _Plan:
    """A plan on a GPU, as far as its object looks at it."""

    is_cuda = True
    device = torch.device("cuda", 0)

    def __init__(self):
        self.recorded = []

    def record_stream(self, stream):
        self.recorded.append(stream)


def test_use_on_another_stream_is_recorded(monkeypatch):
    from bastile_b200 import _lib
    from bastile_b200.ops.packed_attention import PackedSequences

    now = [7]
    monkeypatch.setattr(_lib, "stream_ptr", lambda dev: now[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: f"stream {now[0]}")
    seqs = PackedSequences(_Plan(), 1, 4)
    seqs.keep_for(seqs.device)
    assert seqs.plan.recorded == []
    now[0] = 9
    seqs.keep_for(seqs.device)
    assert seqs.plan.recorded == ["stream 9"]
