"""The packed attention under transformers where a row's sequences are told by its position ids alone."""

import pytest
import torch

from test_gpu_post_training import BAR, _hidden, _rel, models  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("start", [0, 5])  # sequences that begin at 0, or further on (a jump ahead is a border too)
def test_position_ids_without_offsets(models, start):  # noqa: F811
    from bastile_b200 import _lib

    ours, eager = models
    lens = [37, 1, 128, 90]
    ids = torch.randint(0, 4096, (2, sum(lens)), device=DEV)
    pos = torch.cat([torch.arange(n) + start * i * 31 for i, n in enumerate(lens)])[None].to(DEV)
    rows = torch.cat((pos, torch.arange(sum(lens), device=DEV)[None]))  # the second row is one sequence
    packed = _hidden(ours, input_ids=ids, position_ids=rows, use_cache=False)
    want = _hidden(eager, input_ids=ids, position_ids=rows, use_cache=False)
    with torch.no_grad():
        assert _rel(packed, want) < BAR
        at = 0
        for n in lens:
            alone = _hidden(ours, input_ids=ids[:1, at:at + n], position_ids=pos[:, at:at + n], use_cache=False)
            assert _rel(packed[:1, at:at + n], alone) < BAR / 4
            at += n
    g = torch.randn_like(packed)
    packed.backward(g), want.backward(g)
    for (n, p), (_, q) in zip(ours.model.named_parameters(), eager.model.named_parameters()):
        assert _rel(p.grad, q.grad) < 2 * BAR, n
    with pytest.raises(_lib.BastileB200Error, match="position ids alone.*kept apart"):
        _lib.check_all_status()
    with torch.no_grad():  # nothing to report with offsets, or with one sequence a row
        cu = torch.tensor([0, 37, 38, 166, 256], dtype=torch.int32, device=DEV)
        _hidden(ours, input_ids=ids[:1], position_ids=pos, use_cache=False, cu_seq_lens_q=cu, cu_seq_lens_k=cu,
                max_length_q=128, max_length_k=128)
        _hidden(ours, input_ids=ids, use_cache=False)
    _lib.check_all_status()
