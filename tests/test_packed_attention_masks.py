"""What transformers' masks become for the packed attention (no GPU needed)."""

import pytest
import torch


def _config():
    from bastile_b200.ops.packed_attention import register_with_transformers
    from golden.make_golden import tiny_qwen3_config

    cfg = tiny_qwen3_config()
    cfg._attn_implementation = register_with_transformers()
    return cfg


def _mask(b, t, position_ids=None, make="create_causal_mask", **kw):
    from transformers import masking_utils

    kw = {"attention_mask": None, "past_key_values": None, **kw}
    if make != "create_bidirectional_mask":
        kw["position_ids"] = position_ids
    return getattr(masking_utils, make)(kw.pop("config", None) or _config(), torch.zeros(b, t, 8), **kw)


def test_one_sequence_per_row_needs_no_mask():
    assert _mask(2, 7, torch.arange(7)[None]) is None
    assert _mask(2, 7) is None


@pytest.mark.parametrize("ids,cu", [
    ([[0, 1, 2, 0, 1, 0]], [0, 3, 5, 6]), ([[0, 1, 2, 7, 8, 9]], [0, 3, 6]),  # restarts, and a jump ahead
    ([[3, 4, 4, 5]], [0, 2, 4]), ([[0, 1, 2, 3], [0, 0, 1, 2]], [0, 4, 5, 8]), ([[0, 0, 0]], [0, 1, 2, 3]),
])
def test_position_ids_that_start_several_sequences(ids, cu):
    """Where transformers keeps tokens apart without a cache, offsets say so."""
    ids = torch.tensor(ids)
    got = _mask(*ids.shape, ids)
    assert got.dtype == torch.int32 and got.tolist() == cu


def test_offsets_agree_with_the_mask_that_others_get():
    ids = torch.cat([torch.arange(n) for n in (5, 1, 9, 2)])[None]
    cfg = _config()
    cu = _mask(1, 17, ids, config=cfg).tolist()
    cfg._attn_implementation = "eager"
    want = _mask(1, 17, ids, config=cfg)[0, 0] == 0
    seq = torch.searchsorted(torch.tensor(cu[1:]), torch.arange(17), right=True)
    assert torch.equal((seq[:, None] == seq[None]) & torch.ones(17, 17, dtype=torch.bool).tril(), want)


def test_other_masks_are_refused():
    cfg = _config()
    cfg.sliding_window, cfg.attention_chunk_size = 4, 4
    overlay = lambda b, h, q, k: k < 3  # noqa: E731
    for kw in (dict(make="create_bidirectional_mask"), dict(make="create_sliding_window_causal_mask"),
               dict(make="create_chunked_causal_mask"), dict(or_mask_function=overlay),
               dict(and_mask_function=overlay)):
        with pytest.raises(ValueError, match="full causal"):
            _mask(1, 8, torch.arange(8)[None], config=cfg, **kw)


def test_what_the_attention_refuses():
    from bastile_b200.ops.packed_attention import hf_packed_attention

    q, k = torch.zeros(1, 4, 8, 64), torch.zeros(1, 2, 8, 64)
    encoder = torch.nn.Module()
    encoder.is_causal = False
    for module, mask, kw, text in ((encoder, None, {}, "full causal"), (None, None, dict(is_causal=False), "full causal"),
                                   (None, None, dict(s_aux=torch.zeros(4)), "sinks"),
                                   (None, torch.zeros(1, 1, 8, 8), {}, "hf_packed_mask"),
                                   (None, torch.ones(1, 8), {}, "hf_packed_mask")):
        with pytest.raises(ValueError, match=text):
            hf_packed_attention(module, q, k, k, mask, **kw)
