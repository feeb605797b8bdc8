"""The post-training ops in a model: attention as transformers' ``bastile_packed`` implementation on
packed, padded and plain batches, and the step they are made for - score, then take a policy-loss
step - against the same model on torch's own attention and a plain loss."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture()
def models():
    """(ours, eager): the tiny model of the fixtures, patched with packed attention, and unpatched, both bf16."""
    import bastile_b200
    from golden.make_golden import build_tiny_qwen3, tiny_qwen3_config
    from transformers import Qwen3ForCausalLM

    bastile_b200.reset()
    stock = build_tiny_qwen3()
    eager = Qwen3ForCausalLM(tiny_qwen3_config())
    eager.load_state_dict(stock.state_dict())
    eager = eager.to(DEV, torch.bfloat16).train()
    applied = bastile_b200.apply(fused_layers=True, packed_attention=True)
    assert "bastile_packed" in applied
    cfg = tiny_qwen3_config()
    cfg._attn_implementation = "bastile_packed"
    ours = Qwen3ForCausalLM(cfg)
    ours.load_state_dict(stock.state_dict())
    ours = ours.to(DEV, torch.bfloat16).train()
    yield ours, eager
    bastile_b200.reset()


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _hidden(model, **kw):
    return model.model(**kw)[0]


# bf16 activations through two layers: each of ~20 roundings of 2^-8 at most, as independent errors
# sqrt(20) 2^-9 = 9e-3 on either side; the bar for the distance of the two sides is twice their sum
BAR = 4e-2


def test_plain_batch_matches_eager(models):
    ours, eager = models
    ids = torch.randint(0, 4096, (2, 128), device=DEV)
    a, b = _hidden(ours, input_ids=ids), _hidden(eager, input_ids=ids)
    assert _rel(a, b) < BAR
    g = torch.randn_like(a)
    a.backward(g), b.backward(g)
    for (n, p), (_, q) in zip(ours.model.named_parameters(), eager.model.named_parameters()):
        assert _rel(p.grad, q.grad) < 2 * BAR, n


def test_packed_row_is_its_sequences(models):
    from bastile_b200 import _lib

    ours, _ = models
    lens = [37, 1, 128, 90]
    ids = torch.randint(0, 4096, (1, sum(lens)), device=DEV)
    cu = torch.tensor([0, 37, 38, 166, 256], dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(n) for n in lens])[None].to(DEV)
    with torch.no_grad():
        packed = _hidden(ours, input_ids=ids, position_ids=pos, cu_seq_lens_q=cu, cu_seq_lens_k=cu, max_length_q=128,
                         max_length_k=128)
        start = 0
        for n in lens:
            alone = _hidden(ours, input_ids=ids[:, start:start + n])
            # the same rows through the same kernels; only the library products may choose other tiles
            assert _rel(packed[:, start:start + n], alone) < BAR / 4
            start += n
    _lib.check_all_status()
    with torch.no_grad():  # restarting positions without offsets: noticed
        _hidden(ours, input_ids=ids, position_ids=pos)
    with pytest.raises(_lib.BastileB200Error, match="position ids"):
        _lib.check_all_status()


@pytest.mark.parametrize("side", ["right", "left"])
def test_padded_batch(models, side):
    from bastile_b200 import _lib

    ours, _ = models
    lens, t = [50, 128, 3], 128
    ids = torch.randint(0, 4096, (3, t), device=DEV)
    mask = torch.zeros(3, t, dtype=torch.int64, device=DEV)
    for i, n in enumerate(lens):
        mask[i, :n] = 1
    mask = mask if side == "right" else mask.flip(1)
    pos = (mask.cumsum(1) - 1).clamp(min=0)
    with torch.no_grad():
        out = _hidden(ours, input_ids=ids, attention_mask=mask, position_ids=pos)
        for i, n in enumerate(lens):
            at = slice(0, n) if side == "right" else slice(t - n, t)
            alone = _hidden(ours, input_ids=ids[i:i + 1, at])
            assert _rel(out[i:i + 1, at], alone) < BAR / 4
    _lib.check_all_status()
    mask[1, 60:70] = 0
    with torch.no_grad():
        _hidden(ours, input_ids=ids, attention_mask=mask)
    with pytest.raises(_lib.BastileB200Error, match="holes"):
        _lib.check_all_status()


def test_what_the_model_path_refuses(models):
    ours, _ = models
    ids = torch.randint(0, 4096, (1, 16), device=DEV)
    ours.eval()
    with torch.no_grad():
        first = ours.model(input_ids=ids, use_cache=True)  # a prompt fills a cache
        with pytest.raises(ValueError, match="cache"):
            ours.model(input_ids=ids[:, :1], past_key_values=first.past_key_values, use_cache=True)
    from bastile_b200.ops.packed_attention import hf_packed_attention

    q = torch.zeros(1, 4, 8, 64, dtype=torch.bfloat16, device=DEV)
    for kw, text in ((dict(dropout=0.1), "dropout"), (dict(sliding_window=4), "full causal"),
                     (dict(is_causal=False), "full causal")):
        with pytest.raises(ValueError, match=text):
            hf_packed_attention(None, q, q[:, :2], q[:, :2], None, **kw)
    with pytest.raises(ValueError, match="one packed row"):
        hf_packed_attention(None, q.expand(2, -1, -1, -1), q[:, :2].expand(2, -1, -1, -1),
                            q[:, :2].expand(2, -1, -1, -1), None, cu_seq_lens_q=torch.zeros(2, dtype=torch.int32))


def test_policy_step_on_a_packed_batch(models):
    """Score with the ops under no_grad, then loss and gradients of the whole model, against the unpatched
    model run sequence by sequence with a plain fp32 loss."""
    from bastile_b200 import _lib
    from bastile_b200.ops.fused_linear_policy_loss import fused_linear_log_probs, fused_linear_policy_loss

    ours, eager = models
    torch.manual_seed(0)
    lens = [40, 75, 13]
    t = sum(lens)
    ids = torch.randint(0, 4096, (1, t), device=DEV)
    cu = torch.tensor([0, 40, 115, 128], dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(n) for n in lens])[None].to(DEV)
    target = torch.full((1, t), -100, device=DEV)
    start = 0
    for n in lens:  # next tokens; the first five of a sequence are its prompt
        target[0, start + 4:start + n - 1] = ids[0, start + 5:start + n]
        start += n
    adv = torch.repeat_interleave(torch.tensor([1.0, -0.5, 2.0], device=DEV), torch.tensor(lens, device=DEV))[None]
    pack = dict(position_ids=pos, cu_seq_lens_q=cu, cu_seq_lens_k=cu, max_length_q=75, max_length_k=75)
    with torch.no_grad():
        old = fused_linear_log_probs(_hidden(ours, input_ids=ids, **pack), ours.lm_head.weight, target)
    ref = old + 0.1 * torch.randn_like(old)
    got = fused_linear_policy_loss(_hidden(ours, input_ids=ids, **pack), ours.lm_head.weight, target, old, adv, ref,
                                   kl_coef=0.1, cu_seqlens=cu)
    assert torch.equal(got.log_probs, old)  # the policy has not moved: its ratio is exactly 1
    live = target[0] != -100
    d = (ref - old)[0].double()
    kl = torch.expm1(d) - d
    want = sum(((-adv[0] + 0.1 * kl)[s:e][live[s:e]]).mean() for s, e in ((0, 40), (40, 115), (115, 128))) / 3
    assert abs(got.loss.item() - want.item()) <= 1e-5 and got.clip_fraction == 0
    got.loss.backward()
    _lib.check_all_status()

    loss, start = 0.0, 0
    for n in lens:
        at = slice(start, start + n)
        logits = eager(input_ids=ids[:, at]).logits[0].float()
        lp = torch.log_softmax(logits, -1).gather(1, target[0, at].clamp(min=0)[:, None])[:, 0]
        # ratios of the eager model to itself: the step of a policy that has not moved
        r, gap = (lp - lp.detach()).exp(), (ref - old)[0, at] + lp.detach() - lp
        loss = loss + (-r * adv[0, at] + 0.1 * (torch.expm1(gap) - gap))[live[at]].mean() / 3
        start += n
    loss.backward()
    for (n, p), (_, q) in zip(ours.named_parameters(), eager.named_parameters()):
        assert _rel(p.grad, q.grad) < 2 * BAR, n
