"""Teacher-forced scores with 4-bit weights and 8-bit caches against the same model in full
precision."""

from __future__ import annotations

import pytest
import torch

from vflorence_b200 import paged_ops

F32, BF16 = torch.float32, torch.bfloat16


def make_model(dtype, device):
    """A small BART whose decoder weights are whole steps of 4 bits: every group of 64 holds a
    +-7 and its scale is a power of two, so the 4-bit layers are the model's own layers. The K/V
    of every head vary enough for the attention to matter."""
    from transformers import BartConfig, BartForConditionalGeneration

    cfg = BartConfig(vocab_size=301, d_model=64, encoder_layers=1, decoder_layers=2, encoder_attention_heads=2,
                     decoder_attention_heads=2, encoder_ffn_dim=128, decoder_ffn_dim=128, max_position_embeddings=128,
                     dropout=0.0, attention_dropout=0.0, activation_dropout=0.0, init_std=0.4, pad_token_id=1,
                     bos_token_id=0, eos_token_id=2, decoder_start_token_id=2, forced_eos_token_id=None)
    torch.manual_seed(5)
    model = BartForConditionalGeneration(cfg).eval()
    linears = [x for x in model.model.decoder.modules() if isinstance(x, torch.nn.Linear)] + [model.lm_head]
    with torch.no_grad():
        for x in linears:
            w = x.weight.view(x.weight.shape[0], -1, 64)
            codes = (torch.randn(w.shape) * 2.5).round().clamp(-7, 7)
            codes[..., 0] = 7.0
            x.weight.copy_((codes * 2.0 ** -5).view_as(x.weight))
    return model.to(device=device, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scores_follow_the_full_precision_model(dtype):
    """The 4-bit weights are exact here, so what differs is the cache's rounding (a step is 1/127
    of a block's largest magnitude, about 3 times its typical one: half a step at most, some 1 %
    of a K/V row) in four attention layers, and for bfloat16 the 2^-9 roundings of some 30
    operators: 4 % and 2 % of the logits' spread. A wrong token, position, slot or mask moves them
    by their whole spread."""
    from vflorence_b200.engine import LowBitScorer, Request

    device = torch.device("cuda", 0)
    torch.backends.cuda.matmul.allow_tf32 = False
    model = make_model(dtype, device)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(4, 301, (n,), generator=gen).tolist() for n in (5, 37, 16, 23)]
    targets = [torch.randint(4, 301, (n,), generator=gen).tolist() for n in (33, 1, 16, 20)]
    scorer = LowBitScorer(model, max_decoder_len=40)
    for layer, hf in zip(scorer.layers, model.model.decoder.layers):  # the premise
        codes, scales = layer["fc2"].codes, layer["fc2"].scales
        w = torch.stack([codes & 15, codes >> 4], -1).flatten(1).float() - 8
        assert torch.equal(w * scales.float().repeat_interleave(64, 1), hf.fc2.weight.float())
    got = scorer.score([Request(p) for p in prompts], targets, alternatives=3)
    full = model.float()
    for prompt, target, scores in zip(prompts, targets, got):
        fed = torch.tensor([[2] + target[:-1]], device=device)
        with torch.inference_mode():
            logits = full(input_ids=torch.tensor([prompt], device=device), decoder_input_ids=fed).logits[0].double()
        spread = float(logits.std())
        want = torch.log_softmax(logits, -1).cpu()
        picked = want[torch.arange(len(target)), torch.tensor(target)]
        assert scores.logprobs.shape == scores.entropy.shape == (len(target),)
        off = (scores.logprobs.double() - picked).square().mean().sqrt()
        assert off <= (0.04 if dtype == F32 else 0.06) * spread, (float(off), spread)
        moved = (scores.logprobs.double() - picked.roll(1)).square().mean().sqrt()
        assert len(target) == 1 or moved > 0.5 * spread  # another position's scores would not pass
        entropy = -(want.exp() * want).sum(-1)
        assert (scores.entropy.double() - entropy).abs().max() <= 0.5 * spread
        # the alternatives are the likeliest under the scorer: none below the target, and in order
        assert scores.values.shape == scores.indices.shape == (len(target), 3)
        assert (scores.values[:, 0] >= scores.logprobs - 1e-5).all() and (scores.values.diff(dim=1) <= 0).all()
        same = scores.indices == torch.tensor(target, dtype=torch.int32)[:, None]
        assert torch.allclose(scores.values[same], scores.logprobs[:, None].expand(-1, 3)[same], rtol=0, atol=1e-5)
    assert paged_ops.read_device_errors(device) == 0


@pytest.mark.gpu
def test_scores_of_a_batch_equal_those_of_each_request_alone():
    """Rows do not meet: a request's scores do not depend on its neighbours beyond the order of
    float32 sums (the encoder's padded batch, splits of a context): 2^-10 of a log probability's
    scale, unless a code sits at a rounding edge - one step of 1/127 then, 1 % of a score."""
    from vflorence_b200.engine import LowBitScorer, Request

    model = make_model(F32, torch.device("cuda", 0))
    torch.backends.cuda.matmul.allow_tf32 = False
    scorer = LowBitScorer(model, max_decoder_len=24, group_size=32)
    prompts, targets = [[7, 8, 9], [20] * 18], [[30, 31, 32, 33], [40] * 19]
    both = scorer.score([Request(p) for p in prompts], targets)
    for p, t, want in zip(prompts, targets, both):
        alone, = scorer.score([Request(p)], [t])
        off = (alone.logprobs - want.logprobs).abs()
        assert (off <= 0.01 * want.logprobs.abs().clamp(min=1)).all()
        assert alone.values.shape == (len(t), 0)


@pytest.mark.gpu
def test_scorer_refusals():
    from vflorence_b200.engine import LowBitScorer, Request

    scorer = LowBitScorer(make_model(F32, torch.device("cuda", 0)), max_decoder_len=8)
    r = Request([4, 5])
    for requests, targets in (([r], []), ([], []), ([r], [[]]), ([r], [[5] * 9]), ([r], [[301]]), ([r], [[-1]]),
                              ([Request([])], [[5]])):
        with pytest.raises(ValueError):
            scorer.score(requests, targets)


def test_scorer_wants_a_cuda_model():
    from vflorence_b200.engine import LowBitScorer

    with pytest.raises(ValueError, match="CUDA device"):
        LowBitScorer(make_model(F32, torch.device("cpu")), max_decoder_len=8)
