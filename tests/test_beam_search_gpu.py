"""Beam search on the device: kernels of the paged cache together, recorded and not."""
import pytest
import torch

from dart_pytorch_b200.models import GPT, GPTConfig, Llama, LlamaConfig
from test_beam_search_cpu import gpt, llama, plain_search, same

pytestmark = pytest.mark.gpu
PROMPTS = [[3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8, 9, 7, 9, 3, 2], [11], [2, 7, 18]]


@pytest.mark.parametrize("make", [llama, gpt])
@pytest.mark.parametrize("beams,new,eos", [(1, 6, None), (3, 20, None), (4, 24, 7), (5, 1, 0)])
def test_fp32_beams_match_whole_forward_passes(make, beams, new, eos):
    model = make("cuda")
    got = model.generate_beams(PROMPTS, new, beams, eos)
    # on the CPU, as the forward pass there does not share a kernel with the search
    plain = make()
    for mine, p in zip(got, PROMPTS):
        same(mine, plain_search(plain, p, new, beams, eos), p, new, 1e-4)


@pytest.mark.parametrize("family", ["llama", "gpt"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_recorded_steps_are_the_same_steps(family, dtype, monkeypatch):
    if family == "llama":
        model = Llama(LlamaConfig(1000, 128, 256, 3, 4, 2, 512, device="cuda", dtype=dtype, seed=1, init_std=0.1))
    else:
        model = GPT(GPTConfig(vocab_size=1000, max_ctx=128, embed_dim=256, num_layers=3, num_heads=4, device="cuda", dtype=dtype, seed=1,
                              init_std=0.1))
    prompts = [list(range(1, 60)), [5] * 16, [9, 8, 7]]
    recorded = model.generate_beams(prompts, 40, 4, 3)
    again = model.generate_beams(prompts, 40, 4, 3)
    monkeypatch.setenv("DPTB200_DECODE_GRAPH", "0")
    assert recorded == again == model.generate_beams(prompts, 40, 4, 3)


def test_bf16_scores_are_the_sequences_log_probabilities():
    """In bf16 a search may branch otherwise than in fp32, but what it returns must have the score that it says: the sum of the
    log-probabilities that a pass over the whole sequence gives, within what bf16 logits of this size (up to 8: steps of 2^-5,
    some of them apart in every token) leave of it."""
    model = Llama(LlamaConfig(1000, 128, 256, 3, 8, 2, 512, device="cuda", dtype=torch.bfloat16, seed=1, init_std=0.1))
    prompts = [list(range(1, 60)), [9, 8, 7]]
    for p, beams in zip(prompts, model.generate_beams(prompts, 24, 4)):
        assert all(x[1] >= y[1] for x, y in zip(beams, beams[1:])) and len({tuple(s) for s, _ in beams}) == 4
        for seq, score in beams:
            assert seq[:len(p)] == p and len(seq) == len(p) + 24
            with torch.no_grad():
                lp = torch.log_softmax(model(torch.tensor(seq[:-1], device="cuda")).double(), -1)
            want = lp[torch.arange(len(p) - 1, len(seq) - 1), torch.tensor(seq[len(p):])].sum()
            assert abs(float(want) - score) <= 24 * 2.0 ** -4
