"""What a search answers when there is nothing to answer with, or when it is asked for what cannot be."""
import pytest
import torch

from dart_pytorch_b200.apps.servers import GenerationService
from test_beam_search_cpu import gpt, llama


def broken(make, token):
    model = make()
    with torch.no_grad():
        (model.embed_in if make is llama else model.token_emb).weight[token] = float("nan")
    return model


@pytest.mark.parametrize("make", [llama, gpt])
def test_no_continuation_at_all_is_an_error_with_a_name(make):
    model = broken(make, 5)
    with pytest.raises(ArithmeticError, match="generate_beams: no continuation of prompt 0"):
        model.generate_beams([[3, 5], [1, 2]], 4, 2)
    code, out = GenerationService(model, None, "tiny").run({"tokens": [3, 5], "maxNewTokens": 4, "beams": 2})
    assert code == 500 and "no continuation" in out["error"]


def test_an_end_that_is_no_token_is_a_bad_request():
    svc = GenerationService(llama(), None, "tiny")
    for eos in (-1, 37, 10 ** 9):
        code, out = svc.run({"tokens": [3], "maxNewTokens": 2, "beams": 2, "eos": eos})
        assert code == 400 and '"eos"' in out["error"]
    for eos in (0, 36, None):
        assert svc.run({"tokens": [3], "maxNewTokens": 2, "beams": 2, "eos": eos})[0] == 200
    for eos in (99, "none"):                             # sampling has no use for it
        assert svc.run({"tokens": [3], "maxNewTokens": 2, "eos": eos})[0] == 200


def test_more_than_one_call_takes_is_refused_before_it_starts(monkeypatch):
    model = llama()
    monkeypatch.setattr(type(model), "paged_hidden", lambda *a: pytest.fail("the model ran"))
    with pytest.raises(ValueError, match="generate_beams: 129 prompts of 32 beams .* 4128 rows .* 4096 rows"):
        model.generate_beams([[1]] * 129, 4, 32)
    model.config.max_ctx = 1 << 16                      # (128 rows of 2^12 pages, and those of the prompts)
    with pytest.raises(ValueError, match="524288 pages"):
        model.generate_beams([[1]] * 4, 1 << 16, 32)
