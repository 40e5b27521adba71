"""Beam search through a paged cache against the same search by whole forward passes, and the cache class."""
import math

import pytest
import torch

from dart_pytorch_b200.apps.servers import GenerationService
from dart_pytorch_b200.models import GPT, GPTConfig, Llama, LlamaConfig
from dart_pytorch_b200.nn import PagedCache


def llama(device=None, dtype=torch.float32, heads=4, kv=2, dim=32):
    return Llama(LlamaConfig(37, 48, dim, 2, heads, kv, 48, device=device, dtype=dtype, seed=3, init_std=0.4))


def gpt(device=None, dtype=torch.float32):
    return GPT(GPTConfig(vocab_size=37, max_ctx=48, embed_dim=32, num_layers=2, num_heads=4, device=device, dtype=dtype, seed=5, init_std=0.4))


def plain_search(model, prompt, new, beams, eos=None):
    """Every beam's whole sequence through the model at every step; ``(tokens, score)`` best first."""
    live = [(list(prompt), 0.0, False)]
    for _ in range(new):
        every = []
        for w, (seq, score, done) in enumerate(live):
            if done:
                every.append((-score, w, eos, seq, True))
                continue
            with torch.no_grad():
                logits = model(torch.tensor(seq, device=model.device))[-1].double().cpu()
            lp = torch.log_softmax(logits, 0).tolist()
            every += [(-(score + x), w, t, seq + [t], t == eos) for t, x in enumerate(lp)]
        every.sort(key=lambda e: e[:3])
        live = [(seq, -s, done) for s, _, _, seq, done in every[:beams]]
    return [(seq, score) for seq, score, _ in live]


def same(got, want, prompt, new, tol):
    assert [seq for seq, _ in got] == [seq for seq, _ in want]
    for (_, a), (_, b) in zip(got, want):
        assert math.isclose(a, b, abs_tol=tol * new, rel_tol=tol)


@pytest.mark.parametrize("make", [llama, gpt])
@pytest.mark.parametrize("beams,new,eos", [(1, 6, None), (3, 9, None), (4, 20, 7), (5, 1, 0)])
def test_beams_match_whole_forward_passes(make, beams, new, eos):
    model = make()
    prompts = [[3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8, 9, 7, 9, 3, 2], [11], [2, 7, 18]]
    got = model.generate_beams(prompts, new, beams, eos)
    for mine, p in zip(got, prompts):
        same(mine, plain_search(model, p, new, beams, eos), p, new, 1e-4)


def test_one_beam_is_greedy_and_the_context_bounds_it():
    model = llama()
    p = [5, 6, 7]
    assert model.generate_beams([p], 10, 1)[0][0][0] == [int(t) for t in model.generate(p, 10, temperature=0.0)]
    assert len(model.generate_beams([p], 100, 2)[0][0][0]) == len(model.generate(p, 100, temperature=0.0)) == 49
    assert model.generate_beams([p], 0, 2) == [[(p, 0.0)]]


def test_length_penalty_orders_the_beams():
    model = llama()
    flat, long = (model.generate_beams([[3, 1]], 12, 5, 7, length_penalty=x)[0] for x in (0.0, 3.0))
    assert sorted(map(str, flat)) == sorted(map(str, long))
    value = lambda seq, score: score / (len(seq) - 2) ** 3  # noqa: E731
    assert [value(*x) for x in long] == sorted((value(*x) for x in long), reverse=True)


def test_refusals():
    model = llama()
    for args in (([],), ([[]],), ([[1]], 4, 0), ([[1]], 4, 33), ([[1] * 49], 4), ([[1]], 4, 2, 37)):
        with pytest.raises(ValueError):
            model.generate_beams(*(args if len(args) > 1 else args + (4,)))
    with pytest.raises(ValueError):
        PagedCache(1, 1, 8, 0, 8)
    c = PagedCache(1, 1, 8, 3, 8, 4)
    for lengths, rows in (([3], [3]), ([3, 2], [1, 1]), ([0], [0]), ([9], [0]), ([3], [0, 1])):
        with pytest.raises(ValueError):
            c.prompts(lengths, rows)
    c.prompts([7], [1])
    c.fork()
    with pytest.raises(ValueError):
        c.fork()
    with pytest.raises(ValueError):
        c.layers[0].attend(torch.zeros(2, 24), 2, 1, 1)


def test_cache_rows_come_and_go():
    """Rows that start later, end earlier and are packed in between answer as on their own."""
    model = llama()
    cache = PagedCache(2, 2, 8, 3, 48, 4, num_pages=14)

    def feed(lists, rows=None):
        n = max(len(x) for x in lists)
        t = torch.tensor([x + [0] * (n - len(x)) for x in lists])
        with torch.no_grad():
            h = model.paged_hidden(t, cache)
        return [h[i, len(x) - 1] for i, x in enumerate(lists)]

    def alone(seq):
        with torch.no_grad():
            return model.hidden(torch.tensor(seq))[-1]
    a, b, d = [1, 2, 3, 4, 5, 6], [9, 8, 7], [4, 4, 4, 4, 4]
    cache.prompts([6, 3], [0, 2])
    for h, s in zip(feed([a, b]), (a, b)):
        assert torch.allclose(h, alone(s), atol=1e-5)
    cache.fork(torch.tensor([0, 0, 2], dtype=torch.int32))
    a0, a1, b = a + [10], a + [11], b + [12]
    for h, s in zip(feed([[10], [11], [12]]), (a0, a1, b)):
        assert torch.allclose(h, alone(s), atol=1e-5)
    cache.free([0])
    assert int(cache.compact()) == 3 and int(cache.lens[0]) == 0
    cache.prompts([5], [0])
    assert torch.allclose(feed([d])[0], alone(d), atol=1e-5)
    cache.fork(torch.tensor([2, 1, -1], dtype=torch.int32))
    got = feed([[13], [14], [0]])
    assert torch.allclose(got[0], alone(b + [13]), atol=1e-5) and torch.allclose(got[1], alone(a1 + [14]), atol=1e-5)


def test_a_cache_outlives_many_rows():
    """What has ended does not count: rows that come and go for longer than any of them may be."""
    model = llama()
    cache = PagedCache(2, 2, 8, 2, 8, 4)
    for i in range(5):
        cache.prompts([3], [i % 2])
        with torch.no_grad():
            model.paged_hidden(torch.tensor([[1, 2, 3]]), cache)
        for _ in range(4):
            cache.fork()
            with torch.no_grad():
                model.paged_hidden(torch.zeros(2, 1, dtype=torch.long), cache)
        assert cache.lens.tolist() == ([7, 0] if i % 2 == 0 else [0, 7])
        cache.free([i % 2])


def test_service_answers_with_beams():
    svc = GenerationService(llama(), None, "tiny")
    code, out = svc.run({"tokens": [3, 1, 4], "maxNewTokens": 5, "beams": 3, "eos": 7})
    assert code == 200 and len(out["beams"]) == 3 and out["newTokens"] == out["beams"][0]["newTokens"]
    assert out["beams"][0]["score"] >= out["beams"][1]["score"]
    assert svc.run({"tokens": [3], "beams": 40})[0] == 400
