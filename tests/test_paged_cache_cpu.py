"""What a paged cache has room for, and what a model's context has."""
import pytest
import torch

from dart_pytorch_b200.models import GPT, GPTConfig, Llama, LlamaConfig
from dart_pytorch_b200.models.beam import _Search
from dart_pytorch_b200.nn import MultiHeadAttention, PagedCache, RopeCache


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_a_full_row_may_end_while_others_go_on():
    c = PagedCache(1, 1, 8, 2, 8, 4)
    c.prompts([8, 3], [0, 1])
    with pytest.raises(ValueError, match="9 tokens"):
        c.fork()
    with pytest.raises(ValueError, match="9 tokens"):
        c.fork(ints(1, 0))
    assert c.lens.tolist() == [8, 3] and c.longest == 8
    c.fork(ints(-1, 1))
    assert c.lens.tolist() == [0, 4] and c.longest == 4
    c.fork(ints(1, 1))
    assert c.lens.tolist() == [5, 5] and c.table[0, 1] != c.table[1, 1] and c.table[0, 0] == c.table[1, 0]
    c.fork(ints(-1, -1))
    assert c.lens.tolist() == [0, 0]
    for _ in range(9):
        c.fork()                                       # nothing grows
    c.prompts([8], [1])
    c.fork(ints(0, -1))
    assert c.lens.tolist() == [0, 0]


def test_a_recorded_step_looks_at_the_lengths_too():
    c = PagedCache(1, 1, 8, 2, 8, 4)
    c.prompts([8, 3], [0, 1])
    c.free([0])
    search = _Search.__new__(_Search)
    search.cache, search.out = c, "out"

    class Graph:
        def replay(self):
            c.lens = torch.where(c.lens > 0, c.lens + 1, 0).int()
    search.graph = Graph()
    for n in range(4, 9):
        assert search.replay() == "out" and c.longest == n
    with pytest.raises(ValueError, match="9 tokens"):
        search.replay()
    assert c.lens.tolist() == [0, 8]


def family(name):
    if name == "gpt":
        return GPT(GPTConfig(vocab_size=37, max_ctx=8, embed_dim=32, num_layers=2, num_heads=4, seed=5, init_std=0.4))
    return Llama(LlamaConfig(37, 8, 32, 2, 4, 4, 48, seed=3, init_std=0.4))


@pytest.mark.parametrize("name", ["gpt", "llama"])
def test_a_cache_may_be_longer_than_the_context_but_not_its_rows(name):
    model = family(name)
    c = PagedCache(2, 4, 8, 2, 64, 4)
    step = lambda *rows: model.paged_hidden(torch.tensor(rows), c)  # noqa: E731
    with torch.no_grad():
        c.prompts([6, 2], [0, 1])
        step([1, 2, 3, 4, 5, 6], [7, 8, 0, 0, 0, 0])
        for _ in range(2):
            c.fork()
            step([1], [2])
        assert c.lens.tolist() == [8, 4]
        c.fork(ints(-1, 1))                            # the row that has as many as there may be ends
        for _ in range(4):
            h = step([1], [2])
            c.fork()
        assert torch.allclose(h[1, 0], model.hidden(torch.tensor([7, 8, 2, 2, 2, 2, 2, 2]))[-1], atol=1e-5)
        with pytest.raises(ValueError, match="sequence of 9 tokens exceeds maxCtx 8"):
            step([1], [2])
        c.prompts([9], [0])
        with pytest.raises(ValueError, match="exceeds maxCtx 8"):
            step([1] * 9)


def test_rotary_attention_over_pages_keeps_to_its_window():
    m = MultiHeadAttention(32, 4, rope=RopeCache(8, 8), seed=1)
    c = PagedCache(1, 4, 8, 1, 64, 4)
    with torch.no_grad():
        c.prompts([8], [0])
        m(torch.randn(1, 8, 32), cache=c.layers[0], causal=True)
        c.fork()
        with pytest.raises(ValueError, match="RopeCache: sequence of 9 tokens"):
            m(torch.randn(1, 1, 32), cache=c.layers[0])


def test_a_step_that_nothing_was_extended_for_is_refused():
    c = PagedCache(1, 1, 8, 2, 8, 4)
    step = lambda: c.layers[0].attend(torch.zeros(2, 24), 2, 1, 1)  # noqa: E731
    with pytest.raises(ValueError, match="extend"):
        step()
    c.prompts([3, 2], [0, 1])
    c.fork()
    step()
    c.free([1])
    with pytest.raises(ValueError, match="extend"):
        step()


def test_rows_that_are_not_there_do_not_end():
    c = PagedCache(1, 1, 8, 2, 8, 4)
    c.prompts([3, 2], [0, 1])
    for rows in ([2], [-1], [0, 5]):
        with pytest.raises(ValueError, match="rows"):
            c.free(rows)
    assert c.lens.tolist() == [3, 2]
    c.free([1, 1])
    assert c.lens.tolist() == [3, 0]
