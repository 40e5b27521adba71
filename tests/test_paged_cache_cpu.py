"""What a paged cache has room for, and what a model's context has."""
import pytest
import torch

from dart_pytorch_b200.models.beam import _Search
from dart_pytorch_b200.nn import PagedCache


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
