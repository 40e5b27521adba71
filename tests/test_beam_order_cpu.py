"""Within a beam the logits decide, also where its totals are too coarse to tell them apart."""
import pytest
import torch

import paged_oracle as oracle
from dart_pytorch_b200 import ops
from test_beam_cpu import agree

INF = float("inf")


def cases(dtype, vocab, beams):
    """``(logits, scores, finished, eos)`` whose totals are equal, or in large steps, within a beam; larger logits at higher tokens."""
    g = torch.Generator().manual_seed(vocab * 100 + beams)
    live = torch.full((1, beams), -INF)
    live[0, 0] = 0.0
    late = torch.zeros(beams, vocab)
    late[:, -1] = 1e-20
    yield late, live, None, None
    yield late, torch.zeros(1, beams), None, None
    tiny = torch.randn(beams, vocab, generator=g) * 1e-20
    yield tiny, live, None, None
    yield tiny, torch.zeros(1, beams), torch.arange(beams).view(1, beams) % 3 == 1, vocab // 2
    low = torch.full((beams, vocab), torch.finfo(dtype).min)
    low[:, vocab // 3], low[:, vocab - 2] = 12.0, 17.0
    yield low, live - 1e30, None, None
    apart = torch.randn(beams, vocab, generator=g) * 8
    for score in (-1e30, -1e17, -3e16):                      # steps of the totals: more than all logits, 16, 4
        yield apart, live + score, None, None
        yield apart, torch.full((1, beams), score), torch.arange(beams).view(1, beams) % 4 == 2, 1
    yield apart.roll(1, 0), torch.linspace(-1e17, -1.0000001e17, beams).view(1, beams), None, None


SIZES = [(2, 1), (9, 3), (10, 4), (33, 32), (130, 8), (700, 4), (1003, 16), (20001, 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,beams", SIZES)
def test_equal_totals_of_a_beam_go_by_logit(dtype, vocab, beams):
    for logits, scores, finished, eos in cases(dtype, vocab, beams):
        logits = logits.to(dtype)
        agree(ops.beam_step(logits, scores, finished, eos), oracle.beam(logits, scores, finished, -1 if eos is None else eos))
