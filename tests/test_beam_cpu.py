"""Beam selection on CPU tensors against brute force, and its refusals."""
import pytest
import torch

import paged_oracle as oracle
from dart_pytorch_b200 import ops


def agree(got, want):
    scores, parents, tokens, finished = got
    assert parents.tolist() == want[1] and tokens.tolist() == want[2] and finished.tolist() == want[3]
    w = torch.tensor(want[0], dtype=torch.float64)
    s = scores.double().cpu()
    assert torch.equal(s.isinf(), w.isinf())
    # one rounding to fp32 of a total whose logarithm is of fp32 exponentials at worst: 2^-24 of the total, and 2^-21
    fine = w.isfinite()
    assert bool(((s - w).abs()[fine] <= w.abs()[fine] * 2.0 ** -24 + 2.0 ** -21).all())


@pytest.mark.parametrize("items,beams,vocab", [(1, 1, 1), (2, 3, 2), (3, 4, 17), (2, 5, 200)])
def test_beam_step_matches_brute_force(items, beams, vocab):
    g = torch.Generator().manual_seed(items * 100 + vocab)
    logits = (torch.randn(items * beams, vocab, generator=g) * 2).bfloat16().float()      # ties among them
    scores = -torch.rand(items, beams, generator=g) * 5
    finished = torch.rand(items, beams, generator=g) < 0.4
    agree(ops.beam_step(logits, scores), oracle.beam(logits, scores, None, -1))
    agree(ops.beam_step(logits, scores, finished, vocab // 2), oracle.beam(logits, scores, finished, vocab // 2))
    first = torch.full((items, beams), -float("inf"))
    first[:, 0] = 0
    agree(ops.beam_step(logits, first, None, 0), oracle.beam(logits, first, None, 0))


def test_rows_without_a_distribution_have_nothing_to_offer():
    logits = torch.randn(4, 6)
    logits[0, 2], logits[1, 3], logits[2] = float("nan"), float("inf"), -float("inf")
    scores = torch.zeros(1, 4)
    agree(ops.beam_step(logits, scores), oracle.beam(logits, scores, None, -1))
    scores[0, 3] = float("nan")
    got = ops.beam_step(logits, scores)
    assert got[0].tolist() == [[-float("inf")] * 4] and got[1].tolist() == [[0] * 4] and got[2].tolist() == [[0, 1, 2, 3]]


def test_refusals():
    logits, scores = torch.randn(6, 9), torch.zeros(2, 3)
    done = torch.zeros(2, 3, dtype=torch.bool)
    for error, args in [(ValueError, (logits[:5], scores)), (ValueError, (logits, scores[0])), (ValueError, (logits, scores.double())),
                        (TypeError, (logits.double(), scores)), (TypeError, (logits.half(), scores)), (ValueError, (logits, scores, done)),
                        (ValueError, (logits, scores, done[:1], 0)), (ValueError, (logits, scores, done.int(), 0)),
                        (ValueError, (logits, scores, None, 9)), (ValueError, (logits, scores, None, -1)),
                        (ValueError, (logits[:, :0], scores)), (ValueError, (torch.randn(33, 9), torch.zeros(1, 33))),
                        (ValueError, (logits.clone().requires_grad_(), scores))]:
        with pytest.raises(error):
            ops.beam_step(*args)
