"""Beam selection kernels against brute force."""
import pytest
import torch

import paged_oracle as oracle
from dart_pytorch_b200 import ops
from test_beam_cpu import agree

pytestmark = pytest.mark.gpu
INF = float("inf")


def data(items, beams, vocab, dtype, seed, done=0.3):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(items * beams, vocab, generator=g) * 3).to(dtype)
    scores = -torch.rand(items, beams, generator=g) * 8
    finished = torch.rand(items, beams, generator=g) < done
    return logits.cuda(), scores.cuda(), finished.cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("items,beams,vocab", [(1, 1, 1), (1, 1, 9), (2, 3, 2), (3, 4, 31), (2, 5, 321), (1, 8, 8191), (1, 8, 8192), (2, 4, 8193),
                                               (1, 4, 50257), (3, 32, 1000), (2, 32, 33), (1, 16, 17), (40, 2, 2049), (1, 3, 100003)])
def test_beam_step(dtype, items, beams, vocab):
    logits, scores, finished = data(items, beams, vocab, dtype, items + vocab)
    agree(ops.beam_step(logits, scores), oracle.beam(logits, scores, None, -1))
    agree(ops.beam_step(logits, scores, finished, vocab // 2), oracle.beam(logits, scores, finished, vocab // 2))
    first = torch.full((items, beams), -INF, device="cuda")
    first[:, 0] = 0
    agree(ops.beam_step(logits, first, None, vocab - 1), oracle.beam(logits, first, None, vocab - 1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [40, 5000, 20001])
def test_ties_go_to_the_first(dtype, vocab):
    logits = torch.zeros(8, vocab, device="cuda", dtype=dtype)
    scores = torch.zeros(2, 4, device="cuda")
    agree(ops.beam_step(logits, scores), oracle.beam(logits, scores, None, -1))
    logits[:, ::2] = -0.0                                      # the same number
    agree(ops.beam_step(logits, scores), oracle.beam(logits, scores, None, -1))
    logits[:, vocab // 2:] = 1.0
    logits[3, 7] = 1.0
    agree(ops.beam_step(logits, scores), oracle.beam(logits, scores, None, -1))
    logits[:] = torch.arange(vocab, device="cuda") // 50       # ascending, with ties
    agree(ops.beam_step(logits, scores), oracle.beam(logits, scores, None, -1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab,pad", [(127, 3), (128, 0), (9000, 0), (9001, 2)])
@pytest.mark.parametrize("beams", [3, 8, 9])
def test_fewer_tokens_than_beams_above_the_lowest_value(dtype, vocab, pad, beams):
    """What has to be reached lies below the lowest fp32 value then."""
    logits = torch.full((2 * beams, vocab + pad), torch.finfo(dtype).min, dtype=dtype, device="cuda")[:, :vocab]
    logits[:, vocab // 3], logits[:, vocab - 2] = 17.0, 12.0
    scores = torch.full((2, beams), -INF, device="cuda")
    scores[:, 0] = torch.tensor([0.0, -1.0e30], device="cuda")
    finished = torch.arange(2 * beams, device="cuda").view(2, beams) % 3 == 2
    agree(ops.beam_step(logits, scores), oracle.beam(logits, scores, None, -1))
    agree(ops.beam_step(logits, scores, finished, 5), oracle.beam(logits, scores, finished, 5))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask", ["-inf", "lowest"])
@pytest.mark.parametrize("vocab", [9, 321, 50257, 128256])
def test_a_token_without_choice_costs_nothing(dtype, mask, vocab):
    """Rows of one token keep their scores to the bit, and beams of equal scores their order; no score grows."""
    beams = 6
    logits = torch.full((beams, vocab), -INF if mask == "-inf" else torch.finfo(dtype).min, device="cuda", dtype=dtype)
    only = torch.tensor([vocab - 1, 0, 7, vocab // 2, 3, vocab // 3], device="cuda")
    logits[torch.arange(beams, device="cuda"), only] = torch.tensor([0.3, -7.7, 17.3, 1e-3, -41.0, 1e4], device="cuda").to(dtype)
    for scores in (torch.full((1, beams), -0.7, device="cuda"), -torch.arange(beams, device="cuda").view(1, beams).float() / 3):
        got, parents, tokens, _ = ops.beam_step(logits, scores)
        assert torch.equal(got, scores) and parents[0].tolist() == list(range(beams)) and tokens[0].tolist() == only.tolist()
    g = torch.Generator().manual_seed(vocab)
    peaked = (torch.randn(beams, vocab, generator=g) * 30).to(dtype).cuda()
    assert bool((ops.beam_step(peaked, torch.zeros(1, beams, device="cuda"))[0] <= 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [12, 9000])
def test_masked_and_broken_rows(dtype, vocab):
    logits, scores, finished = data(2, 6, vocab, dtype, 1)
    low = torch.finfo(dtype).min
    logits[0, 2], logits[1, 3], logits[2], logits[3, 1:] = float("nan"), INF, -INF, -INF
    logits[4] = low                                            # all masked by the type's lowest value: a flat distribution
    logits[5, vocab // 2:] = low
    logits[6, :] = -INF
    logits[6, vocab - 2] = -5.0
    agree(ops.beam_step(logits, scores), oracle.beam(logits, scores, None, -1))
    agree(ops.beam_step(logits, scores, finished, 3), oracle.beam(logits, scores, finished, 3))
    scores[0, 5], scores[1, 2], scores[0, 3] = float("nan"), -INF, INF
    finished[1, 2] = True
    agree(ops.beam_step(logits, scores, finished, 3), oracle.beam(logits, scores, finished, 3))
    scores[:] = -INF
    agree(ops.beam_step(logits, scores, finished, 3), oracle.beam(logits, scores, finished, 3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(dtype):
    logits, scores, finished = data(2, 4, 1003, dtype, 5)
    want = ops.beam_step(logits, scores, finished, 9)
    wide = torch.full((8, 1100), INF, dtype=dtype, device="cuda")
    for first in (0, 1, 3, 8):
        view = wide[:, first:first + 1003]
        wide.fill_(INF)
        view.copy_(logits)
        got = ops.beam_step(view, scores.t().contiguous().t(), finished.t().contiguous().t(), 9)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = ops.beam_step(logits.t().contiguous().t(), scores, finished, 9)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    rep = logits[:1].expand(8, 1003)                           # one row for all
    agree(ops.beam_step(rep, scores), oracle.beam(rep, scores, None, -1))


def test_streams_and_graphs():
    a, b = data(3, 8, 30011, torch.bfloat16, 1), data(1, 4, 50257, torch.float32, 2)
    want_a, want_b = ops.beam_step(*a, 5), ops.beam_step(*b, 5)
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for x in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.beam_step(*x, 5))
        graphs.append(g)
    for _ in range(4):
        torch.cuda.synchronize()
        got = []
        for g, s, x in zip(graphs, streams, (a, b)):
            with torch.cuda.stream(s):
                g.replay()
                got.append(ops.beam_step(*x, 5))
        torch.cuda.synchronize()
        for have, want in zip(outs + got, (want_a, want_b) * 2):
            assert all(torch.equal(x, y) for x, y in zip(have, want))
    a[0].normal_()
    graphs[0].replay()
    agree(outs[0], oracle.beam(a[0], a[1], a[2], 5))


def test_scores_beyond_float_and_far_apart():
    logits, scores, _ = data(1, 3, 700, torch.float32, 3)
    scores[0] = torch.tensor([-1e30, -3.0, -2e38])
    agree(ops.beam_step(logits, scores), oracle.beam(logits, scores, None, -1))
    scores[0] = torch.tensor([-1e6, -1e6 + 1, -1e6 - 2])
    agree(ops.beam_step(logits * 30, scores), oracle.beam(logits * 30, scores, None, -1))


def test_more_items_than_there_are_counters():
    logits, scores, finished = data(5000, 2, 37, torch.float32, 11)
    got = ops.beam_step(logits, scores, finished, 4)
    agree(got, oracle.beam(logits, scores, finished, 4))
    part = ops.beam_step(logits[:20], scores[:10].contiguous(), finished[:10].contiguous(), 4)
    assert all(torch.equal(a[:10], b) for a, b in zip(got, part))


@pytest.mark.parametrize("beams,vocab", [(8, 50000), (32, 30000)])
def test_few_valid_tokens_and_few_live_beams(beams, vocab):
    """Constrained decoding: all but a few tokens masked, by -inf or by the lowest value, in the first step too."""
    logits, scores, finished = data(2, beams, vocab, torch.float32, 3)
    for low in (-INF, torch.finfo(torch.float32).min):
        masked = torch.full_like(logits, low)
        masked[:, 17::9973] = logits[:, 17::9973]
        agree(ops.beam_step(masked, scores), oracle.beam(masked, scores, None, -1))
        agree(ops.beam_step(masked, scores, finished, 17), oracle.beam(masked, scores, finished, 17))
        first = torch.full_like(scores, -INF)
        first[:, 0] = 0
        agree(ops.beam_step(masked, first), oracle.beam(masked, first, None, -1))


def test_many_close_totals():
    """Thousands of logits within a few steps of one another, more than are ranked at once, in no order."""
    g = torch.Generator().manual_seed(2)
    for dtype, spread in ((torch.bfloat16, 4), (torch.float32, 300)):
        logits = torch.randint(0, spread, (8, 20000), generator=g).float().mul_(1 / 64).to(dtype).cuda()
        scores = torch.zeros(1, 8, device="cuda")
        agree(ops.beam_step(logits, scores), oracle.beam(logits, scores, None, -1))
