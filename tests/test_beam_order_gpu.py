"""Within a beam the logits decide: the kernel, with few candidates and with many."""
import pytest
import torch

import paged_oracle as oracle
from dart_pytorch_b200 import ops
from test_beam_cpu import agree
from test_beam_order_cpu import SIZES, cases

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,beams", SIZES)
def test_equal_totals_of_a_beam_go_by_logit(dtype, vocab, beams):
    for logits, scores, finished, eos in cases(dtype, vocab, beams):
        logits, scores = logits.to(dtype).cuda(), scores.cuda()
        finished = None if finished is None else finished.cuda()
        agree(ops.beam_step(logits, scores, finished, eos), oracle.beam(logits, scores, finished, -1 if eos is None else eos))
