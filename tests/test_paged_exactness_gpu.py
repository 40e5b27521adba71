"""What the paged kernels may lose to rounding, where it shows: in differences of nearly equal numbers."""
import pytest
import torch

from dart_pytorch_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,heads,page", [(64, 1, 16), (128, 4, 16), (64, 16, 8), (128, 12, 1), (256, 2, 32), (33, 1, 4)])
def test_weights_have_all_their_bits(hd, heads, page):
    """Two keys of weights 1 and exp(-x) with values 1 and -1 leave tanh(x / 2), a few 2^-18 of either.

    exp2 is off by 2^-22 of its result at most, a sum of 32 bits that truncates by 2^-23 for each of the three parts of a weight, and the
    quotient by less; half of that reaches the output, which is rounded to 8 bits.  Weights of 16 bits would be off by up to 2^-18."""
    x = torch.arange(1, 128, 2, device="cuda", dtype=torch.float32) * 2.0 ** -18       # (exact in bf16; 16 bits would end at 2^-17)
    rows = len(x)
    pages = -(-2 // page)
    k, v = (torch.zeros(rows * pages, 1, page, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.arange(rows * pages, dtype=torch.int32, device="cuda").view(rows, pages)
    second = (table[:, -1].long(), 0, 1 % page)
    k[second + (0,)] = -x.bfloat16()
    v[table[:, 0].long(), 0, 0] = 1.0
    v[second] = -1.0
    q = torch.zeros(rows, heads, hd, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0
    got = ops.paged_attention(q, k, v, table, torch.full((rows,), 2, dtype=torch.int32, device="cuda"), scale=1.0).double()
    want = torch.tanh(x.double() / 2)[:, None, None]
    assert bool(((got - want).abs() <= want * 2.0 ** -8 + 5 * 2.0 ** -24).all())
