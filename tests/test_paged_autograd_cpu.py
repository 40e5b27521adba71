"""The paged operators have no gradients: what autograd would have to know of is refused, and it learns of what they write."""
import pytest
import torch

from dart_pytorch_b200 import ops


def attention(device):
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(4, 2, 4, 8, generator=g).to(device) for _ in range(2))
    table, lens = (torch.tensor(x, dtype=torch.int32, device=device) for x in ([[0, 2], [3, 1]], [6, 8]))
    return torch.randn(2, 4, 8, generator=g).to(device), k, v, table, lens


def out_is_known_to_autograd(device):
    args = attention(device)
    y, w = torch.randn(2, 4, 8, device=device), torch.randn(2, 4, 8, device=device, requires_grad=True)
    z = (w * y).sum()                                    # saves y
    version = y._version
    ops.paged_attention(*args, out=y)
    assert y._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    before = w.detach().clone()
    with pytest.raises(ValueError, match="gradients"):
        ops.paged_attention(*args, out=w)
    assert torch.equal(w.detach(), before)
    with torch.no_grad():
        assert ops.paged_attention(*args, out=w) is w and torch.equal(w.detach(), y)


def test_out_is_known_to_autograd():
    out_is_known_to_autograd("cpu")
