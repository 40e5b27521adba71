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


def forward_mode_is_refused(device):
    """A tangent would be dropped by a kernel, and a transform would hand it a wrapper."""
    from torch.autograd import forward_ad as fw
    q, k, v, table, lens = attention(device)
    one = torch.tensor([1], dtype=torch.int32, device=device)
    qkv, logits, scores = torch.randn(2, 64, device=device), torch.randn(6, 9, device=device), torch.zeros(2, 3, device=device)
    calls = [(lambda x: ops.paged_attention(x, k, v, table, lens), q), (lambda x: ops.paged_attention(q, x, v, table, lens), k),
             (lambda x: ops.paged_attention(q, k, x, table, lens), v), (lambda x: ops.paged_attention(q, k, v, table, lens, out=x), q),
             (lambda x: ops.paged_append(x, k, v, table, lens - 1, 4), qkv), (lambda x: ops.paged_append(qkv, x, v, table, lens - 1, 4), k),
             (lambda x: ops.paged_append(qkv, k, x, table, lens - 1, 4), v), (lambda x: ops.copy_pages(x, one, one + 1), k),
             (lambda x: ops.beam_step(x, scores), logits), (lambda x: ops.beam_step(logits, x), scores)]
    for call, x in calls:
        x = x.clone()
        with fw.dual_level():
            plain = call(x)                                     # no tangent: as ever
            with pytest.raises(ValueError, match="tangent"):
                call(fw.make_dual(x, torch.ones_like(x)))
        again = call(x)
        if plain is not None:
            for a, b in zip(*((y,) if isinstance(y, torch.Tensor) else y for y in (plain, again))):
                assert torch.equal(a, b)
        for transform in (torch.func.vmap, torch.func.grad):
            with pytest.raises(ValueError, match="transforms|gradients"):
                transform(call)(x[None] if transform is torch.func.vmap else x)
        with pytest.raises(ValueError, match="transforms|gradients"):
            torch.func.jvp(call, (x,), (x,))


def test_forward_mode_is_refused():
    forward_mode_is_refused("cpu")
