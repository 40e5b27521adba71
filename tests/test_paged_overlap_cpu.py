"""Results that lie over themselves, over the queries or over what else is read."""
import pytest
import torch

from dart_pytorch_b200 import ops


def attention(device, rows=5):
    """Arguments in one stretch of memory, as the queries and values there are read."""
    g = torch.Generator().manual_seed(0)
    room = torch.randn(20000, generator=g).to(device)
    k, v = room[:7 * 2 * 4 * 8].view(7, 2, 4, 8), room[1000:1000 + 7 * 2 * 4 * 8].view(7, 2, 4, 8)
    table = torch.tensor([[0, 2, 6], [3, 1, 0], [5, -1, -1], [0, 1, 2], [4, 4, 4]], dtype=torch.int32, device=device)
    lens = torch.tensor([6, 12, 1, 9, 11], dtype=torch.int32, device=device)
    return room, room[3000:3000 + rows * 6 * 8].view(rows, 6, 8), k, v, table, lens


def out_lies_anywhere(device):
    room, *args = attention(device)
    want = ops.paged_attention(*args)
    size = want.numel()
    for first in (3000, 3000 - 48, 3000 + 48, 3001, 0, 1000 + 5, 900, 10000):      # the queries, a row off, an element off, keys, values
        room, *args = attention(device)
        out = room[first:first + size].view(want.shape)
        assert ops.paged_attention(*args, out=out) is out and torch.equal(out, want)
    room, q, *args = attention(device)
    mixed = torch.zeros(5, 9, 8, device=device)
    mixed[:, :6] = q
    ops.paged_attention(mixed[:, :6], *args, out=mixed[:, 3:])                      # heads of the same rows
    assert torch.equal(mixed[:, 3:], want) and torch.equal(mixed[:, :3], q[:, :3])


def out_over_itself_is_refused(device):
    _, *args = attention(device)
    for out in (torch.zeros(1, 6, 8, device=device).expand(5, 6, 8), torch.zeros(5, 1, 8, device=device).expand(5, 6, 8),
                torch.zeros(500, device=device).as_strided((5, 6, 8), (40, 8, 1)), torch.zeros(500, device=device).as_strided((5, 6, 8), (48, 7, 1))):
        with pytest.raises(ValueError, match="overlap"):
            ops.paged_attention(*args, out=out)
    assert torch.equal(ops.paged_attention(*args, out=torch.zeros(6, 5, 8, device=device).transpose(0, 1)), ops.paged_attention(*args))


def test_out_lies_anywhere():
    out_lies_anywhere("cpu")


def test_out_over_itself_is_refused():
    out_over_itself_is_refused("cpu")


def append_to_pages_over_themselves_is_refused(device):
    table, at = torch.tensor([[0, 2], [1, -1]], dtype=torch.int32, device=device), torch.tensor([5, 0], dtype=torch.int32, device=device)
    qkv = torch.randn(2, 8 * 8, device=device)
    zeros = lambda *shape: torch.zeros(*shape, device=device)  # noqa: E731
    k = zeros(3, 2, 4, 8)
    for bad in (zeros(3, 1, 4, 8).expand(3, 2, 4, 8), zeros(3, 2, 1, 8).expand(3, 2, 4, 8), zeros(1, 2, 4, 8).expand(3, 2, 4, 8),
                zeros(300).as_strided((3, 2, 4, 8), (64, 32, 7, 1)), zeros(300).as_strided((3, 2, 4, 8), (63, 32, 8, 1))):
        for pages in ((bad, k), (k, bad)):
            with pytest.raises(ValueError, match="overlap"):
                ops.paged_append(qkv, *pages, table, at, 4)
    with pytest.raises(ValueError, match="overlap"):
        ops.paged_append(qkv, k, k, table, at, 4)
    assert not k.any()
    want = torch.zeros(2, 3, 2, 4, 8, device=device)
    ops.paged_append(qkv, *want, table, at, 4)
    # one head at any stride, pages of a pool of keys and values, tokens and heads the other way round
    for shape, axes in (((2, 3, 2, 4, 8), (0, 1, 2, 3, 4)), ((3, 2, 2, 4, 8), (1, 0, 2, 3, 4)), ((2, 3, 4, 2, 8), (0, 1, 3, 2, 4)),
                        ((4, 3, 2, 2, 8), (3, 1, 2, 0, 4)), ((2, 2, 4, 3, 8), (0, 3, 1, 2, 4))):
        pool = torch.zeros(*shape, device=device).permute(*axes)
        ops.paged_append(qkv, *pool, table, at, 4)
        assert torch.equal(pool, want)


def test_append_to_pages_over_themselves_is_refused():
    append_to_pages_over_themselves_is_refused("cpu")
