"""Tensors that are not where the first one is."""
import pytest
import torch

from dart_pytorch_b200 import ops

pytestmark = pytest.mark.gpu


def refuse(call, *args):
    for i, t in enumerate(args):
        if isinstance(t, torch.Tensor):
            with pytest.raises(ValueError, match="device"):
                call(*(a.cpu() if j == i else a for j, a in enumerate(args)))


def test_arguments_on_another_device_are_refused():
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    table, lens, k, v = ints(0, 1)[:, None].contiguous(), ints(1, 2), z(3, 2, 4, 8), z(3, 2, 4, 8)
    refuse(ops.paged_attention, z(2, 4, 8), k, v, table, lens)
    refuse(lambda *a: ops.paged_attention(*a[:-1], out=a[-1]), z(2, 4, 8), k, v, table, lens, z(2, 4, 8))
    refuse(ops.paged_append, z(2, 64), k, v, table, lens, 4)
    refuse(ops.paged_append, z(2, 64), k, v, table, lens, 4, lens * 0)
    refuse(ops.fork_pages, table, lens, 3, 4, lens * 0, lens * 0)
    refuse(ops.copy_pages, k, lens, lens + 2)
    refuse(ops.beam_step, z(6, 9), z(2, 3), z(2, 3).bool(), 1)
    assert not k.any() and not v.any()
