"""Each operator states what it takes twice: in full, with a reason for each refusal, and in short, for calls that have nothing wrong with
them.  What the short form lets through, the full one must: here on thousands of combinations of good and bad arguments."""
import itertools
import random

import pytest
import torch

from dart_pytorch_b200.ops import beam, paged


@pytest.fixture(autouse=True)
def cpu_is_the_device(monkeypatch):
    for module in (paged, beam):
        monkeypatch.setattr(module, "_current_device", lambda: -1)         # (what a CPU tensor says of its device)


def together(off, check, choices, ordinary, count=6000, more=()):
    """``choices``: for every argument its values, the ordinary ones (as many as ``ordinary`` says) first."""
    rng = random.Random(1)
    taken = refused = 0
    every = list(more)                                                     # what takes several values to see
    every += itertools.product(*([c[0]] for c in choices))
    for i, c in enumerate(choices):                                        # each value on its own among ordinary ones
        every += [tuple(x if j == i else d[0] for j, d in enumerate(choices)) for x in c]
    for i, j in itertools.combinations(range(len(choices)), 2):            # and pairs of them
        every += [tuple(x if n == i else y if n == j else d[0] for n, d in enumerate(choices)) for x in choices[i] for y in choices[j]]
    while len(every) < count:
        every.append(tuple(rng.choice(c) for c in choices))
    for args in every:
        try:
            check(*args)
        except (ValueError, TypeError):
            assert off(*args), args
            refused += 1
        else:
            taken += not off(*args)
    assert refused > 100 and taken >= ordinary
    for args in itertools.product(*(c[:1] for c in choices)):
        assert not off(*args)


ints = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
wants = lambda t: t.clone().requires_grad_()  # noqa: E731
LENS = [ints(3), ints(3)[:, None].expand(3, 1)[:, 0], ints(6)[::2], ints(1).expand(3), ints(3).long(), ints(3, 1), ints(2), ints(4), ints(0), ints(())]
TABLES = [ints(3, 4), ints(3, 9)[:, 2:6], ints(1, 4).expand(3, 4), ints(4, 3).t(), ints(3, 8)[:, ::2], ints(3, 1).expand(3, 4), ints(3, 1), ints(3, 0), ints(2, 4),
          ints(3), ints(3, 4, 1), ints(3, 4).long(), ints(4097, 1), ints(1, 3).t(), ints(2, 3).t()]


def pages(dtype=torch.float32):
    z = lambda *s: torch.zeros(*s, dtype=dtype)  # noqa: E731
    return [z(5, 2, 4, 8), z(2, 5, 2, 4, 8)[1], z(5, 4, 2, 8).transpose(1, 2), z(5, 2, 4, 9)[..., 1:], z(4, 2, 5, 8).permute(2, 1, 0, 3), z(5, 1, 4, 8),
            z(5, 2, 1, 8), z(0, 2, 4, 8), z(5, 1, 4, 8).expand(5, 2, 4, 8), z(1, 2, 4, 8).expand(5, 2, 4, 8), z(5, 2, 8, 4).transpose(2, 3),
            z(5, 2, 4, 8, 1), z(2, 4, 8), z(5, 2, 4, 16), z(5, 2, 4, 16)[..., ::2], z(5, 0, 4, 8), z(5, 2, 0, 8), z(5, 2, 4, 0), z(5, 3, 4, 8), z(1, 2, 1, 264),
            wants(z(5, 2, 4, 8)), z(5, 2, 4, 8).half(), z(5, 2, 4, 8).double(), z(5, 2, 4, 8).to(torch.bfloat16 if dtype == torch.float32 else torch.float32),
            z((1 << 19) + 1, 2, 1, 8).expand((1 << 19) + 1, 2, 4, 8), z(5, 2, 4, 1), z(5, 2, 4, 2)[..., ::2]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention(dtype):
    z = lambda *s: torch.zeros(*s, dtype=dtype)  # noqa: E731
    q = [z(3, 4, 8), z(3, 9, 8)[:, 2:6], z(1, 4, 8).expand(3, 4, 8), z(3, 4, 16)[..., ::2], z(3, 3, 8), z(2, 4, 8), z(3, 0, 8), z(3, 4, 8, 1), z(3, 32), z(3, 4, 16),
         z(3, 4, 1), z(3, 4, 2)[..., ::2], wants(z(3, 4, 8)), z(3, 4, 8).half(), z(3, 4, 8).double(), z(3, 2, 264), z(0, 4, 8), z(3, 8, 4).transpose(1, 2)]
    together(lambda *a: paged._attention_sizes(*a, -1) is None, lambda *a: paged._check_attention(*a, None), [q, pages(dtype), pages(dtype), TABLES, LENS], 100,
             more=[(z(n, 4, 8), *pages(dtype)[:2], ints(n, 1), ints(n)) for n in (4096, 4097)])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append(dtype):
    z = lambda *s: torch.zeros(*s, dtype=dtype)  # noqa: E731
    qkv = [z(3, 64), z(3, 70)[:, 6:], z(1, 64).expand(3, 64), z(64, 3).t(), z(3, 128)[:, ::2], z(3, 63), z(3, 48), z(2, 64), z(0, 64), z(3, 64, 1), z(64),
           wants(z(3, 64)), z(3, 64).half(), z(3, 64).double(), z(4, 64)]
    rows = [None] + LENS
    one = pages(dtype)
    other = one[:1] + pages(dtype)                             # the first of these: the same tensor for both
    together(lambda *a: paged._append_sizes(*a, -1) is None, paged._check_append,
             [qkv, one, other[1:] + other[:1], TABLES, LENS, [4, 2, 0, -4, 3, 6], rows, [8, 0, 4, 2, 3, 10, -2], [1e4, 0.0, -1.0, float("nan"), 1.0]], 100, 9000,
             more=[(z(n, 64), *pages(dtype)[:2], ints(n, 1), ints(n), 4, None, 8, 1e4) for n in (4096, 4097)])


def test_fork():
    grow = [0, 1, -1, 1 << 31, (1 << 31) - 1] + LENS
    off = lambda t, n, pages, page, parents, g: paged._fork_is_off(t, n, pages, page, parents, g, isinstance(g, torch.Tensor), -1)  # noqa: E731
    check = lambda t, n, pages, page, parents, g: paged._check_fork(t, n, pages, page, parents, g, isinstance(g, torch.Tensor))  # noqa: E731
    together(off, check, [TABLES, LENS, [9, 0, 1 << 19, (1 << 19) + 1, -1], [4, 1, 0, -4], [None, ints(4097)] + LENS, grow], 100,
             more=[(ints(n, 1), ints(n), 9, 4, None, 0) for n in (4096, 4097)])


def test_compact():
    together(lambda *a: paged._compact_is_off(*a, -1), paged._check_compact, [TABLES, [9, 0, 1 << 19, (1 << 19) + 1, -1]], 10, 1000)


def test_copy():
    z = torch.zeros
    pool = [z(2, 5, 2, 4, 8), z(5, 2, 4, 8), z(5, 2, 4, 8, dtype=torch.bfloat16), z(2, 4, 8), z(2, 5, 2, 4, 9)[..., 1:], z(5, 2, 2, 4, 8).transpose(0, 1),
            z(1, 5, 2, 4, 8).expand(2, 5, 2, 4, 8), wants(z(5, 2, 4, 8)), z(5, 2, 4, 8).half(), z(5, 2, 4, 8).double(), z(0, 2, 4, 8), z(5, 2, 4, 8).int()]
    together(lambda *a: paged._copy_is_off(*a, -1), paged._check_copy, [pool, LENS + TABLES, LENS + TABLES], 10)


def test_beam():
    z = torch.zeros
    scores = [z(2, 3), z(3, 2).t(), z(2, 1).expand(2, 3), z(2, 6)[:, ::2], z(6), z(2, 3, 1), z(2, 3).double(), z(2, 3).bfloat16(), z(2, 0), z(0, 3), z(1, 6), z(1, 33),
              wants(z(2, 3)), z(3, 2)]
    logits = [z(6, 9), z(6, 9).bfloat16(), z(6, 12)[:, 1:10], z(1, 9).expand(6, 9), z(9, 6).t(), z(6, 18)[:, ::2], z(5, 9), z(6, 0), z(6), z(6, 9, 1), z(6, 9).half(),
              z(6, 9).double(), wants(z(6, 9)), z(33, 9), z(6, 1), z(0, 9), z(6, 1).expand(6, (1 << 30) + 1)]
    done = [None, z(2, 3).bool(), z(3, 2).bool().t(), z(2, 3), z(2, 3).int(), z(1, 3).bool(), z(6).bool(), z(1, 3).bool().expand(2, 3), z(3, 2).bool()]

    def off(x, s, d, eos):
        return x.dim() != 2 or s.dim() != 2 or beam._beam_is_off(x, s, d, eos, -1)
    together(off, beam._check_beam, [logits, scores, done, [None, 0, 8, 9, -1]], 20,
             more=[(z(1, 1).expand(n, 1), z(n, 1), None, None) for n in (1 << 20, (1 << 20) + 1)] + [(z(b, 9), z(1, b), None, 0) for b in (32, 33)])
