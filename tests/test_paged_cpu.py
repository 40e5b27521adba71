"""The operators of the paged cache on CPU tensors, their refusals, and what must hold of tables after any of them."""
import random

import pytest
import torch

import paged_oracle as oracle
from dart_pytorch_b200 import ops


def _pages(pages=9, heads=2, page=4, hd=8, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(pages, heads, page, hd, generator=g).to(dtype) for _ in range(2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_is_softmax_over_the_pages(dtype):
    k, v = _pages(dtype=dtype)
    lens = torch.tensor([0, 1, 9, 12], dtype=torch.int32)
    table = oracle.tables(lens.tolist(), 4, 9, 4, 1)
    q = torch.randn(4, 6, 8).to(dtype)
    want, size, top = oracle.attention(q, k, v, table, lens)
    got = ops.paged_attention(q, k, v, table, lens)
    assert got.dtype == dtype and bool(((got.double() - want).abs() <= oracle.attention_bound(want, size, top, 8, 12, dtype)).all())
    assert not got[0].any()
    out = torch.empty_like(q)
    assert ops.paged_attention(q, k, v, table, lens, out=out) is out and torch.equal(out, got)


def test_attention_ignores_what_lies_behind_a_sequence():
    k, v = _pages()
    lens = torch.tensor([5], dtype=torch.int32)
    table = torch.tensor([[3, 7, -1]], dtype=torch.int32)
    q = torch.randn(1, 2, 8)
    want = ops.paged_attention(q, k, v, table, lens)
    for t in (k, v):
        t[7, :, 1:] = float("nan")
        t[[0, 1, 2]] = float("inf")
    assert torch.equal(ops.paged_attention(q, k, v, table, lens), want)


def test_append_rotates_and_places():
    hd, heads, hkv, page = 8, 4, 2, 4
    for rotary in (0, 4, 8):
        k, v = (torch.full((9, hkv, page, hd), 7.0) for _ in range(2))
        table = torch.tensor([[3, 5], [8, -1]], dtype=torch.int32)
        qkv = torch.randn(4, (heads + 2 * hkv) * hd)
        pos, rows = torch.tensor([6, -1, 0, 3], dtype=torch.int32), torch.tensor([0, 0, 1, 1], dtype=torch.int32)
        q, keys = ops.paged_append(qkv, k, v, table, pos, heads, rows=rows, rotary_dim=rotary, rope_base=500.0, keys=True)
        x = qkv.view(4, -1, hd)
        want = oracle.rotate(x[:, :heads + hkv], pos.tolist(), rotary, 500.0) if rotary else x[:, :heads + hkv].double()
        assert torch.allclose(q.double(), want[:, :heads], atol=1e-6) and torch.allclose(keys.double(), want[:, heads:], atol=1e-6)
        for t, (page_at, off) in {0: (5, 2), 2: (8, 0), 3: (8, 3)}.items():
            assert torch.equal(k[page_at, :, off], keys[t]) and torch.equal(v[page_at, :, off], x[t, heads + hkv:])
        assert int((k != 7.0).any(-1).any(1).sum()) == 3 and int((v != 7.0).any(-1).any(1).sum()) == 3


class Story:
    """Sequences as lists of tokens beside a cache whose pages hold them: every operation is done on both."""

    def __init__(self, rows, width, pages, page, seed):
        self.rng = random.Random(seed)
        self.page, self.pages, self.width = page, pages, width
        self.pool = torch.zeros(1, 1, pages, 1, page, 1)
        self.table = torch.full((rows, width), -1, dtype=torch.int32)
        self.lens = torch.zeros(rows, dtype=torch.int32)
        self.text = [[] for _ in range(rows)]
        self.next = 1.0

    def fork(self, parents, grow):
        old_lens = self.lens.tolist()
        par = None if parents is None else torch.tensor(parents, dtype=torch.int32)
        more = torch.tensor(grow, dtype=torch.int32) if isinstance(grow, list) else grow
        self.table, self.lens, src, dst = ops.fork_pages(self.table, self.lens, self.pages, self.page, par, more)
        ops.copy_pages(self.pool, src, dst)
        who = list(range(len(old_lens))) if parents is None else parents
        self.text = [list(self.text[p]) if p >= 0 else [] for p in who]
        more = grow if isinstance(grow, list) else [grow if p >= 0 and old_lens[p] > 0 else 0 for p in who]
        for r, n in enumerate(more):
            for _ in range(n):
                at = len(self.text[r])
                assert self.lens[r] > at
                self.pool[0, 0, self.table[r, at // self.page], 0, at % self.page, 0] = self.next
                self.text[r].append(self.next)
                self.next += 1

    def compact(self):
        self.table, src, dst, live = ops.compact_pages(self.table, self.pages)
        ops.copy_pages(self.pool, src, dst)
        held = {p for p in self.table.flatten().tolist() if p >= 0}
        assert held == set(range(int(live)))

    def check(self):
        for r, text in enumerate(self.text):
            assert int(self.lens[r]) == len(text)
            held = -(-len(text) // self.page)
            row = self.table[r].tolist()
            assert row[held:] == [-1] * (self.width - held) and all(0 <= p < self.pages for p in row[:held])
            assert [float(self.pool[0, 0, row[j // self.page], 0, j % self.page, 0]) for j in range(len(text))] == text


@pytest.mark.parametrize("page", [1, 3, 4, 16])
@pytest.mark.parametrize("seed", range(6))
def test_pages_hold_every_sequence_through_forks_frees_and_compaction(page, seed):
    s = Story(6, 40 // page + 8, 6 * (40 // page + 8), page, seed)
    s.fork([-1] * 6, [s.rng.randint(0, 9) for _ in range(6)])
    s.check()
    for _ in range(12):
        what = s.rng.random()
        if what < 0.2:
            s.compact()
        elif what < 0.4:
            s.fork(None, [s.rng.randint(0, 2) for _ in range(6)])
        elif what < 0.5:
            s.fork([s.rng.randint(-1, 5) for _ in range(6)], 0)
        else:
            s.fork([s.rng.choice([r, r, s.rng.randint(-1, 5)]) for r in range(6)], 1)
        s.check()


def test_fork_takes_the_lowest_free_pages_in_the_order_of_the_rows():
    table = torch.tensor([[5, 2], [0, -1]], dtype=torch.int32)
    lens = torch.tensor([6, 4], dtype=torch.int32)
    new, n, src, dst = ops.fork_pages(table, lens, 8, 4, torch.tensor([0, 0, 1, -1], dtype=torch.int32), 1)
    assert new.tolist() == [[5, 2], [5, 1], [0, 3], [-1, -1]] and n.tolist() == [7, 7, 5, 0]
    assert src.tolist() == [-1, 2, -1, -1] and dst.tolist() == [-1, 1, -1, -1]
    # a row that does not grow still reads the shared page, so the one that does takes the copy
    new, n, src, dst = ops.fork_pages(table, lens, 8, 4, torch.tensor([0, 0], dtype=torch.int32),
                                      torch.tensor([1, 0], dtype=torch.int32))
    assert new.tolist() == [[5, 0], [5, 2]] and src.tolist() == [2, -1] and dst.tolist() == [0, -1]
    assert table.tolist() == [[5, 2], [0, -1]]


def test_a_full_pool_and_bad_tables_raise():
    one = torch.tensor([[0, 1]], dtype=torch.int32)
    four = torch.tensor([4], dtype=torch.int32)
    with pytest.raises(ValueError, match="no free one"):
        ops.fork_pages(one[:, :2], torch.tensor([8], dtype=torch.int32), 2, 4, torch.tensor([0, -1], dtype=torch.int32),
                       torch.tensor([0, 1], dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.fork_pages(one, four, 1, 2)                                       # lists page 1 of a pool of one
    with pytest.raises(ValueError):
        ops.fork_pages(one, four, 2, 2, None, 1)                              # grows beyond the table
    with pytest.raises(ValueError):
        ops.fork_pages(one, four, 2, 2, torch.tensor([1], dtype=torch.int32))  # no such parent
    with pytest.raises(ValueError):
        ops.compact_pages(one, 1)
    k, v = _pages()
    q = torch.randn(1, 2, 8)
    for table, n in (([[9]], 1), ([[-1]], 1), ([[0]], 5)):
        with pytest.raises(ValueError):
            ops.paged_attention(q, k, v, torch.tensor(table, dtype=torch.int32), torch.tensor([n], dtype=torch.int32))
    qkv = torch.randn(1, 48)
    for table, p in (([[9]], 0), ([[-1]], 0), ([[0]], 4)):
        with pytest.raises(ValueError):
            ops.paged_append(qkv, k, v, torch.tensor(table, dtype=torch.int32), torch.tensor([p], dtype=torch.int32), 2)


def test_refusals_of_arguments():
    k, v = _pages()
    table, lens, q = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.randn(2, 4, 8)
    bad = [(ValueError, dict(q=q[:1])), (ValueError, dict(q=q[:, :3])), (ValueError, dict(q=torch.randn(2, 4, 16))),
           (TypeError, dict(q=q.bfloat16())), (TypeError, dict(k=k.half(), v=v.half(), q=q.half())), (TypeError, dict(v=v.bfloat16())),
           (ValueError, dict(v=v[:8])), (TypeError, dict(table=table.long())), (TypeError, dict(lens=lens.long())),
           (ValueError, dict(lens=lens[:1])), (ValueError, dict(table=table[0])), (ValueError, dict(k=k.transpose(2, 3), v=v.transpose(2, 3))),
           (ValueError, dict(q=q.clone().requires_grad_())), (ValueError, dict(out=torch.empty(2, 4, 9))),
           (ValueError, dict(table=torch.zeros(3, 2, dtype=torch.int32).t()))]
    for error, change in bad:
        with pytest.raises(error):
            ops.paged_attention(**{**dict(q=q, k_pages=change.pop("k", k), v_pages=change.pop("v", v), table=table, lens=lens), **change})
    wide = torch.zeros(3, 1, 2, 264)
    with pytest.raises(ValueError, match="256"):
        ops.paged_attention(torch.zeros(2, 1, 264), wide, wide, table, lens)
    qkv = torch.randn(2, 64)
    for error, change in [(ValueError, dict(heads=3)), (ValueError, dict(rotary_dim=3)), (ValueError, dict(rotary_dim=10)),
                          (ValueError, dict(rope_base=0.0)), (TypeError, dict(qkv=qkv.bfloat16())), (ValueError, dict(positions=lens[:1])),
                          (TypeError, dict(positions=lens.long())), (ValueError, dict(rows=lens[:1])),
                          (ValueError, dict(qkv=qkv[:1], positions=lens[:1])), (ValueError, dict(qkv=qkv.clone().requires_grad_()))]:
        with pytest.raises(error):
            ops.paged_append(**{**dict(qkv=qkv, k_pages=k, v_pages=v, table=table, positions=lens, heads=4), **change})
    for error, change in [(ValueError, dict(grow=-1)), (TypeError, dict(parents=lens.long())), (ValueError, dict(page=0)),
                          (ValueError, dict(pages=(1 << 19) + 1)), (ValueError, dict(grow=lens[:1])), (TypeError, dict(grow=lens.long())),
                          (ValueError, dict(lens=lens[:1])), (ValueError, dict(table=torch.zeros(4097, 1, dtype=torch.int32),
                                                                              lens=torch.zeros(4097, dtype=torch.int32)))]:
        with pytest.raises(error):
            ops.fork_pages(**{**dict(table=table, lens=lens, pages=9, page=4), **change})
    with pytest.raises(ValueError):
        ops.compact_pages(table, -1)
    two = torch.zeros(2, dtype=torch.int32)
    for error, args in [(ValueError, (k[0], two, two)), (ValueError, (k.transpose(0, 1), two, two)), (TypeError, (k.half(), two, two)),
                        (ValueError, (k, two, two[:1])), (TypeError, (k, two.long(), two)), (ValueError, (k, table, table)),
                        (ValueError, (k, two + 9, two)), (ValueError, (k.clone().requires_grad_(), two, two))]:
        with pytest.raises(error):
            ops.copy_pages(*args)


def test_empty_calls():
    k, v = _pages()
    none = torch.zeros(0, 3, dtype=torch.int32)
    zero = torch.zeros(0, dtype=torch.int32)
    assert ops.paged_attention(torch.zeros(0, 4, 8), k, v, none, zero).shape == (0, 4, 8)
    assert ops.paged_append(torch.zeros(0, 64), k, v, none, zero, 4).shape == (0, 4, 8)
    t, n, src, dst = ops.fork_pages(none, zero, 9, 4)
    assert t.shape == (0, 3) and n.numel() == src.numel() == dst.numel() == 0
    t, src, dst, live = ops.compact_pages(none, 9)
    assert t.shape == (0, 3) and src.tolist() == dst.tolist() == [-1] * 4 and int(live) == 0
    ops.copy_pages(k, zero, zero)
