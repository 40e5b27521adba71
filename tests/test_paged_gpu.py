"""The paged-cache kernels against 64-bit oracles and against the CPU formulas."""
import random

import pytest
import torch

import paged_oracle as oracle
from dart_pytorch_b200 import _native, ops

pytestmark = pytest.mark.gpu
NAN = float("nan")


def make(lens, heads, hkv, hd, page, dtype, seed=0, width=None, spare=2, layout="heads"):
    """Queries, pages and tables; whatever no sequence owns is NaN."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lens]
    width = max(held + [1]) if width is None else width
    pages = sum(held) + spare
    table = oracle.tables(lens, page, pages, width, seed)
    k, v = (torch.randn(pages, hkv, page, hd, generator=g).to(dtype) for _ in range(2))
    owned = torch.zeros(pages, page, dtype=torch.bool)
    for r, n in enumerate(lens):
        for j in range(n):
            owned[table[r, j // page], j % page] = True
    for t in (k, v):
        t.masked_fill_(~owned[:, None, :, None], NAN)
    q = (2 * torch.randn(len(lens), heads, hd, generator=g)).to(dtype)
    k, v = k.cuda(), v.cuda()
    if layout == "tokens":         # [pages, page, heads, hd] in memory
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    elif layout == "off":          # rows that start 16 bytes apart from nothing
        k, v = (torch.empty(pages, hkv, page, hd + 1, dtype=dtype, device="cuda").fill_(NAN)[..., 1:].copy_(t) for t in (k, v))
    return q.cuda(), k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def check(q, k, v, table, lens, scale=None, got=None):
    want, size, top = oracle.attention(q, k, v, table, lens, scale)
    got = ops.paged_attention(q, k, v, table, lens, scale) if got is None else got
    bound = oracle.attention_bound(want, size, top, q.shape[2], int(lens.max()), q.dtype)
    off = (got.double().cpu() - want).abs()
    assert got.shape == q.shape and got.dtype == q.dtype
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-30)).max())
    return got


LENS = [1, 0, 17, 63, 64, 130, 2, 300]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,hkv,hd", [(1, 1, 64), (12, 12, 64), (8, 2, 128), (7, 1, 80), (16, 2, 40), (12, 1, 96), (16, 1, 64),
                                          (24, 1, 32), (40, 2, 128), (4, 2, 256), (9, 1, 200), (6, 3, 8), (4, 4, 7), (2, 1, 1), (6, 2, 36)])
def test_attention_heads(dtype, heads, hkv, hd):
    check(*make(LENS, heads, hkv, hd, 16, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [1, 2, 3, 4, 8, 24, 32, 64, 128])
def test_attention_page_sizes(dtype, page):
    check(*make(LENS, 8, 2, 64, page, dtype, seed=page))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["tokens", "off"])
@pytest.mark.parametrize("hd", [64, 72, 128])
def test_attention_layouts(dtype, layout, hd):
    q, k, v, table, lens = make(LENS, 4, 2, hd, 16, dtype, layout=layout)
    check(q, k, v, table, lens)
    wide = torch.randn(len(LENS), 9, hd + 3, device="cuda").to(dtype)
    view = wide[:, 2:6, :hd]                                   # rows and heads at strides of their own, off 16 bytes
    view.copy_(q)
    out = torch.full((len(LENS), 6, hd + 1), 5.0, dtype=dtype, device="cuda")
    got = ops.paged_attention(view, k, v, table, lens, out=out[:, 1:5, :hd])
    check(q, k, v, table, lens, got=got)
    assert bool((out[:, 0] == 5).all()) and bool((out[:, 5] == 5).all()) and bool((out[..., hd] == 5).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,hkv,hd,page", [(1, 1, 33, 16), (8, 1, 100, 5), (12, 1, 64, 32), (40, 2, 128, 16), (9, 3, 255, 24), (6, 1, 256, 1)])
def test_attention_heads_off_16_bytes(dtype, heads, hkv, hd, page):
    check(*make(LENS + [3000], heads, hkv, hd, page, dtype, layout="off"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [[4097], [2500, 1, 0, 0, 3001], [0, 0], [1] * 50, [16 * i for i in range(40)],
                                  [random.Random(3).randint(0, 90) for _ in range(300)]])
def test_attention_lengths(dtype, lens):
    check(*make(lens, 8, 2, 64, 16, dtype, seed=len(lens)))


def test_attention_scale_and_unused_columns():
    q, k, v, table, lens = make(LENS, 4, 2, 64, 16, torch.bfloat16, width=60)
    check(q, k, v, table, lens, scale=0.5)
    check(q, k, v, table, lens, scale=0.0)
    garbage = torch.where(table < 0, torch.randint_like(table, -2**31, 2**31 - 1), table)      # nothing behind a sequence is looked at
    assert torch.equal(ops.paged_attention(q, k, v, garbage, lens), ops.paged_attention(q, k, v, table, lens))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_large_scores(dtype):
    """One key takes all the weight, or all keys the same."""
    q, k, v, table, lens = make([200, 33], 4, 2, 64, 16, dtype)
    check((q * 50).clone(), k, v, table, lens)
    k.fill_(0.25)
    check(q, k, v, table, lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_non_finite_values_and_keys(dtype):
    q, k, v, table, lens = make([40, 40, 40, 40], 2, 2, 64, 16, dtype)
    at = lambda r, j: (int(table[r, j // 16]), j % 16)  # noqa: E731
    p, o = at(0, 20)
    v[p, 0, o, 3] = float("inf")           # an infinite value that has a weight
    p, o = at(1, 39)
    k[p, 1, o, 0] = NAN                    # a score that is none
    p, o = at(2, 5)
    v[p, 1, o, 7] = NAN
    got = ops.paged_attention(q, k, v, table, lens)
    want, _, _ = oracle.attention(q, k, v, table, lens)
    assert torch.equal(got.isnan().cpu(), want.isnan()) and torch.equal(got.isinf().cpu(), want.isinf())
    fine = want.isfinite()
    assert bool(((got.double().cpu() - want).abs()[fine] <= 0.05).all())


def test_attention_repeats_to_the_bit_on_any_stream_and_in_graphs():
    a = make(LENS + [900], 8, 2, 128, 16, torch.bfloat16)
    b = make([700, 5, 0], 8, 2, 128, 16, torch.bfloat16, seed=5)
    want_a, want_b = (ops.paged_attention(*x) for x in (a, b))
    assert torch.equal(ops.paged_attention(*a), want_a)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, x in zip(streams * 4, (a, b) * 4):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(ops.paged_attention(*x))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(got, (want_a, want_b) * 4))
    graphs, outs = [], []
    for x in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_attention(*x))
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):                       # two captured graphs at once
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want_a) and torch.equal(outs[1], want_b)
    b[4].copy_(torch.tensor([3, 700, 1], dtype=torch.int32))    # lengths are read on the device at every replay
    b[3].copy_(b[3][[1, 0, 1]])
    graphs[1].replay()
    check(*b, got=outs[1])


def test_attention_bad_pages_are_passed_over_and_reported():
    q, k, v, table, lens = make([40, 40, 40], 4, 2, 64, 16, torch.bfloat16)
    want = ops.paged_attention(q, k, v, table, lens)
    for bad in (-1, k.shape[0], 2**31 - 1, -2**31):
        t = table.clone()
        t[1, 1] = bad
        got = ops.paged_attention(q, k, v, t, lens)
        with pytest.raises(_native.KernelError, match="page"):
            _native.raise_on_device_error()
        assert torch.equal(got[[0, 2]], want[[0, 2]]) and bool(got[1].isfinite().all())
    long = lens.clone()
    long[2] = 49                                                 # beyond the table
    got = ops.paged_attention(q, k, v, table, long)
    with pytest.raises(_native.KernelError):
        _native.raise_on_device_error()
    assert torch.equal(got[:2], want[:2])
    long[2] = -5                                                 # no tokens
    assert not ops.paged_attention(q, k, v, table, long)[2].any()


# ------------------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,hkv,hd,rotary", [(8, 2, 64, 64), (4, 4, 128, 128), (6, 2, 80, 32), (3, 1, 36, 36), (2, 2, 7, 6),
                                                 (4, 2, 256, 256), (4, 2, 64, 0)])
@pytest.mark.parametrize("layout", ["heads", "tokens", "off"])
def test_append(dtype, heads, hkv, hd, rotary, layout):
    g = torch.Generator().manual_seed(hd)
    page, rows, width = 4, 5, 6
    q_, k, v, _, _ = make([24] * rows, heads, hkv, hd, page, dtype, layout=layout)
    pages = k.shape[0]
    table = oracle.tables([24] * rows, page, pages, width, 3).cuda()
    places = [(r, p) for r in range(rows) for p in range(24)]
    random.Random(1).shuffle(places)
    places = places[:37] + [(2, -1), (0, -7)]
    row, pos = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in zip(*places))
    qkv = torch.randn(len(places), (heads + 2 * hkv) * hd + 3, generator=g).to(dtype).cuda()[:, 3:]
    before, k0, v0 = qkv.clone(), k.clone(), v.clone()
    q, keys = ops.paged_append(qkv, k, v, table, pos, heads, rows=row, rotary_dim=rotary, rope_base=10000.0, keys=True)
    assert torch.equal(qkv, before)
    x = qkv.reshape(len(places), -1, hd).cpu()
    want = oracle.rotate(x[:, :heads + hkv], pos.tolist(), rotary, 10000.0)
    # two products and a sum, sine and cosine to a few ulp, one rounding
    size = x[:, :heads + hkv].double().abs().amax(-1, keepdim=True)
    bound = 8 * 2.0 ** -24 * size + want.abs() * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24)
    got = torch.cat([q, keys], 1).double().cpu()
    assert bool(((got - want).abs() <= bound).all())
    for t, (r, p) in enumerate(places):
        if p >= 0:
            at = int(table[r, p // page])
            k0[at, :, p % page], v0[at, :, p % page] = keys[t], x[t, heads + hkv:].cuda()
    same = lambda a, b: torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0))  # noqa: E731
    assert same(k, k0) and same(v, v0)


def test_append_far_positions_keep_their_angle():
    """Position 131071 turns the first pair by 131071 radians: 32-bit products of the other frequencies would be off by 2^-8."""
    heads, hkv, hd = 2, 1, 64
    k, v = (torch.zeros(2, hkv, 64, hd, device="cuda") for _ in range(2))
    table = torch.zeros(1, 2048, dtype=torch.int32, device="cuda")
    qkv = torch.randn(1, 4 * hd, device="cuda")
    q = ops.paged_append(qkv, k, v, table, torch.tensor([131071], dtype=torch.int32, device="cuda"), heads)
    want = oracle.rotate(qkv.view(1, 4, hd)[:, :3], [131071], hd, 10000.0)
    assert float((q.double().cpu() - want[:, :2]).abs().max()) <= 8 * 2.0 ** -24 * float(qkv.abs().max())
    assert float((k[0, :, 63].double().cpu() - want[0, 2:]).abs().max()) <= 8 * 2.0 ** -24 * float(qkv.abs().max())


def test_append_bad_places_write_nothing():
    k, v = (torch.zeros(4, 2, 4, 64, device="cuda") for _ in range(2))
    table = torch.tensor([[0, 9], [-1, 2]], dtype=torch.int32, device="cuda")
    qkv = torch.randn(5, 8 * 64, device="cuda")
    rows = torch.tensor([0, 0, 1, 2, -1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([8, 4, 0, 0, 0], dtype=torch.int32, device="cuda")
    ops.paged_append(qkv, k, v, table, pos, 4, rows=rows)
    with pytest.raises(_native.KernelError, match="page"):
        _native.raise_on_device_error()
    assert not k.any() and not v.any()


# ------------------------------------------------------------------------------------------------------------ pages
def same_fork(table, lens, pages, page, parents, grow):
    want = ops.fork_pages(table, lens, pages, page, parents, grow)
    cuda = lambda x: x.cuda() if isinstance(x, torch.Tensor) else x  # noqa: E731
    got = ops.fork_pages(*(cuda(x) for x in (table, lens, pages, page, parents, grow)))
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    return want


@pytest.mark.parametrize("page", [1, 3, 16])
@pytest.mark.parametrize("rows,width", [(1, 3), (6, 40), (70, 33), (300, 5), (1100, 7)])
def test_fork_matches_the_cpu_formulas(rows, width, page):
    rng = random.Random(rows * 31 + page)
    pages = rows * width + 5
    t, n = torch.full((rows, width), -1, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32)
    most = max(1, width * page // 3)
    ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    t, n, _, _ = same_fork(t, n, pages, page, ints([-1] * rows), ints([rng.randint(0, most) for _ in range(rows)]))
    for step in range(6):
        if step % 3 == 2:
            parents = None if step == 2 else ints([rng.randint(-1, rows - 1) for _ in range(rows)])
            t, n, _, _ = same_fork(t, n, pages, page, parents, ints([rng.randint(0, page) for _ in range(rows)]) if width * page > 3 * most + 4 * page + 2 else 0)
        else:
            parents = ints([rng.choice([r, r - r % 4, rng.randint(-1, rows - 1)]) for r in range(rows)])
            t, n, _, _ = same_fork(t, n, pages, page, parents, 1 if int(n.max()) < width * page else 0)


def test_fork_reads_any_table_view_and_changes_row_count():
    wide = torch.full((5, 12), 77, dtype=torch.int32)
    wide[:, 2:6] = torch.tensor([[0, 4, -1, -1], [1, 9, 3, -1], [0, 4, -1, -1], [-1] * 4, [7, -1, -1, -1]])
    table, lens = wide[:, 2:6], torch.tensor([6, 9, 7, 0, 4], dtype=torch.int32)
    view = wide.cuda()[:, 2:6]
    for parents in ([1], [0, 1, 2, 3, 4, 0, 1, 2, 2, -1], [3, 3, -1]):
        p = torch.tensor(parents, dtype=torch.int32)
        want = ops.fork_pages(table, lens, 40, 4, p, 1)
        got = ops.fork_pages(view, lens.cuda(), 40, 4, p.cuda(), 1)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_fork_at_the_largest_sizes():
    rows, pages = 4096, 1 << 19
    table = torch.arange(rows * 2, dtype=torch.int32).view(rows, 2) * 64
    lens = torch.arange(rows, dtype=torch.int32) % 24
    parents = torch.arange(rows, dtype=torch.int32) // 2
    table[lens <= 16, 1] = -1
    table[lens == 0, 0] = -1
    same_fork(table, lens, pages, 16, parents, 1)


def test_fork_reports_what_only_the_device_sees():
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    t, n, src, dst = ops.fork_pages(ints([[0, 1], [1, -1]]), ints([8, 4]), 2, 4, ints([-1, 1]), ints([5, 1]))
    with pytest.raises(_native.KernelError, match="free page"):
        _native.raise_on_device_error()
    assert t.tolist() == [[0, -1], [1, -1]] and n.tolist() == [5, 5] and src.tolist() == dst.tolist() == [-1, -1]
    for table, lens, parents, grow in (([[0, 9]], [8], [0], 0), ([[0, 1]], [9], [0], 0), ([[0, 1]], [8], [1], 0), ([[0, 1]], [8], [0], 1),
                                       ([[0, -1]], [8], [0], 0)):
        t, n, src, dst = ops.fork_pages(ints(table), ints(lens), 5, 4, ints(parents), grow)
        with pytest.raises(_native.KernelError, match="page"):
            _native.raise_on_device_error()
        assert int(t.max()) < 5 and int(n) <= 8


@pytest.mark.parametrize("rows,width,pages,live", [(1, 1, 1, 1), (3, 5, 16, 9), (40, 30, 5000, 1100), (7, 200, 1400, 1400), (5, 5, 64, 0),
                                                   (4, 70, 1 << 19, 200)])
def test_compact_matches_the_cpu_formulas(rows, width, pages, live):
    rng = random.Random(pages)
    ids = rng.sample(range(pages), live)
    cells = ids + [rng.choice(ids) if ids and rng.random() < 0.3 else -1 for _ in range(rows * width - live)]
    rng.shuffle(cells)
    table = torch.tensor(cells, dtype=torch.int32).view(rows, width)
    want = ops.compact_pages(table, pages)
    got = ops.compact_pages(table.cuda(), pages)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    padded = torch.full((rows, width + 3), 5, dtype=torch.int32, device="cuda")
    padded[:, 1:width + 1] = table.cuda()
    got = ops.compact_pages(padded[:, 1:width + 1], pages)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_compact_reports_pages_outside_the_pool():
    got = ops.compact_pages(torch.tensor([[3, 8, -1]], dtype=torch.int32, device="cuda"), 4)
    with pytest.raises(_native.KernelError, match="page"):
        _native.raise_on_device_error()
    assert got[0].tolist() == [[0, -1, -1]] and int(got[3]) == 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lead,shape", [((3, 2), (4, 16, 64)), ((), (1, 3, 5)), ((2,), (1, 1, 1)), ((5,), (3, 16, 200))])
def test_copy_pages(dtype, lead, shape):
    pages = 60
    pool = torch.randn(*lead, pages, *shape, device="cuda").to(dtype)
    order = random.Random(2).sample(range(pages), pages)
    src = torch.tensor([order[i] if i % 3 else -1 for i in range(30)], dtype=torch.int32, device="cuda")
    dst = torch.tensor([order[30 + i] if i % 3 else -1 for i in range(30)], dtype=torch.int32, device="cuda")
    src[1], dst[1] = order[2], order[31]                         # one page to two places
    want = pool.clone()
    version = pool._version
    for s, d in zip(src.tolist(), dst.tolist()):
        if s >= 0:
            want[..., d, :, :, :] = want[..., s, :, :, :]
    ops.copy_pages(pool, src, dst)
    assert torch.equal(pool, want) and pool._version > version
    off = torch.empty(pool.numel() + 1, dtype=dtype, device="cuda")[1:].view(pool.shape).copy_(want)    # off 16 bytes
    ops.copy_pages(off, dst, src)
    for s, d in zip(dst.tolist(), src.tolist()):
        if s >= 0:
            want[..., d, :, :, :] = want[..., s, :, :, :]
    assert torch.equal(off, want)


def test_copy_pages_reports_pages_outside_the_pool():
    pool = torch.randn(2, 4, 1, 4, 8, device="cuda")
    want = pool.clone()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.copy_pages(pool, ints([4, 0, 1]), ints([2, 4, 3]))
    with pytest.raises(_native.KernelError, match="page"):
        _native.raise_on_device_error()
    want[:, 3] = want[:, 1]
    assert torch.equal(pool, want)


def test_pages_in_captured_graphs():
    """A captured step of fork, copy, append and attention follows what is in its inputs at every replay."""
    rows, page, pages, width, hd = 4, 4, 40, 6, 64
    pool = torch.randn(1, 2, pages, 2, page, hd, device="cuda").bfloat16()
    table = oracle.tables([9] * rows, page, pages, width, 7).cuda()
    lens = torch.full((rows,), 9, dtype=torch.int32, device="cuda")
    parents = torch.arange(rows, dtype=torch.int32, device="cuda")
    qkv = torch.randn(rows, 8 * hd, device="cuda").bfloat16()

    def step(pool, table, lens):
        t, n, src, dst = ops.fork_pages(table, lens, pages, page, parents, 1)
        ops.copy_pages(pool, src, dst)
        q = ops.paged_append(qkv, pool[0, 0], pool[0, 1], t, lens[parents.long()], 4)
        o = ops.paged_attention(q, pool[0, 0], pool[0, 1], t, n)
        table.copy_(t)
        lens.copy_(n)
        return o
    twin = [t.clone() for t in (pool, table, lens)]
    g = torch.cuda.CUDAGraph()
    warm = [t.clone() for t in twin]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(*warm)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = step(pool, table, lens)
    for i in range(6):
        parents.copy_(torch.tensor([[0, 0, 1, 3], [3, 2, 1, 0], [1, 1, 1, 1], [0, 1, 2, 3]][i % 4], dtype=torch.int32))
        qkv.normal_()
        g.replay()
        want = step(*twin)
        assert torch.equal(out, want) and torch.equal(table, twin[1]) and torch.equal(lens, twin[2])
        assert torch.equal(pool, twin[0])


def test_tensors_of_another_device_are_refused():
    q, k, v, table, lens = make([5], 2, 2, 64, 16, torch.float32)
    for args in ((q.cpu(), k, v, table, lens), (q, k, v.cpu(), table, lens), (q, k, v, table.cpu(), lens), (q, k, v, table, lens.cpu())):
        with pytest.raises(ValueError, match="device"):
            ops.paged_attention(*args)
    with pytest.raises(ValueError, match="device"):
        ops.fork_pages(table, lens.cpu(), 4, 4)
    with pytest.raises(ValueError, match="device"):
        ops.copy_pages(k, lens.cpu(), lens.cpu())


# ------------------------------------------------------------------------------------------------------------ far ends
@pytest.mark.parametrize("dtype,heads,hkv,hd", [(torch.bfloat16, 4, 1, 128), (torch.bfloat16, 16, 1, 128), (torch.float32, 8, 1, 128),
                                                (torch.float32, 1, 1, 8)])
def test_attention_of_as_many_rows_as_there_may_be(dtype, heads, hkv, hd):
    rng = random.Random(heads)
    lens = [rng.choice((0, 1, 2, 7, 33)) for _ in range(4096)]
    check(*make(lens, heads, hkv, hd, 8, dtype))


def test_pools_beyond_32_bits():
    """Pages of a pool whose elements and bytes do not fit 32 bits: 2.4e9 bf16 values."""
    pages, page, hd = 300_000, 64, 128
    pool = torch.empty(2, pages, 1, page, hd, dtype=torch.bfloat16, device="cuda")
    k, v = pool
    lens = torch.tensor([130, 64], dtype=torch.int32, device="cuda")
    table = torch.tensor([[pages - 1, 5, pages - 3], [pages - 2, -1, -1]], dtype=torch.int32, device="cuda")
    used = table[table >= 0].long()
    pool[:, used] = torch.randn(2, len(used), 1, page, hd, device="cuda").bfloat16()
    q = torch.randn(2, 4, hd, device="cuda").bfloat16()
    small = torch.tensor([[0, 1, 2], [3, -1, -1]], dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, k, v, table, lens)
    assert torch.equal(got, ops.paged_attention(q, *(t[used] for t in (k, v)), small, lens))
    ops.copy_pages(pool, table[0, :1].contiguous(), torch.tensor([pages - 7], dtype=torch.int32, device="cuda"))
    assert torch.equal(pool[:, pages - 7], pool[:, pages - 1])
    qkv = torch.randn(2, 6 * hd, device="cuda").bfloat16()
    ops.paged_append(qkv, k, v, table, torch.tensor([191, 0], dtype=torch.int32, device="cuda"), 4, rotary_dim=0)
    assert torch.equal(k[pages - 3, 0, 63], qkv[0, 4 * hd:5 * hd]) and torch.equal(v[pages - 2, 0, 0], qkv[1, 5 * hd:])
    odd = k.view(-1)[1:1 + (pages - 1) * page * hd].view(pages - 1, 1, page, hd)          # off 16 bytes: filled element by element
    odd[pages - 2] = torch.randn(1, page, hd, device="cuda").bfloat16()
    last, n = torch.full((2, 1), pages - 2, dtype=torch.int32, device="cuda"), torch.tensor([64, 9], dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, odd, odd, last, n).float()
    twin = odd[pages - 2:].clone()
    assert torch.allclose(got, ops.paged_attention(q, twin, twin, last * 0, n).float(), rtol=2.0 ** -7, atol=2.0 ** -9)


def test_results_over_the_queries_and_inference_mode():
    q, k, v, table, lens = make(LENS + [3000], 8, 2, 64, 16, torch.bfloat16)
    want = ops.paged_attention(q, k, v, table, lens)
    with torch.inference_mode():
        twin = q.clone()
        assert ops.paged_attention(twin, k, v, table, lens, out=twin) is twin and torch.equal(twin, want)
        kk, vv = torch.zeros_like(k), torch.zeros_like(v)
        ops.paged_append(torch.randn(len(lens), 12 * 64, device="cuda").bfloat16(), kk, vv, table, (lens - 1).int(), 8)
        ops.copy_pages(kk, table[2, :1].contiguous(), table[3, :1].contiguous())
        assert torch.equal(kk[table[2, 0]], kk[table[3, 0]])


def test_one_page_in_many_places():
    """A table may list a page any number of times, in one row and in others."""
    q, k, v, _, _ = make([64, 64, 64], 4, 2, 64, 16, torch.float32)
    table = torch.tensor([[1, 1, 1, 1], [1, 0, 1, 0], [0, 0, 1, 1]], dtype=torch.int32, device="cuda")
    k.normal_(), v.normal_()
    check(q, k, v, table, torch.tensor([64, 60, 33], dtype=torch.int32, device="cuda"))
