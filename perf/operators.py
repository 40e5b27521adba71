"""Performance cases of the paged serving operators: a key / value cache in pages and beam search over it.

Five operators, as a decoding loop uses them one after the other:

* ``attention``: one new token of every sequence attends over its pages (``ops.paged_attention``);
* ``append``: the step's keys and values go to their pages, with the rotary embedding (``ops.paged_append``);
* ``fork``: every beam becomes a copy of its parent, with room for a token (``ops.fork_pages`` and ``ops.copy_pages``);
* ``compact``: the live pages move to the front of the pool (``ops.compact_pages`` and ``ops.copy_pages``);
* ``beam``: the best continuations over beams and vocabulary (``ops.beam_step``).

``own`` chooses between these calls and their plain form in elementary torch operations.  Sequence lengths, beams' parents and
what is live in a pool follow from the case alone, values and page numbers from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp32": 4}
ROPE_BASE = 500000.0


def _attention(name, dtype, rows, heads, kv_heads, head_dim, page, shortest, longest):
    c = dict(op="attention", dtype=dtype, rows=rows, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
             shortest=shortest, longest=longest)
    return {"name": name, **c} if name else c


def _append(name, dtype, rows, tokens, heads, kv_heads, head_dim, page, past):
    """``tokens`` of each row at once: 1 while decoding (behind up to ``past`` tokens), the padded length of a prompt batch."""
    c = dict(op="append", dtype=dtype, rows=rows, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
             page=page, past=past)
    return {"name": name, **c} if name else c


def _fork(name, dtype, items, beams, prompt, new, layers, kv_heads, head_dim, page):
    c = dict(op="fork", dtype=dtype, items=items, beams=beams, prompt=prompt, new=new, layers=layers, kv_heads=kv_heads,
             head_dim=head_dim, page=page)
    return {"name": name, **c} if name else c


def _compact(name, dtype, pages, live, rows, layers, kv_heads, head_dim, page):
    """``live`` per cent of the pool's pages are still held, by ``rows`` sequences."""
    c = dict(op="compact", dtype=dtype, pages=pages, live=live, rows=rows, layers=layers, kv_heads=kv_heads,
             head_dim=head_dim, page=page)
    return {"name": name, **c} if name else c


def _beam(name, dtype, items, beams, vocab, finished):
    c = dict(op="beam", dtype=dtype, items=items, beams=beams, vocab=vocab, finished=finished)
    return {"name": name, **c} if name else c


def listed():
    return [
        # one user of the GPT-2 124M shape, just after a short prompt: the smallest call, where only latency counts
        _attention("attn_gpt2_one_user", "bf16", 1, 12, 12, 64, 16, 65, 65),
        # 32 users of a Llama-3-8B-shaped model (32 heads on 8 key heads of 128) at contexts of all lengths up to 4096
        _attention("attn_llama_32_users", "bf16", 32, 32, 8, 128, 16, 1, 4096),
        # four long documents close to that shape's context of 131072 tokens, in larger pages
        _attention("attn_llama_long", "bf16", 4, 32, 8, 128, 64, 65000, 131072),
        # the default dtype, heads of 80 features and pages of 8: odd sizes on every axis
        _attention("attn_fp32_odd", "fp32", 13, 10, 5, 80, 8, 0, 1531),
        # one decoding step of the 32 users: a launch-bound append
        _append("append_llama_decode", "bf16", 32, 1, 32, 8, 128, 16, 4096),
        # eight prompts of different lengths, padded to the longest, in fp32
        _append("append_prompts_fp32", "fp32", 8, 777, 16, 4, 64, 16, 0),
        # four beams of one GPT-2-shaped request
        _fork("fork_gpt2_4_beams", "bf16", 1, 4, 201, 9, 12, 12, 64, 16),
        # 32 requests of eight beams on a Llama-shaped model of six layers, prompts up to 1531 tokens
        _fork("fork_llama_256_beams", "bf16", 32, 8, 1531, 41, 6, 4, 128, 16),
        # a pool that was 40 % live when its requests ended is packed, six layers of 4 x 128 features
        _compact("compact_llama_pool", "bf16", 6144, 40, 48, 6, 4, 128, 16),
        # the first kind of beam search: a single request over the GPT-2 vocabulary, in the default dtype
        _beam("beam_gpt2_4", "fp32", 1, 4, 50257, 0),
        # a batch of requests over a Llama-3 vocabulary
        _beam("beam_llama_256", "bf16", 32, 8, 128256, 20),
        # a character model's beams, an odd vocabulary and finished beams among them
        _beam("beam_char_odd", "fp32", 7, 5, 321, 30),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "append", "fork", "compact", "beam"))
    dtype = rng.choice(("bf16", "fp32"))
    kv = rng.choice((1, 2, 3, 4, 5, 8, 12))
    hd = rng.choice((32, 40, 64, 64, 80, 96, 128, 128))
    page = rng.choice((4, 8, 16, 16, 32, 64))
    if op == "attention":
        rows = _spread(rng, 1, 96)
        group = rng.choice((1, 1, 2, 3, 4, 7, 8, 12))
        most = 1.2e9 / (rows * kv * hd * 2 * SIZES[dtype])       # bytes of keys and values, as the largest listed case has
        longest = _spread(rng, 1, max(2, min(100000, most)))
        return _attention(None, dtype, rows, kv * group, kv, hd, page, rng.choice((0, 1, longest)), longest)
    if op == "append":
        group = rng.choice((1, 2, 4))
        if rng.random() < 0.5:
            return _append(None, dtype, _spread(rng, 1, 256), 1, kv * group, kv, hd, page, _spread(rng, 1, 20000))
        return _append(None, dtype, _spread(rng, 1, 16), _spread(rng, 2, 1500), kv * group, kv, hd, page, 0)
    if op == "fork":
        return _fork(None, dtype, _spread(rng, 1, 32), rng.randint(1, 12), _spread(rng, 1, 1500), rng.randint(1, 90),
                     rng.randint(1, 12), min(kv, 8), min(hd, 64), page)
    if op == "compact":
        return _compact(None, dtype, _spread(rng, 16, 6000), rng.randint(1, 99), rng.randint(1, 64), rng.randint(1, 6),
                        min(kv, 4), min(hd, 64), min(page, 16))
    return _beam(None, dtype, _spread(rng, 1, 32), rng.randint(1, 16), _spread(rng, 33, 60000), rng.choice((0, 10, 50)))


# ------------------------------------------------------------------------------- what follows from the case alone
def _fixed(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case):
    """Keys of every sequence, from the shortest to the longest, in an order of their own."""
    lo, hi, n = case["shortest"], case["longest"], case["rows"]
    got = [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]
    _fixed(case).shuffle(got)
    return got


def _append_plan(case):
    """(row, position) of every token of the padded batch; position -1: padding."""
    rng = _fixed(case)
    if case["tokens"] == 1:
        return [(r, rng.randrange(case["past"])) for r in range(case["rows"])]
    n = [case["tokens"]] + [rng.randint(1, case["tokens"]) for _ in range(case["rows"] - 1)]
    return [(r, t if t < n[r] else -1) for r in range(case["rows"]) for t in range(case["tokens"])]


def _fork_plan(case):
    """(tables, lengths, parents, pages): every request's beams share the pages that its prompt filled; the others are a beam's own."""
    rng, ps, w = _fixed(case), case["page"], case["beams"]
    tables, lengths, parents, fresh = [], [], [], 0
    for item in range(case["items"]):
        prompt = case["prompt"] if item == 0 else rng.randint(max(1, case["prompt"] // 3), case["prompt"])
        full, held = prompt // ps, -(-(prompt + case["new"]) // ps)
        shared = list(range(fresh, fresh + full))
        fresh += full
        for _ in range(w):
            tables.append(shared + list(range(fresh, fresh + held - full)))
            fresh += held - full
            lengths.append(prompt + case["new"])
            parents.append(item * w + min(rng.randrange(w), rng.randrange(w)))     # better beams have more children
    return tables, lengths, parents, fresh + 2 * len(tables)


def _fork_copies(case):
    _, lengths, parents, _ = _fork_plan(case)
    part = [p for p in parents if lengths[p] % case["page"]]
    return len(part) - len(set(part))


def _compact_plan(case):
    """Tables of the sequences that still hold pages; page numbers are dealt out of a shuffled pool."""
    rng = _fixed(case)
    held = max(1, case["pages"] * case["live"] // 100)
    rows = min(case["rows"], held)
    cuts = sorted(rng.sample(range(1, held), rows - 1)) if rows > 1 else []
    sizes = [b - a for a, b in zip([0] + cuts, cuts + [held])]
    ids = rng.sample(range(case["pages"]), held)
    tables, at = [], 0
    for n in sizes:
        tables.append(ids[at:at + n])
        at += n
    return tables


def _padded(tables, width, device):
    return torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32, device=device)


# ------------------------------------------------------------------------------- inputs
def _pool(shape, dtype, gen):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype) if math.prod(shape) < 1 << 26 else \
        torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=gen)


def _renumber(table, pages, gen):
    """The same tables over page numbers in another order: a pool that has been in use deals them out anyhow."""
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    return torch.where(table >= 0, order[table.clamp(min=0).long()], table)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, op = DTYPES[case["dtype"]], case["op"]
    s = {"op": op}
    if op == "attention":
        lens, ps, hkv, hd = _lengths(case), case["page"], case["kv_heads"], case["head_dim"]
        held = [-(-n // ps) for n in lens]
        pages, width = sum(held) + 1, max(1, max(held))
        firsts = [sum(held[:r]) for r in range(len(held))]
        table = _padded([list(range(f, f + n)) for f, n in zip(firsts, held)], width, "cuda")
        s["table"] = _renumber(table, pages, gen)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["k"], s["v"] = (_pool((pages, hkv, ps, hd), dtype, gen) for _ in range(2))
        s["q"] = 2.0 * _pool((case["rows"], case["heads"], hd), dtype, gen)
    elif op == "append":
        plan, ps, hkv, hd = _append_plan(case), case["page"], case["kv_heads"], case["head_dim"]
        width = max(p for _, p in plan) // ps + 1
        pages = case["rows"] * width + 1
        table = torch.arange(case["rows"] * width, dtype=torch.int32, device="cuda").view(case["rows"], width)
        s["table"] = _renumber(table, pages, gen)
        s["rows"] = torch.tensor([r for r, _ in plan], dtype=torch.int32, device="cuda")
        s["positions"] = torch.tensor([p for _, p in plan], dtype=torch.int32, device="cuda")
        s["k"], s["v"] = (torch.zeros(pages, hkv, ps, hd, dtype=dtype, device="cuda") for _ in range(2))
        s["qkv"] = _pool((len(plan), (case["heads"] + 2 * hkv) * hd), dtype, gen)
        s["heads"], s["page"] = case["heads"], ps
    elif op == "fork":
        tables, lens, parents, pages = _fork_plan(case)
        width = max(len(t) for t in tables) + 2
        s["table"] = _renumber(_padded(tables, width, "cuda"), pages, gen)
        s["lens"], s["parents"] = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lens, parents))
        s["pool"] = _pool((case["layers"], 2, pages, case["kv_heads"], case["page"], case["head_dim"]), dtype, gen)
        s["page"] = case["page"]
    elif op == "compact":
        tables = _compact_plan(case)
        s["table"] = _renumber(_padded(tables, max(len(t) for t in tables) + 1, "cuda"), case["pages"], gen)
        s["pool"] = _pool((case["layers"], 2, case["pages"], case["kv_heads"], case["page"], case["head_dim"]), dtype, gen)
    else:
        b, w, v = case["items"], case["beams"], case["vocab"]
        s["logits"] = 3.0 * _pool((b * w, v), dtype, gen)
        s["scores"] = -20.0 * torch.rand(b, w, generator=gen, device="cuda").sort(-1).values
        s["finished"] = torch.rand(b, w, generator=gen, device="cuda") * 100 < case["finished"]
        s["eos"] = v // 2
    return s


# ------------------------------------------------------------------------------- the operators in their plain form
def _plain_attention(s):
    q, k, v, table, lens = s["q"], s["k"], s["v"], s["table"].clamp(min=0).long(), s["lens"]
    rows, heads, hd = q.shape
    hkv, ps = k.shape[1], k.shape[2]
    seen = torch.arange(table.shape[1] * ps, device=q.device) < lens[:, None]
    keys = k[table].transpose(1, 2).reshape(rows, hkv, -1, hd).float()
    scores = q.float().view(rows, hkv, heads // hkv, hd) @ keys.transpose(-1, -2) / math.sqrt(hd)
    del keys
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    best = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = torch.exp(scores - best)
    total = weights.sum(-1, keepdim=True)
    values = v[table].transpose(1, 2).reshape(rows, hkv, -1, hd).float()
    values.masked_fill_(~seen[:, None, :, None], 0.0)
    out = weights @ values / total
    return torch.where(lens[:, None, None] > 0, out.view(rows, heads, hd), 0.0).to(q.dtype)


def _plain_append(s):
    k, v, positions = s["k"], s["v"], s["positions"].long()
    hkv, ps, hd = k.shape[1:]
    heads = s["heads"]
    x = s["qkv"].view(-1, heads + 2 * hkv, hd)
    angle = positions.double()[:, None] * ROPE_BASE ** (-torch.arange(0, hd, 2, device=k.device, dtype=torch.float64) / hd)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[:, :heads + hkv, :hd // 2].float(), x[:, :heads + hkv, hd // 2:].float()
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(k.dtype)
    turned = torch.where(positions[:, None, None] >= 0, turned, x[:, :heads + hkv])     # padding passes as it is
    real = positions >= 0
    at = positions[real]
    page = s["table"][s["rows"].long()[real], at // ps].long()
    k[page, :, at % ps] = turned[real, heads:]
    v[page, :, at % ps] = x[real, heads + hkv:]
    return turned[:, :heads].contiguous(), k, v


def _plain_copy(pool, src, dst):
    real = src >= 0
    pool[:, :, dst[real].long()] = pool[:, :, src[real].long()]


def _plain_fork(s, grow=1):
    table, lens, parents, pages, ps = s["table"], s["lens"], s["parents"].long(), s["pool"].shape[2], s["page"]
    row, slot, dev = torch.arange(len(parents), device=table.device), torch.arange(table.shape[1], device=table.device), table.device
    parent = parents.clamp(min=0)
    old = torch.where(parents >= 0, lens[parent].long(), 0)
    new = torch.where(parents >= 0, old + grow, 0)
    held, want, last = (old + ps - 1) // ps, (new + ps - 1) // ps, old // ps
    t = torch.where(slot < held[:, None], table[parent].long(), -1)
    # the part-filled last page of a row that grows is kept by the first such row that has it, if nobody else reads it
    grows = (new > old) & (old % ps > 0)
    tail = grows[:, None] & (slot == last[:, None])
    used, others = (torch.zeros(pages + 1, dtype=torch.bool, device=dev) for _ in range(2))
    used[torch.where(t >= 0, t, pages)] = True
    others[torch.where((t >= 0) & ~tail, t, pages)] = True
    page = torch.where(grows, t.gather(1, last.clamp(max=len(slot) - 1)[:, None])[:, 0], pages)
    keeper = torch.full((pages + 1,), len(row), device=dev).scatter_reduce_(0, page, row, "amin")
    copies = grows & (others[page] | (keeper[page] != row))
    free = torch.argsort(used[:pages].int(), stable=True)
    need = want - held + copies
    first = torch.cumsum(need, 0) - need
    dst = torch.where(copies, free[first.clamp(max=pages - 1)], -1)
    src = torch.where(copies, page, -1)
    at = (first + copies)[:, None] + slot - held[:, None]
    t = torch.where((slot >= held[:, None]) & (slot < want[:, None]), free[at.clamp(0, pages - 1)], t)
    t = torch.where(tail & copies[:, None], dst[:, None], t)
    _plain_copy(s["pool"], src, dst)
    return t.int(), new.int(), src.int(), dst.int(), s["pool"]


def _plain_compact(s):
    table, pages, dev = s["table"], s["pool"].shape[2], s["table"].device
    used = torch.zeros(pages + 1, dtype=torch.bool, device=dev)
    used[torch.where(table >= 0, table, pages).long()] = True
    used, ids = used[:pages], torch.arange(pages, device=dev)
    live = used.sum()
    moves, holes = used & (ids >= live), ~used & (ids < live)
    real = torch.arange(pages // 2, device=dev) < moves.sum()
    src = torch.where(real, torch.argsort((~moves).int(), stable=True)[:pages // 2], -1)
    dst = torch.where(real, torch.argsort((~holes).int(), stable=True)[:pages // 2], -1)
    number = torch.cat([ids, ids[:1]])
    number[torch.where(real, src, pages)] = torch.where(real, dst, 0)
    packed = torch.where(table >= 0, number[table.clamp(min=0).long()], -1)
    _plain_copy(s["pool"], src, dst)
    return packed.int(), src.int(), dst.int(), live.int().view(1), s["pool"]


def _plain_beam(s):
    """The best of every beam by its logits first (a beam's score adds the same to all of them), then of all beams; 64 bits, for
    scores that lie close together."""
    logits, scores, finished, eos = s["logits"], s["scores"], s["finished"], s["eos"]
    (b, w), v = scores.shape, logits.shape[1]
    x = logits.float() + 0.0                                     # no negative zeros
    best = x.amax(-1, keepdim=True).double()
    norm = best + torch.log(torch.exp(x.double() - best).sum(-1, keepdim=True))
    bits = x.view(torch.int32)
    ids = torch.arange(v, device=x.device)
    rank = (torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() << 32) + (0xffffffff - ids)
    rank = torch.where(finished.view(-1, 1), torch.where(ids == eos, 1, -ids), rank)
    top = rank.topk(min(w, v), -1).indices
    start = scores.view(-1, 1).double()
    total = start + x.gather(1, top).double() - norm
    total = torch.where(finished.view(-1, 1), torch.where(top == eos, start, -math.inf), total).view(b, -1)
    total, order = torch.sort(total, dim=-1, descending=True, stable=True)
    order = order[:, :w]
    token = top.view(b, -1).gather(1, order)
    beam = order // top.shape[1]
    parents = beam + w * torch.arange(b, device=x.device)[:, None]
    return total[:, :w].float(), parents.int(), token, finished.gather(1, beam) | (token == eos)


# ------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        from dart_pytorch_b200 import ops
        if s["op"] == "attention":
            return ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"])
        if s["op"] == "append":
            q = ops.paged_append(s["qkv"], s["k"], s["v"], s["table"], s["positions"], s["heads"], rows=s["rows"], rope_base=ROPE_BASE)
            return q, s["k"], s["v"]
        if s["op"] == "fork":
            table, lens, src, dst = ops.fork_pages(s["table"], s["lens"], s["pool"].shape[2], s["page"], s["parents"], 1)
            ops.copy_pages(s["pool"], src, dst)
            return table, lens, src, dst, s["pool"]
        if s["op"] == "compact":
            table, src, dst, live = ops.compact_pages(s["table"], s["pool"].shape[2])
            ops.copy_pages(s["pool"], src, dst)
            return table, src, dst, live, s["pool"]
        return ops.beam_step(s["logits"], s["scores"], s["finished"], s["eos"])
    return {"attention": _plain_attention, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact,
            "beam": _plain_beam}[s["op"]](s)


def work(case):
    op, e = case["op"], SIZES[case["dtype"]]
    if op == "attention":
        lens, hd = _lengths(case), case["head_dim"]
        io = 2 * case["rows"] * case["heads"] * hd * e + 4 * case["rows"] + 4 * sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * sum(lens) * case["kv_heads"] * hd * e + io, "flops": 4 * sum(lens) * case["heads"] * hd}
    if op == "append":
        tokens = sum(p >= 0 for _, p in _append_plan(case))
        wide = (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        return {"bytes": tokens * (2 * wide * e + 12), "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["head_dim"]}
    if op in ("fork", "compact"):
        page = 2 * case["layers"] * case["kv_heads"] * case["page"] * case["head_dim"] * e
        if op == "fork":
            tables, _, _, _ = _fork_plan(case)
            moved, entries = _fork_copies(case), sum(len(t) for t in tables)
        else:
            tables = _compact_plan(case)
            entries = sum(len(t) for t in tables)
            # of the live pages, those whose number is not below their count; a random order is what a pool in use has
            moved = entries * (case["pages"] - entries) // case["pages"]
        return {"bytes": 2 * moved * page + 8 * entries + 8 * len(tables), "flops": 0}
    n = case["items"] * case["beams"]
    return {"bytes": n * case["vocab"] * e + n * 22, "flops": 4 * n * case["vocab"]}


# ------------------------------------------------------------------------------- the same from the definition, in 64 bits
def _exact_attention(s):
    q, k, v, ps = s["q"], s["k"], s["v"], s["k"].shape[2]
    group, out = q.shape[1] // k.shape[1], torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for r, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        pages = s["table"][r, :-(-n // ps)].long()
        for h in range(k.shape[1]):
            keys, values = (t[pages, h].reshape(-1, t.shape[3])[:n].double() for t in (k, v))
            for j in range(h * group, (h + 1) * group):
                out[r, j] = torch.softmax(keys @ q[r, j].double() / math.sqrt(q.shape[2]), 0) @ values
    return out


def _exact_append(s):
    k, v, heads = s["k"].double(), s["v"].double(), s["heads"]
    hkv, ps, hd = k.shape[1:]
    x = s["qkv"].double().view(-1, heads + 2 * hkv, hd)
    half = hd // 2
    power = torch.tensor([ROPE_BASE ** (-2.0 * i / hd) for i in range(half)], dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), s["positions"].double()[:, None] * power)
    z = torch.complex(x[:, :heads + hkv, :half].contiguous(), x[:, :heads + hkv, half:].contiguous()) * turn[:, None]
    z = torch.cat([z.real, z.imag], -1)
    z[s["positions"] < 0] = x[s["positions"] < 0, :heads + hkv]
    for r in range(s["table"].shape[0]):
        mine = (s["rows"] == r) & (s["positions"] >= 0)
        at = s["positions"][mine].long()
        page = s["table"][r].long()[at // ps]
        k[page, :, at % ps], v[page, :, at % ps] = z[mine, heads:], x[mine, heads + hkv:]
    return z[:, :heads].contiguous(), k, v


def _exact_pages(s):
    """The pool afterwards, by hand: who holds what, which pages are free."""
    pool, table = s["pool"].double(), s["table"].tolist()
    pages = pool.shape[2]
    moves = []
    if s["op"] == "compact":
        held = sorted({p for t in table for p in t if p >= 0})
        holes = [p for p in range(len(held)) if p not in set(held)]
        moves = list(zip([p for p in held if p >= len(held)], holes))
    else:
        ps, lens, taken = s["page"], s["lens"].tolist(), set()
        rows = [(table[p][:-(-lens[p] // ps)], lens[p]) for p in s["parents"].tolist()]
        used = {q for t, _ in rows for q in t}
        whole = {q for t, n in rows for q in t[:n // ps]}
        free = iter([p for p in range(pages) if p not in used])
        for t, n in rows:
            if n % ps == 0:
                next(free)
            elif t[-1] in taken or t[-1] in whole:
                moves.append((t[-1], next(free)))
            else:
                taken.add(t[-1])
    if moves:
        src, dst = (torch.tensor(x, device=pool.device) for x in zip(*moves))
        pool[:, :, dst] = pool[:, :, src]
    return pool


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "attention":
        return _exact_attention(s)
    if s["op"] == "append":
        return _exact_append(s)
    if s["op"] == "fork":
        return None, None, None, None, _exact_pages(s)
    if s["op"] == "compact":
        return None, None, None, None, _exact_pages(s)
    b, w = s["scores"].shape
    logits = s["logits"].double().view(b, w, -1)
    got = []
    for i in range(b):
        all_ = s["scores"][i].double()[:, None] + torch.log_softmax(logits[i], -1)
        for j in s["finished"][i].nonzero().flatten().tolist():
            all_[j] = -math.inf
            all_[j, s["eos"]] = s["scores"][i, j].double()
        got.append(all_.flatten().sort(descending=True).values[:w])
    return torch.stack(got), None, None, None
