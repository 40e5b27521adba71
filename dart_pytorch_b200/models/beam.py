"""Beam search over a paged cache, for the decoders that offer ``paged_hidden`` (GPT, Llama).

The beams of a prompt share its pages; a step chooses among all continuations, makes every beam a copy of its parent and runs
the model once for all beams of all prompts, which may be of different lengths.  Nothing but the final choice leaves the device, and on a
CUDA device the step is recorded once and replayed."""
from __future__ import annotations

import gc
import os
from typing import List, Optional, Sequence, Tuple

import torch

from .. import _native as N
from .. import ops as F
from ..nn.paged import PagedCache
from ..ops.paged import MAX_PAGES, MAX_ROWS


class _Search:
    """The state of a running search and its step."""

    def __init__(self, model, cache: PagedCache, logits, items: int, beams: int, eos: Optional[int]):
        self.model, self.cache, self.eos = model, cache, eos
        self.logits = logits
        self.scores = torch.full((items, beams), -float("inf"), device=logits.device)
        self.scores[:, 0] = 0.0                  # the beams of a prompt are one at first
        self.finished = None if eos is None else torch.zeros(items, beams, dtype=torch.bool, device=logits.device)

    def choose(self):
        self.scores, parents, tokens, finished = F.beam_step(self.logits, self.scores, self.finished, self.eos)
        self.finished = None if self.eos is None else finished
        return parents.view(-1), tokens.view(-1)

    def step(self):
        """Chooses, and runs the model on what was chosen; ``(parents, tokens)`` of every row."""
        parents, tokens = self.choose()
        self.cache.fork(parents)
        h = self.model.paged_hidden(tokens.view(-1, 1), self.cache)
        self.logits = F.linear(h[:, -1, :], self.model.head_weight)
        return parents, tokens

    # ---- the same step recorded: its state lies in buffers of its own, which it updates in place
    def record(self):
        c = self.cache
        held = [c.table, c.lens, self.logits, self.scores] + ([] if self.finished is None else [self.finished])
        held = [t.clone() for t in held]
        stream = torch.cuda.Stream(device=c.table.device)
        stream.wait_stream(torch.cuda.current_stream())
        graph, longest = torch.cuda.CUDAGraph(), c.longest
        gc.collect()                             # an unreachable older graph must not be destroyed while this one is recorded
        collecting = gc.isenabled()
        gc.disable()
        try:
            with torch.cuda.graph(graph, stream=stream):
                c.table, c.lens, self.logits, self.scores = held[:4]
                self.finished = held[4] if len(held) > 4 else None
                c.longest = 0
                out = self.step()
                for to, t in zip(held, [c.table, c.lens, self.logits, self.scores, self.finished]):
                    to.copy_(t)
        finally:
            if collecting:
                gc.enable()
        torch.cuda.current_stream().wait_stream(stream)
        c.table, c.lens, self.logits, self.scores = held[:4]
        self.finished = held[4] if len(held) > 4 else None
        c.longest = longest
        self.graph, self.out = graph, out

    def replay(self):
        self.cache.longest = self.cache.longer_by(1)
        self.graph.replay()
        return self.out


def beam_search(model, prompts: Sequence[Sequence[float]], max_new_tokens: int, beams: int = 4, eos: Optional[int] = None,
                length_penalty: float = 0.0, page_size: int = 16) -> List[List[Tuple[List[int], float]]]:
    """The ``beams`` most probable continuations found for every prompt, best first, as ``(tokens, score)``: prompt and new
    tokens, up to and with ``eos``, and the sum of the new tokens' log-probabilities.  They are ordered by ``score / (new
    tokens) ** length_penalty``.  Prompts may differ in length.  Where the model's logits are no distribution, so that a prompt has no
    continuation at all, that is an ``ArithmeticError``."""
    what = f"{type(model).__name__}.generate_beams"
    prompts = [[int(round(float(t))) for t in p] for p in prompts]
    if not prompts or any(not p for p in prompts):
        raise ValueError(f"{what}: prompts must be non-empty")
    if not 0 < beams <= 32:
        raise ValueError(f"{what}: 1 to 32 beams, got {beams}")
    c, longest = model.config, max(len(p) for p in prompts)
    if longest > c.max_ctx:
        raise ValueError(f"{what}: prompt of {longest} tokens exceeds maxCtx {c.max_ctx}")
    if eos is not None and not 0 <= eos < c.vocab_size:
        raise ValueError(f"{what}: eos {eos} is no token of {c.vocab_size}")
    new = min(max_new_tokens, c.max_ctx - longest + 1)
    if new <= 0:
        return [[(list(p), 0.0)] for p in prompts]
    items, dev, heads = len(prompts), model.device, getattr(c, "num_kv_heads", c.num_heads)
    # pages: what the prompts fill, and each beam's own behind that (with the part-filled one that it copies)
    pages = sum(-(-len(p) // page_size) for p in prompts) + items * beams * (-(-new // page_size) + 1)
    if items * beams > MAX_ROWS or pages > MAX_PAGES:
        raise ValueError(f"{what}: {items} prompts of {beams} beams and {new} new tokens are {items * beams} rows of {pages} pages; one call "
                         f"takes {MAX_ROWS} rows and {MAX_PAGES} pages")
    was_training = model.training
    model.eval()
    try:
        with torch.no_grad():
            # (the last token is chosen and not appended, so no row is longer than the context)
            cache = PagedCache(c.num_layers, heads, model.paged_head_dim, items * beams, longest + new - 1, page_size, pages,
                               dtype=model.head_weight.dtype, device=dev)
            cache.prompts([len(p) for p in prompts], [i * beams for i in range(items)])
            tokens = torch.tensor([p + [0] * (longest - len(p)) for p in prompts], dtype=torch.long, device=dev)
            last = torch.tensor([len(p) - 1 for p in prompts], device=dev)
            h = model.paged_hidden(tokens, cache)[torch.arange(items, device=dev), last]
            logits = F.linear(h, model.head_weight).repeat_interleave(beams, 0)
            search = _Search(model, cache, logits, items, beams, eos)
            del logits, h
            history, recorded = [], False
            graphs = dev.type == "cuda" and os.environ.get("DPTB200_DECODE_GRAPH", "1") != "0"
            for t in range(new):
                if t + 1 == new:
                    history.append([x.clone() for x in search.choose()])
                    break
                # the first steps run as they are: workspaces and kernel attributes are in place when the step is recorded
                if graphs and t == 2 and new - t >= 8:
                    search.record()
                    recorded = True
                history.append([x.clone() for x in (search.replay() if recorded else search.step())])
                if eos is not None and t % 8 == 7 and bool(search.finished.all()):
                    break
            if dev.type == "cuda":
                N.raise_on_device_error()
            parents, tokens = (torch.stack(x).cpu().tolist() for x in zip(*history))
            scores = search.scores.double().cpu().tolist()
    finally:
        if was_training:
            model.train()
    found = []
    for i, p in enumerate(prompts):
        mine = []
        for w in range(beams):
            if scores[i][w] == -float("inf"):
                continue                          # fewer continuations than beams
            row, path = i * beams + w, []
            for t in reversed(range(len(tokens))):
                path.append(tokens[t][row])
                row = parents[t][row]
            path.reverse()
            if eos is not None and eos in path:
                path = path[:path.index(eos) + 1]
            mine.append((p + path, scores[i][w], scores[i][w] / len(path) ** length_penalty))
        if not mine:
            raise ArithmeticError(f"{what}: no continuation of prompt {i} has a probability (the model's logits are not finite)")
        mine.sort(key=lambda x: -x[2])
        found.append([(seq, score) for seq, score, _ in mine])
    return found

