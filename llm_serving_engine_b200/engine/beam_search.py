"""Beam search over the engine's step function.

Every step runs the beams of all prompts as one batch of single tokens; the choice of the next beams, their block tables, pages
and states, and the next step's metadata are made on the device (``ops.beam_select``, ``ops.beam_reorder``,
``ops.step_tables``), so that the host waits for nothing between the prompts and the end.  (The reference generates one sequence
a request, ``src/llmserve/engine.py:29-72``; it has no beam search.)

The full pages of a prompt belong to all its beams; behind them every beam has pages of its own, lent by the cache manager
for as long as the search lasts.  Beams whose parent went on elsewhere leave their page to the children that need one.
"""
from __future__ import annotations

import gc
from dataclasses import dataclass

import torch

from ..cache.manager import CacheFullError
from ..kernels import ops
from .step import LONG_CONTEXT, Segment, StepContext, StepEntry, StepRunner


@dataclass(frozen=True)
class Beam:
    """A finished or cut-off sequence: its generated tokens (without the end token) and the sum of their log probabilities (the end
    token's among them when it ended)."""

    tokens: list[int]
    score: float
    ended: bool


class BeamSearch:
    """``beams`` beams (at most ``ops.MAX_BEAMS``) a prompt, on the runner's model and cache.  ``use_graph``: the step between two
    choices is captured once a search and replayed."""

    def __init__(self, runner: StepRunner, beams: int, end_token: int, use_graph: bool | None = None) -> None:
        if not 1 <= beams <= ops.MAX_BEAMS:
            raise ValueError(f"beams must be between 1 and {ops.MAX_BEAMS}")
        if not 0 <= end_token < runner.model.vocab_size:
            raise ValueError("the end token lies outside the vocabulary")
        if not getattr(runner.model, "graph_safe", False):
            raise ValueError("beam search needs a model whose parts read a step's metadata on the device")
        self.runner, self.beams, self.end_token = runner, beams, end_token
        self.use_graph = runner.use_graphs if use_graph is None else use_graph

    def search(self, prompts: list[list[int]], max_new_tokens: int) -> list[list[Beam]]:
        """The best ``beams`` continuations of every prompt, the best first (fewer where the model's logits leave fewer).
        Pages for ``max_new_tokens`` of every beam, and a state slot a beam, are taken before the first choice: ``CacheFullError`` where
        they are not free.  Raises ``KernelError`` when a kernel's bounded wait gave up meanwhile, or no beam of a prompt is left."""
        runner, cache = self.runner, self.runner.cache
        if not prompts or max_new_tokens <= 0:
            raise ValueError("a search needs prompts and a positive max_new_tokens")
        limit = runner.model.spec.max_position_embeddings
        for prompt in prompts:
            if not prompt or len(prompt) + max_new_tokens > limit:
                raise ValueError(f"a prompt of {len(prompt)} tokens plus {max_new_tokens} does not fit {limit} positions")
        if len(prompts) * self.beams > runner.max_segments:
            raise ValueError(f"{len(prompts)} prompts of {self.beams} beams, at most {runner.max_segments} sequences a step")
        names = [f"__beams_{index}" for index in range(len(prompts))]
        try:
            for name in names:
                cache.create(name)
            logits = torch.stack([self._prompt(name, prompt) for name, prompt in zip(names, prompts)])
            return self._beams(names, [len(prompt) for prompt in prompts], logits, max_new_tokens)
        except BaseException:
            torch.cuda.current_stream().synchronize()
            ops.kernel_status_reset()        # what this search's kernels left does not fail the next steps
            raise
        finally:
            torch.cuda.current_stream().synchronize()
            for name in names:
                if name in cache.requests:
                    cache.free(name)

    def _prompt(self, name: str, prompt: list[int]) -> torch.Tensor:
        """Logits behind the prompt's last token."""
        most = self.runner.max_tokens
        for first in range(0, len(prompt), most):
            portion = prompt[first:first + most]
            last = first + most >= len(prompt)
            logits = self.runner.run([StepEntry(name, portion, [len(portion) - 1] if last else [])])
        return logits[0].clone()

    def _beams(self, names, lengths, logits, max_new_tokens) -> list[list[Beam]]:
        cache, beams, device = self.runner.cache, self.beams, self.runner.device
        requests, page = len(names), cache.page_size
        rows = requests * beams
        ints = {"dtype": torch.int32, "device": device}
        # block tables: the prompt's full pages for all beams, then pages of a beam's own, for all tokens to come
        width = max(-(-(length + max_new_tokens) // page) for length in lengths)
        tables = [[] for _ in cache.groups]
        slots = []
        for name, length in zip(names, lengths):
            if not cache.grow(name, max_new_tokens):
                raise CacheFullError("paged KV cache has no free blocks for the beams")
            full, own = length // page, -(-(length + max_new_tokens) // page) - length // page
            lent, more = cache.lend(name, own * (beams - 1), beams - 1)
            slots += [cache.requests[name].state_slot, *more]
            for g, pages in enumerate(lent):
                first = cache.block_table(g, name)
                for beam in range(beams):
                    table = list(first) if beam == 0 else [*first[:full], *pages[(beam - 1) * own:beam * own]]
                    tables[g].append(table + [-1] * (width - len(table)))
        held = _Held(self.runner, beams, [torch.tensor(table, **ints) for table in tables], torch.tensor(slots, **ints),
                     torch.tensor(lengths, **ints))
        # one beam a prompt at first: the others have nothing to offer
        scores = torch.full((requests, beams), -torch.inf, dtype=torch.float32, device=device)
        scores[:, 0] = 0.0
        held.scores.copy_(scores)
        chosen, status = [], ops.kernel_status_words()
        step = _Step(held, self.end_token, self.use_graph and max_new_tokens > 3)
        logits = logits.repeat_interleave(beams, 0)
        for index in range(max_new_tokens):
            chosen.append(step.choose(logits))
            if index + 1 < max_new_tokens:
                logits = step.run()
            if index % 16 == 15:                # (a look at the device now and then)
                ops.kernel_status_async(status)
                over = bool(held.ended.all())
                ops.kernel_status_check(status)
                if over:
                    break
        ops.kernel_status_async(status)         # arrives with what was chosen
        chosen, scores, ended = torch.stack(chosen).cpu(), held.scores.cpu().tolist(), held.ended.cpu().tolist()
        ops.kernel_status_check(status)
        found = self._traced([[part.tolist() for part in pair] for pair in chosen], scores, ended)
        if not all(found):
            raise ops.KernelError(f"prompt {found.index([])}: the model's logits are not numbers, no beam is left")
        return found

    def _traced(self, chosen, scores, ended) -> list[list[Beam]]:
        found = []
        for request, (row, over) in enumerate(zip(scores, ended)):
            found.append([])
            for beam, (score, done) in enumerate(zip(row, over)):
                if score == float("-inf"):
                    continue
                tokens, at = [], beam
                for step_tokens, parents in reversed(chosen):
                    tokens.append(step_tokens[request][at])
                    at = parents[request][at]
                tokens.reverse()
                if done:
                    tokens = tokens[:tokens.index(self.end_token)]
                found[-1].append(Beam(tokens, score, bool(done)))
        return found


class _Held:
    """What a search keeps on the device: scores and flags of the beams, block tables, state slots, and the next step's metadata."""

    def __init__(self, runner, beams: int, tables: list, slots: torch.Tensor, lengths: torch.Tensor) -> None:
        device, cache = runner.device, runner.cache
        requests, rows = lengths.shape[0], slots.shape[0]
        ints = {"dtype": torch.int32, "device": device}
        self.runner, self.requests, self.beams, self.rows = runner, requests, beams, rows
        self.scores = torch.empty((requests, beams), dtype=torch.float32, device=device)
        self.ended, self.tokens, self.parents = (torch.zeros((requests, beams), **ints) for _ in range(3))
        self.lengths, self.row_lengths = lengths, lengths.repeat_interleave(beams)
        self.tables, self.new_tables = tables, [torch.empty_like(table) for table in tables]
        self.slots, self.new_slots = slots[:, None].contiguous(), torch.empty_like(slots)[:, None].contiguous()
        self.one, self.ones, self.width = torch.ones(requests, **ints), torch.ones(rows, **ints), tables[0].shape[1] if tables else 1
        self.page_start = torch.arange(0, rows * self.width + 1, self.width, **ints)
        self.storages = []
        for group in cache.groups:
            parts = [group.storage.flatten(0, 1)]
            if group.scale_storage is not None:
                parts.append(group.scale_storage.flatten(0, 1))
            if group.value_storage is not None:
                parts.append(group.value_storage)
            self.storages.append(parts)
        self.states = [tensor[None] if tensor.dim() > 1 else tensor[None, :, None] for tensor in cache.states.tensors.values()]
        # the step: a row a beam
        self.step = step = StepContext()
        step.num_tokens = step.num_segments = step.num_wanted = rows
        step.token_ids = self.tokens.view(-1)
        step.positions, step.segment_of_token, step.segment_context = (torch.empty(rows, **ints) for _ in range(3))
        step.segment_start = torch.empty(rows + 1, **ints)
        step.segment_first_position = self.row_lengths
        step.segment_state_slot = self.slots[:, 0]
        step.want_rows = torch.arange(rows, **ints)
        step.max_segment_tokens, step.max_context = 1, None
        step.decode_only = step.every_row_wanted = True
        step.long_context = self.width * cache.page_size > LONG_CONTEXT
        step.many_keys = self.width * cache.page_size >= ops.DECODE_MANY_KEYS
        step.segments = [Segment(f"beam {row}", 0, 0, 1, row) for row in range(rows)]
        self.maps = [torch.empty(rows, **ints) for _ in cache.groups]
        self.spare_tables = torch.empty((rows, self.width), **ints)
        self.caches = runner.layer_caches(self.maps, self.tables)


class _Step:
    """A choice and the step behind it, launch by launch first, then from a graph (every address stays the same)."""

    def __init__(self, held: _Held, end_token: int, use_graph: bool) -> None:
        self.held, self.end_token, self.use_graph = held, end_token, use_graph
        self.graph, self.logits, self.steps = None, None, 0

    def choose(self, logits: torch.Tensor) -> torch.Tensor:
        """The next beams: scores, flags, tokens and parents are replaced, and what was chosen comes back [2, requests, beams]."""
        held = self.held
        ops.beam_select(logits, held.scores, held.ended, self.end_token, held.scores, held.tokens, held.parents, held.ended)
        return torch.stack((held.tokens, held.parents))

    def _launch(self) -> torch.Tensor:
        held, cache, step = self.held, self.held.runner.cache, self.held.step
        for tables, new, storages in zip(held.tables, held.new_tables, held.storages):
            ops.beam_reorder(held.parents, tables, held.lengths, new, cache.page_size, storages)
            tables.copy_(new)
        if held.states:
            ops.beam_reorder(held.parents, held.slots, held.one, held.new_slots, 2, held.states)
            held.slots.copy_(held.new_slots)
        for index in range(max(1, len(held.tables))):
            pages = held.tables[index].view(-1) if held.tables else held.spare_tables.view(-1)
            ops.step_tables(held.row_lengths, held.ones, pages, held.page_start, cache.page_size, step.segment_start,
                            step.segment_of_token, step.positions, held.maps[index] if held.maps else torch.empty_like(step.positions),
                            step.segment_context, held.spare_tables)
        # An ordinary launch between the tables and the step: the step's first kernels may start before the launch behind which they are
        # queued has ended and read the step's metadata at once, so the tables have to be complete and visible before that launch begins.
        held.lengths += 1
        logits = held.runner.model.forward(step, held.caches)
        held.row_lengths += 1
        return logits

    def run(self) -> torch.Tensor:
        """The step of the beams' tokens: logits [rows, vocabulary]."""
        self.steps += 1
        if not self.use_graph or self.steps == 1:       # (what is set up at a first use is set up here)
            return self._launch()
        if self.graph is None:
            current, stream = torch.cuda.current_stream(), torch.cuda.Stream()
            current.synchronize()
            stream.wait_stream(current)
            graph = torch.cuda.CUDAGraph()
            collecting = gc.isenabled()
            gc.disable()         # (a collection that destroys CUDA objects would invalidate the capture)
            try:
                with torch.cuda.stream(stream):
                    graph.capture_begin()
                    try:
                        self.logits = self._launch()
                    finally:
                        graph.capture_end()
            finally:
                if collecting:
                    gc.enable()
            current.wait_stream(stream)
            self.graph = graph
        self.graph.replay()
        return self.logits
