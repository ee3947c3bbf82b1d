"""Beam search's choice, what follows from it for tables and pages, and a step's tables, against plain forms."""
import math
import random

import pytest
import torch

from llm_serving_engine_b200.kernels import ops
from plain import int4_plain as plain

pytestmark = pytest.mark.gpu


def choose(logits, scores, ended, end_token):
    shape = scores.shape
    out = (torch.full(shape, 9.0, device="cuda"), *(torch.full(shape, -9, dtype=torch.int32, device="cuda") for _ in range(3)))
    ops.beam_select(logits, scores, ended, end_token, *out)
    return out


def compare(logits, scores, ended, end_token):
    got = [t.cpu() for t in choose(logits.cuda() if not logits.is_cuda else logits, scores.cuda(), ended.cuda(), end_token)]
    want = plain.select(logits.cpu(), scores, ended, end_token)
    for r, rows in enumerate(want):
        assert len({(int(got[1][r, k]), int(got[2][r, k])) for k, row in enumerate(rows) if row[0] > -math.inf}) == sum(row[0] > -math.inf for row in rows)
        for k, (value, token, parent, over) in enumerate(rows):
            there = int(got[1][r, k]), int(got[2][r, k]), int(got[3][r, k])
            if there != (token, parent, over):
                # An exponential is off by up to 2^-22 of itself, so a row's lse by as much: offers of two beams that are closer than
                # twice that may come in either order (offers of one beam share its lse, and may not).
                assert there[1] != parent and there[2] == int(bool(ended[r, there[1]]) or there[0] == end_token), (r, k)
                row = logits[r * scores.shape[1] + there[1]].double().cpu()
                offered = float(scores[r, there[1]]) + (0.0 if ended[r, there[1]] else float(row[there[0]] - torch.logsumexp(row, 0)))
                assert abs(offered - value) <= 2.0 ** -21, (r, k)
            # one rounding to float32, and the exponentials' (2^-22 each, of a sum of them)
            assert got[0][r, k] == value or abs(float(got[0][r, k]) - value) <= 2.0 ** -24 * abs(value) + 2.0 ** -21


@pytest.mark.parametrize("requests,beams,vocab", [(1, 1, 1), (1, 4, 5), (2, 3, 1000), (3, 32, 4099), (5, 8, 50_257), (1, 16, 151_936), (40, 5, 33_001), (2, 32, 40)])
def test_select(requests, beams, vocab):
    g = torch.Generator().manual_seed(vocab)
    logits = 2.5 * torch.randn((requests * beams, vocab), generator=g)
    scores = -3 * torch.rand((requests, beams), generator=g)
    ended = (torch.rand((requests, beams), generator=g) < 0.2).int()
    if beams > 2:
        scores[0, 1] = -math.inf                     # a beam that offers nothing
    compare(logits, scores, ended, min(2, vocab - 1))


def test_select_of_strided_and_unaligned_rows():
    g = torch.Generator().manual_seed(1)
    wide = torch.randn((12, 9001), generator=g).cuda()
    for start in (0, 1, 2, 3, 5):
        compare(wide[:, start:start + 8190], -torch.rand((3, 4), generator=g), torch.zeros((3, 4), dtype=torch.int32), 0)
        compare(wide[::2, start:start + 2048], -torch.rand((2, 3), generator=g), torch.zeros((2, 3), dtype=torch.int32), 0)


def test_equal_rows_make_equal_offers():
    """Beams that all hold the same prompt: rows that begin at every place relative to a 16-byte boundary, the same to the last bit."""
    g = torch.Generator().manual_seed(12)
    row = 3 * torch.randn(70_001, generator=g)
    logits = row.repeat(8, 1)
    tokens = torch.topk(row, 1).indices.tolist() * 8
    got = choose(logits.cuda(), torch.zeros((1, 8)).cuda(), torch.zeros((1, 8), dtype=torch.int32).cuda(), 3)
    assert got[1][0].tolist() == tokens and got[2][0].tolist() == list(range(8)) and len(set(got[0][0].tolist())) == 1


def test_select_of_ties():
    """Equal logits: the lower beam, then the lower token, however many are equal."""
    for beams, vocab in ((4, 20_000), (32, 9_000), (3, 100)):
        zeros = torch.zeros((beams, vocab))
        compare(zeros, torch.zeros((1, beams)), torch.zeros((1, beams), dtype=torch.int32), 1)
        few = torch.zeros((beams, vocab))
        few[:, vocab // 2::7] = 1.0
        compare(few, torch.zeros((1, beams)), torch.zeros((1, beams), dtype=torch.int32), 1)
        steps = (torch.arange(vocab) % 5).float().repeat(beams, 1)
        compare(steps, torch.zeros((1, beams)), torch.zeros((1, beams), dtype=torch.int32), 1)


def test_select_of_infinities_and_what_is_not_a_number():
    g = torch.Generator().manual_seed(5)
    logits = torch.randn((6, 3000), generator=g)
    logits[0, 7] = math.nan                          # this beam offers nothing
    logits[1, 9] = math.inf                          # nor does this
    logits[2] = -math.inf                            # nor this
    logits[3, 1:] = -math.inf                        # one offer
    logits[4, ::2] = -math.inf
    scores, ended = torch.zeros((2, 3)), torch.zeros((2, 3), dtype=torch.int32)
    scores[1, 0] = -50.0
    compare(logits, scores, ended, 4)
    ended[1] = 1                                     # all of a request's beams have ended
    compare(logits, scores, ended, 4)


def test_select_captured():
    g = torch.Generator().manual_seed(6)
    logits = torch.randn((8, 30_001), generator=g).cuda()
    scores, ended = -torch.rand((2, 4), generator=g).cuda(), torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    want = choose(logits, scores, ended, 3)
    out = [torch.empty_like(t) for t in want]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.beam_select(logits, scores, ended, 3, *out)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


# ------------------------------------------------------------------ tables and pages
@pytest.mark.parametrize("requests,beams,page_size,lengths", [
    (1, 4, 16, [21]), (3, 8, 8, [1, 8, 37]), (2, 32, 16, [15, 160]), (4, 1, 16, [3, 16, 17, 0]), (2, 5, 3, [31, 33])])
def test_reorder(requests, beams, page_size, lengths):
    rng = random.Random(beams)
    for _ in range(4):
        parents = [[min(int(beams * rng.random() ** 2), beams - 1) for _ in range(beams)] for _ in range(requests)]
        width = max(lengths) // page_size + 2
        rows = requests * beams
        pages = rows * width
        free = list(range(pages))
        rng.shuffle(free)
        tables = []
        for r in range(requests):
            shared = [free.pop() for _ in range(lengths[r] // page_size)]
            tables += [shared + [free.pop() for _ in range(width - len(shared))] for _ in range(beams)]
        storages = [torch.randn((3, pages, 2, 4)).cuda(), torch.randint(0, 255, (2, pages, 5), dtype=torch.uint8).cuda(),      # 5 bytes a page
                    torch.randn((2, pages, 1, 3)).cuda(), torch.randn((4, 2, pages, 8)).bfloat16().cuda()[:, 1]]                # outer parts further apart
        want, copies = plain.reorder(parents, tables, lengths, page_size)
        expected = [s.clone() for s in storages]
        for source, target in copies:
            for new, old in zip(expected, storages):
                new[:, target] = old[:, source]
        new_tables = torch.full((rows, width), -7, dtype=torch.int32, device="cuda")
        ops.beam_reorder(torch.tensor(parents).int().cuda(), torch.tensor(tables).int().cuda(), torch.tensor(lengths).int().cuda(), new_tables,
                         page_size, storages)
        assert new_tables.tolist() == want
        assert all(torch.equal(a, b) for a, b in zip(storages, expected))


def test_reorder_of_states_of_many_layers():
    """Slots of fixed-size states: tables of one column; more tensors than one launch takes."""
    beams, rows = 6, 12
    parents = [[0, 0, 3, 0, 3, 5], [1, 1, 1, 1, 1, 1]]
    slots = torch.randperm(rows + 2)[:rows].tolist()
    states = [torch.randn((1, rows + 2, 3, 5)).cuda() for _ in range(ops.MAX_REORDER_STORAGES + 3)]
    old = [s.clone() for s in states]
    new = torch.empty((rows, 1), dtype=torch.int32, device="cuda")
    ops.beam_reorder(torch.tensor(parents).int().cuda(), torch.tensor(slots).int().cuda()[:, None], torch.ones(2).int().cuda(), new, 2, states)
    want, copies = plain.reorder(parents, [[s] for s in slots], [1, 1], 2)
    assert new.tolist() == want and len(copies) == 3 + 5
    for state, before in zip(states, old):
        for r in range(rows):      # every beam has its parent's state
            source = slots[r // beams * beams + parents[r // beams][r % beams]]
            assert torch.equal(state[0, want[r][0]], before[0, source])


def test_reorder_leaves_pages_alone_that_are_none():
    """Entries outside the storage are not copied, parents outside the beams are taken as the nearest one."""
    storage = torch.randn((1, 4, 8)).cuda()
    before = storage.clone()
    new = torch.empty((3, 1), dtype=torch.int32, device="cuda")
    ops.beam_reorder(torch.tensor([[-5, 0, 9]]).int().cuda(), torch.tensor([[-1], [3], [7]]).int().cuda(), torch.tensor([1]).int().cuda(), new, 4, [storage])
    assert new.tolist() == [[-1], [3], [7]] and torch.equal(storage, before)


# ------------------------------------------------------------------ a step's tables
@pytest.mark.parametrize("requests,page_size", [(1, 16), (3, 1), (64, 16), (255, 8), (256, 7), (700, 16)])
def test_step_tables(requests, page_size):
    rng = random.Random(requests)
    first = [rng.choice([0, 1, page_size - 1, page_size, rng.randrange(500)]) for _ in range(requests)]
    counts = [rng.choice([1, 1, 0, 5, rng.randrange(1, 200)]) for _ in range(requests)]
    held = [max(0, -(-(f + n) // page_size) + rng.choice([0, 0, 0, 2, -1])) for f, n in zip(first, counts)]
    page_start = [0]
    for n in held:
        page_start.append(page_start[-1] + n)
    pages = [rng.choice([rng.randrange(10_000), rng.randrange(10_000), -1]) for _ in range(page_start[-1])]
    tokens, width = sum(counts) + rng.choice([0, 3, 300]), max(held) + 1
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")      # noqa: E731
    out = [torch.full((n,), -77, dtype=torch.int32, device="cuda") for n in (requests + 1, tokens, tokens, tokens, requests)]
    tables = torch.full((requests, width + 3), -77, dtype=torch.int32, device="cuda")[:, :width]     # rows further apart
    ops.step_tables(ints(first), ints(counts), ints(pages), ints(page_start), page_size, *out, tables)
    want = plain.step_tables(first, counts, pages, page_start, page_size, tokens, width)
    for got, expected in zip((*out, tables), want):
        assert got.tolist() == expected


def test_step_tables_of_no_rows():
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")      # noqa: E731
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    start, contexts, tables = ints(5, 5, 5), ints(5, 5), torch.full((2, 2), 5, dtype=torch.int32, device="cuda")
    ops.step_tables(ints(3, 4), ints(0, 0), ints(8, 9), ints(0, 1, 2), 16, start, none, none.clone(), none.clone(), contexts, tables)
    assert start.tolist() == [0, 0, 0] and contexts.tolist() == [3, 4] and tables.tolist() == [[8, -1], [9, -1]]


def test_select_of_logits_far_below_zero():
    """A vocabulary of which parts are ruled out, the rest far below zero: sums of exponentials that only powers of two keep apart."""
    logits = torch.full((4, 9000), -math.inf)
    logits[0, 5000:5100] = -20_000.0 + torch.arange(100.0)
    logits[1, ::3] = 30_000.0 - torch.arange(3000.0)
    logits[2, 8999] = -3e38
    logits[3, :] = -1000.0
    compare(logits, torch.zeros((2, 2)), torch.zeros((2, 2), dtype=torch.int32), 0)
