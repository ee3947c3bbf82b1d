"""Keys and values in 4 bits on the GPU: the write, the way back, and attention of single rows, against plain 64-bit forms."""
import math

import pytest
import torch

from llm_serving_engine_b200.kernels import ops
from plain import int4_plain as plain

pytestmark = pytest.mark.gpu

D64 = torch.float64


def empty_cache(pages, n_kv, page_size, dim, fill=False):
    """Four tensors; with ``fill`` every code is 0xA5 and every scale not a number, as a page may hold anything before it is written."""
    codes = [torch.full((pages, n_kv, page_size, dim // 2), 0xA5, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.full((pages, n_kv, page_size, 2), math.nan if fill else 0.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    return codes[0], scales[0], codes[1], scales[1]


@pytest.mark.parametrize("tokens,n_q,n_kv,dim,page_size,dtype,pairing,bias", [
    (1, 2, 1, 64, 16, torch.bfloat16, 1, True), (3, 12, 2, 128, 5, torch.float32, 0, True), (65, 28, 4, 128, 16, torch.bfloat16, 0, False),
    (130, 5, 5, 64, 8, torch.float32, 1, True), (700, 40, 8, 128, 32, torch.bfloat16, 1, True), (600, 3, 1, 64, 16, torch.float32, 0, True)])
def test_write_and_read(tokens, n_q, n_kv, dim, page_size, dtype, pairing, bias):
    g = torch.Generator().manual_seed(tokens)
    width = (n_q + 2 * n_kv) * dim
    wide = torch.randn((tokens, width + 8), generator=g).to(dtype).cuda()
    qkv = wide[:, :width]                                      # rows further apart than they are long
    offset = torch.randn(width, generator=g).cuda() if bias else None
    pages = -(-tokens // page_size) + 3
    slots = torch.randperm(pages * page_size, generator=g)[:tokens].int().cuda()
    if tokens > 2:
        slots[1] = -1                                          # a padding row
    positions = (torch.arange(tokens) * 37 + 90_000).int().cuda()
    inv_freq = (10000.0 ** (-torch.arange(0, dim, 2, dtype=D64) / dim)).float().cuda()
    cache = empty_cache(pages, n_kv, page_size, dim)
    before = [t.clone() for t in cache]
    q = torch.empty((tokens, n_q, dim), dtype=torch.bfloat16, device="cuda")
    ops.rope_kv_write_int4(qkv, offset, positions, slots, inv_freq, q, *cache, n_q, n_kv, dim, pairing)

    x = qkv.to(D64) + (offset.to(D64) if bias else 0.0)
    x = x.view(tokens, n_q + 2 * n_kv, dim)
    turned = plain.rotate(x[:, :n_q + n_kv], positions, inv_freq, pairing)
    # queries: a float32 rotation (four roundings of the larger addend) and one rounding to bfloat16
    reach = x[:, :n_q].abs().amax(-1, keepdim=True) * 2
    assert ((q.to(D64) - turned[:, :n_q]).abs() <= 2.0 ** -8 * turned[:, :n_q].abs() + 2.0 ** -21 * reach).all()
    # codes, scales and centres: the same numbers, and nothing else written
    page, at = slots.long() // page_size, slots.long() % page_size
    kept = slots >= 0
    want = [t.clone() for t in before]
    for rows, codes, scales in ((turned[:, n_q:], want[0], want[1]), (x[:, n_q + n_kv:], want[2], want[3])):
        u, s, c = plain.quantise(rows[kept])
        codes[page[kept], :, at[kept]] = plain.pack(u)
        scales[page[kept], :, at[kept]] = torch.stack([s, c], -1).bfloat16()
    for got, expected in zip(cache, want):
        assert torch.equal(got, expected)
    # the way back: one rounding to bfloat16; rows without a slot are left alone
    k, v = (torch.full((tokens, n_kv, dim), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.kv_read_int4(*cache, slots, k, v)
    for got, codes, scales in ((k, want[0], want[1]), (v, want[2], want[3])):
        expected = plain.values(codes[page[kept], :, at[kept]], scales[page[kept], :, at[kept]])
        # (the product's addend: one float32 rounding before the bfloat16 one)
        assert ((got[kept].to(D64) - expected).abs() <= (2.0 ** -8 + 2.0 ** -23) * expected.abs() + 2.0 ** -126).all()
        assert (got[~kept] == 7.0).all()


def test_write_takes_partial_sums():
    g = torch.Generator().manual_seed(3)
    tokens, n_q, n_kv, dim = 9, 6, 2, 128
    stack = torch.randn((5, tokens, (n_q + 2 * n_kv) * dim), generator=g).cuda()
    total = torch.zeros_like(stack[0])
    for part in stack:
        total = total + part          # in index order, from zero, as the kernel adds them
    inv_freq = torch.full((dim // 2,), 0.01, device="cuda")
    positions, slots = torch.arange(tokens).int().cuda(), torch.arange(tokens).int().cuda()
    made = []
    for qkv in (stack, total):
        cache = empty_cache(2, n_kv, 16, dim)
        q = torch.empty((tokens, n_q, dim), dtype=torch.bfloat16, device="cuda")
        ops.rope_kv_write_int4(qkv, None, positions, slots, inv_freq, q, *cache, n_q, n_kv, dim, 1)
        made.append((q, *cache))
    for a, b in zip(*made):
        assert torch.equal(a, b)


def test_write_of_rows_that_are_alike_or_not_finite():
    n_q, n_kv, dim, tokens = 1, 1, 64, 7
    qkv = torch.zeros((tokens, 3 * dim))
    v = qkv[:, 2 * dim:]
    v[0] = 2.5                                    # all alike: the centre alone
    v[1] = torch.randn(dim); v[1, 5] = math.inf
    v[2] = torch.randn(dim); v[2, 63] = math.nan
    v[3] = torch.linspace(-3e38, 3e38, dim)       # (steps of a range beyond float32: the ramp itself is not finite)
    v[4] = 1e-38 * torch.arange(dim)              # a scale that hardly is one
    v[5] = 1000 + torch.arange(dim) / 64          # a small range far from zero
    v[6] = 3e38 * torch.linspace(-1, 1, dim)      # a range beyond float32
    cache = empty_cache(1, n_kv, 8, dim)
    q = torch.empty((tokens, n_q, dim), dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(tokens).int().cuda()
    ops.rope_kv_write_int4(qkv.cuda(), None, slots, slots, torch.ones(dim // 2, device="cuda"), q, *cache, n_q, n_kv, dim, 0)
    u, s, c = plain.quantise(v)
    assert torch.equal(cache[2][0, 0, :tokens].cpu(), plain.pack(u))
    assert torch.equal(torch.nan_to_num(cache[3][0, 0, :tokens].cpu().float(), nan=1e9), torch.nan_to_num(torch.stack([s, c], -1).bfloat16().float(), nan=1e9))
    back = plain.values(cache[2][0, 0, :tokens].cpu(), cache[3][0, 0, :tokens].cpu())
    whole = torch.isfinite(v).all(-1)
    assert (back[0] == 2.5).all() and torch.equal(torch.isfinite(back).all(-1), whole) and back[~whole].isnan().all()
    assert whole.tolist() == [True, False, False, False, True, True, True]


# ------------------------------------------------------------------ attention of single rows
def fill_cache(g, pages, n_kv, page_size, dim):
    made = []
    for _ in range(2):
        x = torch.randn((pages, n_kv, page_size, dim), generator=g) + 0.3 * torch.randn((1, n_kv, 1, dim), generator=g)
        u, s, c = plain.quantise(x)
        made += [plain.pack(u).cuda(), torch.stack([s, c], -1).bfloat16().cuda()]
    return made


def request_rows(cache, table, length, page_size):
    """Keys and values of a request, [length, n_kv, D], float64."""
    pages = table[: -(-length // page_size)].long()
    return [plain.values(c[pages], s[pages]).transpose(1, 2).flatten(0, 1)[:length] for c, s in ((cache[0], cache[1]), (cache[2], cache[3]))]


def bound(expected, weighed):
    """The result's rounding (2^-8 of it), the weights' (2^-8 of every term), and float32's in scores of up to 40 in base two:
    2^-24 of them a handful of times, in numerator and denominator (2^-14 of the terms)."""
    return 2.0 ** -8 * expected.abs() + (2.0 ** -8 + 2.0 ** -14) * weighed + 1e-30


ROWS = [
    # contexts, query heads, kv heads, head size, page size, splits
    ([1, 2, 15, 16, 17, 33], 12, 2, 128, 16, 1), ([1, 64, 65, 200], 8, 8, 64, 16, 3), ([333, 7, 90], 20, 2, 128, 32, None),
    ([1000, 1, 2100], 7, 1, 128, 16, 8), ([2100, 31, 640], 6, 2, 64, 8, 20), ([77, 130], 4, 4, 64, 5, 2), ([5000], 28, 4, 128, 16, None),
    ([900, 3], 9, 1, 64, 24, 11), ([300, 1, 40], 3, 3, 128, 128, 1)]


@pytest.mark.parametrize("contexts,n_q,n_kv,dim,page_size,splits", ROWS)
def test_rows(contexts, n_q, n_kv, dim, page_size, splits):
    g = torch.Generator().manual_seed(sum(contexts))
    held = [-(-n // page_size) for n in contexts]
    width = max(held) + 2
    cache = fill_cache(g, sum(held) + 2, n_kv, page_size, dim)
    order = (torch.randperm(sum(held), generator=g) + 1).tolist()
    tables = torch.full((len(contexts), width), -1, dtype=torch.int32)
    for s, n in enumerate(held):
        tables[s, :n] = torch.tensor([order.pop() for _ in range(n)])
        # what lies behind the last key of a request is anything at all
        page, rest = int(tables[s, n - 1]), contexts[s] - (n - 1) * page_size
        for scales in (cache[1], cache[3]):
            scales[page, :, rest:] = math.nan
    # rows in another order than the requests, a padding row and one that sees nothing
    rows = list(range(len(contexts)))[::-1]
    segments = torch.tensor(rows[:1] + [-1] + rows[1:] + [0], dtype=torch.int32)
    positions = torch.tensor([contexts[rows[0]] - 1, 5] + [contexts[r] - 1 for r in rows[1:]] + [-1], dtype=torch.int32)
    q = (2 * torch.randn((len(segments), n_q, dim), generator=g)).bfloat16().cuda()
    out = torch.full_like(q, 3.0)
    scale = dim ** -0.5
    ops.paged_attention_decode_int4(q, *cache, out, tables.cuda(), segments.cuda(), positions.cuda(), scale,
                                    max_context=max(contexts), num_splits=splits)
    for row, (s, p) in enumerate(zip(segments.tolist(), positions.tolist())):
        if s < 0:
            assert (out[row] == 3.0).all()
            continue
        k, v = request_rows(cache, tables[s].cuda(), max(p + 1, 0), page_size)
        expected, weighed = plain.attend(q[row], k, v, p, scale)
        assert ((out[row].to(D64) - expected).abs() <= bound(expected, weighed)).all(), (row, s, p)


@pytest.mark.parametrize("splits", [1, 4, 9])
def test_rows_beside_portions(splits):
    """Requests of one token among portions and empty ones: their rows, wherever these lie, and no other."""
    counts, firsts = [5, 1, 0, 1, 70, 1], [0, 300, 0, 0, 20, 77]
    g, cache, tables, start, _ = portion_case(counts, firsts, 2, 64, 16, 6)
    segments = torch.repeat_interleave(torch.arange(6), torch.tensor(counts)).int().cuda()
    positions = torch.cat([torch.arange(n) + f for n, f in zip(counts, firsts)]).int().cuda()
    q = torch.randn((sum(counts), 6, 64), generator=g).bfloat16().cuda()
    out = torch.full_like(q, 3.0)
    ops.paged_attention_decode_int4(q, *cache, out, tables, segments, positions, 0.125, num_splits=splits, segment_start=start)
    for row, (s, p) in enumerate(zip(segments.tolist(), positions.tolist())):
        if counts[s] != 1:
            assert (out[row] == 3.0).all()
            continue
        k, v = request_rows(cache, tables[s], p + 1, 16)
        expected, weighed = plain.attend(q[row], k, v, p, 0.125)
        assert ((out[row].to(D64) - expected).abs() <= bound(expected, weighed)).all()


def test_rows_with_scores_far_apart():
    """Maxima that grow from tile to tile by far more than what is put off, and scores of minus and plus a thousand."""
    g = torch.Generator().manual_seed(8)
    dim, n = 128, 700
    cache = fill_cache(g, n // 16 + 1, 1, 16, dim)
    slope = torch.linspace(0.01, 60, n // 16 * 16 + 16).view(-1, 1, 16)
    cache[1][..., 0] = (slope / 16).bfloat16().cuda()
    cache[1][..., 1] = (slope / 40 * (-1) ** torch.arange(16)).bfloat16().cuda()
    tables = torch.arange(n // 16 + 1).int().cuda()[None]
    q = torch.randn((2, 8, dim), generator=g).bfloat16().cuda()
    for splits in (1, 5, 16):
        out = torch.empty_like(q)
        ops.paged_attention_decode_int4(q, *cache, out, tables, torch.zeros(2).int().cuda(), torch.tensor([n - 1, 40]).int().cuda(), 0.09, num_splits=splits)
        for row, p in enumerate((n - 1, 40)):
            k, v = request_rows(cache, tables[0], p + 1, 16)
            expected, weighed = plain.attend(q[row], k, v, p, 0.09)
            # scores up to about 10,000 in base two: float32 holds them to 2^-10 at best, so weights near the maximum are off by that
            assert ((out[row].to(D64) - expected).abs() <= bound(expected, weighed) + 2.0 ** -8 * weighed).all()


def test_a_row_that_is_not_a_number_reaches_who_reads_it():
    g = torch.Generator().manual_seed(9)
    cache = fill_cache(g, 8, 2, 16, 64)
    cache[1][3, 1, 5] = torch.tensor([0.0, math.nan])          # a key of head 1, position 53
    tables = torch.arange(8).int().cuda()[None]
    q = torch.randn((2, 4, 64), generator=g).bfloat16().cuda()
    for splits in (1, 2, 10):
        out = torch.empty_like(q)
        ops.paged_attention_decode_int4(q, *cache, out, tables, torch.zeros(2).int().cuda(), torch.tensor([127, 52]).int().cuda(), 0.125, num_splits=splits)
        assert out[0, 2:].isnan().all() and torch.isfinite(out[0, :2].float()).all() and torch.isfinite(out[1].float()).all()


def test_offsets_beyond_32_bits():
    """Codes of 2.4 GB: a page's place in bytes does not fit 31 bits."""
    n_kv, page_size, dim, pages = 8, 16, 128, 300_000
    codes = [torch.empty((pages, n_kv, page_size, dim // 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.empty((pages, n_kv, page_size, 2), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cache = (codes[0], scales[0], codes[1], scales[1])
    g = torch.Generator().manual_seed(2)
    tokens = 20
    qkv = torch.randn((tokens, 24 * dim), generator=g).bfloat16().cuda()
    table = torch.tensor([[pages - 1, 5]], dtype=torch.int32)
    slots = torch.tensor([int(table[0, j // 16]) * 16 + j % 16 for j in range(tokens)]).int().cuda()
    q = torch.empty((tokens, 8, dim), dtype=torch.bfloat16, device="cuda")
    at = torch.arange(tokens).int().cuda()
    ops.rope_kv_write_int4(qkv, None, at, slots, torch.ones(dim // 2, device="cuda"), q, *cache, 8, n_kv, dim, 1)
    out = torch.empty_like(q)
    ops.paged_attention_decode_int4(q, *cache, out, table.cuda(), torch.zeros_like(at), at, 0.1)
    k, v = request_rows(cache, table[0].cuda(), tokens, 16)
    for p in range(tokens):
        expected, weighed = plain.attend(q[p], k, v, p, 0.1)
        assert ((out[p].to(D64) - expected).abs() <= bound(expected, weighed)).all()


def test_rows_captured_and_on_another_stream():
    g = torch.Generator().manual_seed(4)
    cache = fill_cache(g, 80, 2, 16, 128)
    tables = torch.arange(80).int().cuda().view(2, 40)
    q = torch.randn((2, 12, 128), generator=g).bfloat16().cuda()
    segments, positions = torch.arange(2).int().cuda(), torch.tensor([600, 77]).int().cuda()

    def launch(out, splits):
        return ops.paged_attention_decode_int4(q, *cache, out, tables, segments, positions, 0.09, num_splits=splits)

    for splits in (1, 6, 24):
        want = launch(torch.empty_like(q), splits).clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = launch(torch.empty_like(q), splits)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(there, want)
        # two graphs of the same call, replayed side by side: neither has a workspace of the other's
        graphs, outs = [], []
        for _ in range(2):
            out = torch.zeros_like(q)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                launch(out, splits)
            graphs.append(graph)
            outs.append(out)
        positions.copy_(torch.tensor([300, 90]).int())
        want = launch(torch.empty_like(q), splits).clone()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for stream in streams:
            stream.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        positions.copy_(torch.tensor([600, 77]).int())


# ------------------------------------------------------------------ attention of prompt portions
def f16_bound(expected, weighed):
    """The result's rounding (2^-8 of it); values and weights in float16 (2^-11 of every term each); keys in float16, which move a score
    by up to 2^-11 of the sum of |q k| (see ``portions``: given there as a factor of the terms)."""
    return 2.0 ** -8 * expected.abs() + (2.0 ** -10 + 2.0 ** -14) * weighed + 1e-30


def portions(cache, tables, counts, firsts, q, out, scale, page_size, skip_single=False):
    """Every row of ``out`` against the plain form; returns how many were compared."""
    row, compared = 0, 0
    for s, (count, first) in enumerate(zip(counts, firsts)):
        if count:
            k, v = request_rows(cache, tables[s], first + count, page_size)
        for i in range(count):
            if not (skip_single and count == 1) and (i < 3 or i >= count - 3 or i % 29 == 0):
                expected, weighed = plain.attend(q[row], k, v, first + i, scale)
                # a key's rounding moves a score by at most 2^-11 sum |q k| scale, up and down: twice that in a weight's share
                reach = torch.einsum("hd,nhd->hn", q[row].to(D64).abs(), k[:first + i + 1].abs().repeat_interleave(q.shape[1] // k.shape[1], 1)).amax(-1) * scale
                assert ((out[row].to(D64) - expected).abs() <= f16_bound(expected, weighed) + 2.0 ** -10 * reach[:, None] * weighed).all(), (s, i)
                compared += 1
            row += 1
    return compared


def portion_case(counts, firsts, n_kv, dim, page_size, seed):
    g = torch.Generator().manual_seed(seed)
    held = [-(-(n + f) // page_size) if n else 0 for n, f in zip(counts, firsts)]
    cache = fill_cache(g, sum(held) + 1, n_kv, page_size, dim)
    order = torch.randperm(sum(held), generator=g).tolist()
    tables = torch.full((len(counts), max(held) + 1), -1, dtype=torch.int32)
    for s, n in enumerate(held):
        tables[s, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        if n:      # what lies behind the last key is anything at all
            rest = counts[s] + firsts[s] - (n - 1) * page_size
            for scales in (cache[1], cache[3]):
                scales[int(tables[s, n - 1]), :, rest:] = math.nan
    start = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()]).int().cuda()
    return g, cache, tables.cuda(), start, torch.tensor(firsts).int().cuda()


@pytest.mark.parametrize("counts,firsts,n_q,n_kv,dim,page_size", [
    ([1], [0], 2, 2, 64, 16), ([130], [0], 4, 4, 128, 16), ([3, 1, 0, 40], [5, 0, 0, 700], 12, 2, 128, 16), ([200, 77, 2], [0, 300, 1500], 28, 4, 128, 8),
    ([5], [4000], 40, 8, 128, 32), ([260], [33], 7, 1, 64, 5), ([129, 128, 127], [127, 128, 1], 5, 5, 64, 128), ([20, 9], [0, 250], 128, 1, 64, 16),
    ([400], [2000], 9, 3, 128, 24)])
def test_portions(counts, firsts, n_q, n_kv, dim, page_size):
    g, cache, tables, start, first = portion_case(counts, firsts, n_kv, dim, page_size, sum(counts))
    tokens = sum(counts)
    q = (1.5 * torch.randn((tokens + 3, n_q, dim), generator=g)).bfloat16().cuda()
    scale = dim ** -0.5
    for keys in (0, sum(counts) + sum(firsts)):
        out = torch.full_like(q, 3.0)
        ops.paged_attention_prefill_int4(q, *cache, out, tables, start, first, scale, keys=keys)
        assert portions(cache, tables, counts, firsts, q, out, scale, page_size) >= min(tokens, 5)
        assert (out[tokens:] == 3.0).all()          # rows behind the last sequence
    single = torch.full_like(q, 3.0)
    ops.paged_attention_prefill_int4(q, *cache, single, tables, start, first, scale, skip_single=True, max_portions=sum(n > 1 for n in counts))
    row = 0
    for n in counts:
        assert (single[row:row + n] == 3.0).all() if n == 1 else torch.equal(single[row:row + n], out[row:row + n])
        row += n


def test_portions_some_heads_at_a_time(monkeypatch):
    counts, firsts = [50, 30], [300, 0]
    g, cache, tables, start, first = portion_case(counts, firsts, 5, 64, 16, 1)
    q = torch.randn((80, 10, 64), generator=g).bfloat16().cuda()
    want = ops.paged_attention_prefill_int4(q, *cache, torch.empty_like(q), tables, start, first, 0.125)
    monkeypatch.setattr(ops, "INT4_WORKSPACE_BYTES", 1)
    out = ops.paged_attention_prefill_int4(q, *cache, torch.empty_like(q), tables, start, first, 0.125)
    portions(cache, tables, counts, firsts, q, out, 0.125, 16)
    portions(cache, tables, counts, firsts, q, want, 0.125, 16)


def test_portions_with_scores_far_apart():
    """Maxima that grow by more than float16 reaches from one tile to the next."""
    counts, firsts = [300], [600]
    g, cache, tables, start, first = portion_case(counts, firsts, 1, 128, 16, 2)
    pages = tables[0, :57].long()
    ramp = torch.linspace(0.05, 6.0, 57).view(-1, 1, 1).cuda()
    cache[1][pages, :, :, 0] = (ramp * cache[1][pages, :, :, 0].float().nan_to_num(0.3)).bfloat16()
    cache[1][pages, :, :, 1] = 0.0
    q = (4 * torch.randn((300, 6, 128), generator=g)).bfloat16().cuda()
    out = ops.paged_attention_prefill_int4(q, *cache, torch.empty_like(q), tables, start, first, 0.09)
    portions(cache, tables, counts, firsts, q, out, 0.09, 16)


def test_portions_reach_of_what_is_not_a_number():
    """A key or value that is not a number, or beyond float16, reaches the rows that see it and no others."""
    for index, wrong in ((1, math.nan), (3, math.nan), (3, 1e5), (3, math.inf), (1, 1e8)):
        counts, firsts = [140], [20]
        g, cache, tables, start, first = portion_case(counts, firsts, 2, 64, 16, 3)
        cache[index][int(tables[0, 5]), 1, 4, 1] = wrong          # position 84 of head 1
        q = torch.randn((140, 4, 64), generator=g).bfloat16().cuda()
        out = ops.paged_attention_prefill_int4(q, *cache, torch.empty_like(q), tables, start, first, 0.125)
        sees = torch.arange(20, 160).cuda() >= 84
        assert torch.isfinite(out[:, :2].float()).all() and torch.isfinite(out[~sees].float()).all() and out[sees][:, 2:].isnan().all()


def test_portions_beyond_the_announced_keys_are_not_made_up():
    counts, firsts = [10, 10, 10], [300, 300, 300]
    g, cache, tables, start, first = portion_case(counts, firsts, 1, 64, 16, 4)
    q = torch.randn((30, 2, 64), generator=g).bfloat16().cuda()
    out = ops.paged_attention_prefill_int4(q, *cache, torch.empty_like(q), tables, start, first, 0.125, keys=310)     # room for 2 + 3 tiles, 9 are held
    assert torch.isfinite(out[:10].float()).all() and out[10:].isnan().all()


def test_portions_captured():
    counts, firsts = [33, 64], [500, 10]
    g, cache, tables, start, first = portion_case(counts, firsts, 2, 128, 16, 5)
    q = torch.randn((97, 8, 128), generator=g).bfloat16().cuda()
    outs, graphs = [torch.empty_like(q) for _ in range(2)], []
    want = ops.paged_attention_prefill_int4(q, *cache, torch.empty_like(q), tables, start, first, 0.09)
    for out in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention_prefill_int4(q, *cache, out, tables, start, first, 0.09)
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for graph, stream in zip(graphs, streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(3):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@pytest.mark.parametrize("splits", [1, 4, 24])
def test_attention_behind_the_write_of_its_queries(splits):
    """A graph of writes and attention that share a buffer for their queries, launches without a gap: each sees the write before it."""
    g = torch.Generator().manual_seed(6)
    layers, rows, n_q, n_kv, dim = 4, 3, 6, 2, 128
    caches = [fill_cache(g, 24, n_kv, 16, dim) for _ in range(layers)]
    tables = torch.arange(24).int().cuda().view(rows, 8)
    segments, positions = torch.arange(rows).int().cuda(), torch.tensor([41, 100, 7]).int().cuda()
    slots = (tables[segments.long(), positions.long() // 16] * 16 + positions % 16).int()
    inv_freq = torch.full((dim // 2,), 0.01, device="cuda")
    qkv = torch.empty((layers, rows, (n_q + 2 * n_kv) * dim), device="cuda")
    q = torch.empty((rows, n_q, dim), dtype=torch.bfloat16, device="cuda")
    outs = torch.empty((layers, rows, n_q, dim), dtype=torch.bfloat16, device="cuda")

    def run(between):
        for cache, x, out in zip(caches, qkv, outs):
            ops.rope_kv_write_int4(x, None, positions, slots, inv_freq, q, *cache, n_q, n_kv, dim, 1)
            between()
            ops.paged_attention_decode_int4(q, *cache, out, tables, segments, positions, 0.09, num_splits=splits)
            between()

    run(torch.cuda.synchronize)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(lambda: None)
    for _ in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        run(torch.cuda.synchronize)
        want = outs.clone()
        q.fill_(math.nan)
        outs.zero_()
        graph.replay()
        assert torch.equal(outs, want)


@pytest.mark.parametrize("dim,pairing", [(64, 0), (128, 1)])
def test_write_of_rows_on_the_borders_of_rounding(dim, pairing):
    """Ranges and centres half way between two bfloat16 numbers, or a last place of float32 beside, and values half way between codes."""
    g = torch.Generator().manual_seed(dim)
    tokens, n_q, n_kv = 400, 1, 4
    x = torch.randint(-128, 128, (tokens, n_q + 2 * n_kv, dim), generator=g).float() / 16
    lows = torch.randint(-64, 0, (tokens, n_q + 2 * n_kv), generator=g).float() / 8
    steps = (torch.randint(256, 512, lows.shape, generator=g).float() + 0.5) / 512           # half way between two of 8 bits
    x = torch.maximum(torch.minimum(x, (lows + 15 * steps)[..., None]), lows[..., None])
    x[..., 5], x[..., dim - 3] = lows, lows + 15 * steps
    beside = torch.randint(-1, 2, lows.shape, generator=g)
    x[..., 5] = torch.where(beside == 0, x[..., 5], torch.nextafter(x[..., 5], beside.float() * 1e9))
    slots = torch.arange(tokens).int().cuda()
    cache = empty_cache(tokens // 16, n_kv, 16, dim)
    q = torch.empty((tokens, n_q, dim), dtype=torch.bfloat16, device="cuda")
    zero = torch.zeros(dim // 2, device="cuda")               # no angles: a rotation that changes nothing
    ops.rope_kv_write_int4(x.flatten(1).cuda(), None, slots, slots, zero, q, *cache, n_q, n_kv, dim, pairing)
    page, at = slots.long() // 16, slots.long() % 16
    for rows, codes, scales in ((x[:, n_q:n_q + n_kv], cache[0], cache[1]), (x[:, n_q + n_kv:], cache[2], cache[3])):
        u, s, c = plain.quantise(rows.to(D64).cuda())
        assert torch.equal(scales[page, :, at], torch.stack([s, c], -1).bfloat16())
        assert torch.equal(codes[page, :, at], plain.pack(u))


def test_portions_of_many_requests():
    """More requests than a warp has lanes, with none, one or many rows."""
    counts = [(s * 7) % 23 if s % 5 else s % 2 for s in range(75)]
    firsts = [(s * 37) % 190 for s in range(75)]
    g, cache, tables, start, first = portion_case(counts, firsts, 2, 64, 16, 9)
    tokens = sum(counts)
    q = torch.randn((tokens, 10, 64), generator=g).bfloat16().cuda()
    for singles in (False, True):
        out = torch.full_like(q, 3.0)
        ops.paged_attention_prefill_int4(q, *cache, out, tables, start, first, 0.125, keys=tokens + sum(firsts), skip_single=singles)
        assert portions(cache, tables, counts, firsts, q, out, 0.125, 16, singles) > 200
        if singles:
            alone = torch.tensor([n == 1 for n in counts for _ in range(n)]).cuda()
            assert (out[alone] == 3.0).all() and alone.any()


@pytest.mark.parametrize("splits", [2, 24])
def test_rows_of_many_requests(splits):
    """More rows than a block has threads, padding and empty rows among them."""
    g = torch.Generator().manual_seed(12)
    rows = 300
    cache = fill_cache(g, 4 * rows, 1, 16, 64)
    tables = torch.randperm(4 * rows, generator=g).int().view(rows, 4).cuda()
    positions = torch.randint(0, 64, (rows,), generator=g)
    positions[::17] = -1
    segments = torch.randperm(rows, generator=g)
    segments[5::31] = -1
    q = torch.randn((rows, 3, 64), generator=g).bfloat16().cuda()
    out = torch.full_like(q, 3.0)
    ops.paged_attention_decode_int4(q, *cache, out, tables, segments.int().cuda(), positions.int().cuda(), 0.125, num_splits=splits)
    for row, (segment, position) in enumerate(zip(segments.tolist(), positions.tolist())):
        if segment < 0:
            assert (out[row] == 3.0).all()
        elif position < 0:
            assert (out[row] == 0.0).all()
        else:
            k, v = request_rows(cache, tables[segment], position + 1, 16)
            expected, weighed = plain.attend(q[row], k, v, position, 0.125)
            # What is rounded to bfloat16 (2^-8) is weight times scale, of which a value takes u - 8: a term is off by 2^-8 of the value's
            # distance from its row's centre, which with few keys is more than 2^-8 of the value where the two have other signs.
            pages = tables[segment, :position // 16 + 1].long()
            centre = cache[3][pages][..., 1].to(D64).transpose(1, 2).flatten(0, 1)[:position + 1, :, None]
            _, apart = plain.attend(q[row], k, v - centre, position, 0.125)
            assert ((out[row].to(D64) - expected).abs() <= bound(expected, apart) + 2.0 ** -14 * weighed).all(), row
