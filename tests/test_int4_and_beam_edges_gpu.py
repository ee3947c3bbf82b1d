"""The 4-bit cache, beam search and a step's tables at their edges, on the GPU."""
import random

import pytest
import torch

import helpers
from llm_serving_engine_b200.kernels import ops
from plain import int4_plain as plain
from test_beam_engine_gpu import engine_of, models
from test_int4_cache_gpu import fill_cache, portions, portion_case

pytestmark = pytest.mark.gpu

D64 = torch.float64


def shifted(tensor):
    """The same numbers four bytes further from a 16-byte boundary."""
    room = torch.empty(tensor.numel() + 2, dtype=tensor.dtype, device=tensor.device)
    view = room[2:].view(tensor.shape)
    view.copy_(tensor)
    assert view.data_ptr() % 16 == 4
    return view


@pytest.mark.parametrize("dim", [64, 128])
def test_scales_of_small_pages_begin_anywhere(dim):
    """Pages whose rows are no multiple of four: a layer's scales begin at a multiple of four bytes, not of sixteen."""
    counts, firsts, page_size = [40, 3], [7, 60], 5
    g, cache, tables, start, first = portion_case(counts, firsts, 2, dim, page_size, dim)
    odd = [cache[0], shifted(cache[1]), cache[2], shifted(cache[3])]
    q = torch.randn((43, 6, dim), generator=g).bfloat16().cuda()
    segments = torch.tensor([0] * 40 + [1] * 3).int().cuda()
    positions = torch.cat([torch.arange(n) + f for n, f in zip(counts, firsts)]).int().cuda()
    slots = (tables[segments.long(), positions.long() // page_size] * page_size + positions % page_size).int()
    qkv = torch.randn((43, (6 + 4) * dim), generator=g).cuda()
    frequencies = torch.full((dim // 2,), 0.01, device="cuda")
    made = []
    for pages in (cache, odd):
        got = [torch.empty_like(q)]
        ops.rope_kv_write_int4(qkv, None, positions, slots, frequencies, got[0], *pages, 6, 2, dim, 1)
        got += [torch.empty((43, 2, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        ops.kv_read_int4(*pages, slots, *got[1:])
        got += [ops.paged_attention_decode_int4(q, *pages, torch.empty_like(q), tables, segments, positions, 0.1, num_splits=n) for n in (1, 4, 20)]
        got.append(ops.paged_attention_prefill_int4(q, *pages, torch.empty_like(q), tables, start, first, 0.1))
        made.append([*got, pages[1].clone(), pages[3].clone()])
    for a, b in zip(*made):
        assert torch.equal(torch.nan_to_num(a, nan=1e4), torch.nan_to_num(b, nan=1e4))


def test_an_engine_of_small_pages_and_an_odd_number_of_them():
    from llm_serving_engine_b200 import GenerationConfig
    model, rng = models(), random.Random(8)
    prompts = [helpers.random_tokens(rng, 512, n) for n in (3, 41)]
    made = []
    for pages in (100, 101):           # 100: every layer's scales begin at a multiple of 16 bytes
        engine = engine_of(model, page=5, pages=pages, kv_bits=4)
        aligned = all(view.value_scales.data_ptr() % 16 == 0 for view in (engine.cache.layer_view(layer) for layer in range(3)))
        assert aligned == (pages == 100)
        made.append(engine.generate_many(prompts, GenerationConfig(max_new_tokens=9)))
        made[-1].append([beam.tokens for beams in engine.beam_search(prompts, 3, 6, 9) for beam in beams])
    assert made[0] == made[1]


# ------------------------------------------------------------------ searches whose steps are not valid
@pytest.mark.parametrize("count", [3, 24])
def test_a_search_whose_kernels_gave_up_raises_and_leaves_the_engine_usable(count):
    """The few-rows product is made to give up a wait (a test hook: a tile that never arrives and a small limit; the kernel
    returns): beams of such steps are not handed out, and neither the pages nor the word are left to the next caller."""
    from llm_serving_engine_b200 import GenerationConfig
    from test_engine_gpu import engine_for, prompts_for
    engine = engine_for("D", dtype="bfloat16", batch=6)
    prompts = prompts_for("D", (9, 21), seed=4)
    good, tokens = engine.beam_search(prompts, 3, count, 5), engine.generate_many(prompts, GenerationConfig(max_new_tokens=4))
    ops.gemm_bf16_skinny_test_hooks(spin_limit=2000, withhold=True)
    try:
        with pytest.raises(ops.KernelError, match="bounded wait inside the few-rows product"):
            engine.beam_search(prompts, 3, count, 5)
    finally:
        ops.gemm_bf16_skinny_test_hooks()
    assert ops.gemm_bf16_skinny_status() == 0
    assert not engine.cache.requests and engine.cache.groups[0].pool.used_pages == 0
    assert engine.generate_many(prompts, GenerationConfig(max_new_tokens=4)) == tokens
    assert engine.beam_search(prompts, 3, count, 5) == good


@pytest.mark.parametrize("word", range(6))
def test_every_status_word_fails_a_search(word, monkeypatch):
    """Whichever kernel's word comes back set, at the look in between (16 tokens) or at the end."""
    engine = engine_of(models(), kv_bits=4)
    plain_read = ops.kernel_status_async

    def spoilt(words):
        plain_read(words)
        torch.cuda.current_stream().synchronize()
        words[word] = 1

    for count in (4, 20):
        monkeypatch.setattr(ops, "kernel_status_async", spoilt)
        with pytest.raises(ops.KernelError, match=f"bounded wait inside {ops._STATUS_NAMES[word]}"):
            engine.beam_search([[3, 5, 8]], 4, count, 9)
        monkeypatch.setattr(ops, "kernel_status_async", plain_read)
        assert not engine.cache.requests and len(engine.beam_search([[3, 5, 8]], 4, count, 9)[0]) == 4


def test_logits_that_are_not_numbers_leave_no_beam_and_are_told():
    model = models()
    engine = engine_of(model)
    kept = model.final_norm.weight.clone()
    model.final_norm.weight.fill_(float("nan"))
    with pytest.raises(ops.KernelError, match="not numbers"):
        engine.beam_search([[3, 5, 8], [1]], 4, 5, 9)
    model.final_norm.weight.copy_(kept)
    assert not engine.cache.requests and [len(beams) for beams in engine.beam_search([[3, 5, 8], [1]], 4, 5, 9)] == [4, 4]


# ------------------------------------------------------------------ prompt portions over numbers of any size
def times(cache, keys, values):
    """The cache of ``keys`` times its keys and ``values`` times its values (powers of two: scales and centres hold them exactly)."""
    return cache[0], (cache[1].float() * keys).bfloat16(), cache[2], (cache[3].float() * values).bfloat16()


@pytest.mark.parametrize("counts,firsts,n_q,n_kv,dim", [([130, 1, 9], [20, 5, 700], 6, 2, 64), ([70], [3000], 5, 1, 128)])
@pytest.mark.parametrize("key,query,value", [(-14, 0, -14), (-28, 6, -28), (-10, -20, -40), (6, 100, -5), (-50, 50, 8), (0, -60, 3)])
def test_portions_know_no_size(counts, firsts, n_q, n_kv, dim, key, query, value):
    """Keys, queries and values times powers of two, the score's scale divided by them: the same results, to the last bit, times the values'.
    (Every rounding is relative: nothing is small enough to lose bits, and nothing large enough to leave the range.)"""
    g, cache, tables, start, first = portion_case(counts, firsts, n_kv, dim, 16, 11)
    q = torch.randn((sum(counts), n_q, dim), generator=g).bfloat16().cuda()
    want = ops.paged_attention_prefill_int4(q, *cache, torch.empty_like(q), tables, start, first, 0.125)
    assert portions(cache, tables, counts, firsts, q, want, 0.125, 16) >= 8
    got = ops.paged_attention_prefill_int4((q.float() * 2.0 ** query).bfloat16(), *times(cache, 2.0 ** key, 2.0 ** value), torch.empty_like(q), tables, start, first,
                                           0.125 * 2.0 ** (-key - query))
    assert torch.isfinite(want.float()).all() and torch.equal(got, (want.float() * 2.0 ** value).bfloat16())


@pytest.mark.parametrize("page_size", [16, 5])
def test_portions_whose_requests_and_heads_are_of_different_sizes(page_size):
    """A request's numbers do not decide about another's bits, nor a head's about another's; within a request, keys and values that
    grow by 2^20 from its first to its last, so that early rows see small ones only."""
    counts, firsts, n_kv, dim = [40, 150, 33], [0, 200, 600], 2, 64
    g, cache, tables, start, first = portion_case(counts, firsts, n_kv, dim, page_size, 12)
    q = torch.randn((sum(counts), 6, dim), generator=g).bfloat16().cuda()
    for s, (size, steepness) in enumerate(((-20, 0), (2, 0), (-12, 20))):
        pages = tables[s][tables[s] >= 0].long()
        ramp = 2.0 ** (size + torch.linspace(-steepness, 0, len(pages)).round().cuda()).view(-1, 1, 1, 1)
        heads = torch.tensor([1.0, 2.0 ** -9], device="cuda").view(1, 2, 1, 1)
        for scales in (cache[1], cache[3]):
            scales[pages] = (scales[pages].float() * ramp * heads).bfloat16()
    q[:40] *= 2.0 ** 18
    out = ops.paged_attention_prefill_int4(q, *cache, torch.empty_like(q), tables, start, first, 0.5)
    assert portions(cache, tables, counts, firsts, q, out, 0.5, page_size) >= 15


def test_portions_over_zeros():
    """Keys that are all zero weigh alike; values that are all zero give zeros."""
    counts, firsts = [40], [100]
    g, cache, tables, start, first = portion_case(counts, firsts, 1, 64, 16, 13)
    q = torch.randn((40, 2, 64), generator=g).bfloat16().cuda()
    for keys, values in ((0.0, 1.0), (1.0, 0.0), (0.0, 0.0)):
        some = times(tuple(t.nan_to_num(0.0) if t.is_floating_point() else t for t in cache), keys, values)
        out = ops.paged_attention_prefill_int4(q, *some, torch.empty_like(q), tables, start, first, 0.125)
        assert portions(some, tables, counts, firsts, q, out, 0.125, 16) >= 6
        assert values or not out.any()


# ------------------------------------------------------------------ the checked variant of the kernels
CHECKED = r"""
import random, sys
sys.path.insert(0, {tests!r}); sys.path.insert(0, {root!r})
import torch
import helpers
from test_beam_engine_gpu import engine_of, models
from llm_serving_engine_b200 import GenerationConfig
from llm_serving_engine_b200.engine import StepEntry
from llm_serving_engine_b200.kernels import library

model, rng = models(), random.Random(3)
for page in (16, 8, 5):
    engine = engine_of(model, page=page, pages=301, kv_bits=4)
    engine.generate_many([helpers.random_tokens(rng, 512, n) for n in (3, 70, 130, 33)], GenerationConfig(max_new_tokens=12))
    engine.beam_search([helpers.random_tokens(rng, 512, n) for n in (21, 37)], 5, 9, 7)
    assert library.check_report() == [], library.check_report()
for source in ("int4_cache", "attention_int4", "attention_int4_tcgen05", "beam_search", "step_tables"):
    assert library.load().source_loaded(source), source
print("clean: nothing recorded")

# a table entry of -1 inside the context, made on the host: replaced and recorded by the kernels of portions and of rows
for page, kernel in ((16, "attention_int4_tc"), (16, "attention_int4"), (5, "attention_int4_tc"), (5, "attention_int4")):
    engine = engine_of(model, page=page, pages=100, kv_bits=4)
    engine.runner.use_graphs = False
    cache, tokens = engine.cache, helpers.random_tokens(rng, 512, 70)
    cache.create("r")
    engine.runner.run([StepEntry("r", tokens[:60], [])])
    request = cache.requests["r"]
    kept = request.tables[0][1]
    request.tables[0][1] = request.tables_np[0][1] = -1
    engine.runner.run([StepEntry("r", tokens[60:62] if kernel.endswith("tc") else tokens[60:61], [0])])
    torch.cuda.synchronize()
    report = library.check_report()
    assert [line for line in report if line.startswith(kernel + ":")] and all("block-table entry -1" in line for line in report), report
    request.tables[0][1] = request.tables_np[0][1] = kept
    cache.free("r")
    print("recorded:", report)
"""


def test_the_checked_kernels_of_the_4_bit_cache_record_nothing_on_good_steps_and_a_bad_table_entry():
    import os
    import subprocess
    import sys
    tests = os.path.dirname(os.path.abspath(__file__))
    done = subprocess.run([sys.executable, "-c", CHECKED.format(tests=tests, root=os.path.dirname(tests))], env=dict(os.environ, LSE_CHECK="1"),
                          capture_output=True, text=True, timeout=900)
    assert done.returncode == 0, done.stdout[-3000:] + done.stderr[-3000:]
    assert "clean: nothing recorded" in done.stdout and done.stdout.count("recorded:") == 4


# ------------------------------------------------------------------ what a beam's cache holds
def held_rows(cache, layer, table, length):
    """Keys and values [length, heads, D] of a layer behind a block table, and the step of the codes (zero in bfloat16) [length, heads]."""
    view, places = cache.layer_view(layer), torch.arange(length, device="cuda")
    slots = (table[places // cache.page_size] * cache.page_size + places % cache.page_size).int()
    if view.key_scales is None:
        page, at = slots.long() // cache.page_size, slots.long() % cache.page_size
        return [(t[page, :, at].double(), torch.zeros((length, t.shape[1]), device="cuda")) for t in (view.keys, view.values)]
    k, v = (torch.empty((length, view.keys.shape[1], 2 * view.keys.shape[3]), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.kv_read_int4(view.keys, view.key_scales, view.values, view.value_scales, slots, k, v)
    page, at = slots.long() // cache.page_size, slots.long() % cache.page_size
    return [(k.double(), view.key_scales[page, :, at, 0].double()), (v.double(), view.value_scales[page, :, at, 0].double())]


def same_rows(got, want) -> bool:
    """Rows of two steps over the same tokens: numbers of a bfloat16 model within the suite's bound of what another batch gives (8 units of
    2^-8 of the largest of a row); held in 4 bits, each off by half a step of its own row, and by what the rounded scale (15 steps of
    2^-8) and centre (2^-8 of the number) move the range's ends; 2^-8 once more from reading back."""
    for (a, step_a), (b, step_b) in zip(got, want):
        most = torch.maximum(a.abs(), b.abs()).amax(-1, keepdim=True)
        steps = torch.maximum(step_a, step_b)[..., None]
        if not ((a - b).abs() <= (8 + 3) * 2.0 ** -8 * most + (1 + 2 * 15 * 2.0 ** -8) * steps).all():
            return False
    return True


@pytest.mark.parametrize("kv_bits,page,beams,lengths", [(4, 16, 6, (37, 80)), (4, 5, 3, (21, 40)), (0, 16, 6, (37, 80)), (0, 16, 4, (30,))])
def test_a_beams_pages_hold_the_keys_and_values_of_its_own_tokens(kv_bits, page, beams, lengths, monkeypatch):
    """After any number of choices, pages shared, taken over and copied: layer by layer what one plain step over a beam's whole sequence
    writes, and not what another beam's would."""
    from llm_serving_engine_b200.engine import BeamSearch, StepEntry, beam_search
    engine = engine_of(models(), page=page, pages=400, kv_bits=kv_bits)
    steps = []

    class Watched(beam_search._Step):
        def __init__(self, *args):
            super().__init__(*args)
            self.chosen = []
            steps.append(self)

        def choose(self, logits):
            out = super().choose(logits)
            self.chosen.append(out.clone())
            return out

    monkeypatch.setattr(beam_search, "_Step", Watched)
    rng = random.Random(7)
    prompts = [helpers.random_tokens(rng, 512, n) for n in lengths]
    for count in (2, 25):
        for use_graph in (False, True):
            BeamSearch(engine.runner, beams, 9, use_graph=use_graph).search(prompts, count)
            watched = steps.pop()
            held, told = watched.held, {}
            fed = [part.tolist() for part in torch.stack(watched.chosen[:count - 1]).cpu()]      # the last choice was not run
            told = {}
            for request, prompt in enumerate(prompts):
                for beam in range(beams):
                    at, tokens = beam, []
                    for chosen, parents in reversed(fed):
                        tokens.append(chosen[request][at])
                        at = parents[request][at]
                    told[request, beam] = [*prompt, *reversed(tokens)]
            assert held.row_lengths.tolist() == [len(told[key]) for key in sorted(told)]
            tables = held.tables[0].clone()
            kept = {key: [held_rows(engine.cache, layer, tables[key[0] * beams + key[1]], len(sequence)) for layer in range(3)] for key, sequence in told.items()}
            plain_rows = {}
            for key, sequence in told.items():
                engine.cache.create("told")
                engine.runner.run([StepEntry("told", sequence, [])])
                table = torch.tensor(engine.cache.block_table(0, "told"), device="cuda")
                plain_rows[key] = [held_rows(engine.cache, layer, table, len(sequence)) for layer in range(3)]
                engine.cache.free("told")
            for key, sequence in told.items():
                assert all(same_rows(got, want) for got, want in zip(kept[key], plain_rows[key])), (key, count)
                for other, another in told.items():
                    if other[0] == key[0] and another != sequence:       # the bound tells one beam's rows from another's, in every layer
                        assert not any(same_rows(got, want) for got, want in zip(kept[key], plain_rows[other])), (key, other)
