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
