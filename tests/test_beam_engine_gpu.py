"""Beam search and caches of 4 bits through the engine: the choice, the pages and states behind it, whole models."""
import math
import random

import pytest
import torch

import helpers
from plain import qwen2_plain
from tiny_configs import ALL

pytestmark = pytest.mark.gpu


def engine_of(model, page=16, pages=400, batch=24, budget=256, kv_bits=0):
    from llm_serving_engine_b200 import CacheConfig, LLMEngine, SchedulerConfig
    return LLMEngine(model, None, cache_config=CacheConfig(page, pages, kv_bits=kv_bits),
                     scheduler_config=SchedulerConfig(max_batch_size=batch, max_tokens_per_step=budget))


def plain_beams(name, prompt, beams, count, end_token):
    """Beam search by sorting, every step from the whole sequences."""
    cfg, weights = qwen2_plain.load_folder(helpers.model_folder(name))
    held = [([], 0.0, False)]
    for _ in range(count):
        offers = []
        for index, (tokens, score, ended) in enumerate(held):
            if ended:
                offers.append((score, index, end_token, tokens, True))
                continue
            logits = torch.as_tensor(qwen2_plain.forward_full(cfg, weights, [*prompt, *tokens])[-1]).double()
            logs = torch.log_softmax(logits, -1)
            for token in torch.topk(logs, beams).indices.tolist():
                offers.append((score + float(logs[token]), index, token, [*tokens, token], token == end_token))
        offers.sort(key=lambda o: (-o[0], o[1], o[2]))
        held = [(tokens, score, ended) for score, _, _, tokens, ended in offers[:beams]]
    return held


@pytest.mark.parametrize("name,lengths,beams,count", [("A", (5, 16, 30), 4, 9), ("B", (7, 25), 3, 12)])
def test_beams_equal_the_plain_search(name, lengths, beams, count):
    from llm_serving_engine_b200 import load_model
    rng = random.Random(1)
    vocab = ALL[name][0]["vocab_size"]
    prompts = [helpers.random_tokens(rng, vocab, n) for n in lengths]
    engine = engine_of(load_model(helpers.model_folder(name), dtype="float32", device="cuda"), page=8)
    for end_token in (3, vocab - 1):
        found = engine.beam_search(prompts, beams, count, end_token)
        assert not engine.cache.requests and engine.cache.groups[0].pool.used_pages == 0
        for prompt, got in zip(prompts, found):
            want = plain_beams(name, prompt, beams, count, end_token)
            assert [beam.tokens for beam in got] == [tokens[:tokens.index(end_token)] if ended else tokens for tokens, _, ended in want]
            assert [beam.ended for beam in got] == [ended for _, _, ended in want]
            # float32 logits of about a unit: 256 units of rounding each, over the tokens
            assert all(abs(beam.score - score) <= count * 256 * 2.0 ** -24 * 4 for beam, (_, score, _) in zip(got, want))


def told_scores(engine, prompt, beam, end_token):
    """The sum of the log probabilities of a beam's tokens, from one step over the whole sequence."""
    from llm_serving_engine_b200.engine import StepEntry
    tokens = beam.tokens + ([end_token] if beam.ended else [])
    engine.cache.create("told")
    try:
        sequence = [*prompt, *tokens]
        logits = engine.runner.run([StepEntry("told", sequence[:-1], list(range(len(prompt) - 1, len(sequence) - 1)))])
        logs = torch.log_softmax(logits.double(), -1)
        return float(sum(logs[i, token] for i, token in enumerate(tokens)))
    finally:
        engine.cache.free("told")


@pytest.mark.parametrize("design", ["tiny", "givelix", "tufevik", "kofipel", "daferax", "sebudra", "fororax"])
def test_a_beams_score_is_what_the_model_gives_its_tokens(design):
    """Pages, windows, latents, states of every design: after any number of choices a beam's cache is that of its own tokens."""
    from llm_serving_engine_b200 import random_model
    from llm_serving_engine_b200.cli import tiny_config
    rng = random.Random(2)
    model = random_model(tiny_config(300, design), 5, dtype="float32", device="cuda")
    engine = engine_of(model, page=16)
    prompts = [helpers.random_tokens(rng, model.vocab_size, n) for n in (21, 64, 3)]
    for use_graph in (False, True):
        from llm_serving_engine_b200.engine import BeamSearch
        found = BeamSearch(engine.runner, 5, 7, use_graph=use_graph).search(prompts, 40)
        for prompt, beams in zip(prompts, found):
            assert len({tuple(beam.tokens) for beam in beams}) == len(beams) and [b.score for b in beams] == sorted((b.score for b in beams), reverse=True)
            for beam in beams[:3]:
                # logits of up to about 8, forty of them, each off by 256 float32 roundings at most
                assert abs(told_scores(engine, prompt, beam, 7) - beam.score) <= 40 * 8 * 256 * 2.0 ** -24


def test_beams_refuse():
    from llm_serving_engine_b200 import random_model
    from llm_serving_engine_b200.cache.manager import CacheFullError
    from llm_serving_engine_b200.cli import tiny_config
    engine = engine_of(random_model(tiny_config(300, "tiny"), 5, dtype="float32", device="cuda"), pages=12, batch=8)
    for prompts, beams, count, end in (([[1]], 0, 4, 2), ([[1]], 33, 4, 2), ([[1]], 4, 4, 999_999), ([[]], 4, 4, 2), ([[1]], 4, 0, 2), ([[1]] * 3, 4, 4, 2), ([[-1]], 4, 4, 2)):
        with pytest.raises(ValueError):
            engine.beam_search(prompts, beams, count, end)
    with pytest.raises(CacheFullError):
        engine.beam_search([[1] * 20], 8, 60, 2)
    assert engine.cache.groups[0].pool.used_pages == 0 and not engine.cache.requests
    assert len(engine.beam_search([[1] * 20], 8, 4, 2)[0]) == 8


# ------------------------------------------------------------------ caches of 4 bits
CONFIG = {"architectures": ["Qwen2ForCausalLM"], "model_type": "qwen2", "vocab_size": 512, "hidden_size": 256, "intermediate_size": 512,
          "num_hidden_layers": 3, "num_attention_heads": 6, "num_key_value_heads": 2, "head_dim": 128, "max_position_embeddings": 2048,
          "rope_theta": 10000.0, "rms_norm_eps": 1e-6, "tie_word_embeddings": True, "attention_bias": True}


def models(seed=3):
    from llm_serving_engine_b200 import random_model
    return random_model(CONFIG, seed, dtype="bfloat16", device="cuda")


def test_a_cache_of_4_bits_is_one_of_the_values_that_it_holds(monkeypatch):
    """Logits over 4-bit pages against a bfloat16 cache into which the same values are written: portions, rows and both together."""
    from llm_serving_engine_b200.engine import StepEntry
    from llm_serving_engine_b200.kernels import ops
    from llm_serving_engine_b200.parts.rope import RotaryEncoding
    model = models()
    rng = random.Random(4)
    first, second = helpers.random_tokens(rng, 512, 150), helpers.random_tokens(rng, 512, 40)

    def steps(engine):
        run, got = engine.runner.run, []
        for name in "ab":
            engine.cache.create(name)
        got.append(run([StepEntry("a", first[:90], [0, 50, 89])]).clone())
        got.append(run([StepEntry("a", first[90:91], [0]), StepEntry("b", second[:30], [29])]).clone())
        got.append(run([StepEntry("a", first[91:130], [38]), StepEntry("b", second[30:31], [0])]).clone())
        for i in range(9):
            got.append(run([StepEntry("a", first[130 + i:131 + i], [0]), StepEntry("b", second[31 + i:32 + i], [0])]).clone())
        return torch.cat(got).double()

    four = steps(engine_of(model, kv_bits=4))
    plain_store = RotaryEncoding.encode_and_store

    def store(self, qkv, bias, step, cache, q_out, n_q, n_kv, head_dim):
        pages, heads, page_size, dim = cache.keys.shape
        held = [torch.zeros((pages, heads, page_size, dim // 2), dtype=torch.uint8, device="cuda"), torch.zeros((pages, heads, page_size, 2), dtype=torch.bfloat16, device="cuda")]
        held += [t.clone() for t in held]
        ops.rope_kv_write_int4(qkv, bias, step.positions, cache.slot_mapping, self.inv_freq, q_out, *held, n_q, n_kv, head_dim, self.pairing)
        rows = q_out.shape[0]
        k, v = (torch.empty((rows, n_kv, head_dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        ops.kv_read_int4(*held, cache.slot_mapping, k, v)
        slots = cache.slot_mapping[:rows].long()
        live = slots >= 0
        cache.keys[slots[live] // page_size, :, slots[live] % page_size] = k[live]
        cache.values[slots[live] // page_size, :, slots[live] % page_size] = v[live]

    monkeypatch.setattr(RotaryEncoding, "encode_and_store", store)
    wide_engine = engine_of(model)
    wide_engine.runner.use_graphs = False
    wide = steps(wide_engine)
    monkeypatch.setattr(RotaryEncoding, "encode_and_store", plain_store)
    # the bfloat16 bounds of the whole suite (helpers): both sides round activations and probabilities to bfloat16
    assert (four - wide).abs().max() <= helpers.tolerance("bfloat16", wide)
    assert helpers.rms_ratio(four, wide) <= 2 * helpers.RMS_RATIO["bfloat16"]


def test_generation_with_4_bits():
    """Through admission, portions, mixed steps and graphs: the same tokens however many requests run side by side."""
    from llm_serving_engine_b200 import GenerationConfig
    model = models()
    rng = random.Random(5)
    prompts = [helpers.random_tokens(rng, 512, n) for n in (3, 70, 130, 33, 64)]
    engine = engine_of(model, kv_bits=4)
    assert engine.cache.kv_bytes_per_token() == 3 * 2 * 2 * (64 + 4)
    got = engine.generate_many(prompts, GenerationConfig(max_new_tokens=24))
    again = engine.generate_many(prompts, GenerationConfig(max_new_tokens=24))
    assert [len(tokens) for tokens in got] == [24] * 5 and got == again
    assert engine.cache.groups[0].pool.used_pages == 0 and engine.runner.graph_replays > 0


@pytest.mark.parametrize("kv_bits", [0, 4])
def test_beams_over_either_cache(kv_bits):
    """Beam search, 4-bit write and attention, reordering and the step's tables as one run."""
    engine = engine_of(models(), kv_bits=kv_bits)
    rng = random.Random(6)
    prompts = [helpers.random_tokens(rng, 512, n) for n in (37, 80)]
    found = engine.beam_search(prompts, 6, 30, 9)
    for prompt, beams in zip(prompts, found):
        assert len(beams) == 6
        for beam in beams[:3]:
            # a bfloat16 model's logits, each within the suite's bound of what another batch gives (8 units of 2^-8 of logits of about 2),
            # and errors that do not all point one way: a third of the sum of the bounds
            assert abs(told_scores(engine, prompt, beam, 9) - beam.score) <= 30 * 8 * 2.0 ** -8 * 2 / 3


def test_caches_of_4_bits_refuse():
    from llm_serving_engine_b200 import CacheConfig, random_model
    from llm_serving_engine_b200.cli import tiny_config
    with pytest.raises(ValueError, match="kv_bits"):
        CacheConfig(16, 8, kv_bits=8)
    with pytest.raises(ValueError, match="bfloat16"):
        engine_of(random_model(CONFIG, 1, dtype="float32", device="cuda"), kv_bits=4)
    for design in ("givelix", "fororax", "daferax"):
        with pytest.raises(ValueError, match="4 bits"):
            engine_of(random_model(tiny_config(300, design), 1, dtype="bfloat16", device="cuda"), kv_bits=4)
