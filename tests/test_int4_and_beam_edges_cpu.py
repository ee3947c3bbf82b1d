"""The 4-bit cache, beam search and a step's tables at their edges: what needs no GPU."""
import pytest
import torch

from llm_serving_engine_b200.kernels import ops
from llm_serving_engine_b200.kernels.library import KernelError


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("tables", [ints(1, 4).expand(3, 4), ints(12).as_strided((3, 4), (2, 1))])
def test_tables_whose_rows_overlap_are_not_written(tables):
    """Rows that share memory (an expanded tensor) have no room for a row each: writing them ``width`` apart would leave the tensor."""
    with pytest.raises(KernelError, match="overlap"):
        ops.step_tables(ints(3), ints(3), ints(9), ints(4), 16, ints(4), ints(5), ints(5), ints(5), ints(3), tables)
    with pytest.raises(KernelError, match="overlap"):
        ops.beam_reorder(ints(1, 3), ints(3, 4), ints(1), tables, 16, [])
    # the tables that are only read may be one row for all; a single row has no distance
    with pytest.raises(KernelError, match="CUDA tensors only"):
        ops.beam_reorder(ints(1, 3), tables, ints(1), ints(3, 4), 16, [])
    with pytest.raises(KernelError, match="CUDA tensors only"):
        ops.step_tables(ints(1), ints(1), ints(9), ints(2), 16, ints(2), ints(5), ints(5), ints(5), ints(1), tables[:1])


def test_an_ordinary_launch_lies_between_a_steps_tables_and_its_kernels(monkeypatch):
    """The step's kernels may read tables, positions and slots before their wait for the launch before them: that launch is none of those
    that write these."""
    from types import SimpleNamespace

    from llm_serving_engine_b200.engine import beam_search

    order = []

    class Counted:
        def __init__(self, name):
            self.name = name

        def __iadd__(self, one):
            order.append(self.name)
            return self

        def copy_(self, other):
            order.append(self.name)

        def view(self, *shape):
            return self

    monkeypatch.setattr(beam_search.ops, "beam_reorder", lambda *a: order.append("reorder"))
    monkeypatch.setattr(beam_search.ops, "step_tables", lambda *a: order.append("tables"))
    for states in ([], ["state"]):
        order.clear()
        runner = SimpleNamespace(cache=SimpleNamespace(page_size=16), model=SimpleNamespace(forward=lambda *a: order.append("step")))
        step = SimpleNamespace(segment_start=None, segment_of_token=None, positions=None, segment_context=None)
        held = SimpleNamespace(runner=runner, step=step, states=states, tables=[Counted("own tables")] * 2, new_tables=[None] * 2, storages=[[]] * 2,
                               parents=None, lengths=Counted("lengths"), row_lengths=Counted("row lengths"), one=None, ones=None, slots=Counted("slots"),
                               new_slots=None, page_start=None, maps=[None] * 2, spare_tables=None, caches=None)
        beam_search._Step(held, 0, False)._launch()
        at = order.index("step")
        assert {"own tables", "tables"} <= set(order[:at]) and order[at - 1] == "lengths" and "row lengths" in order[at:]


def test_parts_of_their_own_are_not_given_pages_of_4_bits(monkeypatch):
    """A rotation or an attention that replaces the one which knows 4-bit pages would write and read them as if they held bfloat16 numbers:
    what was said of the other class does not hold for it."""
    from llm_serving_engine_b200.cache.manager import CacheManager
    from llm_serving_engine_b200.config import CacheConfig
    from llm_serving_engine_b200.parts.attention import GroupedQueryAttention
    from llm_serving_engine_b200.parts.base import POSITION_ENCODINGS, PositionEncoding
    from llm_serving_engine_b200.parts.rope import RotaryEncoding

    class Own(RotaryEncoding):
        def encode_and_store(self, *args):
            raise AssertionError

    class OwnOf4Bits(RotaryEncoding):
        int4 = True

        def encode_and_store(self, *args):
            raise AssertionError

    class Named(RotaryEncoding):
        pass

    class Stranger:          # no PositionEncoding at all
        pass

    class OwnAttention(GroupedQueryAttention):
        def forward(self, x, step, cache):
            raise AssertionError

    kinds = {"rope": RotaryEncoding, "own": Own, "own4": OwnOf4Bits, "named": Named, "stranger": Stranger, "wave": PositionEncoding}
    monkeypatch.setattr(POSITION_ENCODINGS, "get", kinds.__getitem__)
    for kind, taken in (("rope", True), ("own", False), ("own4", True), ("named", True), ("stranger", False), ("wave", False)):
        params = {"num_heads": 4, "num_kv_heads": 2, "head_dim": 64, "position": {"kind": kind}}
        for mixer, of_mixer in ((GroupedQueryAttention, True), (OwnAttention, False)):
            need = mixer.cache_requirement(params, 256)
            assert need.int4 == (taken and of_mixer), (kind, mixer)
            CacheManager([need], CacheConfig(16, 4), torch.bfloat16, "cpu", 64)            # a bfloat16 cache in any case
            if need.int4:
                CacheManager([need], CacheConfig(16, 4, kv_bits=4), torch.bfloat16, "cpu", 64)
            else:
                with pytest.raises(ValueError, match="4 bits"):
                    CacheManager([need], CacheConfig(16, 4, kv_bits=4), torch.bfloat16, "cpu", 64)


def test_lent_pages_count_in_the_most_that_were_used():
    from llm_serving_engine_b200.cache.manager import CacheFullError, CacheManager
    from llm_serving_engine_b200.config import CacheConfig
    from llm_serving_engine_b200.parts.base import PagedKV

    cache = CacheManager([PagedKV(2, 64), PagedKV(2, 128)], CacheConfig(16, 40), torch.float32, "cpu", 640, num_state_slots=4)
    cache.create("a")
    cache.reserve("a", 40)                       # three pages of either group
    assert cache.grow("a", 30)                   # five
    lent, slots = cache.lend("a", 6, 2)
    assert [len(pages) for pages in lent] == [6, 6] and len(slots) == 2
    with pytest.raises(CacheFullError):
        cache.lend("a", 30, 0)
    for _ in range(2):                           # while they are held, and afterwards
        stats = cache.stats(contiguous_max_length=640)
        assert stats["peak_blocks_used"] == 22 and stats["contiguous_waste_tokens"] == 640 - 40
        if "a" in cache.requests:
            assert stats["blocks_used"] == 22
            cache.free("a")
    assert cache.stats()["blocks_used"] == 0
    cache.create("b")
    cache.reserve("b", 16)
    cache.lend("b", 1, 0)
    assert cache.stats()["peak_blocks_used"] == 22
