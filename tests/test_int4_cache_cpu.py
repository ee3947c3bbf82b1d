"""What the entry points of the 4-bit cache, beam search and a step's tables refuse (no GPU: arguments are looked at first)."""
import pytest
import torch

from llm_serving_engine_b200.kernels import ops
from llm_serving_engine_b200.kernels.library import KernelError


def cache(pages=4, n_kv=2, page_size=16, dim=128):
    codes = lambda: torch.zeros((pages, n_kv, page_size, dim // 2), dtype=torch.uint8)      # noqa: E731
    scales = lambda: torch.zeros((pages, n_kv, page_size, 2), dtype=torch.bfloat16)         # noqa: E731
    return [codes(), scales(), codes(), scales()]


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def write(**changes):
    pages = changes.pop("pages", cache())
    kept = {"qkv": torch.zeros((3, 8 * 128), dtype=torch.bfloat16), "bias": None, "positions": ints(3), "slot_mapping": ints(3),
            "inv_freq": torch.zeros(64), "q_out": torch.zeros((3, 4, 128), dtype=torch.bfloat16), "n_q": 4, "n_kv": 2, "head_dim": 128, "pairing": 1}
    kept.update(zip(("k_codes", "k_scales", "v_codes", "v_scales"), pages))
    ops.rope_kv_write_int4(**{**kept, **changes})


@pytest.mark.parametrize("changes,what", [
    ({"qkv": torch.zeros((3, 7 * 128), dtype=torch.bfloat16)}, "rows of 1024"),
    ({"qkv": torch.zeros((3, 8 * 128), dtype=torch.float16)}, "unsupported dtype"),
    ({"qkv": torch.zeros((2, 3, 8 * 128), dtype=torch.bfloat16)}, "partial sums"),
    ({"pages": cache(dim=96)}, "head size 96"), ({"pages": cache(n_kv=1)}, "1 heads of 128"), ({"pages": cache(dim=64)}, "2 heads of 64"),
    ({"positions": ints(2)}, "positions"), ({"slot_mapping": torch.zeros(3, dtype=torch.int64)}, "slots"),
    ({"inv_freq": torch.zeros(63)}, "frequencies"), ({"q_out": torch.zeros((3, 4, 128))}, "q_out"), ({"bias": torch.zeros(5)}, "bias"),
    ({}, "CUDA tensors only")])
def test_write_refuses(changes, what):
    with pytest.raises(KernelError, match=what):
        write(**changes)


def test_a_cache_of_other_kinds_is_refused():
    good = cache()
    out = torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    for index, other in ((0, good[0].to(torch.int32)), (0, good[0][:, :, ::2]), (1, good[1].float()), (2, good[2][:3]), (3, good[3][..., :1])):
        pages = list(good)
        pages[index] = other
        with pytest.raises(KernelError, match="codes|scales|contiguous"):
            ops.kv_read_int4(*pages, ints(3), out, out.clone())
    with pytest.raises(KernelError, match="outputs"):
        ops.kv_read_int4(*good, ints(3), out, out[:2])
    with pytest.raises(KernelError, match="slots"):
        ops.kv_read_int4(*good, ints(2), out, out.clone())


def rows(**changes):
    kept = {"q": torch.zeros((3, 4, 128), dtype=torch.bfloat16), "out": torch.zeros((3, 4, 128), dtype=torch.bfloat16),
            "block_tables": ints(2, 4), "segment_of_token": ints(3), "positions": ints(3), "scale": 0.1}
    kept.update(zip(("k_codes", "k_scales", "v_codes", "v_scales"), cache()))
    ops.paged_attention_decode_int4(**{**kept, **changes})


@pytest.mark.parametrize("changes,what", [
    ({"q": torch.zeros((3, 4, 128))}, "bfloat16"), ({"q": torch.zeros((3, 3, 128), dtype=torch.bfloat16), "out": torch.zeros((3, 3, 128), dtype=torch.bfloat16)}, "do not fit"),
    ({"q": torch.zeros((3, 8, 128), dtype=torch.bfloat16)[:, ::2]}, "contiguous"), ({"block_tables": ints(8)}, "block tables"),
    ({"block_tables": torch.zeros((2, 4), dtype=torch.int64)}, "block tables"), ({"segment_of_token": ints(2)}, "segments"),
    ({"positions": ints(2)}, "positions"), ({"scale": -1.0}, "scale"), ({"scale": 0.0}, "scale"), ({}, "CUDA tensors only")])
def test_rows_refuse(changes, what):
    with pytest.raises(KernelError, match=what):
        rows(**changes)


def select(**changes):
    kept = {"logits": torch.zeros((6, 50)), "scores": torch.zeros((2, 3)), "ended": ints(2, 3), "end_token": 4, "out_scores": torch.zeros((2, 3)),
            "out_tokens": ints(2, 3), "out_parents": ints(2, 3), "out_ended": ints(2, 3)}
    ops.beam_select(**{**kept, **changes})


@pytest.mark.parametrize("changes,what", [
    ({"logits": torch.zeros((5, 50))}, "logits"), ({"logits": torch.zeros((6, 50), dtype=torch.bfloat16)}, "logits"), ({"logits": torch.zeros((50, 6)).t()}, "logits"),
    ({"scores": torch.zeros((2, 33)), "logits": torch.zeros((66, 50))}, "33 beams"), ({"end_token": 50}, "end token"), ({"end_token": -1}, "end token"),
    ({"ended": torch.zeros((2, 3), dtype=torch.bool)}, "int32"), ({"out_tokens": ints(3, 2)}, "int32"), ({"scores": torch.zeros(6)}, "scores"), ({}, "CUDA tensors only")])
def test_select_refuses(changes, what):
    with pytest.raises(KernelError, match=what):
        select(**changes)


def reorder(**changes):
    kept = {"parents": ints(2, 3), "block_tables": ints(6, 4), "lengths": ints(2), "new_tables": ints(6, 4), "page_size": 16, "storages": [torch.zeros((2, 8, 4))]}
    ops.beam_reorder(**{**kept, **changes})


SAME = ints(6, 4)


@pytest.mark.parametrize("changes,what", [
    ({"parents": ints(1, 40), "block_tables": ints(40, 4), "new_tables": ints(40, 4)}, "40 beams"), ({"parents": torch.zeros((2, 3))}, "parents"),
    ({"new_tables": ints(6, 3)}, "block tables"), ({"block_tables": SAME, "new_tables": SAME}, "another tensor"), ({"lengths": ints(1)}, "lengths"),
    ({"page_size": 0}, "page size"), ({"storages": [torch.zeros((8, 4))]}, "storages"), ({"storages": [torch.zeros((2, 8, 4, 6)).transpose(2, 3)]}, "storages"), ({}, "CUDA tensors only")])
def test_reorder_refuses(changes, what):
    with pytest.raises(KernelError, match=what):
        reorder(**changes)


def tables(**changes):
    kept = {"first": ints(2), "counts": ints(2), "pages": ints(9), "page_start": ints(3), "page_size": 16, "segment_start": ints(3), "segment_of_token": ints(5),
            "positions": ints(5), "slot_mapping": ints(5), "contexts": ints(2), "block_tables": ints(2, 4)}
    ops.step_tables(**{**kept, **changes})


@pytest.mark.parametrize("changes,what", [
    ({"first": ints(0)}, "first positions"), ({"counts": ints(1)}, "counts"), ({"page_start": ints(2)}, "page starts"), ({"pages": torch.zeros(9)}, "pages"),
    ({"segment_start": ints(2)}, "segment starts"), ({"positions": ints(4)}, "positions"), ({"contexts": ints(1)}, "contexts"), ({"page_size": 0}, "page size"),
    ({"block_tables": ints(3, 4)}, "block tables"), ({}, "CUDA tensors only")])
def test_step_tables_refuse(changes, what):
    with pytest.raises(KernelError, match=what):
        tables(**changes)


def test_status_words_are_read_by_declared_entry_points():
    from llm_serving_engine_b200.kernels import library
    for _, entry in ops._STATUS_WORDS:
        for name in (entry, entry + "_async", entry + "_reset"):
            assert name in library._SIGNATURES, name
