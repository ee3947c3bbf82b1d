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
