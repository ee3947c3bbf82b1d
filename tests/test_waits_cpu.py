"""What kernels read before and behind their wait for the kernels before them, as far as the sources show it (no GPU)."""
import re
from pathlib import Path

import llm_serving_engine_b200

CSRC = Path(llm_serving_engine_b200.__file__).parent / "csrc"

# What no kernel of a step writes: weights and tables of the model, and the step's own arrays (uploaded, or complete behind an ordinary
# launch, before the step begins).
OF_THE_MODEL = {"a_log", "after_alpha", "after_b", "after_w", "B", "before_alpha", "before_b", "before_w", "bias", "conv_weight", "correction", "delta_weight",
                "dt_bias", "f_bias", "freq", "gate_bias", "head_bias", "i_bias", "inv_freq", "k_norm", "kv_norm", "logit_bias", "mix", "norm", "pos_table", "q_norm",
                "read_w", "scale", "sink", "skip", "table", "w", "weight", "weight_t", "write_w"}
OF_THE_STEP = {"block_tables", "bt", "context", "first", "first_pos", "positions", "rows", "segment_first", "segment_first_pos", "segment_first_position",
               "segment_of_token", "segment_slot", "segment_start", "slot_mapping", "temperature", "top_p"}


def test_what_earlier_kernels_wrote_is_read_through_plain_pointers():
    """Memory behind a ``const T* __restrict__`` parameter counts as unchanged during the whole launch: such a load may be moved above the
    wait, and then sees what the kernel before has not written yet."""
    seen = set()
    for source in sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")]):
        text = re.sub(r"//[^\n]*", "", source.read_text())
        for name in re.findall(r"const\s+\w+\s*\*\s*(?:const\s+)?__restrict__\s+(\w+)", text):
            assert name in OF_THE_MODEL | OF_THE_STEP, f"{source.name}: {name}"
            seen.add(name)
        if source.name != "decode_layers.cu":       # (its kernel loads the model's vectors so, by name, behind the wait)
            assert not re.search(r"__ldg\s*\(|ld\.global\.nc", text), source.name
        else:
            assert set(re.findall(r"__ldg\(([\w.]+)", text)) <= {"L.qkv_bias", "next_norm"}
    assert seen == OF_THE_MODEL | OF_THE_STEP          # no name that is not used any more
