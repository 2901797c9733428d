"""CPU tests of what the attention sources have to hold in their written-out
instructions, where the compiler neither knows nor checks it."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ai_engine_amd", "csrc")


def test_every_written_out_copy_waits_for_its_descriptor():
    # a copy reads scalar registers that a vector instruction (v_readlane of a
    # spilled register) may have written just before the text: five wait states
    with open(os.path.join(CSRC, "attn_impl.h")) as f:
        texts = re.findall(r'__asm__ volatile\(((?:"[^"]*"|\s|\w+\("[^"]*"\))*)', f.read())
    copies = [t for t in texts if "buffer_load" in t or "COPY" in t]
    assert copies
    for t in copies:
        assert t.startswith('"s_mov_b32 m0, %0\\n\\ts_nop 4\\n\\t'), t
