"""What the attention's interface says, against its sources (no GPU)."""
import os
import re

from unpopped_b200 import _lib
from unpopped_b200.interface import kernel_interface

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unpopped_b200", "csrc")


def test_dynamic_shared_memory_is_the_largest_launchs():
    """The kernel for many query rows at size 128: two tiles of 128 queries, K and V as two halves of 64 tokens in two parts
    or stages each, all rows of 128 f16; a pair of scales a token and 32 dimensions, of K and V; 1024 bytes to align."""
    row = 128 * 2
    many = 2 * 128 * row + 2 * 2 * 2 * 64 * row + 2 * 128 * (128 // 32) * 4 + 1024
    few = 4 * 2 * (2 * 16 * 256 + 2 * 2 * 256)  # four warps' two stages of 32 tokens at size 256
    ki = kernel_interface(_lib.SERVING_KERNEL["KV4_ATTENTION"])
    assert ki.launch["dynamic_shared_bytes"] == f"up to {max(many, few)}"


def test_fidelity_notes_name_the_roundings_that_are_made():
    with open(os.path.join(CSRC, "kv4_prompt.cu")) as f:
        two = re.search(r"const bool two = (.*?);", f.read()).group(1)
    assert two == "!BF16 || z == 0"  # both parts of a scale: K always, V unless the output is bf16
    notes = kernel_interface(_lib.SERVING_KERNEL["KV4_ATTENTION"]).fidelity_notes[0]
    assert "many: p, and with bf16 outputs nibble * v_scale" in notes and "few query rows: p * v_scale" in notes
