"""The rules that let the paged attention kernel end when a bounded wait gives up, read off its source.

Running out of a wait's limit cannot be arranged on a healthy device, so the control flow is checked here: whole warps
give up together, and a barrier without a limit is reached whether or not a wait before it gave up."""

from __future__ import annotations

import re
from pathlib import Path

KERNELS = Path(__file__).resolve().parent.parent / "fast-kernels_b200" / "csrc" / "kernels" / "paged_kv"


def _kernel() -> str:
    source = (KERNELS / "paged_attention_tc.cuh").read_text()
    source = re.sub(r"//(?! ----).*", "", source)  # the headings of the roles stay
    return source[source.index("paged_attention_tc_kernel("):]


def test_only_single_lanes_decide_by_themselves() -> None:
    """wait_for's verdict is one lane's. The MMA issuers are single lanes; every other role is whole warps."""
    kernel = _kernel()
    begin, end = kernel.index("---- MMA issuers"), kernel.index("---- copies")
    assert "lane == 0 && count > 0" in kernel[kernel.rindex("if (", 0, begin):begin]
    assert "wait_for(" in kernel[begin:end]
    assert "wait_for(" not in kernel[:begin] + kernel[end:]


def test_converting_warps_meet_at_their_barrier_after_a_wait_gave_up() -> None:
    """Between the head of the conversion's loop and its bar.sync there is no way out of the loop, and the loop's head
    does not look at the verdict of one warp's waits."""
    kernel = _kernel()
    role = kernel[kernel.index("---- 8-bit tiles to 16 bits"):]
    head = re.search(r"for \(int i = 0; ([^;]*); \+\+i\) \{", role)
    assert head is not None and "ok" not in head.group(1)
    barrier = role.index("bar.sync 2")
    before = role[head.end():barrier]
    assert not re.search(r"\b(break|continue|return|goto)\b", before)
    assert "wait_all(" in before and re.search(r"if \(!ok\) \{\s*continue;", role[barrier:])


def test_copies_in_flight_land_before_the_block_ends() -> None:
    """Behind the block's last barrier, where every role's verdict is known."""
    kernel = _kernel()
    end = kernel[kernel.rindex("__syncthreads();"):]
    assert re.search(r"if \(\*fail_flag != 0u\) \{.*wait_all\(drain.*\*issued_slot.*wait_all\(\(QUANT \? raw_full : full\)", end, re.S)
    assert end.index("wait_all(drain") < end.index("tmem_dealloc")
