"""The decode kernel's joined instances (results that other kernels have over a request's first tokens) beside the plain
ones."""

from __future__ import annotations

import re
from pathlib import Path

KERNELS = Path(__file__).resolve().parent.parent / "fast-kernels_b200" / "csrc" / "kernels" / "clustered_page_decode"


def test_the_plain_instances_have_nothing_of_the_join() -> None:
    """The join took registers, and time, from every plain call that was compiled with it."""
    source = re.sub(r"//.*", "", (KERNELS / "page_decode_kernel.cuh").read_text())
    plain = re.search(r"struct DecodeParams \{(.*?)\n\};", source, re.S)
    assert plain is not None and "prior" not in plain.group(1)
    kernel = source[source.index("page_decode_kernel("):]
    assert "conditional_t<JOIN, JoinedDecodeParams, DecodeParams> p" in kernel
    open_blocks: list[bool] = []  # of the blocks around a line: whether one is compiled for joined instances only
    uses = 0
    for line in kernel.splitlines():
        if re.search(r"\bp\.prior", line):
            uses += 1
            assert any(open_blocks), line
        for brace in re.findall(r"if constexpr \(JOIN\) \{|[{}]", line):
            if brace != "}":
                open_blocks.append(brace != "{")
            elif open_blocks:  # (the namespace's own brace closes last)
                open_blocks.pop()
    assert uses >= 3


def test_a_warp_gives_up_a_wait_as_a_whole() -> None:
    """The limit of a unit's wait runs out lane by lane, and what follows it are shuffles and products of whole warps. (The
    waits behind the loop only let copies land: nothing hangs on their verdicts.)"""
    source = re.sub(r"//.*", "", (KERNELS / "page_decode_kernel.cuh").read_text())
    kernel = source[source.index("page_decode_kernel("):]
    waits = re.findall(r"([^\n;{}]*)mbar_wait_bounded\(", kernel)
    assert len(waits) == 2
    assert "if (!__all_sync(0xffffffffu, " in waits[0] and "(void)" in waits[1]
