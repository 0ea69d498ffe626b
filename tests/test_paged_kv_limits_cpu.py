"""Lengths that the attention over pages cannot count."""

from __future__ import annotations

import importlib
import re
from pathlib import Path

import pytest
import torch

ops = importlib.import_module("fast_kernels.ops")
KERNELS = Path(__file__).resolve().parent.parent / "fast-kernels_b200" / "csrc" / "kernels" / "paged_kv"


@pytest.mark.parametrize("plan", [ops.plan_paged_prompt_attention, ops.plan_shared_prefix_decode])
def test_a_length_whose_tiles_pass_31_bits_is_refused(plan) -> None:
    arguments = dict(page_table=torch.tensor([[0]]), num_q_heads=4, num_kv_heads=2, head_dim=64, page_size=16, kv_layout="bf16_kv")
    if plan is ops.plan_paged_prompt_attention:
        arguments["query_lens"] = torch.tensor([1])
    with pytest.raises(ValueError, match="at most 2\\^31 - 128"):
        plan(seq_lens=torch.tensor([2**31 - 127]), **arguments)
    with pytest.raises(ValueError, match="fewer columns"):  # counted, and then its pages are missed
        plan(seq_lens=torch.tensor([2**31 - 128]), **arguments)


def test_the_kernel_leaves_out_items_that_it_cannot_count() -> None:
    """Its tiles of 128 tokens, rounded up, stay below 2^31 for the largest end token that it takes."""
    header = (KERNELS.parents[3] / "include" / "fk_paged_kv.h").read_text()
    most = re.search(r"#define FK_PAGED_KV_MAX_TOKENS \((0x[0-9a-f]+) - (\d+)\)", header)
    assert most is not None
    most_tokens = int(most.group(1), 16) - int(most.group(2))
    assert (most_tokens + 127) // 128 * 128 < 2**31 and most_tokens + 128 > 2**31 - 1
    assert "item.end_token <= FK_PAGED_KV_MAX_TOKENS" in (KERNELS / "paged_attention.cuh").read_text()
