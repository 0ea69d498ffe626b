"""The operators around the paged cache, the parts that need no GPU: plans, refusals, the C ABI's surface."""

from __future__ import annotations

import ctypes
import importlib
import re
from pathlib import Path

import pytest
import torch

REPO = Path(__file__).resolve().parent.parent
ops = importlib.import_module("fast_kernels.ops")
LIB = REPO / "fast-kernels_b200" / "src" / "fast_kernels" / "lib" / "libfk_paged_kv.so"


def _append_plan(table, lens, new, **kwargs):
    arguments = dict(page_table=torch.tensor(table, dtype=torch.int32), seq_lens=torch.tensor(lens, dtype=torch.int32),
                     append_lens=torch.tensor(new, dtype=torch.int32), num_kv_heads=2, head_dim=64, page_size=16,
                     kv_layout="bf16_kv", use_cache=False)
    return ops.plan_paged_kv_append(**{**arguments, **kwargs})


def test_library_exports_every_declared_symbol() -> None:
    lib = ctypes.CDLL(str(LIB))
    names = set(re.findall(r"\b(fk_paged_kv_\w+)\s*\(", (REPO / "include" / "fk_paged_kv.h").read_text()))
    assert "fk_paged_kv_append" in names
    for name in names:
        assert hasattr(lib, name), f"{name} is declared in include/ but not exported"


def test_append_plan_cuts_tokens_into_pages() -> None:
    """20 tokens behind 10 (slots 10-15 of page 7, 0-13 of page 3), none, and one in a page's last slot."""
    plan = _append_plan([[7, 3], [9, -1], [4, 5]], [10, 3, 31], [20, 0, 1])
    assert plan.segments_cpu.tolist() == [[7, 10 | 6 << 16, 0, 10], [3, 0 | 14 << 16, 6, 16], [5, 15 | 1 << 16, 20, 31]]
    assert plan.num_tokens == 21 and plan.largest_page == 7 and plan.seq_lens_after_cpu.tolist() == [30, 3, 32]
    nothing = _append_plan([[7, 3]], [10], [0])
    assert nothing.num_segments == 0 and nothing.largest_page == -1
    none = _append_plan(torch.zeros((0, 4)).tolist() or [[0]], [0], [0])
    assert none.num_segments == 0


def test_append_plans_are_remembered_by_their_contents() -> None:
    arguments = dict(use_cache=True)
    first = _append_plan([[0, 1]], [3], [4], **arguments)
    assert _append_plan([[0, 1]], [3], [4], **arguments) is first
    assert _append_plan([[0, 2]], [3], [4], **arguments) is not first
    assert _append_plan([[0, 1]], [3], [5], **arguments) is not first


def test_append_plan_refusals() -> None:
    with pytest.raises(ValueError, match="same page"):
        _append_plan([[1, 2], [1, 2]], [16, 17], [1, 1])
    with pytest.raises(ValueError, match="no page for some"):
        _append_plan([[1, -1]], [10], [7])
    with pytest.raises(ValueError, match="fewer columns"):
        _append_plan([[1]], [10], [7])
    with pytest.raises(ValueError, match="append_lens must not be negative"):
        _append_plan([[1]], [10], [-1])
    with pytest.raises(ValueError, match="one entry per request"):
        _append_plan([[1]], [10, 3], [1])
    with pytest.raises(ValueError, match="head_dim must be 64 or 128"):
        _append_plan([[1]], [10], [1], head_dim=96)
    with pytest.raises(ValueError, match="page_size must be 16 or 32"):
        _append_plan([[1]], [10], [1], page_size=64)
    with pytest.raises(ValueError, match="layout must be one of"):
        _append_plan([[1]], [10], [1], kv_layout="fp4_kv")
    with pytest.raises(TypeError, match="must hold integers"):
        _append_plan([[1]], [10], [1], page_table=torch.tensor([[1.0]]))
    with pytest.raises(ValueError, match="fit 32 bits"):
        _append_plan([[1]], [2**31 - 1], [1], page_table=torch.zeros((1, 1), dtype=torch.int32))


def test_append_needs_lengths_or_a_plan() -> None:
    cache = ops.empty_paged_kv(num_pages=1, page_table=torch.tensor([[0]]), seq_lens=torch.tensor([0]), num_kv_heads=2, head_dim=64,
                               page_size=16, kv_layout="int8_kv", device="cpu")
    assert cache.key_scales.shape == (1, 2, 1) and cache.value_scales.shape == (1, 2, 16, 1) and cache.reference_key_pages is None
    rows = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="append_lens or a plan"):
        ops.paged_kv_append(rows, rows, cache)
    with pytest.raises(ValueError, match="not both"):
        ops.paged_kv_append(rows, rows, cache, append_lens=torch.tensor([1]), plan=_append_plan([[0]], [0], [1], kv_layout="int8_kv"))
    with pytest.raises(ValueError, match="key_pages must be a CUDA tensor"):
        ops.paged_kv_append(rows, rows, cache, append_lens=torch.tensor([1]))
    with pytest.raises(ValueError, match="the plan was made for kv_layout"):
        ops.paged_kv_append(rows, rows, cache, plan=_append_plan([[0]], [0], [1]))


def test_native_append_checks_its_arguments_before_the_device() -> None:
    from fast_kernels.native import native_module

    call = native_module().paged_kv_append_forward
    good = dict(keys_ptr=256, values_ptr=256, key_token_stride=128, key_head_stride=64, value_token_stride=128,
                value_head_stride=64, key_pages_ptr=256, value_pages_ptr=256, key_scales_ptr=256, value_scales_ptr=256,
                segments_ptr=256, num_segments=1, num_tokens=1, num_pages=1, num_kv_heads=2, head_dim=64, page_size=16,
                kv_format=2, rotate_keys=1, rope_theta=10000.0, stream_ptr=0)
    call(**{**good, "num_segments": 0, "keys_ptr": 0})  # nothing to do
    for change, message in (({"head_dim": 96}, "head_dim"), ({"page_size": 8}, "page_size"), ({"kv_format": 3}, "kv_format"),
                            ({"num_kv_heads": 0}, "num_kv_heads"), ({"num_tokens": -1}, "non-negative"),
                            ({"rope_theta": 0.0}, "rope_theta"), ({"rope_theta": float("inf")}, "rope_theta"),
                            ({"keys_ptr": 0}, "NULL"), ({"segments_ptr": 0}, "NULL"), ({"value_scales_ptr": 0}, "scales"),
                            ({"keys_ptr": 264}, "aligned"), ({"key_scales_ptr": 258}, "aligned"),
                            ({"key_token_stride": 12}, "multiples of 8")):
        with pytest.raises(ValueError, match=message):
            call(**{**good, **change})
