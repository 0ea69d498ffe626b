"""Plans of the paged-cache operators that are remembered by their contents."""

from __future__ import annotations

import importlib
from collections import OrderedDict

import torch
from fast_kernels.ops import _paged

ops = importlib.import_module("fast_kernels.ops")


def test_a_plan_in_use_outlives_others() -> None:
    plans: OrderedDict = OrderedDict()
    make = lambda name: _paged.remembered(plans, (name,), object, True, most=2)  # noqa: E731
    first = make("first")
    for other in ("second", "third", "fourth"):
        make(other)
        assert make("first") is first
    assert list(plans) == [("fourth",), ("first",)]


def test_plans_of_a_loop_are_dropped() -> None:
    """A decode loop makes a plan a step, each with its page table and, on a device, its tables."""
    module = importlib.import_module("fast_kernels.ops.paged_kv_append")
    for step in range(100):
        ops.plan_paged_kv_append(page_table=torch.arange(8, dtype=torch.int32)[None], seq_lens=torch.tensor([step]),
                                 append_lens=torch.tensor([1]), num_kv_heads=2, head_dim=64, page_size=16, kv_layout="bf16_kv")
    assert len(module._PLANS) <= 32


def test_a_plan_that_a_captured_call_found_is_kept(monkeypatch) -> None:
    plan = object()
    monkeypatch.setattr(_paged, "_IN_GRAPHS", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    _paged.keep_for_graphs(plan)
    assert not _paged._IN_GRAPHS
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    _paged.keep_for_graphs(plan)
    _paged.keep_for_graphs(plan)
    assert list(_paged._IN_GRAPHS.values()) == [plan]
