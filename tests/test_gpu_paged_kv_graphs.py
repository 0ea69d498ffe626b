"""Graphs of the paged-cache operators."""

from __future__ import annotations

import gc
import importlib

import pytest
import torch
from fast_kernels.native import native_module
from paged_kv_testlib import fragmented_table, random_cache

pytestmark = pytest.mark.gpu
ops = importlib.import_module("fast_kernels.ops")


def _status_ok() -> None:
    torch.cuda.synchronize()
    assert native_module().paged_kv_device_status() == 0 and native_module().page_decode_device_status() == 0


def _rows(tokens: int, heads: int, dim: int, seed: int) -> torch.Tensor:
    return torch.randn((tokens, heads, dim), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


def _same_bits(got: torch.Tensor, want: torch.Tensor) -> bool:
    return torch.equal(got.view(torch.uint8), want.view(torch.uint8))


def test_a_graph_outlives_the_memory_of_the_plans_that_its_calls_found() -> None:
    """Calls without a plan of the caller's, captured; then plans of many other lengths, and whatever was freed written over."""
    lens = [300, 37]
    table, pages = fragmented_table([20, 4], 1)
    cache = random_cache(layout="int8_kv", pages=pages, heads=2, page_size=16, dim=64, table=table, lens=lens, theta=10000.0, seed=2)
    keys, values = _rows(3, 2, 64, 3), _rows(3, 2, 64, 4)
    prompts, decoded = _rows(8, 4, 64, 5), _rows(2, 4, 64, 6)
    new, queries = torch.tensor([1, 2]), torch.tensor([6, 2])

    def step(at: torch.Tensor, out: list[torch.Tensor]) -> None:
        ops.paged_kv_append(keys, values, cache, append_lens=at)
        ops.paged_prompt_attention(prompts, cache, query_lens=queries, output=out[0])
        ops.shared_prefix_decode(decoded, cache, output=out[1])

    want, got = ([torch.empty_like(prompts), torch.empty_like(decoded)] for _ in range(2))
    step(new, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(new, got)
    # (positions near the end of the requests' pages, so that these lengths are only asked for, never used)
    for length in range(1, 120):
        arguments = dict(page_table=cache.page_table, seq_lens=torch.tensor([length, 1]), num_kv_heads=2, head_dim=64, page_size=16, kv_layout="int8_kv")
        ops.plan_paged_kv_append(append_lens=new, **arguments)
        ops.plan_paged_prompt_attention(query_lens=torch.tensor([1, 1]), num_q_heads=4, **arguments)
        ops.plan_shared_prefix_decode(num_q_heads=4, **arguments)
    gc.collect()
    rubbish = [torch.full((128 * n,), -1, dtype=torch.int32, device="cuda") for n in range(1, 40) for _ in range(4)]
    graph.replay()
    torch.cuda.synchronize()
    assert all(_same_bits(a, b) for a, b in zip(got, want))
    del rubbish
    _status_ok()


def test_without_sharing_captured_calls_are_the_eager_one_with_scratch_of_their_own() -> None:
    """Two long requests on few heads: split over as many blocks as the device has room for, through scratch. The same
    bits as the plain decode, eager and from two graphs that replay side by side on queries of their own."""
    table, pages = fragmented_table([500, 450], 1)
    cache = random_cache(layout="bf16_kv", pages=pages, heads=2, page_size=32, dim=128, table=table, lens=[15_990, 14_400], theta=10000.0, seed=2)
    plan = ops.plan_shared_prefix_decode(page_table=cache.page_table, seq_lens=cache.seq_lens, num_q_heads=8, num_kv_heads=2, head_dim=128,
                                         page_size=32, kv_layout="bf16_kv", use_cache=False)
    assert plan.runs == []
    queries = [_rows(2, 8, 128, seed) for seed in (3, 4)]
    wants = [ops.clustered_page_decode(query, cache) for query in queries]
    for query, want in zip(queries, wants):
        assert _same_bits(ops.shared_prefix_decode(query, cache, plan=plan), want)
    torch.cuda.synchronize()
    graphs, side = [], torch.cuda.Stream()
    for query in queries:
        graph, output = torch.cuda.CUDAGraph(), torch.empty_like(query)
        with torch.cuda.graph(graph, stream=side):
            ops.shared_prefix_decode(query, cache, plan=plan, output=output)
        graphs.append((graph, output))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for stream, (graph, output) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                output.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for (_, output), want in zip(graphs, wants):
        assert _same_bits(output, want)
    _status_ok()


def test_without_sharing_large_head_groups_and_short_requests_are_the_plain_decode() -> None:
    for group, lens in ((12, [40, 3]), (60, [33, 700]), (3, [1, 0])):
        counts = [-(-n // 16) for n in lens]
        table, pages = fragmented_table(counts, 1)
        cache = random_cache(layout="int8_kv", pages=pages, heads=2, page_size=16, dim=64, table=table, lens=lens, theta=10000.0, seed=2)
        query = _rows(2, 2 * group, 64, 3)
        assert _same_bits(ops.shared_prefix_decode(query, cache), ops.clustered_page_decode(query, cache))
    _status_ok()
