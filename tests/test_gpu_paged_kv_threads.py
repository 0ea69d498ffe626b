"""Several host threads, each on a stream of its own, that use one plan for the first time together."""

from __future__ import annotations

import importlib
import threading
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch
from fast_kernels.native import native_module
from paged_kv_testlib import fragmented_table, random_cache

pytestmark = pytest.mark.gpu
ops = importlib.import_module("fast_kernels.ops")
THREADS = 4


def test_threads_share_a_plan_from_its_first_use_on() -> None:
    lens, new = [700, 90, 33], [20, 90, 1]
    table, pages = fragmented_table([-(-n // 16) for n in lens], 1)
    cache = random_cache(layout="int8_kv", pages=pages, heads=2, page_size=16, dim=64, table=table, lens=lens, theta=10000.0, seed=2)
    query = torch.randn((sum(new), 8, 64), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    decode = query[:3].contiguous()
    arguments = dict(page_table=cache.page_table, seq_lens=cache.seq_lens, num_q_heads=8, num_kv_heads=2, head_dim=64, page_size=16,
                     kv_layout="int8_kv", use_cache=False)
    want = ops.paged_prompt_attention(query, cache, query_lens=torch.tensor(new)), ops.shared_prefix_decode(decode, cache)
    torch.cuda.synchronize()
    together = threading.Barrier(THREADS)

    def worker(plans, stream):
        results = []
        with torch.cuda.stream(stream):
            for prompt, shared in plans:
                together.wait(timeout=60)
                results.append((ops.paged_prompt_attention(query, cache, plan=prompt), ops.shared_prefix_decode(decode, cache, plan=shared)))
        stream.synchronize()
        return results

    plans = [(ops.plan_paged_prompt_attention(query_lens=torch.tensor(new), **arguments), ops.plan_shared_prefix_decode(**arguments))
             for _ in range(30)]
    with ThreadPoolExecutor(THREADS) as pool:
        calls = [pool.submit(worker, plans, torch.cuda.Stream()) for _ in range(THREADS)]
        for call in calls:
            for got in call.result():
                for a, b in zip(got, want):
                    assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    torch.cuda.synchronize()
    assert native_module().paged_kv_device_status() == 0 and native_module().page_decode_device_status() == 0
