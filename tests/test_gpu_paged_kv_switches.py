"""A shared decode with the decode kernel's switches (environment variables, read once per process) set."""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent
CHILD = """
import importlib
import torch
from fast_kernels.native import native_module
from paged_kv_testlib import attention_terms64, default_scale, random_cache

ops = importlib.import_module("fast_kernels.ops")
# 2 requests x 2 kv heads, 256 tokens in common, then up to 4000 of their own: blocks of a task merge
for layout in ("bf16_kv", "int8_kv"):
    shared, counts = 16, [250, 130]
    table = torch.full((2, shared + max(counts)), -1, dtype=torch.int32)
    table[:, :shared] = torch.arange(shared)
    table[0, shared : shared + counts[0]] = torch.arange(counts[0]) + shared
    table[1, shared : shared + counts[1]] = torch.arange(counts[1]) + shared + counts[0]
    lens = [(shared + counts[0]) * 16 - 3, (shared + counts[1]) * 16]
    cache = random_cache(layout=layout, pages=shared + sum(counts), heads=2, page_size=16, dim=64, table=table, lens=lens, theta=10000.0, seed=1)
    query = torch.randn((2, 8, 64), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    plan = ops.plan_shared_prefix_decode(page_table=cache.page_table, seq_lens=cache.seq_lens, num_q_heads=8, num_kv_heads=2, head_dim=64,
                                         page_size=16, kv_layout=layout, min_saved_bytes=0)
    assert plan.runs == [(0, shared, (0, 1))]
    got = ops.shared_prefix_decode(query, cache, plan=plan).double().cpu()
    torch.cuda.synchronize()
    assert native_module().paged_kv_device_status() == 0 and native_module().page_decode_device_status() == 0
    terms = attention_terms64(cache, query, [(0, lens[0] - 1), (1, lens[1] - 1)], default_scale(64), 10000.0)
    # the bf16 bound of the shared runs: a query and weights rounded to 2^-8, the row once more
    d = 1.1 * 2.0**-8 * terms["logit"]
    bound = 2.0**-8 * terms["out"].abs() + (2.0**-8 + 2 * d) * terms["a"] + 1e-30
    print(float(((got - terms["out"]).abs() / bound).max()), float((got - terms["out"]).norm() / terms["out"].norm()))
"""


@pytest.mark.parametrize("switch", ["FK_PAGE_DECODE_CLUSTER_MERGE", "FK_PAGE_DECODE_TENSOR_CORES", "FK_PAGE_DECODE_PDL", ""])
def test_shared_decode_with_a_switch_off(switch) -> None:
    paths = [str(ROOT / "tests"), str(ROOT / "fast-kernels_b200" / "src"), os.environ.get("PYTHONPATH", "")]
    environment = {**os.environ, "PYTHONPATH": os.pathsep.join(paths)}
    if switch:
        environment[switch] = "0"
    done = subprocess.run([sys.executable, "-c", CHILD], capture_output=True, text=True, env=environment, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]
    lines = done.stdout.split("\n")[:2]
    assert len(lines) == 2
    for line in lines:
        worst, norm = map(float, line.split())
        assert worst <= 1.0 and norm <= 2.0**-7
