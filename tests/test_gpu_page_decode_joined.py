"""fk_page_decode_forward_merged through the C ABI: a request's first tokens as prior rows, the rest in its runs, against
attention over all of them in 64 bits. Within the decode's own bound, 2e-3 + 8e-3 |y|; prior rows are fp32."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch
from fast_kernels import ops
from fast_kernels import page_decode_capi as pdc
from paged_kv_testlib import cache_values, fragmented_table, random_cache, rotate64

pytestmark = pytest.mark.gpu
THETA = 10000.0
KV_IDS = {"bf16_kv": 0, "fp8_kv": 1, "int8_kv": 2}


def _tokens(cache, request: int, length: int, rotated: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """fp64 [tokens, heads, dim], the keys turned by their positions."""
    pages = cache.page_table[request, : -(-length // cache.page_size)].long()
    keys, values = (x[pages].permute(0, 2, 1, 3).flatten(0, 1)[:length] for x in cache_values(cache))
    return keys if rotated else rotate64(keys, range(length), THETA), values


def _case(layout: str, group: int, rotated: bool, dim: int, ps: int):
    """(cache, query, what the call is given, the exact rows). Of the requests one has prior rows and tokens of its own, one
    only prior rows, one only tokens, one nothing."""
    heads, lens, before = 2, [330, 96, 41, 0], [192, 96, 0, 0]
    counts = [-(-n // ps) for n in lens]
    table, pages = fragmented_table(counts, 3)
    cache = random_cache(layout=layout, pages=pages, heads=heads, page_size=ps, dim=dim, table=table, lens=lens,
                         theta=THETA if rotated else None, seed=1)
    query = torch.randn((len(lens), heads * group, dim), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    scale = 1.0 / math.sqrt(dim)
    rows, of_request, want = [], [], torch.zeros(query.shape, dtype=torch.float64)
    rest = np.full_like(table, -1)
    for b, (n, c) in enumerate(zip(lens, before)):
        rest[b, : counts[b] - c // ps] = table[b, c // ps : counts[b]]
        pieces = [(0, c // 3 // ps * ps), (c // 3 // ps * ps, c)] if c else []  # two prior results, in token order
        of_request.append((len(rows), len(pieces)))
        if n == 0:
            continue
        keys, values = _tokens(cache, b, n, rotated)
        q = rotate64(query[b : b + 1], [n - 1], THETA)[0].reshape(heads, group, dim)
        logits = torch.einsum("hgd,thd->hgt", q, keys) * scale
        want[b] = torch.einsum("hgt,thd->hgd", torch.softmax(logits, dim=-1), values).reshape(want[b].shape)
        for begin, end in pieces:
            part = logits[..., begin:end]
            top = part.amax(dim=-1, keepdim=True)
            weights = torch.exp(part - top)
            row = torch.zeros((heads, group, dim + 4), dtype=torch.float64)
            row[..., :dim] = torch.einsum("hgt,thd->hgd", weights, values[begin:end])
            row[..., dim], row[..., dim + 1] = top[..., 0] / math.log(2.0), weights.sum(dim=-1)
            rows.append(row.reshape(heads * group, dim + 4))
    plan = ops.plan_clustered_page_decode(page_table=torch.from_numpy(rest), seq_lens=torch.tensor([n - c for n, c in zip(lens, before)]),
                                          num_q_heads=heads * group, num_kv_heads=heads, head_dim=dim, page_size=ps, kv_layout=layout, use_cache=False)
    owner = np.repeat(np.arange(len(lens)), np.diff(plan.request_run_offsets_cpu.numpy()))
    starts = plan.run_logical_starts_cpu + torch.tensor([before[b] // ps for b in owner], dtype=torch.int32)
    given = dict(run_base_pages=plan.run_base_pages_cpu, run_page_counts=plan.run_page_counts_cpu, run_logical_starts=starts,
                 run_last_page_lens=plan.run_last_page_lens_cpu, request_run_offsets=plan.request_run_offsets_cpu,
                 seq_lens=torch.tensor(lens, dtype=torch.int32), rows=torch.stack(rows).float(),
                 of_request=torch.tensor(of_request, dtype=torch.int32))
    return cache, query.cuda(), {name: tensor.cuda() for name, tensor in given.items()}, want, scale, plan.max_pages


@pytest.mark.parametrize("layout", ["bf16_kv", "fp8_kv", "int8_kv"])
@pytest.mark.parametrize(("rotated", "dim", "ps"), [(True, 64, 16), (True, 128, 32), (False, 64, 32), (False, 128, 16)])
@pytest.mark.parametrize("group", [1, 2, 3, 8, 12])
def test_prior_rows_join_the_runs(layout, group, rotated, dim, ps) -> None:
    cache, query, given, want, scale, max_pages = _case(layout, group, rotated, dim, ps)
    lib = pdc.load_library()
    batch, q_heads, heads = query.shape[0], query.shape[1], cache.num_kv_heads
    workspace = torch.zeros(lib.fk_page_decode_workspace_bytes(batch, q_heads, heads, dim), dtype=torch.uint8, device="cuda")
    for splits, with_workspace in ((0, False), (1, False), (2, False), (3, True)):
        output = torch.full_like(query, float("nan"))
        args = pdc.PageDecodeArgs(
            query=query.data_ptr(), key_pages=cache.key_pages.data_ptr(), value_pages=cache.value_pages.data_ptr(),
            key_scales=cache.key_scales.data_ptr() if cache.key_scales is not None else None,
            value_scales=cache.value_scales.data_ptr() if cache.value_scales is not None else None,
            **{name: given[name].data_ptr() for name in ("run_base_pages", "run_page_counts", "run_logical_starts", "run_last_page_lens",
                                                         "request_run_offsets", "seq_lens")},
            output=output.data_ptr(), workspace=workspace.data_ptr() if with_workspace else None,
            workspace_bytes=workspace.numel() if with_workspace else 0, batch=batch, num_runs=given["run_base_pages"].numel(),
            num_q_heads=q_heads, num_kv_heads=heads, head_dim=dim, page_size=ps, kv_format=KV_IDS[layout],
            keys_are_rotated=int(rotated), splits=splits, max_pages_hint=max_pages, softmax_scale=scale, rope_theta=THETA,
            stream=torch.cuda.current_stream().cuda_stream)
        prior = pdc.PageDecodePrior(given["rows"].data_ptr(), given["of_request"].data_ptr())
        torch.cuda.synchronize()  # (the rows' own copy is not the kernel before this one)
        pdc.check(lib.fk_page_decode_forward_merged(ctypes.byref(args), ctypes.byref(prior)))
        torch.testing.assert_close(output.double().cpu(), want, rtol=8e-3, atol=2e-3)
    status = ctypes.c_int(-1)
    pdc.check(lib.fk_page_decode_device_status(ctypes.byref(status)))
    assert status.value == 0
