"""8-bit pages whose two 64-dim blocks have very different scales."""

from __future__ import annotations

import dataclasses
import importlib

import pytest
import torch
from fast_kernels.native import native_module
from paged_kv_testlib import cache_values, random_cache

pytestmark = pytest.mark.gpu
ops = importlib.import_module("fast_kernels.ops")


def _means(cache, positions: list[int]) -> torch.Tensor:
    """fp64 [rows, heads, dim]: of the values of tokens 0 .. position."""
    table = cache.page_table[0, : -(-(max(positions) + 1) // cache.page_size)].long()
    values = cache_values(cache)[1][table].permute(0, 2, 1, 3).flatten(0, 1)
    return torch.stack([values[: p + 1].mean(dim=0) for p in positions])


def _cache(layout: str, *, heads: int = 2, dim: int = 128, ps: int = 16, length: int = 2000):
    """One request. Keys of 0 make all weights equal; values' numbers are 16 or more: nothing cancels."""
    pages = length // ps
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32)[None]
    cache = random_cache(layout=layout, pages=pages, heads=heads, page_size=ps, dim=dim, table=table, lens=[length], theta=10000.0, seed=1)
    limit = 127 if layout == "int8_kv" else 448
    numbers = torch.randint(16, limit + 1, cache.value_pages.shape, generator=torch.Generator().manual_seed(2)).float()
    cache.value_pages.copy_(numbers.to(torch.int8) if layout == "int8_kv" else numbers.to(torch.float8_e4m3fn).view(torch.uint8))
    cache.key_pages.zero_()
    return cache


def _assert_means(cache, bound: float) -> None:
    """Prompts and a shared decode give the means of the values, each element within `bound` of itself."""
    heads, dim, ps, length, layout = cache.num_kv_heads, cache.head_dim, cache.page_size, int(cache.seq_lens[0]), cache.kv_layout
    geometry = dict(num_q_heads=2 * heads, num_kv_heads=heads, head_dim=dim, page_size=ps, kv_layout=layout)

    def check(got: torch.Tensor, positions: list[int]) -> None:
        want = _means(cache, positions)[:, :, None].expand(-1, -1, 2, -1).reshape(got.shape)
        off = ((got.double().cpu() - want).abs() / want).amax(dim=(0, 1))
        assert float(off.max()) <= bound, (float(off[:64].max()), float(off[64:].max()), bound)

    query = torch.randn((300, 2 * heads, dim), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    # few queries: the tokens are cut into pieces with partial results; many: rows are written directly
    plan = ops.plan_paged_prompt_attention(page_table=cache.page_table, seq_lens=cache.seq_lens, query_lens=torch.tensor([3]), **geometry)
    assert plan.num_partials > 0
    check(ops.paged_prompt_attention(query[:3], cache, plan=plan), [length - 3 + i for i in range(3)])
    short = torch.tensor([300], dtype=torch.int32)
    plan = ops.plan_paged_prompt_attention(page_table=cache.page_table, seq_lens=short, query_lens=short, **geometry)
    assert plan.num_partials == 0
    check(ops.paged_prompt_attention(query, dataclasses.replace(cache, seq_lens=short), plan=plan), list(range(300)))
    # two requests that share everything but the last page
    both = torch.cat([cache.page_table, cache.page_table])
    twice = dataclasses.replace(cache, page_table=both, seq_lens=torch.tensor([length, length - 5], dtype=torch.int32))
    plan = ops.plan_shared_prefix_decode(page_table=both, seq_lens=twice.seq_lens, min_saved_bytes=0, **geometry)
    assert plan.runs
    check(ops.shared_prefix_decode(query[:2].contiguous(), twice, plan=plan), [length - 1, length - 6])
    torch.cuda.synchronize()
    assert native_module().paged_kv_device_status() == 0 and native_module().page_decode_device_status() == 0


@pytest.mark.parametrize("layout", ["fp8_kv", "int8_kv"])
@pytest.mark.parametrize("exponent", [-4, -18, -20, -22, -24])
@pytest.mark.parametrize("larger", [0, 1])
def test_the_block_with_the_smaller_scales_keeps_its_bits(layout, exponent, larger) -> None:
    """Every rounding counts relative to the result. The row is rounded to bf16 (2^-8), a weight to fp16 (2^-11). Both blocks'
    elements are fp16 times 2^7: the block of the smaller scales by its ratio r, 1.3 * 2^exponent, which is off by up to
    2^-25 / (2^7 r), or 2^-11; the products, of elements of 16 or more, by a sixteenth of that or 2^-11. fp32 sums add less than
    2^-12 for 2000 tokens."""
    cache = _cache(layout)
    ratio = 1.3 * 2.0**exponent
    cache.value_scales[..., larger] = 0.75
    cache.value_scales[..., 1 - larger] = 0.75 * ratio
    bound = 2.0**-8 + 2.0**-11 + 17 / 16 * max(2.0**-25 / (128 * ratio), 2.0**-11) + 2.0**-12
    assert bound < 2.0**-6.9
    _assert_means(cache, bound)


@pytest.mark.parametrize("layout", ["fp8_kv", "int8_kv"])
@pytest.mark.parametrize("exponent", [-18, -20, -22])
def test_a_token_with_one_large_block_takes_no_bits_from_the_others(layout, exponent) -> None:
    """Every other token has its first block's scale far above all others; in the second block all tokens count alike. A
    weight of r = 1.35 * 2^exponent of the heaviest, which is 2^7 or more, is off by up to 2^-25 / (2^7 r), or 2^-11, and so are the
    heavy tokens' ratio and (as above) its products; with the row and the sums as above."""
    cache = _cache(layout)
    ratio = 1.35 * 2.0**exponent
    cache.value_scales[:] = 0.75 * ratio
    cache.value_scales[:, :, ::2, 0] = 0.75
    small = max(2.0**-25 / (128 * ratio), 2.0**-11)
    _assert_means(cache, 2.0**-8 + 2.0**-11 + (2 + 1 / 16) * small + 2.0**-12)
