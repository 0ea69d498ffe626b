"""paged_kv_append on the GPU against its definition in 64 bits.

Tolerances. A stored element is off by at most half a step of its format (bf16 2^-8 of the value; int8 half of 1;
e4m3 2^-4 of the number or half its smallest subnormal, all in units of the scale). On top of that the fp32 turn: cosine
and sine are off by at most 2^-22 (a fraction of a turn rounded to fp32, 2^-25 turns = 2^-22.3 radians, and the function's
own 2^-23), and the two products and their sum add 3 * 2^-24 of the pair's length: SLACK = 2^-21 covers the sum."""

from __future__ import annotations

import dataclasses
import importlib

import numpy as np
import pytest
import torch
from paged_kv_testlib import append64, assert_append, cache_values, fragmented_table, random_cache

pytestmark = pytest.mark.gpu
ops = importlib.import_module("fast_kernels.ops")
LAYOUTS = ("bf16_kv", "fp8_kv", "int8_kv")
SLACK = 2.0**-21


def _copy(cache):
    keep = {name: getattr(cache, name).clone() for name in ("key_pages", "value_pages", "key_scales", "value_scales")
            if getattr(cache, name) is not None}
    return dataclasses.replace(cache, **keep)


def _rows(tokens: int, heads: int, dim: int, seed: int, magnitude: float = 1.0) -> torch.Tensor:
    gen = torch.Generator().manual_seed(seed)
    return (magnitude * torch.randn((tokens, heads, dim), generator=gen)).to(torch.bfloat16).cuda()


def _case(layout, lens, new, *, heads=2, dim=128, ps=16, theta=10000.0, seed=0):
    counts = [-(-(c + n) // ps) for c, n in zip(lens, new)]
    table, pages = fragmented_table(counts, seed)
    cache = random_cache(layout=layout, pages=pages, heads=heads, page_size=ps, dim=dim, table=table, lens=lens, theta=theta,
                         seed=seed + 1)
    return cache, _rows(sum(new), heads, dim, seed + 2), _rows(sum(new), heads, dim, seed + 3)


@pytest.mark.parametrize("theta", [None, 10000.0])
@pytest.mark.parametrize(("dim", "ps"), [(64, 16), (64, 32), (128, 16), (128, 32)])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_every_instantiation(layout, dim, ps, theta) -> None:
    """Requests that begin, fill, cross and end pages, one that gets nothing, one token alone in a page's last slot."""
    lens = [0, 5, 3 * ps - 1, 2 * ps, ps + 7, 0]
    new = [3 * ps + 1, 0, 1, ps, 2 * ps - 7, 1]
    cache, keys, values = _case(layout, lens, new, heads=3, dim=dim, ps=ps, theta=theta, seed=dim + ps)
    before, want = _copy(cache), append64(cache, keys, values, new)
    after = ops.paged_kv_append(keys, values, cache, append_lens=torch.tensor(new))
    assert after.seq_lens.tolist() == [c + n for c, n in zip(lens, new)] and after.key_pages is cache.key_pages
    assert_append(before, after, want, SLACK)


@pytest.mark.parametrize("heads", [1, 8, 9, 17])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_head_counts_around_a_block_of_warps(layout, heads) -> None:
    lens, new = [30, 0], [1, 20]
    cache, keys, values = _case(layout, lens, new, heads=heads, seed=heads)
    before, want = _copy(cache), append64(cache, keys, values, new)
    assert_append(before, ops.paged_kv_append(keys, values, cache, append_lens=torch.tensor(new)), want, SLACK)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_token_by_token_with_growing_and_shrinking_keys(layout) -> None:
    """One page filled a token a step. A step's page is what the definition makes of the page before it, whether its keys
    are larger than all before (the held ones are rounded again) or smaller."""
    cache = random_cache(layout=layout, pages=2, heads=2, page_size=16, dim=64, table=[[1]], lens=[0], theta=10000.0, seed=5)
    for step, magnitude in enumerate([1.0, 0.2, 3.0, 0.01, 3.0, 40.0, 0.0, 1e-9, 41.0]):
        keys, values = _rows(1, 2, 64, 2 * step, magnitude), _rows(1, 2, 64, 2 * step + 1, magnitude)
        before, want = _copy(cache), append64(cache, keys, values, [1])
        cache = ops.paged_kv_append(keys, values, cache, append_lens=torch.tensor([1]))
        assert_append(before, cache, want, SLACK)
    assert cache.seq_lens.tolist() == [9]


@pytest.mark.parametrize("layout", ["fp8_kv", "int8_kv"])
def test_a_reused_page_forgets_its_scale(layout) -> None:
    cache = random_cache(layout=layout, pages=2, heads=2, page_size=16, dim=128, table=[[0]], lens=[0], theta=None, seed=5)
    cache.key_scales.fill_(1e4)
    keys, values = _rows(3, 2, 128, 1), _rows(3, 2, 128, 2)
    after = ops.paged_kv_append(keys, values, cache, append_lens=torch.tensor([3]))
    assert float(after.key_scales[0].max()) < 1.0 and float(after.key_scales[1].min()) == 1e4
    got = cache_values(after)[0][0, :, :3].transpose(0, 1)
    # half a step: of 1 for int8 with scales below 5 / 127, of 2^-4 for e4m3
    torch.testing.assert_close(got, keys.double().cpu(), rtol=2.0**-4, atol=0.5 * 5 / 127)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_a_prompt_appended_at_once_gives_the_bytes_of_the_builders(layout) -> None:
    """Keys stored as they come: same divisions, same roundings, so the same bytes. The builders run on the CPU here:
    torch on a GPU divides by a number by multiplying with its rounded reciprocal, so their scales are then off by up to
    2^-24 (that rounding) + 2^-24 (the product's) against the quotient's own 2^-24."""
    lens, heads, dim, ps = [70, 16, 1], 2, 128, 16
    gen = torch.Generator(device="cuda").manual_seed(1)
    dense = [torch.randn((3, heads, max(lens), dim), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2)]
    build = {"bf16_kv": ops.pack_paged_kv_bf16, "fp8_kv": ops.quantize_paged_kv_fp8, "int8_kv": ops.quantize_paged_kv_int8}[layout]
    built = build(*(x.cpu() for x in dense), torch.tensor(lens, dtype=torch.int32), page_size=ps, fragment_pages=True, seed=3)
    empty = ops.empty_paged_kv(num_pages=built.total_pages, page_table=built.page_table, seq_lens=torch.zeros(3, dtype=torch.int32),
                               num_kv_heads=heads, head_dim=dim, page_size=ps, kv_layout=layout)
    rows = [torch.cat([x[b, :, :n].transpose(0, 1) for b, n in enumerate(lens)]) for x in dense]
    after = ops.paged_kv_append(*rows, empty, append_lens=torch.tensor(lens))
    token = torch.arange(ps)
    for b, n in enumerate(lens):
        for slot, page in enumerate(built.page_table[b, : -(-n // ps)].tolist()):
            real = token < n - slot * ps
            for name in ("key_pages", "value_pages"):
                got, expected = (getattr(cache, name)[page].cpu()[:, real].view(torch.uint8) for cache in (after, built))
                assert torch.equal(got, expected)
            if layout != "bf16_kv":
                assert torch.equal(after.key_scales[page].cpu(), built.key_scales[page])
                assert torch.equal(after.value_scales[page].cpu()[:, real], built.value_scales[page][:, real])


@pytest.mark.parametrize("layout", LAYOUTS)
def test_views_into_the_rows_of_a_fused_projection(layout) -> None:
    lens, new, heads, dim = [0, 40], [33, 2], 2, 64
    cache, _, _ = _case(layout, lens, new, heads=heads, dim=dim)
    fused = _rows(sum(new), 8, dim, 9)
    keys, values = fused[:, 4:6], fused[:, 6:8]
    by_head = fused[:, 4:6].transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost in memory
    before, want = _copy(cache), append64(cache, keys, values, new)
    twin = _copy(cache)
    assert_append(before, ops.paged_kv_append(keys, values, cache, append_lens=torch.tensor(new)), want, SLACK)
    other = ops.paged_kv_append(by_head, values, twin, append_lens=torch.tensor(new))
    assert torch.equal(other.key_pages.view(torch.uint8), cache.key_pages.view(torch.uint8))


@pytest.mark.parametrize("position", [131071, 2**24 + 1, 2**31 - 2])
def test_the_angle_keeps_its_precision_at_far_positions(position) -> None:
    """The pages before the new token are not read, so the table may name any page for them."""
    ps = 32
    table = np.zeros((1, position // ps + 1), dtype=np.int32)
    table[0, -1] = 1
    cache = random_cache(layout="bf16_kv", pages=2, heads=2, page_size=ps, dim=128, table=table, lens=[position], theta=10000.0, seed=1)
    keys, values = _rows(1, 2, 128, 3), _rows(1, 2, 128, 4)
    before, want = _copy(cache), append64(cache, keys, values, [1])
    plan = ops.plan_paged_kv_append(page_table=cache.page_table, seq_lens=cache.seq_lens, append_lens=torch.tensor([1]),
                                    num_kv_heads=2, head_dim=128, page_size=ps, kv_layout="bf16_kv", use_cache=False)
    assert_append(before, ops.paged_kv_append(keys, values, cache, plan=plan), want, SLACK)


@pytest.mark.parametrize("layout", ["bf16_kv", "int8_kv"])
def test_pages_past_32_bit_offsets(layout) -> None:
    """A pool of more than 2^32 bytes of keys: the last page's offset does not fit 32 bits, in elements either for bf16."""
    heads, dim, ps = 8, 128, 32
    pages = 2**31 // (heads * dim * ps) + 2 if layout == "bf16_kv" else 2**32 // (heads * dim * ps) + 2
    element = torch.bfloat16 if layout == "bf16_kv" else torch.int8
    shape = (pages, heads, ps, dim)
    scales = (None, None) if layout == "bf16_kv" else (torch.zeros((*shape[:2], 2), device="cuda"), torch.zeros((*shape[:3], 2), device="cuda"))
    cache = ops.PagedKVCache(
        key_pages=torch.zeros(shape, dtype=element, device="cuda"), value_pages=torch.zeros(shape, dtype=element, device="cuda"),
        page_table=torch.tensor([[pages - 1]], dtype=torch.int32), seq_lens=torch.tensor([0], dtype=torch.int32), key_scales=scales[0],
        value_scales=scales[1], reference_key_pages=None, reference_value_pages=None, kv_layout=layout, page_size=ps,
        num_kv_heads=heads, head_dim=dim)
    keys, values = _rows(5, heads, dim, 1), _rows(5, heads, dim, 2)
    ops.paged_kv_append(keys, values, cache, append_lens=torch.tensor([5]))
    last = dataclasses.replace(cache, **{name: getattr(cache, name)[-1:] for name in ("key_pages", "value_pages", "key_scales", "value_scales")
                                         if getattr(cache, name) is not None})
    for got, rows in zip(cache_values(last), (keys, values)):
        torch.testing.assert_close(got[0, :, :5].transpose(0, 1), rows.double().cpu(), rtol=0, atol=0.5 * 5 / 127)
    assert not bool(cache.key_pages[:-1].any()) and not bool(cache.key_pages[-1, :, 5:].any())


def test_plan_none_and_empty_calls() -> None:
    cache, keys, values = _case("bf16_kv", [4, 0], [0, 0])
    before = _copy(cache)
    after = ops.paged_kv_append(keys, values, cache, append_lens=torch.tensor([0, 0]))
    assert torch.equal(after.key_pages, before.key_pages) and after.seq_lens.tolist() == [4, 0]


def test_lengths_of_a_cache_are_its_own() -> None:
    """A caller that ends a request by setting its length to 0 changes no other call with the same lengths."""
    cache, keys, values = _case("bf16_kv", [4, 7], [2, 1])
    new = torch.tensor([2, 1])
    ops.paged_kv_append(keys, values, cache, append_lens=new).seq_lens.zero_()
    assert ops.paged_kv_append(keys, values, cache, append_lens=new).seq_lens.tolist() == [6, 8]


def test_two_streams_and_a_captured_step() -> None:
    """One plan on two streams into two caches, and a step replayed from a graph into pages that were changed since."""
    lens, new = [5, 33], [1, 1]
    caches = [_case("int8_kv", lens, new, seed=7)[0] for _ in range(3)]
    _, keys, values = _case("int8_kv", lens, new, seed=7)
    plan = ops.plan_paged_kv_append(page_table=caches[0].page_table, seq_lens=caches[0].seq_lens, append_lens=torch.tensor(new),
                                    num_kv_heads=2, head_dim=128, page_size=16, kv_layout="int8_kv", use_cache=False)
    before, want = _copy(caches[0]), append64(caches[0], keys, values, new)
    plan.device_tables(keys.device, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for stream, cache in zip(streams, caches):
        with torch.cuda.stream(stream):
            ops.paged_kv_append(keys, values, cache, plan=plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_kv_append(keys, values, caches[2], plan=plan)
    graph.replay()
    torch.cuda.synchronize()
    for cache in caches:
        assert_append(before, cache, want, SLACK)
    for name in ("key_pages", "value_pages", "key_scales", "value_scales"):
        getattr(caches[2], name).copy_(getattr(before, name))
    graph.replay()
    torch.cuda.synchronize()
    assert_append(before, caches[2], want, SLACK)


def test_refusals_of_tensors() -> None:
    cache, keys, values = _case("bf16_kv", [4], [3])
    new = torch.tensor([3])
    with pytest.raises(TypeError, match="keys must have dtype"):
        ops.paged_kv_append(keys.half(), values, cache, append_lens=new)
    with pytest.raises(ValueError, match="values must be shaped"):
        ops.paged_kv_append(keys, values[:2], cache, append_lens=new)
    with pytest.raises(ValueError, match="keys must be a CUDA tensor"):
        ops.paged_kv_append(keys.cpu(), values, cache, append_lens=new)
    wide = torch.zeros((3, 2, 256), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="contiguous rows"):
        ops.paged_kv_append(wide[:, :, ::2], values, cache, append_lens=new)
    with pytest.raises(ValueError, match="contiguous rows"):
        ops.paged_kv_append(wide[:, :, 4:132], values, cache, append_lens=new)
    with pytest.raises(ValueError, match="the cache has 1$"):
        ops.paged_kv_append(keys, values, dataclasses.replace(cache, key_pages=cache.key_pages[:1], value_pages=cache.value_pages[:1],
                                                              page_table=torch.tensor([[3]])), append_lens=new)
    with pytest.raises(ValueError, match="must be contiguous"):
        ops.paged_kv_append(keys, values, dataclasses.replace(cache, key_pages=cache.key_pages.transpose(2, 3).contiguous().transpose(2, 3)),
                            append_lens=new)
    with pytest.raises(TypeError, match="key_scales must be a torch.Tensor"):
        ops.paged_kv_append(keys, values, dataclasses.replace(cache, kv_layout="int8_kv", key_pages=cache.key_pages.to(torch.int8),
                                                              value_pages=cache.value_pages.to(torch.int8)), append_lens=new)
