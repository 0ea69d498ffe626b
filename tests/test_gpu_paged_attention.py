"""paged_prompt_attention and shared_prefix_decode on the GPU against attention in 64 bits over the same bytes.

Tolerances, with u = 2^-8 (half a step of bf16) and h = 2^-11 (half a step of fp16; 2^-25 below 2^-14). Let a = sum_t p_t |v_t|
with the exact weights p. The row is rounded once: u |y|. The rest, to first order:

bf16 pages: the turned query is rounded to bf16, so that a logit is off by at most d = u * scale * sum_i |q_i k_i| and every
weight by a factor within e^(+-2 d); weights are rounded to bf16: (u + 2 d) a.

8-bit pages: query, keys and values are fp16. The query and the keys' elements are off by h, the elements of the block that has
not the page's larger scale by 2 h more (the ratio of the scales, the product), or by 2^-25 of that scale:
d = scale * (3 h sum_i |q_i k_i| + 2^-25 s_k sum_i |q_i|), one h where there is one block. The same of values and weights:
(3 h + 2 d) a + 2^-25 sum_t p_t s_t, and, since a weight p_t s_t below 2^-14 of the row's largest W is off by up to 2^-25 W
however small it is itself, 2^-25 W sum_t |v_t| / s_t.

d is taken at the largest sum over the row's tokens, times 1.1 for the higher orders; fp32 sums are well below all of these.
The tail of a shared decode rounds less. On top, an element-wise bound that wide says little about a token too many or too
few in a long row; the counting tests do: keys of zero make all weights equal, and each output counts the tokens of one
residue, so that one token more or less is seen at once."""

from __future__ import annotations

import dataclasses
import importlib

import numpy as np
import pytest
import torch
from fast_kernels.native import native_module
from paged_kv_testlib import (
    BLOCK,
    attention_terms64,
    default_scale,
    fragmented_table,
    random_cache,
)

pytestmark = pytest.mark.gpu
ops = importlib.import_module("fast_kernels.ops")
LAYOUTS = ("bf16_kv", "fp8_kv", "int8_kv")
THETA = 10000.0
U = 2.0**-8
H = 2.0**-11


def _status_ok() -> None:
    torch.cuda.synchronize()
    assert native_module().paged_kv_device_status() == 0 and native_module().page_decode_device_status() == 0


def _query(rows: int, heads: int, dim: int, seed: int) -> torch.Tensor:
    return torch.randn((rows, heads, dim), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


def _assert_rows(got: torch.Tensor, cache, query, rows, scale: float) -> None:
    terms = attention_terms64(cache, query, rows, scale, THETA)
    want, a = terms["out"], terms["a"]
    if cache.kv_layout == "bf16_kv":
        d = 1.1 * U * terms["logit"]
        bound = U * want.abs() + (U + 2 * d) * a + 1e-30
    else:
        h = H * (3 if cache.head_dim > BLOCK else 1)
        d = 1.1 * (h * terms["logit"] + 2.0**-25 * abs(scale) * terms["key_scale"] * terms["query"])
        bound = U * want.abs() + (h + 2 * d) * a + 2.0**-25 * (terms["weights"] + terms["weight"] * terms["numbers"]) + 1e-30
    off = (got.double().cpu() - want).abs()
    assert bool(torch.isfinite(got).all())
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.2f} x the bound, off by {float(off.max()):.3e}"
    # roundings are independent, so that as a whole the rows are much nearer than any one element must be
    if off.numel() >= 1000:
        assert float(off.norm() / want.norm()) <= 2.0**-7


def _counting_cache(layout, *, heads, dim, ps, table, lens, pages):
    """Keys 0; value dimension d of token t is 1 where t % dim == d. Slots behind a request's end hold NaN (bf16, e4m3) or
    the largest number."""
    cache = random_cache(layout=layout, pages=pages, heads=heads, page_size=ps, dim=dim, table=table, lens=lens, theta=THETA, seed=1)
    one = {"bf16_kv": 1.0, "fp8_kv": 0x38, "int8_kv": 127}[layout]
    bad = {"bf16_kv": float("nan"), "fp8_kv": 0x7F, "int8_kv": 127}[layout]
    cache.key_pages.fill_(bad)
    cache.value_pages.fill_(bad)
    if layout != "bf16_kv":
        cache.key_scales.fill_(0.5)
        cache.value_scales.fill_(float("nan"))
    table, lens = np.asarray(table), list(lens)
    for b, length in enumerate(lens):
        token = torch.arange(length)
        page = torch.from_numpy(table[b].astype(np.int64))[token // ps].cuda()
        slot = (token % ps).cuda()
        values = torch.zeros((length, dim), dtype=torch.float32)
        values[token, token % dim] = one
        cache.key_pages.transpose(1, 2)[page, slot] = torch.zeros((), dtype=cache.key_pages.dtype, device="cuda")
        cache.value_pages.transpose(1, 2)[page, slot] = values[:, None].expand(-1, heads, -1).to(cache.value_pages.dtype).cuda()
        if layout != "bf16_kv":
            cache.value_scales.transpose(1, 2)[page, slot] = 1.0 if layout == "fp8_kv" else 1.0 / 127.0
    return cache


def _assert_counts(got: torch.Tensor, positions: list[int], dim: int) -> None:
    """A rounding of the weight (1: none; 1/127 times 127: u), of the row, and fp32 sums: 2 u + u^2 covers them."""
    position = torch.tensor(positions, dtype=torch.float64)
    residue = torch.arange(dim, dtype=torch.float64)
    count = torch.clamp(torch.floor((position[:, None] - residue) / dim) + 1, min=0)
    want = (count / torch.clamp(position[:, None] + 1, min=1))[:, None].expand(-1, got.shape[1], -1)
    torch.testing.assert_close(got.double().cpu(), want, rtol=2 * U + U * U, atol=0)


# ---- prompts -----------------------------------------------------------------------------------------


def _prompt(layout, lens, new, *, heads=2, group=4, dim=128, ps=16, seed=0, counting=False, **kwargs):
    table, pages = fragmented_table([-(-n // ps) for n in lens], seed)
    make = dict(layout=layout, heads=heads, dim=dim, table=table, lens=lens, pages=pages)
    cache = _counting_cache(make.pop("layout"), ps=ps, **make) if counting else random_cache(
        page_size=ps, theta=THETA, seed=seed + 1, **make)
    rows = [(b, lens[b] - n + i) for b, n in enumerate(new) for i in range(n)]
    query = _query(len(rows), heads * group, dim, seed + 2)
    got = ops.paged_prompt_attention(query, cache, query_lens=torch.tensor(new), **kwargs)
    return cache, query, rows, got


@pytest.mark.parametrize(("dim", "ps"), [(64, 16), (64, 32), (128, 16), (128, 32)])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("group", [1, 3, 4, 8])
def test_prompts_every_instantiation(group, layout, dim, ps) -> None:
    """Whole prompts, a piece behind a cached part, one token, a request without queries, ends inside and on pages and tiles."""
    lens = [150, 2 * ps, 300, 1, 77, 128, 129]
    new = [150, 1, 40, 1, 0, 128, 2]
    cache, query, rows, got = _prompt(layout, lens, new, group=group, dim=dim, ps=ps, seed=group + dim + ps)
    _assert_rows(got, cache, query, rows, default_scale(dim))
    _status_ok()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize(("group", "dim", "ps", "lens", "new"), [
    (4, 128, 16, [1], [1]),
    (4, 128, 16, [1000, 16, 17], [1000, 16, 17]),
    (1, 64, 32, [513, 3000], [513, 2]),
    (2, 128, 32, [9000], [5]),       # cut into pieces
    (8, 64, 16, [5000, 127], [33, 60]),
    (3, 128, 16, [700, 0, 90], [100, 0, 90]),
])
def test_prompts_count_their_tokens(layout, group, dim, ps, lens, new) -> None:
    _, _, rows, got = _prompt(layout, lens, new, group=group, dim=dim, ps=ps, counting=True)
    _assert_counts(got, [p for _, p in rows], dim)
    _status_ok()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize(("heads", "group"), [(1, 128), (1, 200), (1, 256), (5, 7), (1, 1)])
def test_prompts_head_groups_that_fill_and_overflow_tiles(layout, heads, group) -> None:
    cache, query, rows, got = _prompt(layout, [40, 21], [3, 21], heads=heads, group=group, dim=64, seed=group)
    _assert_rows(got, cache, query, rows, default_scale(64))
    _status_ok()


@pytest.mark.parametrize("layout", LAYOUTS)
def test_prompts_with_uneven_magnitudes(layout) -> None:
    """Large queries (logits to +-100: the maximum moves late and far), tiny and huge value scales side by side, and a
    softmax scale of the caller's."""
    table, pages = fragmented_table([40, 3], 5)
    cache = random_cache(layout=layout, pages=pages, heads=2, page_size=16, dim=128, table=table, lens=[640, 40], theta=THETA, seed=6)
    if layout != "bf16_kv":
        cache.value_scales[..., 0] *= torch.logspace(-6, 3, pages, device="cuda")[:, None, None]
        cache.key_scales[..., 1] *= 1e-3
    query = 8 * _query(130, 8, 128, 7)
    got = ops.paged_prompt_attention(query, cache, query_lens=torch.tensor([100, 30]), softmax_scale=0.1)
    rows = [(0, 540 + i) for i in range(100)] + [(1, 10 + i) for i in range(30)]
    if layout == "bf16_kv":
        # the bound to first order is of no use where d is not small; 2^-8 of logits around 100 is 0.4
        query = query / 8
        got = ops.paged_prompt_attention(query, cache, query_lens=torch.tensor([100, 30]), softmax_scale=0.1)
    _assert_rows(got, cache, query, rows, 0.1)
    _status_ok()


def test_prompts_negative_zero_and_dominant_logits() -> None:
    """A scale of zero gives the mean; one key that dominates by more than fp32's exponents gives its value."""
    cache, query, rows, got = _prompt("bf16_kv", [200], [3], counting=True, softmax_scale=0.0)
    _assert_counts(got, [p for _, p in rows], 128)
    table = np.array([[0, 1]])
    cache = random_cache(layout="bf16_kv", pages=2, heads=1, page_size=16, dim=64, table=table, lens=[32], theta=THETA, seed=1)
    cache.key_pages.zero_()
    query = torch.zeros((1, 1, 64), dtype=torch.bfloat16, device="cuda")
    query[..., 63] = 1000.0  # the slowest pair: hardly turned at position 31
    for token in (0, 15, 16, 31):
        cache.key_pages.zero_()
        cache.key_pages[token // 16, 0, token % 16, 63] = 1000.0
        got = ops.paged_prompt_attention(query, cache, query_lens=torch.tensor([1]))
        assert torch.equal(got[0, 0], cache.value_pages[token // 16, 0, token % 16])
        got = ops.paged_prompt_attention(query, cache, query_lens=torch.tensor([1]), softmax_scale=-1.0)
        others = torch.cat([cache.value_pages[p, 0, s][None] for p in range(2) for s in range(16) if p * 16 + s != token])
        torch.testing.assert_close(got[0, 0].double(), others.double().mean(dim=0), rtol=U, atol=2.0**-20)


def test_prompts_strided_queries_and_given_output() -> None:
    fused = _query(50, 12, 64, 1)
    cache, _, rows, _ = _prompt("bf16_kv", [60], [50], group=2, heads=2, dim=64)
    view = fused[:, 4:8]
    output = torch.full((50, 4, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    got = ops.paged_prompt_attention(view, cache, query_lens=torch.tensor([50]), output=output)
    assert got is output
    same = ops.paged_prompt_attention(view.contiguous(), cache, query_lens=torch.tensor([50]))
    assert torch.equal(got.view(torch.int16), same.view(torch.int16))
    _assert_rows(got, cache, view, rows, default_scale(64))


def test_prompts_far_positions() -> None:
    """A request of 200000 tokens in one page used over and over: positions far out, the same keys all along."""
    length, ps = 200_000, 32
    table = np.zeros((1, -(-length // ps)), dtype=np.int32)
    cache = random_cache(layout="bf16_kv", pages=1, heads=1, page_size=ps, dim=128, table=table, lens=[length], theta=THETA, seed=1)
    query = _query(2, 4, 128, 3)
    got = ops.paged_prompt_attention(query, cache, query_lens=torch.tensor([2]))
    _assert_rows(got, cache, query, [(0, length - 2), (0, length - 1)], default_scale(128))


@pytest.mark.parametrize("layout", ["bf16_kv", "int8_kv"])
def test_prompts_pages_past_32_bit_offsets(layout) -> None:
    heads, dim, ps = 8, 128, 32
    pages = (2**31 if layout == "bf16_kv" else 2**32) // (heads * dim * ps) + 2
    small = random_cache(layout=layout, pages=3, heads=heads, page_size=ps, dim=dim, table=[[0, 2, 1]], lens=[90], theta=THETA, seed=1)
    tensors = {}
    for name in ("key_pages", "value_pages", "key_scales", "value_scales"):
        source = getattr(small, name)
        if source is not None:
            tensors[name] = torch.empty((pages, *source.shape[1:]), dtype=source.dtype, device="cuda")
            tensors[name][-3:] = source
    large = dataclasses.replace(small, page_table=small.page_table + (pages - 3), **tensors)
    query = _query(60, 16, dim, 3)
    want = ops.paged_prompt_attention(query, small, query_lens=torch.tensor([60]))
    got = ops.paged_prompt_attention(query, large, query_lens=torch.tensor([60]))
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    _assert_rows(want, small, query, [(0, 30 + i) for i in range(60)], default_scale(dim))


def test_prompts_same_bits_every_time_on_streams_and_in_graphs() -> None:
    cache, query, rows, first = _prompt("fp8_kv", [4000, 100], [40, 100])
    plan = ops.plan_paged_prompt_attention(page_table=cache.page_table, seq_lens=cache.seq_lens, query_lens=torch.tensor([40, 100]),
                                           num_q_heads=8, num_kv_heads=2, head_dim=128, page_size=16, kv_layout="fp8_kv", use_cache=False)
    assert plan.num_partials > 0
    plan.device_tables(query.device, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    outputs = []
    for stream in [torch.cuda.Stream() for _ in range(4)]:
        with torch.cuda.stream(stream):
            outputs += [ops.paged_prompt_attention(query, cache, plan=plan) for _ in range(3)]
    graphs = []
    for _ in range(2):  # two graphs, replayed side by side
        graph, output = torch.cuda.CUDAGraph(), torch.empty_like(first)
        with torch.cuda.graph(graph):
            ops.paged_prompt_attention(query, cache, plan=plan, output=output)
        graphs.append((graph, output))
    for _ in range(3):
        for stream, (graph, output) in zip([torch.cuda.Stream() for _ in range(2)], graphs):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for output in outputs + [output for _, output in graphs]:
        assert torch.equal(output.view(torch.int16), first.view(torch.int16))
    _assert_rows(first, cache, query, rows, default_scale(128))
    _status_ok()


def test_prompts_over_a_slice_of_a_cache() -> None:
    """All pages but the first, of one head: their scales start 4 bytes behind a boundary."""
    table, pages = fragmented_table([3, 2], 1)
    whole = random_cache(layout="int8_kv", pages=pages + 1, heads=1, page_size=16, dim=64, table=table, lens=[40, 32], theta=THETA, seed=4)
    cache = dataclasses.replace(whole, **{name: getattr(whole, name)[1:] for name in ("key_pages", "value_pages", "key_scales", "value_scales")})
    assert cache.key_scales.data_ptr() % 8 == 4
    query = _query(12, 4, 64, 6)
    rows = [(0, t) for t in range(30, 40)] + [(1, 30), (1, 31)]
    _assert_rows(ops.paged_prompt_attention(query, cache, query_lens=torch.tensor([10, 2])), cache, query, rows, default_scale(64))
    _status_ok()


def test_first_calls_of_a_plan_are_refused_inside_a_capture() -> None:
    table, pages = fragmented_table([3], 1)
    cache = random_cache(layout="bf16_kv", pages=pages, heads=2, page_size=16, dim=64, table=table, lens=[40], theta=THETA, seed=4)
    query = _query(3, 4, 64, 6)
    plan = ops.plan_paged_prompt_attention(page_table=cache.page_table, seq_lens=cache.seq_lens, query_lens=torch.tensor([3]), num_q_heads=4,
                                           num_kv_heads=2, head_dim=64, page_size=16, kv_layout="bf16_kv", use_cache=False)
    output = torch.empty_like(query)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="before the capture"):
            ops.paged_prompt_attention(query, cache, plan=plan, output=output)
        output.zero_()
    _assert_rows(ops.paged_prompt_attention(query, cache, plan=plan), cache, query, [(0, 37), (0, 38), (0, 39)], default_scale(64))
    _status_ok()


def test_prompts_empty_and_refused_calls() -> None:
    cache, query, _, got = _prompt("bf16_kv", [40], [3])
    assert ops.paged_prompt_attention(query[:0], cache, query_lens=torch.tensor([0])).shape == (0, 8, 128)
    new = torch.tensor([3])
    with pytest.raises(ValueError, match="query_lens or a plan"):
        ops.paged_prompt_attention(query, cache)
    with pytest.raises(ValueError, match="query must be shaped"):
        ops.paged_prompt_attention(query[:2], cache, query_lens=new)
    with pytest.raises(TypeError, match="query must have dtype"):
        ops.paged_prompt_attention(query.float(), cache, query_lens=new)
    with pytest.raises(ValueError, match="rotated ahead of time"):
        ops.paged_prompt_attention(query, dataclasses.replace(cache, keys_are_rotated=False), query_lens=new)
    with pytest.raises(ValueError, match="rope_theta must match"):
        ops.paged_prompt_attention(query, cache, query_lens=new, rope_theta=5000.0)
    with pytest.raises(ValueError, match="output must be contiguous"):
        ops.paged_prompt_attention(query, cache, query_lens=new, output=torch.empty((3, 16, 128), dtype=torch.bfloat16, device="cuda")[:, ::2])
    with pytest.raises(ValueError, match="softmax_scale must be finite"):
        ops.paged_prompt_attention(query, cache, query_lens=new, softmax_scale=float("inf"))
    with pytest.raises(ValueError, match="the plan names page"):
        ops.paged_prompt_attention(query, dataclasses.replace(cache, key_pages=cache.key_pages[:1], value_pages=cache.value_pages[:1]),
                                   query_lens=new)


# ---- shared beginnings -------------------------------------------------------------------------------


def _shared(layout, *, ps=16, heads=2, dim=64, prefixes=((0, 160), (0, 144), (1, 320)), seed=3, counting=False):
    """Requests whose pages begin alike: every request names the prefixes that it takes, in order, and a tail."""
    who = [([0], 7), ([], 0), ([0, 1], 33), ([0, 1], 1), ([], 90), ([0], 16), ([0, 1], 40), ([2], 0), ([2], 5), ([0, 1], 0)]
    counter = iter(range(10_000))
    take = lambda tokens: [next(counter) for _ in range(-(-tokens // ps))]  # noqa: E731
    bodies = [take(tokens) for _, tokens in prefixes]
    rows, lens = [], []
    for parts, tail in who:
        shared = [page for part in parts for page in bodies[part]]
        lens.append(len(shared) * ps + tail)
        rows.append(shared + take(tail))
    total = next(counter)
    rename = np.random.RandomState(seed).permutation(total)
    table = np.full((len(rows), max(map(len, rows))), -1, dtype=np.int32)
    for b, pages in enumerate(rows):
        table[b, : len(pages)] = rename[pages]
    if counting:
        return _counting_cache(layout, heads=heads, dim=dim, ps=ps, table=table, lens=lens, pages=total)
    return random_cache(layout=layout, pages=total, heads=heads, page_size=ps, dim=dim, table=table, lens=lens, theta=THETA, seed=seed)


def _shared_plan(cache, q_heads, **kwargs):
    return ops.plan_shared_prefix_decode(page_table=cache.page_table, seq_lens=cache.seq_lens, num_q_heads=q_heads,
                                         num_kv_heads=cache.num_kv_heads, head_dim=cache.head_dim, page_size=cache.page_size,
                                         kv_layout=cache.kv_layout, **{"use_cache": False, "min_saved_bytes": 0, **kwargs})


@pytest.mark.parametrize(("dim", "ps"), [(64, 16), (64, 32), (128, 16), (128, 32)])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("group", [1, 3, 8, 12])
def test_shared_every_instantiation(group, layout, dim, ps) -> None:
    cache = _shared(layout, ps=ps, dim=dim)
    plan = _shared_plan(cache, 2 * group)
    assert len(plan.runs) == 3
    query = _query(10, 2 * group, dim, 5)
    got = ops.shared_prefix_decode(query, cache, plan=plan)
    _assert_rows(got, cache, query, [(b, n - 1) for b, n in enumerate(cache.seq_lens.tolist())], default_scale(dim))
    _status_ok()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize(("group", "prefixes"), [
    (4, ((0, 160), (0, 144), (1, 320))), (1, ((0, 4096), (0, 128), (1, 1024))), (60, ((0, 256), (0, 2560), (1, 128)))])
def test_shared_counts_its_tokens(layout, group, prefixes) -> None:
    cache = _shared(layout, dim=128, prefixes=prefixes, counting=True)
    got = ops.shared_prefix_decode(_query(10, 2 * group, 128, 5), cache, plan=_shared_plan(cache, 2 * group))
    _assert_counts(got, [n - 1 for n in cache.seq_lens.tolist()], 128)
    _status_ok()


def test_shared_agrees_with_the_plain_decode_and_without_sharing_is_it() -> None:
    cache = _shared("int8_kv", dim=128, heads=4)
    query = _query(10, 16, 128, 5)
    plain = ops.clustered_page_decode(query, cache)
    small = ops.shared_prefix_decode(query, cache)  # too little to save: the same call
    assert torch.equal(small.view(torch.int16), plain.view(torch.int16))
    shared = ops.shared_prefix_decode(query, cache, plan=_shared_plan(cache, 16))
    torch.testing.assert_close(shared, plain, rtol=2e-2, atol=2e-2)  # both within the bounds above of the same numbers


def test_shared_same_bits_every_time_on_streams_and_in_graphs() -> None:
    cache = _shared("bf16_kv", dim=128, prefixes=((0, 4096), (0, 144), (1, 1024)))
    query = _query(10, 8, 128, 5)
    plan = _shared_plan(cache, 8)
    first = ops.shared_prefix_decode(query, cache, plan=plan)
    torch.cuda.synchronize()
    outputs = []
    for stream in [torch.cuda.Stream() for _ in range(4)]:
        with torch.cuda.stream(stream):
            outputs += [ops.shared_prefix_decode(query, cache, plan=plan) for _ in range(3)]
    graphs = []
    for _ in range(2):
        graph, output = torch.cuda.CUDAGraph(), torch.empty_like(first)
        with torch.cuda.graph(graph):
            ops.shared_prefix_decode(query, cache, plan=plan, output=output)
        graphs.append((graph, output))
    for _ in range(3):
        for stream, (graph, output) in zip([torch.cuda.Stream() for _ in range(2)], graphs):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for output in outputs + [output for _, output in graphs]:
        assert torch.equal(output.view(torch.int16), first.view(torch.int16))
    _status_ok()


def test_without_sharing_a_captured_call_needs_no_call_before_it() -> None:
    """Long requests on a stream that has made no call yet: the plain decode would want scratch of the stream's."""
    counts = [200, 3]
    table, pages = fragmented_table(counts, 1)
    cache = random_cache(layout="bf16_kv", pages=pages, heads=2, page_size=16, dim=64, table=table, lens=[3199, 40], theta=THETA, seed=2)
    query = _query(2, 8, 64, 3)
    plan = _shared_plan(cache, 8)
    assert plan.runs == []
    plan.device_tables(query.device, torch.cuda.current_stream().cuda_stream)
    output = torch.empty_like(query)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        ops.shared_prefix_decode(query, cache, plan=plan, output=output)
    graph.replay()
    torch.cuda.synchronize()
    _assert_rows(output, cache, query, [(0, 3198), (1, 39)], default_scale(64))
    _status_ok()


def test_shared_refusals() -> None:
    cache = _shared("bf16_kv")
    query = _query(10, 8, 64, 5)
    with pytest.raises(ValueError, match="query must be shaped"):
        ops.shared_prefix_decode(query[:9], cache)
    with pytest.raises(ValueError, match="query must be contiguous"):
        ops.shared_prefix_decode(_query(10, 16, 64, 5)[:, ::2], cache)
    with pytest.raises(ValueError, match="rotated ahead of time"):
        ops.shared_prefix_decode(query, dataclasses.replace(cache, keys_are_rotated=False))
    with pytest.raises(ValueError, match="rope_theta must match"):
        ops.shared_prefix_decode(query, cache, rope_theta=500.0)
    with pytest.raises(ValueError, match="the plan was made for page_size"):
        ops.shared_prefix_decode(query, cache, plan=dataclasses.replace(_shared_plan(cache, 8), page_size=32))


# ---- the operators one after the other ---------------------------------------------------------------


@pytest.mark.parametrize("layout", LAYOUTS)
def test_a_serving_loop_fills_attends_and_decodes(layout) -> None:
    """A system prompt is appended and attended over in two pieces, four requests continue behind its pages with prompts of
    their own, then all decode for a few steps; every stage against attention over the pages as they then are."""
    heads, group, dim, ps = 2, 4, 64, 16
    q_heads = heads * group
    system, own, steps = 288, [5, 40, 17, 33], 3
    gen = torch.Generator(device="cuda").manual_seed(1)

    def fused(tokens):
        rows = torch.randn((tokens, q_heads + 2 * heads, dim), generator=gen, device="cuda").to(torch.bfloat16)
        return rows[:, :q_heads], rows[:, q_heads : q_heads + heads], rows[:, q_heads + heads :]

    per_request = -(-(max(own) + steps) // ps)
    table = torch.arange(system // ps + 4 * per_request, dtype=torch.int32)
    shared_pages = table[: system // ps]
    cache = ops.empty_paged_kv(num_pages=len(table), page_table=shared_pages[None], seq_lens=torch.tensor([0]), num_kv_heads=heads,
                               head_dim=dim, page_size=ps, kv_layout=layout, key_rope_theta=THETA)
    for piece in (130, system - 130):
        q, k, v = fused(piece)
        begin = int(cache.seq_lens[0])
        cache = ops.paged_kv_append(k, v, cache, append_lens=torch.tensor([piece]))
        got = ops.paged_prompt_attention(q, cache, query_lens=torch.tensor([piece]))
        _assert_rows(got, cache, q, [(0, begin + i) for i in range(piece)], default_scale(dim))
    tails = table[system // ps :].reshape(4, per_request)
    cache = dataclasses.replace(cache, page_table=torch.cat([shared_pages.expand(4, -1), tails], dim=1),
                                seq_lens=torch.full((4,), system, dtype=torch.int32))
    q, k, v = fused(sum(own))
    cache = ops.paged_kv_append(k, v, cache, append_lens=torch.tensor(own))
    got = ops.paged_prompt_attention(q, cache, query_lens=torch.tensor(own))
    _assert_rows(got, cache, q, [(b, system + i) for b, n in enumerate(own) for i in range(n)], default_scale(dim))
    for _ in range(steps):
        q, k, v = fused(4)
        cache = ops.paged_kv_append(k, v, cache, append_lens=torch.ones(4, dtype=torch.int32))
        rows = [(b, n - 1) for b, n in enumerate(cache.seq_lens.tolist())]
        plan = _shared_plan(cache, q_heads)
        assert plan.runs == [(0, system // ps, (0, 1, 2, 3))]
        q = q.contiguous()
        got = ops.shared_prefix_decode(q, cache, plan=plan)
        _assert_rows(got, cache, q, rows, default_scale(dim))
        _assert_rows(ops.clustered_page_decode(q, cache), cache, q, rows, default_scale(dim))
    assert cache.seq_lens.tolist() == [system + n + steps for n in own]
    _status_ok()
