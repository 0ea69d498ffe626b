"""Causal attention of prompt tokens over a paged cache.

``clustered_page_decode`` serves one new token per request. This operator serves any number: the last
``query_lens[b]`` of a request's ``seq_lens[b]`` tokens (a whole prompt, a piece of one behind what is
cached already, a few tokens to be checked at once, or a single one), each attending over the
request's tokens up to and including itself. Keys and values are in the pages before the call
(``paged_kv_append``), in any of the cache's formats, with the keys turned by their positions:

    out_i = sum_{t <= pos_i} softmax_t(scale * <R(pos_i) q_i, k_t>) v_t,   pos_i = seq_len - query_len + i

Grouped-query heads share a kernel tile, so a page is read once for all of them. The plan cuts the
work into items (up to 256 query rows of one kv head over a range of tokens) that fill the device, and
cuts long ranges in pieces whose partial results a second kernel adds in order: results do not depend
on timing. Inference only: there is no backward pass.

bf16 pages: the turned query and the weights are rounded to bf16 once (the tensor cores take both operands in
one type), the row is off by 2.5e-3 to 2.9e-3 in the 2-norm where its own rounding is 1.7e-3. 8-bit pages: fp16, the
row's own rounding, as long as the scales of a token's (keys: a page's) two 64-dim blocks are within 2^24 of each other.

A bounded wait inside the kernel that gives up leaves the call's output invalid and raises nothing:
``fast_kernels.native.native_module().paged_kv_device_status()`` is 0 while none has.
"""

from __future__ import annotations

import math
from collections import OrderedDict
from dataclasses import dataclass, field
from typing import Any

import numpy as np

from fast_kernels.ops import _paged, _paged_items
from fast_kernels.ops.clustered_page_decode import KvLayout, PagedKVCache, _layout_id, _torch

_PLANS: OrderedDict = OrderedDict()


@dataclass(slots=True)
class PagedPromptPlan:
    batch: int
    page_size: int
    num_q_heads: int
    num_kv_heads: int
    head_dim: int
    kv_layout: KvLayout
    num_tokens: int
    num_partials: int
    largest_page: int
    page_ids_cpu: Any  # int32: the requests' pages, one request after the other
    vectors_cpu: Any   # int32 [tokens, 4]: row, position, first partial result, partial results
    items_cpu: Any     # int32 [items, 8]
    _device_cache: dict[int, Any] = field(default_factory=dict, repr=False)

    @property
    def num_items(self) -> int:
        return int(self.items_cpu.shape[0])

    def device_tables(self, device: Any, stream: int) -> dict[str, int]:
        """Addresses of the tables on `device`, for a launch on `stream`; uploaded once per device."""
        return _paged.on_device(self._device_cache, device, stream, lambda: {
            "page_ids": self.page_ids_cpu.numpy(), "vectors": self.vectors_cpu.numpy(), "items": self.items_cpu.numpy()})


def plan_paged_prompt_attention(
    *,
    page_table: Any,
    seq_lens: Any,
    query_lens: Any,
    num_q_heads: int,
    num_kv_heads: int,
    head_dim: int,
    page_size: int,
    kv_layout: str,
    use_cache: bool = True,
) -> PagedPromptPlan:
    """`seq_lens` counts every request's tokens, the `query_lens` new ones among them."""
    layout = _paged.require_geometry(num_kv_heads=num_kv_heads, head_dim=head_dim, page_size=page_size, kv_layout=kv_layout,
                                     num_q_heads=num_q_heads)
    if num_q_heads // num_kv_heads > _paged_items.ITEM_ROWS:
        raise ValueError(f"at most {_paged_items.ITEM_ROWS} query heads per kv head")
    table, lens, new = _paged.table_and_lengths(page_table, seq_lens=seq_lens, query_lens=query_lens)
    _paged.require_countable(lens)
    if lens.size and bool((new > lens).any()):
        raise ValueError("query_lens must not exceed seq_lens")
    made_from = (table, lens, new, num_q_heads, num_kv_heads, head_dim, page_size, layout)
    return _paged.remembered(_PLANS, made_from, lambda: _build(*made_from), use_cache)


def _build(table: np.ndarray, lens: np.ndarray, new: np.ndarray, num_q_heads: int, num_kv_heads: int, head_dim: int,
           page_size: int, layout: KvLayout) -> PagedPromptPlan:
    torch = _torch()
    lens = np.where(new > 0, lens, 0)  # a request without queries needs no pages
    pages = -(-lens // page_size)
    if pages.size and int(pages.max()) > table.shape[1]:
        raise ValueError("page_table has fewer columns than the tokens need")
    request = np.repeat(np.arange(len(lens)), pages)
    entries = np.cumsum(pages) - pages
    page_ids = _paged.require_pages(table, request, np.arange(int(pages.sum())) - entries[request])
    # groups of vectors that an item carries
    per_item = _paged_items.ITEM_ROWS // (num_q_heads // num_kv_heads)
    start = np.cumsum(new) - new
    groups = -(-new // per_item)
    owner = np.repeat(np.arange(len(lens)), groups)
    within = (np.arange(int(groups.sum())) - np.repeat(np.cumsum(groups) - groups, groups)) * per_item
    vectors = np.minimum(per_item, new[owner] - within)
    end = lens[owner] - new[owner] + within + vectors
    first = np.zeros_like(end)
    pieces = _paged_items.pieces_for(-(-end // _paged_items.TILE_TOKENS), num_kv_heads, fewest=4)
    group, number, begin, stop = _paged_items.cut(first, end, pieces)
    pieces = np.bincount(group, minlength=len(end))
    items = _paged_items.item_rows(
        first_vector=(start[owner] + within)[group], vectors=vectors[group], entry=entries[owner][group], first=begin, end=stop,
        causal=1, partial=np.where(pieces[group] > 1, number, -1), kv_heads=num_kv_heads)
    # every vector's place among the queries, in the sequence, and among the partial results
    tokens = int(new.sum())
    count = np.repeat(np.where(pieces > 1, pieces, 0), vectors)
    position = np.arange(tokens) - np.repeat(start, new) + np.repeat(lens - new, new)
    rows = np.stack((np.arange(tokens), position, np.cumsum(count) - count, count), axis=1)
    if int(count.sum()) >= 1 << 31 or tokens >= 1 << 31:
        raise ValueError("too many tokens for one call")
    return PagedPromptPlan(
        batch=len(lens), page_size=page_size, num_q_heads=num_q_heads, num_kv_heads=num_kv_heads, head_dim=head_dim,
        kv_layout=layout, num_tokens=tokens, num_partials=int(count.sum()),
        largest_page=int(page_ids.max()) if page_ids.size else -1, page_ids_cpu=torch.from_numpy(page_ids.astype(np.int32)),
        vectors_cpu=torch.from_numpy(rows.astype(np.int32)), items_cpu=torch.from_numpy(items))


def paged_prompt_attention(
    query: Any,
    cache: PagedKVCache,
    *,
    query_lens: Any | None = None,
    plan: PagedPromptPlan | None = None,
    output: Any | None = None,
    softmax_scale: float | None = None,
    rope_theta: float = 10000.0,
) -> Any:
    """`query` is bf16 [tokens, q_heads, head_dim], the requests' new tokens one request after the other (a view into
    a fused projection's rows will do), not yet turned by their positions. Either `query_lens` or a `plan` says how
    many tokens each request has. A NaN or infinity in the keys or values of a request's tokens may reach the outputs of
    all of that request's queries; pages behind its last token may hold anything."""
    torch = _torch()
    native = _paged.backend()
    if not isinstance(query, torch.Tensor):
        raise TypeError("query must be a torch.Tensor")
    if query.ndim != 3:
        raise ValueError("query must be 3D")
    found = plan is None
    if plan is None:
        if query_lens is None:
            raise ValueError("paged_prompt_attention needs query_lens or a plan")
        plan = plan_paged_prompt_attention(
            page_table=cache.page_table, seq_lens=cache.seq_lens, query_lens=query_lens, num_q_heads=int(query.shape[1]),
            num_kv_heads=cache.num_kv_heads, head_dim=cache.head_dim, page_size=cache.page_size, kv_layout=cache.kv_layout)
    elif query_lens is not None:
        raise ValueError("give query_lens or a plan, not both")
    device = _paged.check_cache(cache, plan)
    shape = (plan.num_tokens, plan.num_q_heads, plan.head_dim)
    _paged.check_rows(query, name="query", shape=shape, device=device)
    _paged.check_turned_keys(cache, rope_theta)
    if output is None:
        output = torch.empty(shape, dtype=torch.bfloat16, device=device)
    else:
        _paged.check_output(output, shape=shape, device=device)
    if plan.num_tokens:
        scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(plan.head_dim)
        with _paged.current(device):
            stream = _paged.current_stream(device)
            if found:
                _paged.keep_for_graphs(plan)
            tables = plan.device_tables(device, stream)
            partials = None
            if plan.num_partials:
                partials = torch.empty((plan.num_partials, plan.num_q_heads, plan.head_dim + 4), dtype=torch.float32, device=device)
            native.paged_attention_forward(
                query.data_ptr(), *_paged.row_strides(query), cache.key_pages.data_ptr(), cache.value_pages.data_ptr(),
                _paged.address(cache.key_scales), _paged.address(cache.value_scales), tables["page_ids"], tables["vectors"],
                tables["items"], output.data_ptr(), _paged.address(partials), plan.num_tokens, plan.page_ids_cpu.shape[0],
                plan.num_tokens, plan.num_items, plan.num_partials, cache.key_pages.shape[0], plan.num_q_heads,
                plan.num_kv_heads, plan.head_dim, plan.page_size, _layout_id(plan.kv_layout), float(scale),
                float(rope_theta), stream)
    return output
