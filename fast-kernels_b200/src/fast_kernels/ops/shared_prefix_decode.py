"""Decode attention for a batch whose requests share pages, every shared page read once for all of them.

One new token per request, as in ``clustered_page_decode``, for caches in which page tables begin with
the same physical pages: one system prompt for a batch, a document that some of its requests ask
about, several continuations of one prompt. The plan finds what is shared from the page tables alone, at
any number of levels: runs of full pages that two or more requests have in common become products of
all these requests' query rows with the run's keys and values (one kernel, tensor cores), and what a
request has to itself goes through the paged decode kernel, which merges it with the partial results
of the runs:

    out = (sum_j e^(m_j - m) o_j) / (sum_j e^(m_j - m) l_j),   m = max_j m_j

over the runs that a request takes part in and its own tokens, maxima and sums in fp32, in a fixed
order. Where sharing would not pay (``estimated_saved_hbm_bytes`` below what the second kernel costs)
the plan is the plain decode.

Over shared runs of bf16 pages the turned query and the weights are rounded to bf16 once (the tensor cores
take both operands in one type): a row is off by 2.9e-3 in the 2-norm where the plain decode, which carries
both as 16-bit heads and remainders, has the output's own rounding, 1.7e-3. A request's row is so less exact when its batch
shares than when it does not; ``min_saved_bytes`` beyond any saving keeps the plan plain. 8-bit pages have
fp16 weights and stay at the output's rounding.

A bounded wait inside a kernel that gives up leaves the call's output invalid and raises nothing:
``fast_kernels.native.native_module()`` has ``paged_kv_device_status()`` and ``page_decode_device_status()``, 0 while
none has.

``prefix_union_decode`` keeps the contract of the op of that name, which on this device computes every
request by itself.
"""

from __future__ import annotations

import math
from collections import OrderedDict
from dataclasses import dataclass, field
from typing import Any

import numpy as np

from fast_kernels.ops import _paged, _paged_items
from fast_kernels.ops.clustered_page_decode import (
    ClusteredPageDecodePlan,
    KvLayout,
    PagedKVCache,
    _layout_id,
    _torch,
    plan_clustered_page_decode,
)
from fast_kernels.ops.prefix_union_decode import _shared_page_bytes

_PLANS: OrderedDict = OrderedDict()
# Bytes that a plan has to save before it shares. Measured in graphs, us with sharing / without, requests with 200 tokens of
# their own behind 1024 that they share. 8 kv heads of 128 x 4 query heads, bf16: 63 MB saved 21.9 / 19.1, 130 MB 25.5 / 27.2,
# 264 MB 35.8 / 51.9; int8: 32 MB 26.4 / 21.4, 67 MB 29.7 / 31.7, 136 MB 40.8 / 59.5. 8 heads of 64 x 2, bf16: 31 MB
# 18.7 / 15.7, 65 MB 19.9 / 22.6; int8: 34 MB 23.0 / 21.8, 68 MB 26.2 / 40.4. 32 heads of 128 x 1, bf16: 117 MB 26.3 / 26.3,
# 252 MB 33.2 / 49.9. Not the bytes alone count: 4096 shared tokens pay from 25 to 60 MB on, and few heads with many
# requests later (2 heads of 128 x 8, 64 requests, bf16: 66 MB 26.0 / 20.1).
DEFAULT_MIN_SAVED_BYTES = 64 << 20
# From this length on the plain decode's angle, an fp32 product of position and frequency, is not good enough for keys whose
# own angle is exact (paged_kv_append): off by up to 2e-3 radians here (logits by 1e-4 on average, their outputs' rounding is
# 2e-3), and growing with the position. Shorter requests that share nothing are turned by it all the same, and so have the bits
# of clustered_page_decode.
FAR_TOKENS = 32768
# Shared runs shorter than this stay with the requests (or with longer runs further down).
MIN_RUN_TOKENS = 128


@dataclass(slots=True)
class SharedPrefixDecodePlan:
    batch: int
    page_size: int
    num_q_heads: int
    num_kv_heads: int
    head_dim: int
    kv_layout: KvLayout
    estimated_saved_hbm_bytes: int
    num_partials: int
    largest_page: int
    # per shared run: first page, end page (of the requests' tables), requests in order
    runs: list[tuple[int, int, tuple[int, ...]]]
    page_ids_cpu: Any    # int32: the pages of the requests that stand for a run each
    vectors_cpu: Any     # int32 [batch, 4]: request, position, first partial result, partial results
    items_cpu: Any       # int32 [items, 8]
    of_request_cpu: Any  # int32 [batch, 2]: first partial result, partial results
    tail_plan: ClusteredPageDecodePlan  # what every request has to itself (all of it where nothing is shared)
    far: bool  # some request is longer than FAR_TOKENS
    _device_cache: dict[int, Any] = field(default_factory=dict, repr=False)

    @property
    def num_items(self) -> int:
        return int(self.items_cpu.shape[0])

    def device_tables(self, device: Any, stream: int) -> dict[str, int]:
        """Addresses of the tables on `device`, for a launch on `stream`; uploaded once per device."""
        return _paged.on_device(self._device_cache, device, stream, lambda: {
            "page_ids": self.page_ids_cpu.numpy(), "vectors": self.vectors_cpu.numpy(), "items": self.items_cpu.numpy(),
            "of_request": self.of_request_cpu.numpy(),
            **{name: getattr(self.tail_plan, f"{name}_cpu").numpy() for name in (
                "run_base_pages", "run_page_counts", "run_logical_starts", "run_last_page_lens", "request_run_offsets", "seq_lens")}})


def _shared_runs(table: np.ndarray, full_pages: np.ndarray, min_pages: int) -> tuple[np.ndarray, list[tuple[int, int, int, int]]]:
    """(order, runs): requests sorted so that sharers are neighbours, and (first page, end page, first, end) of the shared
    runs, the outer ones first, as ranges of that order. A run is a maximal stretch of full pages that the same requests
    have in common; one shorter than `min_pages` is left to what comes further down."""
    batch = len(full_pages)
    width = int(full_pages.max()) if batch else 0
    fill = (-1 - np.arange(batch)).astype(table.dtype)[:, None]
    rows = np.where(np.arange(width) < full_pages[:, None], table[:, :width], fill)
    # (by their bytes: any order will do in which equal beginnings are neighbours)
    order = np.array(sorted(range(batch), key=lambda b: rows[b].tobytes()), dtype=np.int64)
    rows = rows[order]
    same = rows[1:] == rows[:-1]
    common = np.where(same.all(axis=1), width, np.argmin(same, axis=1)) if width and batch > 1 else np.zeros(max(0, batch - 1), dtype=np.int64)
    runs: list[tuple[int, int, int, int]] = []
    stack = [(0, batch, 0)]
    while stack:
        low, high, covered = stack.pop()
        if high - low < 2:
            continue
        between = common[low : high - 1]
        shared = int(between.min())
        if shared - covered >= min_pages:
            runs.append((covered, shared, low, high))
            covered = shared
        edges = np.flatnonzero(between == shared) + low + 1
        bounds = [low, *edges.tolist(), high]
        stack += [(a, b, covered) for a, b in zip(bounds[:-1], bounds[1:])][::-1]
    return order, runs


def plan_shared_prefix_decode(
    *,
    page_table: Any,
    seq_lens: Any,
    num_q_heads: int,
    num_kv_heads: int,
    head_dim: int,
    page_size: int,
    kv_layout: str,
    min_saved_bytes: int = DEFAULT_MIN_SAVED_BYTES,
    use_cache: bool = True,
) -> SharedPrefixDecodePlan:
    """`min_saved_bytes` is what sharing must save of a call's traffic before the plan shares at all (0: always). The plan is
    the caller's to keep as long as graphs that were captured with it."""
    layout = _paged.require_geometry(num_kv_heads=num_kv_heads, head_dim=head_dim, page_size=page_size, kv_layout=kv_layout,
                                     num_q_heads=num_q_heads)
    if num_q_heads // num_kv_heads > _paged_items.ITEM_ROWS:
        raise ValueError(f"at most {_paged_items.ITEM_ROWS} query heads per kv head")
    if min_saved_bytes < 0:
        raise ValueError("min_saved_bytes must not be negative")
    table, lens = _paged.table_and_lengths(page_table, seq_lens=seq_lens)
    if lens.size == 0:
        raise ValueError("the batch must not be empty")
    _paged.require_countable(lens)
    made_from = (table, lens, num_q_heads, num_kv_heads, head_dim, page_size, layout, min_saved_bytes)
    return _paged.remembered(_PLANS, made_from, lambda: _build(*made_from), use_cache)


def _build(table: np.ndarray, lens: np.ndarray, num_q_heads: int, num_kv_heads: int, head_dim: int, page_size: int,
           layout: KvLayout, min_saved_bytes: int) -> SharedPrefixDecodePlan:
    torch = _torch()
    batch = len(lens)
    pages = -(-lens // page_size)
    if int(pages.max()) > table.shape[1]:
        raise ValueError("page_table has fewer columns than the tokens need")
    slots = np.arange(int(pages.max()))
    table = table[:, : len(slots)]
    used = table[slots < pages[:, None]]
    if used.size and int(used.min()) < 0:
        raise ValueError("page_table has no page for some of the tokens")
    if used.dtype != np.int32 and used.size and int(used.max()) >= 1 << 31:
        raise ValueError("page_table entries must fit 32 bits")
    order, runs = _shared_runs(table, lens // page_size, -(-MIN_RUN_TOKENS // page_size))
    saved = sum((high - low - 1) * (end - first) for first, end, low, high in runs)
    saved *= num_kv_heads * _shared_page_bytes(page_size, head_dim, layout)
    if saved < min_saved_bytes or saved == 0:
        runs, saved = [], 0

    # items: every run for groups of the requests' rows, cut so that all runs together fill the device
    per_item = _paged_items.ITEM_ROWS // (num_q_heads // num_kv_heads)
    run_pages = np.array([(first, end) for first, end, _, _ in runs], dtype=np.int64).reshape(-1, 2)
    span = np.array([(low, high) for _, _, low, high in runs], dtype=np.int64).reshape(-1, 2)
    entries = np.cumsum(run_pages[:, 1]) - run_pages[:, 1] if len(runs) else np.zeros(0, dtype=np.int64)
    page_ids = np.concatenate([table[order[low], :end] for (_, end), (low, _) in zip(run_pages, span)] or [np.zeros(0, dtype=np.int64)])
    sharers = span[:, 1] - span[:, 0]
    groups = -(-sharers // per_item)
    tiles = -(-((run_pages[:, 1] - run_pages[:, 0]) * page_size) // _paged_items.TILE_TOKENS)
    owner = np.repeat(np.arange(len(runs)), groups)
    pieces = np.ones(len(runs), dtype=np.int64)
    if len(runs):
        by_group = _paged_items.pieces_for(tiles[owner], num_kv_heads)
        pieces[owner] = by_group
    run, number, begin, stop = _paged_items.cut(run_pages[:, 0] * page_size, run_pages[:, 1] * page_size, pieces)
    pieces = np.bincount(run, minlength=len(runs))
    # partial results of a request: its runs from the outermost in, the pieces of each in order
    partials = np.zeros(batch, dtype=np.int64)  # by place in the order
    offset = np.zeros(len(runs), dtype=np.int64)
    for index, (_, _, low, high) in enumerate(runs):  # the outer runs come first
        offset[index] = partials[low]
        partials[low:high] += pieces[index]
    first_partial = np.cumsum(partials) - partials
    fan = groups[run]
    piece = np.repeat(np.arange(len(run)), fan)
    within = (np.arange(int(fan.sum())) - np.repeat(np.cumsum(fan) - fan, fan)) * per_item
    items = _paged_items.item_rows(
        first_vector=span[run][piece, 0] + within, vectors=np.minimum(per_item, sharers[run][piece] - within), entry=entries[run][piece],
        first=begin[piece], end=stop[piece], causal=0, partial=(offset[run] + number)[piece], kv_heads=num_kv_heads)
    vectors = np.stack((order, np.maximum(lens[order] - 1, 0), first_partial, partials), axis=1)
    of_request = np.zeros((batch, 2), dtype=np.int64)
    of_request[order] = np.stack((first_partial, partials), axis=1)

    # what is left to every request: its pages behind the last run that it takes part in
    covered = np.zeros(batch, dtype=np.int64)
    for _, end, low, high in runs:
        covered[order[low:high]] = end
    rest = lens - covered * page_size
    shifted = np.full((batch, max(1, int((-(-rest // page_size)).max()))), -1, dtype=np.int32)
    column = np.arange(shifted.shape[1])
    take = column < (-(-rest // page_size))[:, None]
    shifted[take] = np.take_along_axis(table, np.minimum(column + covered[:, None], max(0, table.shape[1] - 1)), axis=1)[take] if table.shape[1] else 0
    tail_plan = plan_clustered_page_decode(
        page_table=torch.from_numpy(shifted), seq_lens=torch.from_numpy(rest), num_q_heads=num_q_heads, num_kv_heads=num_kv_heads,
        head_dim=head_dim, page_size=page_size, kv_layout=layout, use_cache=False)
    tail_plan.seq_lens_cpu = torch.from_numpy(lens.astype(np.int32))  # the queries sit behind everything
    return SharedPrefixDecodePlan(
        batch=batch, page_size=page_size, num_q_heads=num_q_heads, num_kv_heads=num_kv_heads, head_dim=head_dim, kv_layout=layout,
        estimated_saved_hbm_bytes=saved, num_partials=int(partials.sum()), largest_page=int(used.max()) if used.size else -1,
        runs=[(first, end, tuple(sorted(order[low:high].tolist()))) for first, end, low, high in runs],
        page_ids_cpu=torch.from_numpy(page_ids.astype(np.int32)), vectors_cpu=torch.from_numpy(vectors.astype(np.int32)),
        items_cpu=torch.from_numpy(items), of_request_cpu=torch.from_numpy(of_request.astype(np.int32)), tail_plan=tail_plan,
        far=int(lens.max()) > FAR_TOKENS)


def shared_prefix_decode(
    query: Any,
    cache: PagedKVCache,
    *,
    plan: SharedPrefixDecodePlan | None = None,
    output: Any | None = None,
    softmax_scale: float | None = None,
    rope_theta: float = 10000.0,
) -> Any:
    """`query` is bf16 [batch, q_heads, head_dim], contiguous, not yet turned by its positions; request b's token is the
    last of its `seq_lens[b]`. The cache's keys are turned ahead of time (`key_rope_theta`). Requests that share pages, and
    batches with one beyond `FAR_TOKENS`, have their queries turned by exact angles (as `paged_kv_append` turns keys);
    others by those of `clustered_page_decode`, products in fp32."""
    torch = _torch()
    native = _paged.backend()
    if not isinstance(query, torch.Tensor):
        raise TypeError("query must be a torch.Tensor")
    if query.ndim != 3:
        raise ValueError("query must be 3D")
    found = plan is None
    if plan is None:
        plan = plan_shared_prefix_decode(
            page_table=cache.page_table, seq_lens=cache.seq_lens, num_q_heads=int(query.shape[1]),
            num_kv_heads=cache.num_kv_heads, head_dim=cache.head_dim, page_size=cache.page_size, kv_layout=cache.kv_layout)
    device = _paged.check_cache(cache, plan)
    shape = (plan.batch, plan.num_q_heads, plan.head_dim)
    _paged.check_output(query, shape=shape, device=device, name="query")
    _paged.check_turned_keys(cache, rope_theta)
    if output is None:
        output = torch.empty_like(query)
    else:
        _paged.check_output(output, shape=shape, device=device)
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(plan.head_dim)
    with _paged.current(device):
        stream = _paged.current_stream(device)
        if found:
            _paged.keep_for_graphs(plan)
        tables = plan.device_tables(device, stream)
        tail = plan.tail_plan
        if not plan.runs:  # the launch that clustered_page_decode makes, except for the angle of far queries
            # (it may split long requests through scratch: the stream's, or, since graphs that were captured on one stream
            # may be replayed at the same time, a captured call's own)
            scratch = None
            if torch.cuda.is_current_stream_capturing():
                scratch = torch.empty(native.page_decode_workspace_bytes(plan.batch, plan.num_q_heads, plan.num_kv_heads, plan.head_dim),
                                      dtype=torch.uint8, device=device)
            direct = tail.launch_mode == "direct"
            native.clustered_page_decode_forward(
                query.data_ptr(), cache.key_pages.data_ptr(), cache.value_pages.data_ptr(), _paged.address(cache.key_scales),
                _paged.address(cache.value_scales), tables["run_base_pages"], tables["run_page_counts"], tables["run_logical_starts"],
                tables["run_last_page_lens"], tables["request_run_offsets"], tables["seq_lens"], output.data_ptr(), plan.batch,
                tail.num_runs, plan.num_q_heads, plan.num_kv_heads, plan.head_dim, plan.page_size, tail.group_tile, int(not direct),
                1 if direct else max(2, tail.cluster_size), _layout_id(plan.kv_layout), int(cache.keys_are_rotated), float(scale),
                float(rope_theta), stream, max_pages_hint=tail.max_pages, early_descriptors=1, workspace_ptr=_paged.address(scratch),
                exact_turns=int(plan.far))
            return output
        partials = torch.empty((plan.num_partials, plan.num_q_heads, plan.head_dim + 4), dtype=torch.float32, device=device)
        native.shared_prefix_decode_forward(
            query.data_ptr(), cache.key_pages.data_ptr(), cache.value_pages.data_ptr(), _paged.address(cache.key_scales),
            _paged.address(cache.value_scales), tables["page_ids"], tables["vectors"], tables["items"], tables["of_request"],
            tables["run_base_pages"], tables["run_page_counts"], tables["run_logical_starts"], tables["run_last_page_lens"],
            tables["request_run_offsets"], tables["seq_lens"], output.data_ptr(), _paged.address(partials), plan.batch,
            plan.page_ids_cpu.shape[0], plan.num_items, plan.num_partials, tail.num_runs, tail.max_pages,
            cache.key_pages.shape[0], plan.num_q_heads, plan.num_kv_heads, plan.head_dim, plan.page_size,
            _layout_id(plan.kv_layout), float(scale), float(rope_theta), stream)
    return output
