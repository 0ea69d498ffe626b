"""New keys and values of a batch into the pages of a paged cache, in the cache's own format.

The builders of ``clustered_page_decode`` make a cache out of whole sequences. A server fills one as it
goes: the tokens of a prompt (or of a piece of it), then one token per request and step. For every new
token of request ``b``, at position ``seq_lens[b] + i``, this operator turns the key by its position
(where the cache holds turned keys), and writes key and value into the page and slot that the page table
says:

* ``bf16_kv``: the turned key rounded once, the value as it is;
* ``int8_kv`` / ``fp8_kv`` (L = 127 / 448), per 64-dim block: a value as ``round(v / s)`` with
  ``s = max(max|v| / L, 1e-6)`` of its own token; a key with the scale of its page,
  ``s' = max(s, max|k| / L, 1e-6)``, where ``s`` is what the page has, or 0 where the new tokens begin the
  page (whatever a reused page held is gone). Where the scale grows, the tokens that the page holds
  already become ``round(q s / s')``. A prompt appended at once to fresh pages gives the scales that
  ``quantize_paged_kv_int8`` / ``_fp8`` compute.

The pages are written in place. ``reference_key_pages`` / ``reference_value_pages`` are not: the cache that
is returned has them only where they are the pages themselves (bf16), not where they would lack the new
tokens. A page that two requests
share is the caller's to copy before one of them writes to it; two requests that would write to the
same page are refused.
"""

from __future__ import annotations

import dataclasses
from collections import OrderedDict
from dataclasses import dataclass, field
from typing import Any

import numpy as np

from fast_kernels.ops import _paged
from fast_kernels.ops.clustered_page_decode import (
    _SCALE_BLOCK,
    KvLayout,
    PagedKVCache,
    _layout_id,
    _torch,
)

_PLANS: OrderedDict = OrderedDict()


@dataclass(slots=True)
class PagedKVAppendPlan:
    batch: int
    page_size: int
    num_kv_heads: int
    head_dim: int
    kv_layout: KvLayout
    num_tokens: int
    largest_page: int
    # int32 [segments, 4]: physical page, first slot | count << 16, first row of the new tokens, its position
    segments_cpu: Any
    seq_lens_after_cpu: Any
    _device_cache: dict[int, Any] = field(default_factory=dict, repr=False)

    @property
    def num_segments(self) -> int:
        return int(self.segments_cpu.shape[0])

    def device_tables(self, device: Any, stream: int) -> dict[str, int]:
        """Addresses of the tables on `device`, for a launch on `stream`; uploaded once per device."""
        return _paged.on_device(self._device_cache, device, stream, lambda: {"segments": self.segments_cpu.numpy()})


def empty_paged_kv(*, num_pages: int, page_table: Any, seq_lens: Any, num_kv_heads: int, head_dim: int, page_size: int,
                   kv_layout: str, key_rope_theta: float | None = None, device: Any = "cuda") -> PagedKVCache:
    """A cache of `num_pages` zeroed pages for `paged_kv_append` to fill. With `key_rope_theta` its keys are
    turned by their positions as they are appended, otherwise they are stored as they come."""
    torch = _torch()
    layout = _paged.require_geometry(num_kv_heads=num_kv_heads, head_dim=head_dim, page_size=page_size, kv_layout=kv_layout)
    if num_pages < 0:
        raise ValueError("num_pages must not be negative")
    _paged.table_and_lengths(page_table, seq_lens=seq_lens)
    element = {"bf16_kv": torch.bfloat16, "fp8_kv": torch.uint8, "int8_kv": torch.int8}[layout]
    shape = (num_pages, num_kv_heads, page_size, head_dim)
    keys, values = (torch.zeros(shape, dtype=element, device=device) for _ in range(2))
    key_scales = value_scales = None
    if layout != "bf16_kv":
        blocks = head_dim // _SCALE_BLOCK
        key_scales = torch.zeros((*shape[:2], blocks), dtype=torch.float32, device=device)
        value_scales = torch.zeros((*shape[:3], blocks), dtype=torch.float32, device=device)
    reference = (keys, values) if layout == "bf16_kv" else (None, None)
    return PagedKVCache(
        key_pages=keys, value_pages=values, page_table=page_table, seq_lens=seq_lens, key_scales=key_scales,
        value_scales=value_scales, reference_key_pages=reference[0], reference_value_pages=reference[1],
        kv_layout=layout, page_size=page_size, num_kv_heads=num_kv_heads, head_dim=head_dim,
        keys_are_rotated=key_rope_theta is not None,
        key_rope_theta=None if key_rope_theta is None else float(key_rope_theta))


def plan_paged_kv_append(
    *,
    page_table: Any,
    seq_lens: Any,
    append_lens: Any,
    num_kv_heads: int,
    head_dim: int,
    page_size: int,
    kv_layout: str,
    use_cache: bool = True,
) -> PagedKVAppendPlan:
    """Where `append_lens[b]` new tokens of every request go, behind the `seq_lens[b]` that it has. The plan
    serves every layer whose cache has this page table."""
    layout = _paged.require_geometry(num_kv_heads=num_kv_heads, head_dim=head_dim, page_size=page_size, kv_layout=kv_layout)
    table, lens, new = _paged.table_and_lengths(page_table, seq_lens=seq_lens, append_lens=append_lens)
    made_from = (table, lens, new, num_kv_heads, head_dim, page_size, layout)
    return _paged.remembered(_PLANS, made_from, lambda: _build(table, lens, new, num_kv_heads, head_dim, page_size, layout),
                             use_cache)


def _build(table: np.ndarray, lens: np.ndarray, new: np.ndarray, num_kv_heads: int, head_dim: int, page_size: int,
           layout: KvLayout) -> PagedKVAppendPlan:
    torch = _torch()
    ends = lens + new
    if ends.size and int(ends.max()) >= 1 << 31 or int(new.sum()) >= 1 << 31:
        raise ValueError("seq_lens + append_lens must fit 32 bits")
    first = lens // page_size
    counts = np.where(new > 0, (ends - 1) // page_size - first + 1, 0)
    request = np.repeat(np.arange(len(lens)), counts)
    page = np.arange(int(counts.sum())) - np.repeat(np.cumsum(counts) - counts, counts) + first[request]
    physical = _paged.require_pages(table, request, page)
    if np.unique(physical).size != physical.size:
        raise ValueError("two requests would append to the same page; copy a shared page before writing to it")
    position = np.maximum(page * page_size, lens[request])
    count = np.minimum((page + 1) * page_size, ends[request]) - position
    token = (np.cumsum(new) - new)[request] + position - lens[request]
    segments = np.stack((physical, position - page * page_size | count << 16, token, position), axis=1).astype(np.int32)
    return PagedKVAppendPlan(
        batch=len(lens), page_size=page_size, num_kv_heads=num_kv_heads, head_dim=head_dim, kv_layout=layout,
        num_tokens=int(new.sum()), largest_page=int(physical.max()) if physical.size else -1,
        segments_cpu=torch.from_numpy(segments), seq_lens_after_cpu=torch.from_numpy(ends.astype(np.int32)))


def paged_kv_append(
    keys: Any,
    values: Any,
    cache: PagedKVCache,
    *,
    append_lens: Any | None = None,
    plan: PagedKVAppendPlan | None = None,
) -> PagedKVCache:
    """Writes `keys` and `values` (bf16, [tokens, kv_heads, head_dim], the requests' new tokens one request
    after the other; views into a fused projection's rows will do) into the cache's pages. Either
    `append_lens` or a `plan` says how many tokens each request gets. Returns the cache with the new
    `seq_lens`, as int32 on the CPU wherever the cache had them (plans are made there); its pages are the same tensors."""
    native = _paged.backend()
    found = plan is None
    if plan is None:
        if append_lens is None:
            raise ValueError("paged_kv_append needs append_lens or a plan")
        plan = plan_paged_kv_append(
            page_table=cache.page_table, seq_lens=cache.seq_lens, append_lens=append_lens,
            num_kv_heads=cache.num_kv_heads, head_dim=cache.head_dim, page_size=cache.page_size, kv_layout=cache.kv_layout)
    elif append_lens is not None:
        raise ValueError("give append_lens or a plan, not both")
    device = _paged.check_cache(cache, plan)
    shape = (plan.num_tokens, plan.num_kv_heads, plan.head_dim)
    _paged.check_rows(keys, name="keys", shape=shape, device=device)
    _paged.check_rows(values, name="values", shape=shape, device=device)
    if cache.keys_are_rotated and cache.key_rope_theta is None:
        raise ValueError("rotated key caches must record key_rope_theta")
    if plan.num_tokens:
        with _paged.current(device):
            stream = _paged.current_stream(device)
            if found:
                _paged.keep_for_graphs(plan)
            native.paged_kv_append_forward(
                keys.data_ptr(), values.data_ptr(), *_paged.row_strides(keys), *_paged.row_strides(values),
                cache.key_pages.data_ptr(), cache.value_pages.data_ptr(), _paged.address(cache.key_scales),
                _paged.address(cache.value_scales), plan.device_tables(device, stream)["segments"], plan.num_segments,
                plan.num_tokens, cache.key_pages.shape[0], plan.num_kv_heads, plan.head_dim, plan.page_size,
                _layout_id(plan.kv_layout), int(cache.keys_are_rotated),
                float(cache.key_rope_theta) if cache.keys_are_rotated else 1.0, stream)
    # (a copy: the plan may be used again, and the caller may write to the cache's lengths)
    lens = plan.seq_lens_after_cpu.clone()
    kept = cache.reference_key_pages, cache.reference_value_pages
    if plan.num_tokens and (kept[0] is not None and kept[0] is not cache.key_pages or kept[1] is not None and kept[1] is not cache.value_pages):
        return dataclasses.replace(cache, seq_lens=lens, reference_key_pages=None, reference_value_pages=None)
    return dataclasses.replace(cache, seq_lens=lens)
