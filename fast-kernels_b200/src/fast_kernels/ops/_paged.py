"""What the operators around the paged cache share: checks of shapes and caches, the descriptor tables
of a plan on its devices, and plans remembered by their contents."""

from __future__ import annotations

import threading
from collections import OrderedDict
from contextlib import nullcontext
from typing import Any, Callable

import numpy as np

from fast_kernels.ops.clustered_page_decode import (
    _SCALE_BLOCK,
    PagedKVCache,
    _require_cuda_backend,
    _require_layout,
    _torch,
)

_ROW_ALIGN = 16  # bytes
_UPLOAD_ALIGN = 128  # int32 words: 512 bytes
_backend: Any = None
_HERE = nullcontext()
_REMEMBERING = threading.Lock()
_IN_GRAPHS: dict[int, Any] = {}  # plans by identity


def require_geometry(*, num_kv_heads: int, head_dim: int, page_size: int, kv_layout: str, num_q_heads: int | None = None) -> str:
    layout = _require_layout(kv_layout)
    if num_kv_heads < 1:
        raise ValueError("num_kv_heads must be >= 1")
    if num_q_heads is not None and (num_q_heads < 1 or num_q_heads % num_kv_heads != 0):
        raise ValueError("num_q_heads must be divisible by num_kv_heads")
    if head_dim not in {64, 128}:
        raise ValueError("head_dim must be 64 or 128")
    if page_size not in {16, 32}:
        raise ValueError("page_size must be 16 or 32")
    return layout


def host_ints(tensor: Any, name: str, ndim: int) -> np.ndarray:
    torch = _torch()
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if tensor.ndim != ndim:
        raise ValueError(f"{name} must be {ndim}D")
    if tensor.is_floating_point() or tensor.is_complex():
        raise TypeError(f"{name} must hold integers")
    return tensor.detach().to(device="cpu", dtype=torch.int64).numpy()


def table_and_lengths(page_table: Any, **lengths: Any) -> list[np.ndarray]:
    """The page table (int32 as it mostly comes, or int64) and 1D length tensors as int64 arrays, one non-negative length
    per request."""
    torch = _torch()
    if isinstance(page_table, torch.Tensor) and page_table.dtype == torch.int32 and page_table.ndim == 2:
        table = page_table.detach().cpu().contiguous().numpy()
    else:
        table = host_ints(page_table, "page_table", 2)
    out = [table]
    for name, tensor in lengths.items():
        values = host_ints(tensor, name, 1)
        if values.shape[0] != table.shape[0]:
            raise ValueError(f"{name} must be a 1D tensor with one entry per request")
        if values.size and int(values.min()) < 0:
            raise ValueError(f"{name} must not be negative")
        if values.size and int(values.max()) >= 1 << 31:
            raise ValueError(f"{name} must fit 32 bits")
        out.append(values)
    return out


def require_countable(lens: np.ndarray) -> None:
    """The attention kernel counts a request's tokens in 32 bits, a tile at a time (FK_PAGED_KV_MAX_TOKENS)."""
    if lens.size and int(lens.max()) > (1 << 31) - 128:
        raise ValueError("seq_lens must be at most 2^31 - 128")


def require_pages(table: np.ndarray, request: np.ndarray, slot: np.ndarray) -> np.ndarray:
    """Physical pages of (request, logical page) pairs; every one must be in the table."""
    if slot.size and int(slot.max()) >= table.shape[1]:
        raise ValueError("page_table has fewer columns than the tokens need")
    pages = table[request, slot]
    if pages.size and int(pages.min()) < 0:
        raise ValueError("page_table has no page for some of the tokens")
    if pages.dtype != np.int32 and pages.size and int(pages.max()) >= 1 << 31:
        raise ValueError("page_table entries must fit 32 bits")
    return pages


def remembered(plans: OrderedDict, made_from: tuple, build: Callable[[], Any], use_cache: bool, most: int = 32) -> Any:
    """A plan by the contents that it was made from; the `most` last used ones are kept. (The lengths of a decode step never
    come back, so nearly all plans of a server are dead after their step, each with its page table and device tables.)"""
    if not use_cache:
        return build()
    key = tuple((v.shape, v.tobytes()) if isinstance(v, np.ndarray) else v for v in made_from)
    with _REMEMBERING:
        plan = plans.get(key)
        if plan is not None:
            plans.move_to_end(key)
            return plan
    plan = build()
    with _REMEMBERING:
        plan = plans.setdefault(key, plan)
        plans.move_to_end(key)
        while len(plans) > most:
            plans.popitem(last=False)
    return plan


def keep_for_graphs(plan: Any) -> None:
    """For a call that found its plan by itself: where it is being captured, the graph's replays read the plan's tables, and
    nobody but this module can keep them. (A plan that the caller gave is the caller's to keep.)"""
    if _torch().cuda.is_current_stream_capturing():
        _IN_GRAPHS[id(plan)] = plan


def backend() -> Any:
    """The native module; raises where it is missing or was built without CUDA."""
    global _backend
    if _backend is None:
        _backend = _require_cuda_backend()
    return _backend


def current_stream(device: Any) -> int:
    """Handle of the current stream of `device`."""
    return _torch()._C._cuda_getCurrentRawStream(device.index)


def on_device(kept: dict[int, Any], device: Any, stream: int, host: Callable[[], dict[str, np.ndarray]]) -> dict[str, int]:
    """Addresses of the descriptor tables as int32 arrays on `device`, for a launch on `stream`; uploaded once per device
    in one copy."""
    entry = kept.get(device.index)
    if entry is None:
        torch = _torch()
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a plan's first call on a device uploads its tables: make one before the capture")
        tables = host()
        parts, starts, at = [], {}, 0
        for name, values in tables.items():
            gap = -values.size % _UPLOAD_ALIGN
            parts += [np.ascontiguousarray(values, dtype=np.int32).reshape(-1), np.zeros(gap, dtype=np.int32)]
            starts[name] = at
            at += 4 * (values.size + gap)
        block = torch.from_numpy(np.concatenate(parts)).to(device=device)
        base = block.data_ptr()
        # (two host threads may both get here: the first entry stands, so that nobody is given addresses into a block
        # that the other one's entry has just dropped)
        entry = kept.setdefault(device.index, (block, {name: base + start for name, start in starts.items()}, stream))
    block, addresses, home = entry
    if stream != home:
        torch = _torch()
        if not torch.cuda.is_current_stream_capturing():
            block.record_stream(torch.cuda.current_stream(device))  # the plan may go away before that stream is done with it
    return addresses


def check_rows(tensor: Any, *, name: str, shape: tuple[int, ...], device: Any) -> None:
    """bf16 rows [tokens, heads, head_dim] on `device`: any token and head strides, each row 16-byte aligned."""
    torch = _torch()
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if tensor.ndim != 3:
        raise ValueError(f"{name} must be 3D")
    if tensor.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must have dtype {torch.bfloat16}")
    if tensor.device != device:
        if not tensor.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        raise ValueError(f"all CUDA tensors must be on the same device: {name}={tensor.device}, key_pages={device}")
    if tensor.shape != shape:
        raise ValueError(f"{name} must be shaped {list(shape)}, got {list(tensor.shape)}")
    if 0 in shape:
        return
    rows, heads, elements = tensor.stride()
    if elements != 1 or tensor.data_ptr() % _ROW_ALIGN or (rows % 8 and shape[0] > 1) or (heads % 8 and shape[1] > 1):
        raise ValueError(f"{name} must have contiguous rows that start on 16-byte boundaries")


def check_output(tensor: Any, *, shape: tuple[int, ...], device: Any, name: str = "output") -> None:
    check_rows(tensor, name=name, shape=shape, device=device)
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def check_turned_keys(cache: PagedKVCache, rope_theta: float) -> None:
    if not cache.keys_are_rotated:
        raise ValueError("the cache's keys must be rotated ahead of time")
    if cache.key_rope_theta is None:
        raise ValueError("rotated key caches must record key_rope_theta")
    if float(cache.key_rope_theta) != float(rope_theta):
        raise ValueError("rope_theta must match the key_rope_theta used to build the cache")


def row_strides(tensor: Any) -> tuple[int, int]:
    """Token and head strides in elements; the stride of a dimension of one entry is never walked."""
    rows, heads, _ = tensor.stride()
    return rows if tensor.shape[0] > 1 else 0, heads if tensor.shape[1] > 1 else 0


def check_cache(cache: PagedKVCache, plan: Any) -> Any:
    """The cache's tensors against its own description and the plan's; returns its device."""
    torch = _torch()
    if (cache.num_kv_heads, cache.head_dim, cache.page_size, cache.kv_layout) != (
            plan.num_kv_heads, plan.head_dim, plan.page_size, plan.kv_layout):
        for name in ("num_kv_heads", "head_dim", "page_size", "kv_layout"):
            if getattr(cache, name) != getattr(plan, name):
                raise ValueError(f"the plan was made for {name}={getattr(plan, name)}, the cache has {getattr(cache, name)}")
    device = cache.key_pages.device
    pages = cache.key_pages.shape[0]
    shape = (pages, cache.num_kv_heads, cache.page_size, cache.head_dim)
    if cache.kv_layout == "bf16_kv":
        _check_pages("key_pages", cache.key_pages, torch.bfloat16, shape, device)
        _check_pages("value_pages", cache.value_pages, torch.bfloat16, shape, device)
    else:
        element = torch.uint8 if cache.kv_layout == "fp8_kv" else torch.int8
        blocks = cache.head_dim // _SCALE_BLOCK
        _check_pages("key_pages", cache.key_pages, element, shape, device)
        _check_pages("value_pages", cache.value_pages, element, shape, device)
        _check_pages("key_scales", cache.key_scales, torch.float32, (pages, shape[1], blocks), device)
        _check_pages("value_scales", cache.value_scales, torch.float32, (*shape[:3], blocks), device)
    if plan.largest_page >= pages:
        raise ValueError(f"the plan names page {plan.largest_page}, the cache has {pages}")
    return device


def _check_pages(name: str, tensor: Any, dtype: Any, shape: tuple[int, ...], device: Any) -> None:
    if not isinstance(tensor, _torch().Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if tensor.dtype is not dtype:
        raise TypeError(f"{name} must have dtype {dtype}")
    if tensor.shape != shape:
        raise ValueError(f"{name} must be shaped {list(shape)}, got {list(tensor.shape)}")
    if not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if tensor.device != device:
        raise ValueError(f"all CUDA tensors must be on the same device: {name}={tensor.device}, key_pages={device}")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def current(device: Any) -> Any:
    """Makes `device` the current one for a launch, where it is not already."""
    torch = _torch()
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def address(tensor: Any | None) -> int:
    return 0 if tensor is None else tensor.data_ptr()
