"""Plain 64-bit statements of the operators around the paged cache, and caches to try them on."""

from __future__ import annotations

import importlib
import math
from typing import Any

import numpy as np
import torch

ops = importlib.import_module("fast_kernels.ops")
LIMITS = {"fp8_kv": 448.0, "int8_kv": 127.0}
BLOCK = 64


def rotate64(x: torch.Tensor, positions: Any, theta: float) -> torch.Tensor:
    """x [tokens, heads, dim]: dimensions 2i, 2i + 1 turned by position * theta^(-2i/dim)."""
    x = x.double()
    dim = x.shape[-1]
    frequency = torch.tensor([theta ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64)
    angle = torch.as_tensor(positions, dtype=torch.float64)[:, None, None] * frequency
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack((even * angle.cos() - odd * angle.sin(), even * angle.sin() + odd * angle.cos()), dim=-1).flatten(-2)


def page_numbers(pages: torch.Tensor, layout: str) -> torch.Tensor:
    """What the elements of pages are as numbers, without their scales."""
    pages = pages.cpu()
    return (pages.view(torch.float8_e4m3fn).float() if layout == "fp8_kv" else pages).double()


def cache_values(cache: Any) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values that the pages stand for, fp64 [pages, heads, slots, dim]."""
    keys, values = (page_numbers(p, cache.kv_layout) for p in (cache.key_pages, cache.value_pages))
    if cache.kv_layout != "bf16_kv":
        keys = keys * cache.key_scales.cpu().double().repeat_interleave(BLOCK, dim=-1)[:, :, None]
        values = values * cache.value_scales.cpu().double().repeat_interleave(BLOCK, dim=-1)
    return keys, values


def random_cache(*, layout: str, pages: int, heads: int, page_size: int, dim: int, table: Any, lens: Any, theta: float | None,
                 seed: int, device: str = "cuda") -> Any:
    """Pages full of random numbers, whatever the table says of them."""
    gen = torch.Generator().manual_seed(seed)
    shape = (pages, heads, page_size, dim)
    keys, values = (torch.randn(shape, generator=gen) for _ in range(2))
    scales: list[Any] = [None, None]
    if layout == "bf16_kv":
        keys, values = keys.to(torch.bfloat16), values.to(torch.bfloat16)
    else:
        limit = LIMITS[layout]
        scales = [3.5 / limit * (0.6 + 0.8 * torch.rand((pages, heads, dim // BLOCK), generator=gen)),
                  3.5 / limit * (0.6 + 0.8 * torch.rand((pages, heads, page_size, dim // BLOCK), generator=gen))]
        keys, values = ((x * limit / 4).clamp(-limit, limit) for x in (keys, values))
        keys, values = ((x.to(torch.float8_e4m3fn).view(torch.uint8) if layout == "fp8_kv" else x.round().to(torch.int8))
                        for x in (keys, values))
    move = lambda t: None if t is None else t.to(device)  # noqa: E731
    return ops.PagedKVCache(
        key_pages=move(keys), value_pages=move(values), page_table=torch.as_tensor(np.asarray(table), dtype=torch.int32),
        seq_lens=torch.as_tensor(np.asarray(lens), dtype=torch.int32), key_scales=move(scales[0]), value_scales=move(scales[1]),
        reference_key_pages=None, reference_value_pages=None, kv_layout=layout, page_size=page_size, num_kv_heads=heads,
        head_dim=dim, keys_are_rotated=theta is not None, key_rope_theta=theta)


def fragmented_table(counts: list[int], seed: int, spare: int = 3) -> tuple[np.ndarray, int]:
    """(table with -1 padding, pages of the pool): every request's pages anywhere in the pool."""
    rng = np.random.RandomState(seed)
    total = sum(counts)
    ids = rng.permutation(total + spare)[:total]
    table = np.full((len(counts), max([1, *counts])), -1, dtype=np.int32)
    at = 0
    for row, count in enumerate(counts):
        table[row, :count] = ids[at : at + count]
        at += count
    return table, total + spare


def append64(cache: Any, keys: torch.Tensor, values: torch.Tensor, new: list[int]) -> dict[str, Any]:
    """What an append leaves, token by token from the definition: fp64 keys and values of the tokens written (before
    their own rounding to the page's format), the held tokens' new numbers, scales, and which slots are touched."""
    layout, ps, theta = cache.kv_layout, cache.page_size, cache.key_rope_theta
    lens = cache.seq_lens.tolist()
    position = [lens[b] + i for b, n in enumerate(new) for i in range(n)]
    where = [(int(cache.page_table[b, (lens[b] + i) // ps]), (lens[b] + i) % ps) for b, n in enumerate(new) for i in range(n)]
    k = rotate64(keys.cpu(), position, theta) if theta is not None else keys.cpu().double()
    v = values.cpu().double()
    heads, dim = k.shape[1:]
    numbers_k, numbers_v = (page_numbers(p, layout) for p in (cache.key_pages, cache.value_pages))
    written = torch.zeros(numbers_k.shape[0], numbers_k.shape[2], dtype=torch.bool)
    result: dict[str, Any] = {"written": written}
    if layout == "bf16_kv":
        for t, (page, slot) in enumerate(where):
            numbers_k[page, :, slot], numbers_v[page, :, slot] = k[t], v[t]
            written[page, slot] = True
        return result | {"keys": numbers_k, "values": numbers_v}
    limit = LIMITS[layout]
    blocks = lambda x: x.reshape(*x.shape[:-1], dim // BLOCK, BLOCK)  # noqa: E731
    spread = lambda s: s.repeat_interleave(BLOCK, dim=-1)  # noqa: E731
    key_scales, value_scales = cache.key_scales.cpu().double(), cache.value_scales.cpu().double()
    requantised = torch.zeros(numbers_k.shape[:3], dtype=torch.bool)[..., None].repeat(1, 1, 1, dim)
    by_page: dict[int, list[int]] = {}
    for t, (page, _) in enumerate(where):
        by_page.setdefault(page, []).append(t)
    for page, tokens in by_page.items():
        start = min(where[t][1] for t in tokens)
        fresh = (blocks(k[tokens]).abs().amax(dim=(0, 3)) / limit).clamp(min=1e-6)
        held = torch.zeros_like(fresh) if start == 0 else key_scales[page]
        scale = torch.maximum(held, fresh)
        grown = spread(scale > held)[:, None].expand(heads, start, dim)
        numbers_k[page, :, :start] = torch.where(grown, numbers_k[page, :, :start] * spread(held / scale)[:, None],
                                                 numbers_k[page, :, :start])
        requantised[page, :, :start] = grown
        key_scales[page] = scale
        for t in tokens:
            slot = where[t][1]
            numbers_k[page, :, slot] = k[t] / spread(scale)
            value_scales[page, :, slot] = (blocks(v[t]).abs().amax(dim=-1) / limit).clamp(min=1e-6)
            numbers_v[page, :, slot] = v[t] / spread(value_scales[page, :, slot])
            written[page, slot] = True
    return result | {"keys": numbers_k, "values": numbers_v, "key_scales": key_scales, "value_scales": value_scales,
                     "requantised": requantised}


def assert_append(before: Any, after: Any, want: dict[str, Any], slack: float) -> None:
    """Every slot of every page, scales too, of `after` against `want`; what was not touched against `before`, bit for bit.

    `slack` is what the fp32 turn may be off, relative to the pair's length, which the page's largest element bounds."""
    layout = after.kv_layout
    written = want["written"][:, None, :, None]
    for name, pages in (("keys", after.key_pages), ("values", after.value_pages)):
        got = page_numbers(pages, layout)
        old = page_numbers(getattr(before, "key_pages" if name == "keys" else "value_pages"), layout)
        touched = written.expand_as(got)
        if layout != "bf16_kv" and name == "keys":
            touched = touched | want["requantised"]
        assert torch.equal(got[~touched], old[~touched]), f"{name} outside of the segments"
        exact = want[name]
        if layout == "bf16_kv":  # one rounding, half a step
            bound = exact.abs() * 2.0**-8 + slack * 8.0
        elif layout == "int8_kv":  # half a step of 1, and the turn's and the scale's own error in steps
            bound = 0.5 + 127.0 * 2.0 * slack
        else:  # half a step of e4m3: 2^-4 of the number, or half its smallest subnormal 2^-9
            bound = torch.clamp(exact.abs() * 2.0**-4, min=2.0**-10) + 448.0 * 2.0 * slack
        off = (got - exact).abs()
        bad = touched & (off > bound)
        assert not bool(bad.any()), f"{name}: {int(bad.sum())} elements off, worst {float((off - bound)[touched].max()):.3e}"
    if layout != "bf16_kv":
        for name in ("key_scales", "value_scales"):
            torch.testing.assert_close(getattr(after, name).cpu().double(), want[name], rtol=2.0 * slack + 2.0**-22, atol=0)


def attention64(cache: Any, query: torch.Tensor, rows: list[tuple[int, int]], scale: float, theta: float) -> torch.Tensor:
    """Row i = query[i] [q_heads, dim] of request rows[i][0] at position rows[i][1]: softmax over the request's tokens
    0 .. position in fp64; a position below 0 gives zeros."""
    keys, values = cache_values(cache)
    ps, heads = cache.page_size, cache.num_kv_heads
    q = rotate64(query.cpu(), [max(0, p) for _, p in rows], theta)
    out = torch.zeros_like(q)
    group = q.shape[1] // heads
    gathered: dict[int, tuple[torch.Tensor, torch.Tensor]] = {}
    for i, (request, position) in enumerate(rows):
        if position < 0:
            continue
        if request not in gathered:
            most = max(p for r, p in rows if r == request) + 1
            pages = cache.page_table[request, : -(-most // ps)].long()
            gathered[request] = tuple(x[pages].permute(1, 0, 2, 3).reshape(heads, -1, x.shape[-1]) for x in (keys, values))
        k, v = (x[:, : position + 1] for x in gathered[request])
        logits = torch.einsum("hgd,htd->hgt", q[i].reshape(heads, group, -1), k) * scale
        out[i] = torch.einsum("hgt,htd->hgd", torch.softmax(logits, dim=-1), v).reshape(q.shape[1:])
    return out


def attention_terms64(cache: Any, query: torch.Tensor, rows: list[tuple[int, int]], scale: float, theta: float) -> dict[str, torch.Tensor]:
    """`attention64`, and what its rounding errors are bounded by, per row and query head (and dimension):
    a = sum_t p_t |v_t|; logit = max_t |scale| sum_i |q_i k_i|; query = sum_i |q_i|; with s_t the larger of a token's value
    scales (8-bit pages): weight = max_t p_t s_t, weights = sum_t p_t s_t, numbers = sum_t |v_t| / s_t; and the largest key
    scale of the tokens."""
    keys, values = cache_values(cache)
    ps, heads = cache.page_size, cache.num_kv_heads
    q = rotate64(query.cpu(), [max(0, p) for _, p in rows], theta)
    group, dim = q.shape[1] // heads, q.shape[2]
    quantised = cache.kv_layout != "bf16_kv"
    terms = {name: torch.zeros_like(q) for name in ("out", "a", "numbers")}
    terms |= {name: torch.zeros((*q.shape[:2], 1), dtype=torch.float64) for name in ("logit", "query", "weight", "weights", "key_scale")}
    gathered: dict[int, list[torch.Tensor]] = {}
    for i, (request, position) in enumerate(rows):
        if position < 0:
            continue
        if request not in gathered:
            most = max(p for r, p in rows if r == request) + 1
            pages = cache.page_table[request, : -(-most // ps)].long()
            flat = lambda x: x[pages].permute(1, 0, 2, 3).reshape(heads, -1, x.shape[-1])  # noqa: E731
            gathered[request] = [flat(keys), flat(values)]
            if quantised:
                gathered[request].append(flat(cache.value_scales.cpu().double()).amax(dim=-1, keepdim=True))
                page_scales = cache.key_scales.cpu().double().amax(dim=-1)[:, :, None, None].expand(-1, -1, ps, -1)
                gathered[request].append(flat(page_scales))
        k, v, *scales = (x[:, : position + 1] for x in gathered[request])
        mine = q[i].reshape(heads, group, dim)
        p = torch.softmax(torch.einsum("hgd,htd->hgt", mine, k) * scale, dim=-1)

        def put(name: str, x: torch.Tensor) -> None:
            terms[name][i] = x.reshape(heads * group, -1)

        put("out", torch.einsum("hgt,htd->hgd", p, v))
        put("a", torch.einsum("hgt,htd->hgd", p, v.abs()))
        put("logit", abs(scale) * torch.einsum("hgd,htd->hgt", mine.abs(), k.abs()).amax(dim=-1))
        put("query", mine.abs().sum(dim=-1))
        if quantised:
            put("weight", (p * scales[0].transpose(1, 2)).amax(dim=-1))
            put("weights", (p * scales[0].transpose(1, 2)).sum(dim=-1))
            put("numbers", (v.abs() / scales[0]).sum(dim=1)[:, None].expand(-1, group, -1))
            put("key_scale", scales[1].amax(dim=(1, 2))[:, None].expand(-1, group))
    return terms


def default_scale(dim: int) -> float:
    return 1.0 / math.sqrt(dim)
