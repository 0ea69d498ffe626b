"""The paged KV cache's operators around the decode attention, with sizes of real use.

``kind`` names the operator of a case:

  append   ``ops.paged_kv_append``: new keys and values of a batch go into their pages, the keys turned by
           their positions on the way, in the cache's own format
  prompt   ``ops.paged_prompt_attention``: the new tokens of prompts (or pieces of prompts) attend, each up
           to its own position, over the pages
  shared   ``ops.shared_prefix_decode``: one decode token per request where groups of requests share the
           pages of a long beginning (a system prompt, a document, samples of one prompt)

``own`` says whether ``run`` calls the package or computes the plain form.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

ROPE_THETA = 10000.0
LAYOUTS = ("bf16_kv", "fp8_kv", "int8_kv")
LIMITS = {"fp8_kv": 448.0, "int8_kv": 127.0}
SCALE_BLOCK = 64

# Bounds of the ranges. Multiply-adds of an attention pass: one prompt of 8192 tokens, 32 heads of 128.
MAX_APPEND_TOKENS = 32768
MAX_ATTENTION_MACS = 8192 * 8192 * 32 * 128
MAX_PAIRS = 8192 * 8192 * 32  # (query head, key) pairs with every request as long as the longest
MAX_DENSE = 128 * 16896 * 8 * 128  # elements of one request-by-request copy of the keys


def listed() -> list[dict]:
    return [
        # One request, one token: what a single user's decode step adds per layer. Latency is all there is.
        dict(name="append_one_token", kind="append", layout="bf16_kv", page=16, kv_heads=8, head_dim=128,
             requests=1, shortest=1, longest=1, cached=1000, rotated=True),
        # A serving batch's step into int8 pages: most pages are partly full and their key scale may grow.
        dict(name="append_step_int8", kind="append", layout="int8_kv", page=32, kv_heads=8, head_dim=128,
             requests=96, shortest=1, longest=1, cached=2048, rotated=True),
        # Prompts of uneven lengths into fp8 pages, some behind what an earlier piece left.
        dict(name="append_prompts_fp8", kind="append", layout="fp8_kv", page=16, kv_heads=8, head_dim=128,
             requests=12, shortest=37, longest=2048, cached=77, rotated=True),
        # The most tokens of one prefill step, bf16 pages: bound by memory traffic.
        dict(name="append_prompts_bf16", kind="append", layout="bf16_kv", page=16, kv_heads=8, head_dim=128,
             requests=8, shortest=4096, longest=4096, cached=0, rotated=True),
        # A few tokens checked at once against a short cache, small heads.
        dict(name="prompt_few_tokens_h64", kind="prompt", layout="bf16_kv", page=32, q_heads=16, kv_heads=8,
             head_dim=64, requests=8, shortest=5, longest=5, cached=500),
        # Prompts of uneven lengths in one batch, int8 pages, some behind what is cached already.
        dict(name="prompt_ragged_int8", kind="prompt", layout="int8_kv", page=16, q_heads=32, kv_heads=8,
             head_dim=128, requests=6, shortest=131, longest=1500, cached=333),
        # A piece of a prompt behind a long cached context in fp8 pages.
        dict(name="prompt_piece_fp8_32k", kind="prompt", layout="fp8_kv", page=32, q_heads=32, kv_heads=4,
             head_dim=128, requests=1, shortest=512, longest=512, cached=32768),
        # One whole prompt, the most arithmetic of a pass.
        dict(name="prompt_8k_bf16", kind="prompt", layout="bf16_kv", page=16, q_heads=32, kv_heads=8,
             head_dim=128, requests=1, shortest=8192, longest=8192, cached=0),
        # The shape of the package's own suite for shared beginnings, small heads.
        dict(name="shared_small_h64", kind="shared", layout="bf16_kv", page=32, q_heads=16, kv_heads=8, head_dim=64,
             requests=8, groups=2, prefix=512, sub_sharers=1, sub_prefix=0, shortest=1, longest=200),
        # A serving batch behind one system prompt, int8 pages, an odd group of heads.
        dict(name="shared_int8_48x4k", kind="shared", layout="int8_kv", page=16, q_heads=24, kv_heads=8, head_dim=128,
             requests=48, groups=1, prefix=4096, sub_sharers=1, sub_prefix=0, shortest=17, longest=300),
        # Two levels: one system prompt for all, a document for every eight, and a tail each.
        dict(name="shared_tree_fp8", kind="shared", layout="fp8_kv", page=16, q_heads=32, kv_heads=8, head_dim=128,
             requests=64, groups=1, prefix=2048, sub_sharers=8, sub_prefix=2048, shortest=33, longest=256),
        # The largest batch and prefix.
        dict(name="shared_bf16_128x16k", kind="shared", layout="bf16_kv", page=16, q_heads=32, kv_heads=8, head_dim=128,
             requests=128, groups=1, prefix=16384, sub_sharers=1, sub_prefix=0, shortest=64, longest=512),
    ]


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng) -> dict:
    kind = rng.choice(("append", "prompt", "shared"))
    while True:
        case = dict(kind=kind, layout=rng.choice(LAYOUTS), page=rng.choice((16, 32)), kv_heads=rng.choice((1, 2, 4, 8)),
                    head_dim=rng.choice((64, 128)))
        if kind == "append":
            longest = _log(rng, 1, 4096)
            case.update(requests=_log(rng, 1, 128), shortest=_log(rng, 1, longest), longest=longest,
                        cached=rng.choice((0, _log(rng, 1, 4096))), rotated=rng.random() < 0.8)
            if sum(_lengths(case)) <= MAX_APPEND_TOKENS:
                return case
            continue
        case["q_heads"] = case["kv_heads"] * rng.choice((1, 2, 3, 4, 8))
        if kind == "prompt":
            longest = _log(rng, 1, 6000)
            case.update(requests=_log(rng, 1, 16), shortest=_log(rng, 1, longest), longest=longest,
                        cached=rng.choice((0, _log(rng, 1, 16384))))
            pairs = case["requests"] * longest * (longest + case["cached"]) * case["q_heads"]
            if pairs <= MAX_PAIRS and _pairs(case) * case["head_dim"] * 2 <= MAX_ATTENTION_MACS:
                return case
            continue
        longest = _log(rng, 1, 512)
        sub = rng.choice((1, 1, 2, 4))
        case.update(requests=_log(rng, 2, 128), groups=rng.choice((1, 1, 2)), prefix=_log(rng, 32, 16384),
                    sub_sharers=sub, sub_prefix=0 if sub == 1 else _log(rng, 32, 2048),
                    shortest=rng.randint(0, longest), longest=longest)
        whole = case["requests"] * (case["prefix"] + case["sub_prefix"] + longest)
        if whole * case["kv_heads"] * case["head_dim"] <= MAX_DENSE:
            return case


# ---- sizes that follow from a case -----------------------------------------------------------------


def _lengths(case: dict) -> list[int]:
    """New tokens (append, prompt) or tokens of a request's own (shared): steps from the longest to the shortest."""
    count, low, high = case["requests"], case["shortest"], case["longest"]
    return [high - (high - low) * i // max(1, count - 1) for i in range(count)]


def _cached(case: dict) -> list[int]:
    """Tokens that are in the pages before the call: uneven, and none for every third request of several."""
    base = case["cached"]
    return [0 if case["requests"] > 2 and i % 3 == 2 else base + (7 * i) % max(1, base // 4) if base else 0
            for i in range(case["requests"])]


def _pairs(case: dict) -> int:
    """(query head, key) pairs that a prompt case's tokens see."""
    return case["q_heads"] * sum(n * c + n * (n + 1) // 2 for n, c in zip(_lengths(case), _cached(case)))


def _prefix_pages(case: dict) -> tuple[int, int]:
    return case["prefix"] // case["page"], case["sub_prefix"] // case["page"]


def _shared_lens(case: dict) -> np.ndarray:
    shared, sub = _prefix_pages(case)
    return (shared + sub) * case["page"] + np.array(_lengths(case), dtype=np.int64)


def _family(case: dict) -> tuple[np.ndarray, np.ndarray]:
    """Of every request, the prefix it begins with and the second-level prefix behind that. Sharers are not neighbours."""
    request = np.arange(case["requests"])
    group = request % case["groups"]
    return group, group + case["groups"] * (request // case["groups"] // case["sub_sharers"])


# ---- inputs ----------------------------------------------------------------------------------------


def _pool(case: dict, gen, pages: int) -> dict:
    """`pages` pages as earlier steps left them, in the cache's format."""
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    blocks = case["head_dim"] // SCALE_BLOCK
    keys, values = (torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    if case["layout"] == "bf16_kv":
        return dict(key_pages=keys, value_pages=values, key_scales=None, value_scales=None)
    limit = LIMITS[case["layout"]]
    key_scales = 3.5 / limit * (0.8 + 0.4 * torch.rand((*shape[:2], blocks), generator=gen, device="cuda"))
    value_scales = 2.8 / limit * (0.8 + 0.4 * torch.rand((*shape[:3], blocks), generator=gen, device="cuda"))

    def packed(x, scale):
        x = (x.float().reshape(*shape[:3], blocks, SCALE_BLOCK) / scale).clamp(-limit, limit).reshape(shape)
        return x.to(torch.float8_e4m3fn).view(torch.uint8) if case["layout"] == "fp8_kv" else x.round().to(torch.int8)

    return dict(key_pages=packed(keys, key_scales[:, :, None, :, None]), value_pages=packed(values, value_scales[..., None]),
                key_scales=key_scales, value_scales=value_scales)


def _fused_rows(gen, tokens: int, heads: int, head_dim: int, skip: int):
    """`heads` heads a token out of the rows of a fused projection, `skip` heads in front of them."""
    rows = torch.randn((tokens, skip + heads, head_dim), generator=gen, device="cuda", dtype=torch.bfloat16)
    return rows[:, skip:]


def _cache(case: dict, pool: dict, table, lens, rotated: bool):
    from fast_kernels import ops

    return ops.PagedKVCache(page_table=torch.from_numpy(table), seq_lens=torch.from_numpy(lens.astype(np.int32)),
                            reference_key_pages=None, reference_value_pages=None, kv_layout=case["layout"],
                            page_size=case["page"], num_kv_heads=case["kv_heads"], head_dim=case["head_dim"],
                            keys_are_rotated=rotated, key_rope_theta=ROPE_THETA if rotated else None, **pool)


def _shape_arguments(case: dict) -> dict:
    return dict(num_kv_heads=case["kv_heads"], head_dim=case["head_dim"], page_size=case["page"], kv_layout=case["layout"])


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = np.random.RandomState(seed % (1 << 31))
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "fast-kernels_b200", "src"))
        from fast_kernels import ops
    page = case["page"]
    if case["kind"] == "shared":
        return _prepare_shared(case, gen, order)
    new, cached = np.array(_lengths(case), dtype=np.int64), np.array(_cached(case), dtype=np.int64)
    shuffle = order.permutation(case["requests"])
    new, cached = new[shuffle], cached[shuffle]
    lens = cached + new
    pages = -(-lens // page)
    first = cached // page if case["kind"] == "append" else np.zeros_like(cached)  # an append needs no page before these
    held = int((pages - first).sum())
    ids = order.permutation(held + 1)  # one page stands for all that the call does not touch
    table = np.full((case["requests"], int(pages.max())), -1, dtype=np.int32)
    column = np.arange(table.shape[1])
    table[column < pages[:, None]] = ids[held]
    table[(column >= first[:, None]) & (column < pages[:, None])] = ids[:held]
    state = dict(case=case, pool=_pool(case, gen, held + 1))
    # where each new token goes: (page, slot), and its position
    request = np.repeat(np.arange(case["requests"]), new)
    position = np.arange(int(new.sum())) - np.repeat(np.cumsum(new) - new, new) + np.repeat(cached, new)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int64)).cuda()  # noqa: E731
    state.update(position=to(position), request=to(request))
    if case["kind"] == "append":
        state.update(token_page=to(table[request, position // page]), token_slot=to(position % page),
                     keys=_fused_rows(gen, len(position), case["kv_heads"], case["head_dim"], 4),
                     values=_fused_rows(gen, len(position), case["kv_heads"], case["head_dim"], 4))
        if own:
            state["cache"] = _cache(case, state["pool"], table, cached, case["rotated"])
            state["plan"] = ops.plan_paged_kv_append(page_table=state["cache"].page_table, seq_lens=state["cache"].seq_lens,
                                                     append_lens=torch.from_numpy(new.astype(np.int32)),
                                                     use_cache=False, **_shape_arguments(case))
        return state
    start = np.cumsum(new) - new
    rows = np.arange(int(new.max()))
    state.update(table=to(table), lens=to(lens), new=to(new), padded_token=to(np.minimum(start[:, None] + rows, len(position) - 1)),
                 token_row=to(np.arange(len(position)) - np.repeat(start, new)),
                 query=_fused_rows(gen, len(position), case["q_heads"], case["head_dim"], 0))
    if own:
        state["cache"] = _cache(case, state["pool"], table, lens, True)
        state["plan"] = ops.plan_paged_prompt_attention(page_table=state["cache"].page_table, seq_lens=state["cache"].seq_lens,
                                                        query_lens=torch.from_numpy(new.astype(np.int32)),
                                                        num_q_heads=case["q_heads"], use_cache=False, **_shape_arguments(case))
    return state


def _prepare_shared(case: dict, gen, order) -> dict:
    page, requests = case["page"], case["requests"]
    shared, sub = _prefix_pages(case)
    lens = _shared_lens(case)
    pages = -(-lens // page)
    group, second = _family(case)
    table = np.full((requests, max(1, int(pages.max()))), -1, dtype=np.int32)
    tails = pages - shared - sub
    held = int(case["groups"] * shared + (int(second.max()) + 1) * sub + tails.sum())
    ids = order.permutation(max(1, held)).astype(np.int32)
    table[:, :shared] = ids[: case["groups"] * shared].reshape(case["groups"], shared)[group]
    used = case["groups"] * shared
    table[:, shared : shared + sub] = ids[used : used + (int(second.max()) + 1) * sub].reshape(-1, sub)[second] if sub else 0
    used += (int(second.max()) + 1) * sub
    column = np.arange(table.shape[1])
    table[(column >= shared + sub) & (column < pages[:, None])] = ids[used:held]
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int64)).cuda()  # noqa: E731
    state = dict(case=case, pool=_pool(case, gen, max(1, held)), table=to(table), lens=to(lens), position=to(lens - 1),
                 query=torch.randn((requests, case["q_heads"], case["head_dim"]), generator=gen, device="cuda",
                                   dtype=torch.bfloat16))
    if own:
        from fast_kernels import ops

        state["cache"] = _cache(case, state["pool"], table, lens, True)
        state["plan"] = ops.plan_shared_prefix_decode(page_table=state["cache"].page_table, seq_lens=state["cache"].seq_lens,
                                                      num_q_heads=case["q_heads"], use_cache=False, **_shape_arguments(case))
    return state


# ---- one pass --------------------------------------------------------------------------------------


def run(state: dict):
    case = state["case"]
    if case["kind"] == "append":
        if own:
            from fast_kernels import ops

            ops.paged_kv_append(state["keys"], state["values"], state["cache"], plan=state["plan"])
        else:
            _plain_append(state)
        return _pages_as_values(case, state["pool"])
    if case["kind"] == "prompt":
        if own:
            from fast_kernels import ops

            return ops.paged_prompt_attention(state["query"], state["cache"], plan=state["plan"], rope_theta=ROPE_THETA)
        return _plain_prompt(state)
    if own:
        from fast_kernels import ops

        return ops.shared_prefix_decode(state["query"], state["cache"], plan=state["plan"], rope_theta=ROPE_THETA)
    return _plain_shared(state)


def _pages_as_values(case: dict, pool: dict):
    """The pages after an append: bf16 as they are, e4m3 as numbers beside their scales, int8 as the values they stand for."""
    if case["layout"] == "bf16_kv":
        return pool["key_pages"], pool["value_pages"]
    scales = pool["key_scales"], pool["value_scales"]
    if case["layout"] == "fp8_kv":
        return pool["key_pages"].view(torch.float8_e4m3fn), pool["value_pages"].view(torch.float8_e4m3fn), *scales
    shape = pool["key_pages"].shape
    blocks = (*shape[:3], shape[3] // SCALE_BLOCK, SCALE_BLOCK)
    return ((pool["key_pages"].view(blocks) * scales[0][:, :, None, :, None]).to(torch.bfloat16).view(shape),
            (pool["value_pages"].view(blocks) * scales[1][..., None]).to(torch.bfloat16).view(shape), *scales)


def _rotated(x, position):
    """Dimensions 2i and 2i + 1 turned by position * theta^(-2i/d): angles in 64 bits, the turn in 32."""
    dim = x.shape[-1]
    frequency = ROPE_THETA ** (-torch.arange(0, dim, 2, device=x.device, dtype=torch.float64) / dim)
    angle = position.double()[:, None, None] * frequency
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    even, odd = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack((even * cos - odd * sin, even * sin + odd * cos), dim=-1).flatten(-2)


def _plain_append(state: dict) -> None:
    case, pool = state["case"], state["pool"]
    page, slot = state["token_page"], state["token_slot"]
    keys = _rotated(state["keys"], state["position"]) if case["rotated"] else state["keys"].float()
    values = state["values"]
    key_pages, value_pages = pool["key_pages"].transpose(1, 2), pool["value_pages"].transpose(1, 2)  # [page, slot, head, dim]
    if case["layout"] == "bf16_kv":
        key_pages[page, slot] = keys.to(torch.bfloat16)
        value_pages[page, slot] = values
        return
    limit, heads, dim = LIMITS[case["layout"]], case["kv_heads"], case["head_dim"]
    blocks = (-1, heads, dim // SCALE_BLOCK, SCALE_BLOCK)

    def packed(x):
        x = x.clamp(-limit, limit).reshape(-1, heads, dim)
        return x.to(torch.float8_e4m3fn).view(torch.uint8) if case["layout"] == "fp8_kv" else x.round().to(torch.int8)

    # values: a scale per token and block
    values = values.float().reshape(blocks)
    scale = (values.abs().amax(dim=-1) / limit).clamp(min=1e-6)
    value_pages[page, slot] = packed(values / scale[..., None])
    pool["value_scales"].transpose(1, 2)[page, slot] = scale
    # keys: a scale per page and block, which never shrinks while the page fills up
    keys = keys.reshape(blocks)
    scales = pool["key_scales"]
    largest = torch.zeros_like(scales).index_reduce_(0, page, keys.abs().amax(dim=-1), "amax")
    start = torch.full((len(scales),), case["page"], device=page.device).index_reduce_(0, page, slot, "amin")
    before = torch.where((start == 0)[:, None, None], 0.0, scales)
    fresh = torch.where((start < case["page"])[:, None, None], torch.maximum(before, (largest / limit).clamp(min=1e-6)), scales)
    # what a page holds already is brought to a scale that has grown
    old = pool["key_pages"].view(torch.float8_e4m3fn) if case["layout"] == "fp8_kv" else pool["key_pages"]
    here, at = torch.nonzero((torch.arange(case["page"], device=page.device) < start[:, None]) & (start < case["page"])[:, None],
                             as_tuple=True)
    kept = old.transpose(1, 2)[here, at].float().reshape(blocks)
    again = packed(kept * before[here][..., None] / fresh[here][..., None])
    grown = (fresh > before)[here].repeat_interleave(SCALE_BLOCK, dim=-1)
    key_pages[here, at] = torch.where(grown, again, key_pages[here, at])
    key_pages[page, slot] = packed(keys / fresh[page][..., None])
    scales.copy_(fresh)


def _dense(case: dict, pool: dict, table):
    """[requests, kv_heads, tokens, head_dim] keys and values in 32 bits, request by request."""
    dense = []
    for pages, scales in ((pool["key_pages"], pool["key_scales"]), (pool["value_pages"], pool["value_scales"])):
        if case["layout"] == "fp8_kv":
            pages = pages.view(torch.float8_e4m3fn)
        x = pages.float()
        if scales is not None:
            scales = scales if scales.ndim == 4 else scales[:, :, None, :]
            x = (x.unflatten(-1, (-1, SCALE_BLOCK)) * scales[..., None]).flatten(-2)
        dense.append(x[table.clamp(min=0)].transpose(1, 2).flatten(2, 3))
    return dense


def _attention(query, keys, values, seen):
    """query [requests, kv_heads, rows, dim], seen [requests, 1, rows, tokens]; a row that sees nothing gives zeros."""
    logits = (query / math.sqrt(query.shape[-1])) @ keys.transpose(-1, -2)
    logits = logits.masked_fill_(~seen, -math.inf)
    top = logits.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = torch.exp_(logits.sub_(top))
    total = weights.sum(dim=-1, keepdim=True)
    return torch.where(total > 0, (weights @ values) / total, 0.0)


def _plain_prompt(state: dict):
    case = state["case"]
    heads, group, dim = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["head_dim"]
    keys, values = _dense(case, state["pool"], state["table"])
    token = torch.arange(keys.shape[2], device=keys.device)
    # tokens past a request's end hold nothing: their values must not reach the sums
    values = values.masked_fill_((token >= state["lens"][:, None])[:, None, :, None], 0.0)
    rows = _rotated(state["query"], state["position"])[state["padded_token"]]  # [requests, new, q_heads, dim]
    requests, new = rows.shape[:2]
    rows = rows.reshape(requests, new, heads, group, dim).permute(0, 2, 1, 3, 4).reshape(requests, heads, new * group, dim)
    limit = (state["lens"] - state["new"])[:, None] + torch.arange(new, device=keys.device) + 1
    seen = token < torch.minimum(limit, state["lens"][:, None]).repeat_interleave(group, dim=1)[:, None, :, None]
    out = _attention(rows, keys, values, seen).reshape(requests, heads, new, group, dim).permute(0, 2, 1, 3, 4)
    return out.reshape(requests, new, heads * group, dim)[state["request"], state["token_row"]].to(torch.bfloat16)


def _plain_shared(state: dict):
    case = state["case"]
    heads, dim, requests = case["kv_heads"], case["head_dim"], case["requests"]
    keys, values = _dense(case, state["pool"], state["table"])
    seen = (torch.arange(keys.shape[2], device=keys.device) < state["lens"][:, None])[:, None, None, :]
    values = values.masked_fill_(~seen.transpose(-1, -2), 0.0)
    rows = _rotated(state["query"], state["position"]).reshape(requests, heads, -1, dim)
    return _attention(rows, keys, values, seen).reshape(requests, case["q_heads"], dim).to(torch.bfloat16)


# ---- the same from the definitions, in 64 bits -----------------------------------------------------


def _turn64(x, position):
    dim = x.shape[-1]
    pair = torch.arange(dim // 2, device=x.device, dtype=torch.float64)
    angle = position.double()[:, None] * torch.pow(torch.tensor(ROPE_THETA, dtype=torch.float64, device=x.device), -2 * pair / dim)
    z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], dim // 2, 2).contiguous())
    return torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)[:, None]).reshape(x.shape)


def _real64(case: dict, pages, scales):
    """Pages (any leading dimensions, [heads, slots, dim] last) as the numbers they stand for."""
    if case["layout"] == "bf16_kv":
        return pages.double()
    x = (pages.view(torch.float8_e4m3fn).float() if case["layout"] == "fp8_kv" else pages).double()
    return x * scales.double().repeat_interleave(SCALE_BLOCK, dim=-1)


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(state)
    pool, lens = state["pool"], state["lens"].tolist()
    heads, group, page = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["page"]
    query = _turn64(state["query"], state["position"]) / math.sqrt(case["head_dim"])
    out = torch.zeros_like(query)
    counts = state["new"].tolist() if case["kind"] == "prompt" else [1] * case["requests"]
    first = 0
    for request, (length, count) in enumerate(zip(lens, counts)):
        pages = state["table"][request, : -(-length // page)]
        for head in range(heads):
            if length == 0:
                continue
            key_scales = None if pool["key_scales"] is None else pool["key_scales"][pages, head][:, None]
            value_scales = None if pool["value_scales"] is None else pool["value_scales"][pages, head]
            k = _real64(case, pool["key_pages"][pages, head], key_scales).reshape(-1, case["head_dim"])[:length]
            v = _real64(case, pool["value_pages"][pages, head], value_scales).reshape(-1, case["head_dim"])[:length]
            for q_head in range(head * group, (head + 1) * group):
                logits = query[first : first + count, q_head] @ k.T
                later = torch.arange(length, device=k.device) > (length - count + torch.arange(count, device=k.device))[:, None]
                out[first : first + count, q_head] = torch.softmax(logits.masked_fill_(later, -math.inf), dim=-1) @ v
        first += count
    return out


def _exact_append(state: dict):
    case, pool = state["case"], state["pool"]
    keys = _turn64(state["keys"], state["position"]) if case["rotated"] else state["keys"].double()
    values = state["values"].double()
    token_page, token_slot = state["token_page"].cpu().numpy(), state["token_slot"].cpu().numpy()
    if case["layout"] == "bf16_kv":
        key_pages, value_pages = pool["key_pages"].double(), pool["value_pages"].double()
        flat = torch.from_numpy(token_page * case["page"] + token_slot).cuda()
        for pages, x in ((key_pages, keys), (value_pages, values)):
            rows = pages.transpose(1, 2).reshape(-1, *x.shape[1:])
            rows[flat] = x
            pages.copy_(rows.reshape(pages.transpose(1, 2).shape).transpose(1, 2))
        return key_pages, value_pages
    limit, dim = LIMITS[case["layout"]], case["head_dim"]

    def stored(x):  # the numbers that 8 bits hold
        x = x.clamp(-limit, limit)
        return x.float().to(torch.float8_e4m3fn).double() if case["layout"] == "fp8_kv" else x.round()

    def spread(scale):
        return scale.repeat_interleave(SCALE_BLOCK, dim=-1)

    def largest(x, axes):
        return x.abs().unflatten(-1, (dim // SCALE_BLOCK, SCALE_BLOCK)).amax(dim=axes)

    numbers = [p.view(torch.float8_e4m3fn).float().double() if case["layout"] == "fp8_kv" else p.double()
               for p in (pool["key_pages"], pool["value_pages"])]
    key_scales, value_scales = pool["key_scales"].double(), pool["value_scales"].double()
    scale = (largest(values, -1) / limit).clamp(min=1e-6)
    where = (torch.from_numpy(token_page).cuda(), torch.from_numpy(token_slot).cuda())
    numbers[1].transpose(1, 2)[where] = stored(values / spread(scale))
    value_scales.transpose(1, 2)[where] = scale
    # page by page: tokens of a page follow one another
    bounds = np.flatnonzero(np.r_[True, token_page[1:] != token_page[:-1], True])
    for begin, end in zip(bounds[:-1], bounds[1:]):
        page, slot = int(token_page[begin]), int(token_slot[begin])
        new = (largest(keys[begin:end], (0, -1)) / limit).clamp(min=1e-6)
        if slot > 0:
            held = key_scales[page]
            grown = new > held
            new = torch.maximum(new, held)
            again = stored(numbers[0][page, :, :slot] * spread(held / new)[:, None])
            numbers[0][page, :, :slot] = torch.where(spread(grown)[:, None], again, numbers[0][page, :, :slot])
        key_scales[page] = new
        numbers[0][page, :, slot : slot + end - begin] = stored(keys[begin:end] / spread(new)).transpose(0, 1)
    if case["layout"] == "fp8_kv":
        return numbers[0], numbers[1], key_scales, value_scales
    return (numbers[0] * spread(key_scales)[:, :, None], numbers[1] * spread(value_scales), key_scales, value_scales)


# ---- what a pass cannot do without -----------------------------------------------------------------


def work(case: dict) -> dict:
    """Bytes read and written once, and the multiply-adds of logits and weighted values.

    An append reads its rows and writes them in the cache's format; the scale of a page is read and written.
    Attention reads every page that a request sees once, whoever shares it, and the queries, and writes its rows."""
    heads, dim, page = case["kv_heads"], case["head_dim"], case["page"]
    element, blocks = (2, 0) if case["layout"] == "bf16_kv" else (1, dim // SCALE_BLOCK)
    if case["kind"] == "append":
        tokens = sum(_lengths(case))
        touched = sum((c + n - 1) // page - c // page + 1 for n, c in zip(_lengths(case), _cached(case)) if n)
        moved = tokens * heads * (2 * dim * (2 + element) + 4 * blocks) + touched * heads * 8 * blocks
        return dict(bytes=moved, flops=3 * tokens * heads * dim if case["rotated"] else 0)
    if case["kind"] == "prompt":
        lens = [n + c for n, c in zip(_lengths(case), _cached(case))]
        tokens, pages = sum(lens), sum(-(-n // page) for n in lens)
        rows, flops = sum(_lengths(case)), 4 * _pairs(case) * dim
    else:
        shared, sub = _prefix_pages(case)
        group, second = _family(case)
        own_tokens = _shared_lens(case) - (shared + sub) * page
        common = len(set(group.tolist())) * shared + len(set(second.tolist())) * sub
        tokens, pages = int(own_tokens.sum()) + common * page, int((-(-own_tokens // page)).sum()) + common
        rows, flops = case["requests"], int(4 * _shared_lens(case).sum()) * case["q_heads"] * dim
    moved = tokens * heads * (2 * dim * element + 4 * blocks) + pages * heads * 4 * blocks
    return dict(bytes=moved + 4 * rows * case["q_heads"] * dim, flops=flops)
