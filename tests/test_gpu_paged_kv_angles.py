"""The rotary angles of the paged-cache operators."""

from __future__ import annotations

import importlib
import math
from decimal import Decimal, getcontext

import numpy as np
import pytest
import torch
from fast_kernels.native import native_module
from paged_kv_testlib import cache_values, random_cache, rotate64

pytestmark = pytest.mark.gpu
ops = importlib.import_module("fast_kernels.ops")


def _angles(positions: np.ndarray, dim: int, theta: float) -> tuple[np.ndarray, np.ndarray]:
    """[positions, pairs]: position * theta^(-2i/dim) in radians, the whole turns taken off in exact arithmetic; and what
    rounding half an angle's turns to fp32 leaves out of it."""
    getcontext().prec = 60
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    per_position = [int((Decimal(theta).ln() * Decimal(-2 * i) / dim).exp() / (2 * pi) * 2**64) for i in range(dim // 2)]
    upper = np.array([[((int(p) * t) % 2**64) >> 32 for t in per_position] for p in positions], dtype=np.int64)
    upper = np.where(upper >= 2**31, upper - 2**32, upper)
    rest = upper - upper.astype(np.float32).astype(np.int64)
    return upper * (math.pi / 2**31), rest * (math.pi / 2**31)


def test_an_appended_keys_angle_is_not_rounded_to_fp32() -> None:
    """Every key has a single element of 1, which its turn makes (cos, sin): the page's scale times 127 is the larger of the
    two. It is off by at most 2^-24 (an fp32 cosine within one unit in the last place, below 1) and 2^-24 (the quotient), and
    these have nothing to do with the sign of what rounding the whole angle leaves out: over N keys the mean of the errors,
    each times that sign, stays within 6 * 2^-23 / sqrt(N), 2.8e-9. With the angle rounded the mean is its share of the error,
    about 3e-8 * 0.35.

    What rounding the angle's distance to a quarter turn leaves out (in units u = pi * 2^-31: w(rest), rest brought into +-16
    or less) has no part in the mean where the whole angle's rounding is coarser: w is as often up as down over +-32 or +-64.
    Where it is the same rounding, in the eighth of the turn around 0, its mean is 8 u on |angle| in [1/16, 1/8] of a turn, half
    of that in the interval of half the length before, and so on: 8 u * 1/8 * (1 + 1/4 + 1/16 + ..) * the slope's 0.71 < 1.4e-9."""
    heads, dim, ps, tokens, theta = 32, 64, 16, 2048, 10000.0
    positions = np.random.RandomState(1).randint(0, 100_000 // ps, tokens) * ps
    table = np.full((tokens, 100_000 // ps + 1), -1, dtype=np.int32)
    table[np.arange(tokens), positions // ps] = np.arange(tokens)
    lens = torch.from_numpy(positions.astype(np.int32))
    cache = ops.empty_paged_kv(num_pages=tokens, page_table=torch.from_numpy(table), seq_lens=lens, num_kv_heads=heads, head_dim=dim,
                               page_size=ps, kv_layout="int8_kv", key_rope_theta=theta)
    keys = torch.zeros((tokens, heads, dim), dtype=torch.bfloat16, device="cuda")
    pair = torch.arange(heads, device="cuda")
    keys[:, pair, 2 * pair] = 1.0
    plan = ops.plan_paged_kv_append(page_table=cache.page_table, seq_lens=lens, append_lens=torch.ones(tokens, dtype=torch.int32),
                                    num_kv_heads=heads, head_dim=dim, page_size=ps, kv_layout="int8_kv", use_cache=False)
    ops.paged_kv_append(keys, keys, cache, plan=plan)
    got = cache.key_scales[:, :, 0].double().cpu().numpy() * 127.0
    angle, rest = _angles(positions, dim, theta)
    cos, sin = np.cos(angle), np.sin(angle)
    of_cos = np.abs(cos) >= np.abs(sin)
    want = np.where(of_cos, np.abs(cos), np.abs(sin))
    slope = np.where(of_cos, -sin * np.sign(cos), cos * np.sign(sin))
    off = got - want
    assert np.abs(off).max() <= 2.0**-23
    mean = float((off * np.sign(-rest * slope)).mean())
    assert abs(mean) <= 6 * 2.0**-23 / math.sqrt(off.size), mean


@pytest.mark.parametrize("layout", ["bf16_kv", "fp8_kv", "int8_kv"])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_shared_decode_far_out_turns_its_queries_by_one_angle(layout, dim) -> None:
    """Two requests share a million tokens, one page over and over, whose keys are 0: logits of 0, whatever the angle. Their
    own last tokens have logits to about +-40, and nearly all of the weight.

    Of these the query is a 16-bit head and remainder (2^-17 with bf16) and its turn fp32: d = 2^-16 * scale * max_t sum_i
    |q_i k_i| on a logit, a factor within e^(+-2 d) on a weight; 16-bit heads and remainders of the weights: 2^-16. The shared part's
    weights are rounded to bf16 or fp16, and 8-bit values of the block without the token's larger scale to fp16 twice: 2^-8 of
    its sum. The row is rounded once. An fp32 angle is off by up to 0.05 here."""
    ps, theta, shared, own = 32, 10000.0, 31_250, 25
    table = np.zeros((2, shared + 1), dtype=np.int32)
    table[:, -1] = [1, 2]
    length = shared * ps + own
    cache = random_cache(layout=layout, pages=3, heads=2, page_size=ps, dim=dim, table=table, lens=[length, length - 8], theta=theta, seed=1)
    cache.key_pages[0] = 0
    query = torch.randn((2, 8, dim), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    plan = ops.plan_shared_prefix_decode(page_table=cache.page_table, seq_lens=cache.seq_lens, num_q_heads=8, num_kv_heads=2, head_dim=dim,
                                         page_size=ps, kv_layout=layout, min_saved_bytes=0, use_cache=False)
    assert plan.runs == [(0, shared, (0, 1))]
    scale = 8.0 / math.sqrt(dim)
    got = ops.shared_prefix_decode(query, cache, plan=plan, softmax_scale=scale).double().cpu()
    keys, values = cache_values(cache)
    for b, n in enumerate(cache.seq_lens.tolist()):
        turned = rotate64(query[b : b + 1].cpu(), [n - 1], theta)[0].reshape(2, 4, dim)
        k, v = keys[1 + b, :, : n - shared * ps], values[1 + b, :, : n - shared * ps]
        logits = torch.einsum("hgd,htd->hgt", turned, k) * scale
        top = logits.amax(dim=-1, keepdim=True)
        weights, before = torch.exp(logits - top), torch.exp(-top) * shared
        total = weights.sum(dim=-1, keepdim=True) + before * ps
        mine = torch.einsum("hgt,htd->hgd", weights, v) / total
        others = before * values[0].sum(dim=1)[:, None] / total
        want = mine + others
        d = 2.0**-16 * scale * torch.einsum("hgd,htd->hgt", turned.abs(), k.abs()).amax(dim=-1, keepdim=True)
        a_mine = torch.einsum("hgt,htd->hgd", weights, v.abs()) / total
        a_others = before * values[0].abs().sum(dim=1)[:, None] / total
        bound = 2.0**-8 * want.abs() + (2.0**-16 + 2.2 * d) * (a_mine + a_others) + 2.0**-8 * a_others
        off = (got[b].reshape(2, 4, dim) - want).abs()
        assert float((off / bound).max()) <= 1.0, float((off / bound).max())
    torch.cuda.synchronize()
    assert native_module().paged_kv_device_status() == 0 and native_module().page_decode_device_status() == 0


@pytest.mark.parametrize("layout", ["bf16_kv", "int8_kv"])
def test_a_far_decode_that_shares_nothing_is_turned_by_the_same_angle(layout) -> None:
    """As above with one request, in a graph too. No part of it is rounded to 16 bits but for the row: weights and query are
    16-bit heads and remainders."""
    ps, theta, before_own, own, dim = 32, 10000.0, 31_250, 25, 128
    table = np.zeros((1, before_own + 1), dtype=np.int32)
    table[0, -1] = 1
    length = before_own * ps + own
    cache = random_cache(layout=layout, pages=2, heads=2, page_size=ps, dim=dim, table=table, lens=[length], theta=theta, seed=1)
    cache.key_pages[0] = 0
    query = torch.randn((1, 8, dim), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    plan = ops.plan_shared_prefix_decode(page_table=cache.page_table, seq_lens=cache.seq_lens, num_q_heads=8, num_kv_heads=2, head_dim=dim,
                                         page_size=ps, kv_layout=layout, use_cache=False)
    assert plan.runs == []
    scale = 8.0 / math.sqrt(dim)
    got = ops.shared_prefix_decode(query, cache, plan=plan, softmax_scale=scale)
    graph, again = torch.cuda.CUDAGraph(), torch.empty_like(got)
    with torch.cuda.graph(graph):
        ops.shared_prefix_decode(query, cache, plan=plan, softmax_scale=scale, output=again)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    keys, values = cache_values(cache)
    turned = rotate64(query.cpu(), [length - 1], theta)[0].reshape(2, 4, dim)
    k, v = keys[1, :, :own], values[1, :, :own]
    logits = torch.einsum("hgd,htd->hgt", turned, k) * scale
    top = logits.amax(dim=-1, keepdim=True)
    weights, before = torch.exp(logits - top), torch.exp(-top) * before_own
    total = weights.sum(dim=-1, keepdim=True) + before * ps
    want = (torch.einsum("hgt,htd->hgd", weights, v) + before * values[0].sum(dim=1)[:, None]) / total
    a = (torch.einsum("hgt,htd->hgd", weights, v.abs()) + before * values[0].abs().sum(dim=1)[:, None]) / total
    d = 2.0**-16 * scale * torch.einsum("hgd,htd->hgt", turned.abs(), k.abs()).amax(dim=-1, keepdim=True)
    # (a million fp32 weights of about e^-top each, added one after the other in blocks: 2^-12 of their share at most)
    bound = 2.0**-8 * want.abs() + (2.0**-16 + 2.2 * d) * a + 2.0**-12 * before * values[0].abs().sum(dim=1)[:, None] / total
    off = (got.double().cpu().reshape(2, 4, dim) - want).abs()
    assert float((off / bound).max()) <= 1.0, float((off / bound).max())
    assert native_module().page_decode_device_status() == 0
