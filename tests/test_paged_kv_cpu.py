"""The operators around the paged cache, the parts that need no GPU: plans, refusals, the C ABI's surface."""

from __future__ import annotations

import ctypes
import importlib
import re
from pathlib import Path

import numpy as np
import pytest
import torch
from fast_kernels.ops import _paged
from paged_kv_testlib import attention64, cache_values, fragmented_table, random_cache, rotate64

REPO = Path(__file__).resolve().parent.parent
ops = importlib.import_module("fast_kernels.ops")
LIB = REPO / "fast-kernels_b200" / "src" / "fast_kernels" / "lib" / "libfk_paged_kv.so"


def _append_plan(table, lens, new, **kwargs):
    arguments = dict(page_table=torch.tensor(table, dtype=torch.int32), seq_lens=torch.tensor(lens, dtype=torch.int32),
                     append_lens=torch.tensor(new, dtype=torch.int32), num_kv_heads=2, head_dim=64, page_size=16,
                     kv_layout="bf16_kv", use_cache=False)
    return ops.plan_paged_kv_append(**{**arguments, **kwargs})


def test_library_exports_every_declared_symbol() -> None:
    lib = ctypes.CDLL(str(LIB))
    names = set(re.findall(r"\b(fk_paged_kv_\w+)\s*\(", (REPO / "include" / "fk_paged_kv.h").read_text()))
    assert "fk_paged_kv_append" in names
    for name in names:
        assert hasattr(lib, name), f"{name} is declared in include/ but not exported"


def test_append_plan_cuts_tokens_into_pages() -> None:
    """20 tokens behind 10 (slots 10-15 of page 7, 0-13 of page 3), none, and one in a page's last slot."""
    plan = _append_plan([[7, 3], [9, -1], [4, 5]], [10, 3, 31], [20, 0, 1])
    assert plan.segments_cpu.tolist() == [[7, 10 | 6 << 16, 0, 10], [3, 0 | 14 << 16, 6, 16], [5, 15 | 1 << 16, 20, 31]]
    assert plan.num_tokens == 21 and plan.largest_page == 7 and plan.seq_lens_after_cpu.tolist() == [30, 3, 32]
    nothing = _append_plan([[7, 3]], [10], [0])
    assert nothing.num_segments == 0 and nothing.largest_page == -1
    none = _append_plan(torch.zeros((0, 4)).tolist() or [[0]], [0], [0])
    assert none.num_segments == 0


def test_append_plans_are_remembered_by_their_contents() -> None:
    arguments = dict(use_cache=True)
    first = _append_plan([[0, 1]], [3], [4], **arguments)
    assert _append_plan([[0, 1]], [3], [4], **arguments) is first
    assert _append_plan([[0, 2]], [3], [4], **arguments) is not first
    assert _append_plan([[0, 1]], [3], [5], **arguments) is not first


def test_append_plan_refusals() -> None:
    with pytest.raises(ValueError, match="same page"):
        _append_plan([[1, 2], [1, 2]], [16, 17], [1, 1])
    with pytest.raises(ValueError, match="no page for some"):
        _append_plan([[1, -1]], [10], [7])
    with pytest.raises(ValueError, match="fewer columns"):
        _append_plan([[1]], [10], [7])
    with pytest.raises(ValueError, match="append_lens must not be negative"):
        _append_plan([[1]], [10], [-1])
    with pytest.raises(ValueError, match="one entry per request"):
        _append_plan([[1]], [10, 3], [1])
    with pytest.raises(ValueError, match="head_dim must be 64 or 128"):
        _append_plan([[1]], [10], [1], head_dim=96)
    with pytest.raises(ValueError, match="page_size must be 16 or 32"):
        _append_plan([[1]], [10], [1], page_size=64)
    with pytest.raises(ValueError, match="layout must be one of"):
        _append_plan([[1]], [10], [1], kv_layout="fp4_kv")
    with pytest.raises(TypeError, match="must hold integers"):
        _append_plan([[1]], [10], [1], page_table=torch.tensor([[1.0]]))
    with pytest.raises(ValueError, match="fit 32 bits"):
        _append_plan([[1]], [2**31 - 1], [1], page_table=torch.zeros((1, 1), dtype=torch.int32))


def test_append_needs_lengths_or_a_plan() -> None:
    cache = ops.empty_paged_kv(num_pages=1, page_table=torch.tensor([[0]]), seq_lens=torch.tensor([0]), num_kv_heads=2, head_dim=64,
                               page_size=16, kv_layout="int8_kv", device="cpu")
    assert cache.key_scales.shape == (1, 2, 1) and cache.value_scales.shape == (1, 2, 16, 1) and cache.reference_key_pages is None
    rows = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="append_lens or a plan"):
        ops.paged_kv_append(rows, rows, cache)
    with pytest.raises(ValueError, match="not both"):
        ops.paged_kv_append(rows, rows, cache, append_lens=torch.tensor([1]), plan=_append_plan([[0]], [0], [1], kv_layout="int8_kv"))
    with pytest.raises(ValueError, match="key_pages must be a CUDA tensor"):
        ops.paged_kv_append(rows, rows, cache, append_lens=torch.tensor([1]))
    with pytest.raises(ValueError, match="the plan was made for kv_layout"):
        ops.paged_kv_append(rows, rows, cache, plan=_append_plan([[0]], [0], [1]))


def test_native_append_checks_its_arguments_before_the_device() -> None:
    from fast_kernels.native import native_module

    call = native_module().paged_kv_append_forward
    good = dict(keys_ptr=256, values_ptr=256, key_token_stride=128, key_head_stride=64, value_token_stride=128,
                value_head_stride=64, key_pages_ptr=256, value_pages_ptr=256, key_scales_ptr=256, value_scales_ptr=256,
                segments_ptr=256, num_segments=1, num_tokens=1, num_pages=1, num_kv_heads=2, head_dim=64, page_size=16,
                kv_format=2, rotate_keys=1, rope_theta=10000.0, stream_ptr=0)
    call(**{**good, "num_segments": 0, "keys_ptr": 0})  # nothing to do
    for change, message in (({"head_dim": 96}, "head_dim"), ({"page_size": 8}, "page_size"), ({"kv_format": 3}, "kv_format"),
                            ({"num_kv_heads": 0}, "num_kv_heads"), ({"num_tokens": -1}, "non-negative"),
                            ({"rope_theta": 0.0}, "rope_theta"), ({"rope_theta": float("inf")}, "rope_theta"),
                            ({"keys_ptr": 0}, "NULL"), ({"segments_ptr": 0}, "NULL"), ({"value_scales_ptr": 0}, "scales"),
                            ({"keys_ptr": 264}, "aligned"), ({"key_scales_ptr": 258}, "aligned"),
                            ({"key_token_stride": 12}, "multiples of 8")):
        with pytest.raises(ValueError, match=message):
            call(**{**good, **change})


# ---- attention plans: the descriptors, carried out in fp64, give the attention -------------------------------


def _run_items(plan, cache, query64, scale):
    """What the kernels make of a plan's tables: per vector and query head the partial results (values, maximum, denominator)
    or the finished row, as {row: fp64 [q_heads, dim]}, {partial: ...}."""
    keys, values = cache_values(cache)
    ps, group, dim = plan.page_size, plan.num_q_heads // plan.num_kv_heads, plan.head_dim
    page_ids, vectors = plan.page_ids_cpu, plan.vectors_cpu.tolist()
    direct, partials = {}, {}
    for first_vector, count, head, entry, first, end, causal, partial in plan.items_cpu.tolist():
        assert count * group <= 256 and first % ps == 0 and first < end
        pages = page_ids[entry : entry + -(-end // ps)].long()
        k, v = (x[pages, head].reshape(-1, dim)[first:end] for x in (keys, values))
        for vector in range(first_vector, first_vector + count):
            row, position, first_partial, partial_count = vectors[vector]
            seen = max(0, min(end, position + 1) - first) if causal else end - first
            for q_head in range(head * group, (head + 1) * group):
                logits = (k[:seen] @ query64[row, q_head]) * scale
                top = float(logits.max()) if seen else -np.inf
                weights = torch.exp(logits - top) if seen else logits
                result = (weights @ v[:seen], top, float(weights.sum()))
                key = (row, q_head) if partial < 0 else (first_partial + partial, q_head)
                place = direct if partial < 0 else partials
                assert key not in place and (partial < 0 or partial < partial_count)
                place[key] = result
    return direct, partials


def _merge(parts):
    top = max(m for _, m, _ in parts)
    if top == -np.inf:
        return torch.zeros_like(parts[0][0])
    return sum(o * np.exp(m - top) for o, m, _ in parts) / sum(l * np.exp(m - top) for _, m, l in parts)


@pytest.mark.parametrize(("group", "ps", "lens", "new"), [
    (4, 16, [70, 5, 33], [70, 0, 1]),
    (1, 32, [700], [300]),
    (3, 16, [1, 0, 200], [1, 0, 90]),
    (8, 32, [2100, 40], [3, 40]),
    (256, 16, [20], [3]),
])
def test_prompt_plan_carried_out_in_fp64_is_the_attention(group, ps, lens, new) -> None:
    heads, dim = 2, 64
    table, pages = fragmented_table([-(-n // ps) for n in lens], seed=1)
    cache = random_cache(layout="int8_kv", pages=pages, heads=heads, page_size=ps, dim=dim, table=table, lens=lens, theta=10000.0,
                         seed=2, device="cpu")
    plan = ops.plan_paged_prompt_attention(page_table=cache.page_table, seq_lens=cache.seq_lens, query_lens=torch.tensor(new),
                                           num_q_heads=group * heads, num_kv_heads=heads, head_dim=dim, page_size=ps,
                                           kv_layout="int8_kv", use_cache=False)
    rows = [(b, lens[b] - n + i) for b, n in enumerate(new) for i in range(n)]
    query = torch.randn((len(rows), group * heads, dim), generator=torch.Generator().manual_seed(3)).double()
    want = attention64(cache, query, rows, 0.125, 10000.0)
    direct, partials = _run_items(plan, cache, rotate64(query, [p for _, p in rows], 10000.0), 0.125)
    assert len(partials) == plan.num_partials * group * heads
    for row, (_, position, first, count) in enumerate(plan.vectors_cpu.tolist()):
        assert position == rows[row][1]
        for head in range(group * heads):
            parts = [partials[first + j, head] for j in range(count)] if count else [direct[row, head]]
            torch.testing.assert_close(_merge(parts), want[row, head], rtol=1e-10, atol=1e-12)


def test_long_ranges_are_cut_and_short_ones_are_not() -> None:
    def items(length, new, heads):
        return ops.plan_paged_prompt_attention(
            page_table=torch.arange(-(-length // 16))[None], seq_lens=torch.tensor([length]), query_lens=torch.tensor([new]),
            num_q_heads=heads * 4, num_kv_heads=heads, head_dim=128, page_size=16, kv_layout="bf16_kv", use_cache=False)

    assert items(300, 64, 8).num_items == 8 and items(300, 64, 8).num_partials == 0
    long = items(32768, 64, 8)  # one group of vectors and 8 kv heads: 18 pieces each would be a wave of 144
    assert 100 <= long.num_items <= 148 and long.num_partials == 64 * long.num_items // 8
    assert items(8192, 8192, 8).num_partials == 0  # 1024 items without cutting


def _shared_case(ps=16, layout="fp8_kv", heads=2, dim=64):
    """Nine requests, not sorted: five share 160 tokens of which three share 144 more, two share 320 whole (one of them a
    page boundary's length, one empty tail), one is alone and one is empty."""
    page = iter(range(1000))
    take = lambda tokens: [next(page) for _ in range(tokens // ps)]  # noqa: E731
    system, document, other = take(160), take(144), take(320)
    tails = {0: 7, 2: 33, 3: 1, 5: 16, 6: 40, 7: 0, 8: 5}
    rows = {0: system, 2: system + document, 3: system + document, 5: system, 6: system + document, 7: other, 8: other}
    lens = [0] * 9
    for b, prefix in rows.items():
        lens[b] = len(prefix) * ps + tails[b]
        rows[b] = prefix + take(-(-tails[b] // ps) * ps)
    rows[4], lens[4] = take(96), 90
    rows[1] = []
    table = np.full((9, max(map(len, rows.values()))), -1, dtype=np.int32)
    for b, pages in rows.items():
        table[b, : len(pages)] = pages
    total = next(page)
    table[table >= 0] = np.random.RandomState(0).permutation(total)[table[table >= 0]]
    return random_cache(layout=layout, pages=total, heads=heads, page_size=ps, dim=dim, table=table, lens=lens, theta=10000.0, seed=2,
                        device="cpu")


def _shared_plan(cache, group, **kwargs):
    return ops.plan_shared_prefix_decode(page_table=cache.page_table, seq_lens=cache.seq_lens, num_q_heads=group * cache.num_kv_heads,
                                         num_kv_heads=cache.num_kv_heads, head_dim=cache.head_dim, page_size=cache.page_size,
                                         kv_layout=cache.kv_layout, **{"use_cache": False, "min_saved_bytes": 0, **kwargs})


@pytest.mark.parametrize("group", [1, 3, 100])
def test_shared_plan_carried_out_in_fp64_is_the_attention(group) -> None:
    cache = _shared_case()
    plan = _shared_plan(cache, group)
    assert sorted((first, end, tuple(sorted(who))) for first, end, who in plan.runs) == [
        (0, 10, (0, 2, 3, 5, 6)), (0, 20, (7, 8)), (10, 19, (2, 3, 6))]
    lens = cache.seq_lens.tolist()
    query = torch.randn((9, group * 2, 64), generator=torch.Generator().manual_seed(3)).double()
    rows = [(b, lens[b] - 1) for b in range(9)]
    want = attention64(cache, query, rows, 0.125, 10000.0)
    turned = rotate64(query, [max(0, n - 1) for n in lens], 10000.0)
    direct, partials = _run_items(plan, cache, turned, 0.125)
    assert not direct and len(partials) == plan.num_partials * group * 2
    keys, values = cache_values(cache)
    tail = plan.tail_plan
    assert tail.seq_lens_cpu.tolist() == lens
    offsets = tail.request_run_offsets_cpu.tolist()
    for b, (first, count) in enumerate(plan.of_request_cpu.tolist()):
        slots = []
        for run in range(offsets[b], offsets[b + 1]):
            base, pages, last = (int(getattr(tail, f"run_{n}_cpu")[run]) for n in ("base_pages", "page_counts", "last_page_lens"))
            slots += [(base + i, s) for i in range(pages) for s in range(last if i == pages - 1 else 16)]
        for head in range(group * 2):
            parts = [partials[first + j, head] for j in range(count)]
            if slots:
                k, v = (torch.stack([x[page, head // group, slot] for page, slot in slots]) for x in (keys, values))
                logits = (k @ turned[b, head]) * 0.125
                weights = torch.exp(logits - logits.max())
                parts.append((weights @ v, float(logits.max()), float(weights.sum())))
            got = _merge(parts) if parts else torch.zeros(64, dtype=torch.float64)
            torch.testing.assert_close(got, want[b, head], rtol=1e-10, atol=1e-12)


def test_shared_plan_without_enough_to_save_is_the_plain_decode() -> None:
    cache = _shared_case()
    plan = _shared_plan(cache, 2, min_saved_bytes=1 << 30)
    assert plan.runs == [] and plan.num_items == 0 and plan.num_partials == 0 and plan.estimated_saved_hbm_bytes == 0
    plain = ops.plan_clustered_page_decode(page_table=cache.page_table, seq_lens=cache.seq_lens, num_q_heads=4, num_kv_heads=2, head_dim=64,
                                           page_size=16, kv_layout="fp8_kv", use_cache=False)
    for name in ("run_base_pages", "run_page_counts", "run_last_page_lens", "request_run_offsets", "seq_lens"):
        assert torch.equal(getattr(plan.tail_plan, f"{name}_cpu"), getattr(plain, f"{name}_cpu")), name
    assert plan.tail_plan.max_pages == plain.max_pages
    assert _shared_plan(cache, 2).estimated_saved_hbm_bytes == (4 * 10 + 2 * 9 + 20) * 2 * (2 * 16 * 64 + 4 * 17)


def test_attention_plan_refusals() -> None:
    arguments = dict(page_table=torch.tensor([[0, 1]]), seq_lens=torch.tensor([20]), query_lens=torch.tensor([3]), num_q_heads=4,
                     num_kv_heads=2, head_dim=64, page_size=16, kv_layout="bf16_kv", use_cache=False)
    plan = ops.plan_paged_prompt_attention
    assert plan(**arguments).num_tokens == 3
    for change, message in (({"query_lens": torch.tensor([21])}, "must not exceed"), ({"query_lens": torch.tensor([-1])}, "negative"),
                            ({"num_q_heads": 3}, "divisible"), ({"num_q_heads": 1024}, "at most 256"), ({"head_dim": 32}, "head_dim"),
                            ({"page_table": torch.tensor([[0, -1]])}, "no page"), ({"page_table": torch.tensor([[0]])}, "fewer columns")):
        with pytest.raises(ValueError, match=message):
            plan(**{**arguments, **change})
    arguments.pop("query_lens")
    plan = ops.plan_shared_prefix_decode
    assert plan(**arguments).batch == 1
    for change, message in (({"min_saved_bytes": -1}, "negative"), ({"num_q_heads": 3}, "divisible"),
                            ({"page_table": torch.tensor([[0, -1]])}, "no page"), ({"page_table": torch.tensor([[0]])}, "fewer columns"),
                            ({"page_table": torch.zeros((0, 2), dtype=torch.int32), "seq_lens": torch.zeros(0, dtype=torch.int32)}, "empty")):
        with pytest.raises(ValueError, match=message):
            plan(**{**arguments, **change})


# ---- the entry points refuse before they touch the device ----------------------------------------------------


def test_native_attention_checks_its_arguments_before_the_device() -> None:
    from fast_kernels.native import native_module

    call = native_module().paged_attention_forward
    good = dict(query_ptr=256, query_row_stride=256, query_head_stride=64, key_ptr=256, value_ptr=256, key_scales_ptr=256,
                value_scales_ptr=256, page_ids_ptr=256, vectors_ptr=256, items_ptr=256, output_ptr=256, partials_ptr=256, num_rows=1,
                num_page_ids=1, num_vectors=1, num_items=1, num_partials=1, num_pages=1, num_q_heads=4, num_kv_heads=2, head_dim=64,
                page_size=16, kv_format=2, softmax_scale=0.1, rope_theta=10000.0, stream_ptr=0)
    call(**{**good, "num_items": 0, "query_ptr": 0})  # nothing to do
    call(**{**good, "num_vectors": 0, "query_ptr": 0})
    for change, message in (({"head_dim": 96}, "head_dim"), ({"page_size": 8}, "page_size"), ({"kv_format": 3}, "kv_format"),
                            ({"num_q_heads": 3}, "divisible"), ({"num_q_heads": 1024}, "256 query heads"), ({"num_rows": -1}, "non-negative"),
                            ({"softmax_scale": float("nan")}, "softmax_scale"), ({"rope_theta": -1.0}, "rope_theta"),
                            ({"query_ptr": 0}, "NULL"), ({"items_ptr": 0}, "NULL"), ({"partials_ptr": 0}, "partials"),
                            ({"key_scales_ptr": 0}, "scales"), ({"output_ptr": 264}, "aligned"), ({"key_scales_ptr": 258}, "aligned"),
                            ({"key_scales_ptr": 260, "head_dim": 128}, "key_scales must be aligned"), ({"query_row_stride": 12}, "multiples of 8"), ({"num_pages": 0}, "num_pages"),
                            ({"num_pages": 2**30}, "31 bits"), ({"num_vectors": 2**30}, "31 bits")):
        with pytest.raises(ValueError, match=message):
            call(**{**good, **change})
    # a cache that is a slice of another one starts at any of its pages' scales: the next check is what refuses this
    for change in ({"key_scales_ptr": 260}, {"key_scales_ptr": 264, "head_dim": 128}):
        with pytest.raises(ValueError, match="multiples of 8"):
            call(**{**good, **change, "query_row_stride": 12})


@pytest.mark.parametrize("first_call_captured", [True, False])
def test_tables_of_a_plan_are_not_uploaded_into_a_capture(monkeypatch, first_call_captured: bool) -> None:
    device = torch.device("cpu", 0)  # (an index is all that is asked of it)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    kept: dict = {}
    if not first_call_captured:
        before = _paged.on_device(kept, device, 0, lambda: {"a": np.arange(3), "b": np.arange(4)})
        assert before["b"] - before["a"] == 512
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    if first_call_captured:
        with pytest.raises(RuntimeError, match="before the capture"):
            _paged.on_device(kept, device, 0, lambda: {"a": np.arange(3), "b": np.arange(4)})
        assert not kept
    else:
        assert _paged.on_device(kept, device, 1, lambda: {}) == before


def test_native_shared_decode_wants_items_with_partial_results() -> None:
    from fast_kernels.native import native_module

    call = native_module().shared_prefix_decode_forward
    pointers = {f"{name}_ptr": 256 for name in (
        "query", "key", "value", "key_scales", "value_scales", "page_ids", "vectors", "items", "of_request", "run_base_pages",
        "run_page_counts", "run_logical_starts", "run_last_page_lens", "request_run_offsets", "seq_lens", "output", "partials")}
    good = dict(**pointers, batch=1, num_page_ids=1, num_items=1, num_partials=1, num_runs=0, max_tail_pages=0, num_pages=1,
                num_q_heads=4, num_kv_heads=2, head_dim=64, page_size=16, kv_format=0, softmax_scale=0.1, rope_theta=10000.0, stream_ptr=0)
    for change, message in (({"num_partials": 0}, "come together"), ({"num_items": 0}, "come together"), ({"num_items": -1}, "come together"),
                            ({"head_dim": 32}, "head_dim"), ({"num_kv_heads": 0}, "divisible")):
        with pytest.raises(ValueError, match=message):
            call(**{**good, **change})


def test_merged_decode_checks_the_prior_rows() -> None:
    from fast_kernels import page_decode_capi as pdc

    lib, args = pdc.load_library(), pdc.PageDecodeArgs()
    for rows, of_request, message in ((0, 256, "NULL"), (256, 0, "NULL"), (264, 256, "aligned"), (256, 260, "aligned"), (256, 256, "empty inputs")):
        prior = pdc.PageDecodePrior(rows, of_request)
        assert lib.fk_page_decode_forward_merged(ctypes.byref(args), ctypes.byref(prior)) == pdc.ERR_INVALID_ARGUMENT
        assert message in lib.fk_page_decode_last_error().decode()
    assert lib.fk_page_decode_forward_merged(ctypes.byref(args), None) == pdc.ERR_INVALID_ARGUMENT


def test_a_build_without_cuda_has_the_names(tmp_path: Path) -> None:
    import importlib.util
    import subprocess
    import sys

    spec = importlib.util.spec_from_file_location("fk_build", REPO / "fast-kernels_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    build.build_python_module_without_cuda(tmp_path)
    child = ("import sys; sys.path.insert(0, sys.argv[1]); import _native\n"
             "for name in ('paged_kv_append_forward', 'paged_attention_forward', 'shared_prefix_decode_forward'): assert hasattr(_native, name)\n"
             "try: _native.paged_kv_device_status()\n"
             "except RuntimeError as error: print(error)")
    done = subprocess.run([sys.executable, "-c", child, str(tmp_path)], capture_output=True, text=True, check=True)
    assert done.stdout.strip() == "fast-kernels was built without CUDA support"
