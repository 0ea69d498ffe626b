"""The unquantised pages of a cache that was built from whole sequences, after an append."""

from __future__ import annotations

import dataclasses
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
ops = importlib.import_module("fast_kernels.ops")


def _grown(build):
    dense = [torch.randn((2, 2, 20, 64), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda() for seed in (1, 2)]
    built = build(*dense, torch.tensor([20, 11], dtype=torch.int32), page_size=16, fragment_pages=False)
    rows = [torch.randn((3, 2, 64), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda() for seed in (3, 4)]
    return built, rows, ops.paged_kv_append(*rows, built, append_lens=torch.tensor([2, 1]))


@pytest.mark.parametrize("build", [ops.quantize_paged_kv_int8, ops.quantize_paged_kv_fp8])
def test_an_appended_8_bit_cache_has_no_pages_that_lack_its_tokens(build) -> None:
    built, rows, grown = _grown(build)
    assert built.reference_key_pages is not None
    assert grown.reference_key_pages is None and grown.reference_value_pages is None
    with pytest.raises(ValueError, match="no unquantised pages"):
        ops.reference_clustered_page_decode(torch.zeros((2, 4, 64), dtype=torch.bfloat16, device="cuda"), grown)
    none = torch.tensor([0, 0])
    same = ops.paged_kv_append(rows[0][:0], rows[1][:0], built, append_lens=none)
    assert same.reference_key_pages is built.reference_key_pages


def test_an_appended_bf16_cache_is_its_own_reference() -> None:
    built, rows, grown = _grown(ops.pack_paged_kv_bf16)
    assert grown.reference_key_pages is grown.key_pages
    keys, values = ops.materialize_reference_dense_kv(grown)
    assert torch.equal(keys[0, :, 20:22].transpose(0, 1), rows[0][:2]) and torch.equal(values[1, :, 11], rows[1][2])
    separate = dataclasses.replace(built, reference_key_pages=built.key_pages.clone(), reference_value_pages=built.value_pages.clone())
    assert ops.paged_kv_append(*rows, separate, append_lens=torch.tensor([2, 1])).reference_key_pages is None
