"""8-bit pages whose value scales are all next to nothing, or as large as they can be."""

from __future__ import annotations

import pytest
from test_gpu_paged_kv_blocks import _assert_means, _cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["fp8_kv", "int8_kv"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", [1e-30, 3e-29, 1e-28, 1e-24, 1e-20, 1e-6, 1e20, 1e30])
def test_value_scales_of_any_size(layout, dim, scale) -> None:
    """All tokens have one scale, keys are 0, nothing cancels: the row is rounded to bf16 (2^-8), weights to fp16 (2^-11: at 1e-30
    the heaviest is 2^7 * 1e-6, still a normal number), values times 2^7 exactly; fp32 sums add less than 2^-12."""
    cache = _cache(layout, dim=dim)
    cache.value_scales.fill_(scale)
    _assert_means(cache, 2.0**-8 + 2.0**-11 + 2.0**-12)
