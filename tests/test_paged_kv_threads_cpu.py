"""Plans of the paged-cache operators in a program with several host threads."""

from __future__ import annotations

import threading
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import torch
from fast_kernels.ops import _paged


def test_threads_that_use_a_plan_first_together_get_tables_that_stay(monkeypatch) -> None:
    """Both find no tables and upload some; the addresses of either must lie in the block that the plan keeps."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    device, kept, both = torch.device("cpu", 0), {}, threading.Barrier(2)  # (an index is all that is asked of the device)

    def host() -> dict:
        both.wait(timeout=30)
        return {"a": np.arange(3), "b": np.arange(4)}

    with ThreadPoolExecutor(2) as pool:
        got = [call.result() for call in [pool.submit(_paged.on_device, kept, device, 0, host) for _ in range(2)]]
    block = kept[0][0]
    begin, end = block.data_ptr(), block.data_ptr() + 4 * block.numel()
    for addresses in got:
        assert all(begin <= address < end for address in addresses.values())
