"""What the C ABI of the page decode says of a call's workspace before there is a device."""

from __future__ import annotations

import ctypes

from fast_kernels import page_decode_capi as pdc


def test_the_need_of_a_call_is_checked_like_the_call() -> None:
    lib, args, need = pdc.load_library(), pdc.PageDecodeArgs(), ctypes.c_size_t(1)
    assert lib.fk_page_decode_workspace_need(None, ctypes.byref(need)) == pdc.ERR_INVALID_ARGUMENT
    assert lib.fk_page_decode_workspace_need(ctypes.byref(args), None) == pdc.ERR_INVALID_ARGUMENT
    assert "NULL" in lib.fk_page_decode_last_error().decode()
    assert lib.fk_page_decode_workspace_need(ctypes.byref(args), ctypes.byref(need)) == pdc.ERR_INVALID_ARGUMENT
    assert "empty inputs" in lib.fk_page_decode_last_error().decode()
