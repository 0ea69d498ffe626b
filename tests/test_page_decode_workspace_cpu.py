"""What the C ABI of the page decode says of a call before there is a device: its workspace, its flags."""

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


def test_exact_turns_are_for_rotated_keys() -> None:
    lib, need = pdc.load_library(), ctypes.c_size_t(0)
    args = pdc.PageDecodeArgs(query=256, key_pages=256, value_pages=256, output=256, request_run_offsets=256, seq_lens=256, batch=1,
                              num_q_heads=4, num_kv_heads=2, head_dim=64, page_size=16, softmax_scale=0.1, rope_theta=1e4,
                              flags=pdc.FLAG_EXACT_TURNS)
    assert lib.fk_page_decode_workspace_need(ctypes.byref(args), ctypes.byref(need)) == pdc.ERR_INVALID_ARGUMENT
    assert "exact turns are for keys that are rotated" in lib.fk_page_decode_last_error().decode()
