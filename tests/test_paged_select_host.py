"""Host checks of the page selection's C entry, with made-up pointers."""
import ctypes

import pytest
import torch

import _native

I = ctypes.c_int64


class PageList(ctypes.Structure):
    _fields_ = [("pages", ctypes.c_void_p), ("heads", ctypes.c_void_p), ("counts", ctypes.c_void_p), ("capacity", I)]


@pytest.fixture(scope="module")
def lib():
    lib = _native.c_library()
    lib.popkv_last_error.restype = ctypes.c_char_p
    lib.popkv_paged_select_workspace_bytes.restype = ctypes.c_size_t
    return lib


def select(lib, workspace=4096, batch=1, q_heads=4, kv_heads=2, page_size=16, budget=2, width=64, capacity=64, ws_bytes=None,
           scores=256, pages=256):
    need = lib.popkv_paged_select_workspace_bytes(I(batch), I(q_heads), I(width)) if ws_bytes is None else ws_bytes
    pl = PageList(pages, 256, 256, capacity)
    return lib.popkv_paged_select(ctypes.c_void_p(scores), I(width), ctypes.c_void_p(256), I(batch), I(q_heads), I(kv_heads),
                                  I(page_size), I(budget), ctypes.byref(pl), ctypes.c_void_p(workspace), ctypes.c_size_t(need), None)


@pytest.mark.parametrize("offset", [1, 2, 3, 4, 8, 15])
def test_workspace_needs_16_byte_alignment(lib, offset):
    assert select(lib, workspace=4096 + offset) == 4, lib.popkv_last_error()
    assert b"align" in lib.popkv_last_error()


def test_arguments_are_checked(lib):
    assert select(lib, budget=0) == 1
    assert select(lib, q_heads=3) == 1
    assert select(lib, page_size=0) == 1
    assert select(lib, width=-1) == 1
    assert select(lib, q_heads=66) == 3          # 33 query heads per KV head
    assert select(lib, scores=None) == 1
    assert select(lib, pages=None) == 1
    assert select(lib, capacity=3) == 2          # a group of two may list four pages
    assert select(lib, ws_bytes=64) == 6
    assert select(lib, batch=0) == 0



@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up: nothing may be launched with them")
def test_lists_without_room_need_no_arrays(lib):
    """A block table without columns: nothing is listed, so there is nothing to point to."""
    assert select(lib, width=0, capacity=0, scores=None, pages=None, ws_bytes=1 << 20) == 5, lib.popkv_last_error()  # no GPU
    assert select(lib, width=0, capacity=1, scores=None, pages=None, ws_bytes=1 << 20) == 1
