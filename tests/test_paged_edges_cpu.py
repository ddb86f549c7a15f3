"""More refusals of the paged serving path at the C boundary: no GPU."""
import ctypes

import pytest

P, OTHER = ctypes.c_void_p(4096), ctypes.c_void_p(8192)
I64 = ctypes.c_int64


@pytest.fixture(scope="module")
def lib():
    from sparse_attention_b200_b200 import _lib
    return _lib.lib()


def _refused(lib, rc, word):
    from sparse_attention_b200_b200 import _lib
    assert rc == _lib.ERR_INVALID and word in lib.sparse_b200_last_error(), (rc, lib.sparse_b200_last_error())


@pytest.mark.parametrize("batch,width", [(4096, 1 << 19), (300, 1 << 23), (129, (1 << 24) - 1)])
def test_extend_pages_refuses_more_pages_than_int32(lib, batch, width):
    """The pages of a step are counted in 32 bits (cu_page_offsets)."""
    rc = lib.sparse_b200_extend_pages(P, I64(width), width, P, P, P, 4, P, OTHER, P, P, P, P, P, OTHER, P, batch, 4, 4, None)
    _refused(lib, rc, b"int32")


@pytest.mark.parametrize("pages", [51200, 1 << 26, 1 << 28, (1 << 31) - 1])
def test_select_pages_refuses_more_pages_than_it_holds(lib, pages):
    """Before anything is computed from the size: four lists of 2^28 pages are 2^32 bytes."""
    rc = lib.sparse_b200_select_pages(P, P, P, P, 2, 1, 1, pages, 4, 4, 1, 1, 1, 1, None)
    _refused(lib, rc, b"too many pages")
