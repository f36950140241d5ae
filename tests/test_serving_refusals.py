"""More of what the batched serving operators' C entries refuse on the host, before anything is launched."""
import ctypes

import pytest

import vtq
from tests import _serving_abi as A
from tests.test_serving_args import append_args, attention_args, refused

ENTRIES = [
    lambda kv: (A.function("vtq_append_kv"), ctypes.byref(append_args(kv)), None),
    lambda kv: (A.function("vtq_attention_paged"), ctypes.byref(attention_args(kv)), None, 0, None)]


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("kv", [dict(pages=0, table=None), dict(pages=0, k=None, v=None, table=None)])
def test_a_cache_without_pages_still_needs_its_table(entry, kv):
    """The kernels read a sequence's row of the table before they find that its page does not exist."""
    fn, *args = entry(kv)
    refused(fn, vtq.ERR_INVALID_ARG, "null cache pointer", *args)


@pytest.mark.parametrize("width,page_size", [(1 << 40, 1 << 24), (1 << 62, 4), (1 << 33, (1 << 31) - 1), ((1 << 30) + 1, 1)])
def test_attention_of_tables_too_wide_to_count(width, page_size):
    """Their positions, counted in 64 bits, would come round to few or none."""
    a = attention_args(dict(table_width=width, page_size=page_size))
    refused(A.function("vtq_attention_paged"), vtq.ERR_NOT_IMPLEMENTED, "positions", ctypes.byref(a), None, 0, None)
