"""Pages of 8 bits are written in words and f32 scales: appends refuse pages that are not aligned, as attention, read and keep do, on the CPU."""
import ctypes as C

import pytest

from test_candidates_checks import q8
from test_paged_checks import P, batch, refused


@pytest.mark.parametrize("off", [1, 2, 4, 8])
def test_appends_refuse_pages_that_are_not_aligned(qa, off):
    lib, lay, b = qa.lib, q8(qa), batch(qa)
    refused(qa, lib.qa_paged_append(P, P, P, P, P + off, C.byref(lay), 0, C.byref(b), 16, 1e6, 1e-6, None), "aligned")
    refused(qa, lib.qa_paged_tree_append(P, P, P, P, P + off, C.byref(lay), 0, C.byref(b), P, 16, 1e6, 1e-6, None), "aligned")
    # without rows there is nothing to write
    none = batch(qa, n_rows=0)
    assert lib.qa_paged_append(P, P, P, P, P + off, C.byref(lay), 0, C.byref(none), 16, 1e6, 1e-6, None) == qa.QA_OK
