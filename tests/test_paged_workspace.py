"""The attention's workspace is asked for before the batch is on the device: its size does not depend on the pointers."""
import ctypes as C

import pytest

import paged_ref as ref


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_seqs,n_rows,max_len", [(1, 1, 4000), (32, 32, 3914), (3, 500, 3000), (1, 1024, 3913)])
def test_workspace_of_a_batch_without_pointers(qa, f16, n_seqs, n_rows, max_len):
    lay = ref.layout(qa, 2, 8192, 8, 16, f16)

    def need(*pointers):
        return qa.lib.qa_paged_attn_workspace_bytes(C.byref(lay), C.byref(qa.PagedBatch(*pointers, n_seqs, 300, n_rows, 0, max_len)), 16)

    assert need(None, None, None) == need(4096, 4096, 4096) == need(4096, None, 4096)
    # 1024 tokens on f32 pages are 1024 workgroups in one key range each: nothing to join
    assert (need(None, None, None) > 0) == (f16 or n_rows < 1024)
