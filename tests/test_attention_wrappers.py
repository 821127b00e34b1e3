"""What the Python side of the attention entry points hands over and refuses (no GPU)."""
import ctypes

import pytest
import torch

from gewell_b200 import _lib

P = 1 << 20          # an aligned address


def sequence_batch(table, rows=2, max_rows=1, count=2):
    import gewell_b200 as gw
    offsets, lengths = torch.arange(count + 1, dtype=torch.int32), torch.ones(count, dtype=torch.int32)
    return gw.SequenceBatch(offsets, lengths, table, rows, max_rows)


def test_a_view_of_a_page_table_has_its_own_entries():
    wide = torch.zeros((2, 12), dtype=torch.int32)
    for view, stride, entries in ((wide, 12, 12), (wide[:, :5], 12, 5), (wide[:, 4:9], 12, 5), (wide[:1], 12, 12), (wide[1:, 3:4], 1, 1)):
        held = sequence_batch(view, count=view.shape[0])._struct
        assert (held.page_table, held.page_table_stride, held.page_table_entries) == (view.data_ptr(), stride, entries)
    assert sequence_batch(wide[:, 3:3])._struct.page_table is None                    # no entries: no table


def test_more_entries_than_a_stride_are_refused():
    lib = _lib.load()
    heads = _lib.HeadRows(input=P, input_stride=1024, output=P, output_stride=1024, heads=4)
    cache = _lib.KvCache(P, P, P, P, 8, 4, 16, 256)
    batch = _lib.Sequences(P, P, P, 4, 2, 6, 3, 5)
    status = lib.gw_kv_cache_append(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(heads), ctypes.byref(heads), None, None, None, 1e-6, None)
    assert status == _lib.GW_INVALID_ARGUMENT and b"entries" in lib.gw_last_error()
    status = lib.gw_paged_attention_bf16(ctypes.byref(cache), ctypes.byref(batch), P, 2048, 8, 0.1, 0, P, 2048, P, 1 << 40, None)
    assert status == _lib.GW_INVALID_ARGUMENT and b"entries" in lib.gw_last_error()


@pytest.mark.parametrize("rows,max_rows", [(-1, 1), (2, -1), ((1 << 32) + 2, 1), (2, (1 << 32) + 1), (1 << 40, 1)])
def test_row_counts_that_32_bits_do_not_hold_are_refused(rows, max_rows):
    import gewell_b200 as gw
    with pytest.raises(gw.GewellInvalidArgument):
        sequence_batch(torch.zeros((2, 4), dtype=torch.int32), rows, max_rows)


def test_strides_that_32_bits_do_not_hold_are_refused():
    """A page table 2^32 + 4 entries apart (of the meta device: no memory)."""
    import gewell_b200 as gw
    far = torch.empty_strided((2, 4), ((1 << 32) + 4, 1), dtype=torch.int32, device="meta")
    offsets, lengths = torch.zeros(3, dtype=torch.int32, device="meta"), torch.zeros(2, dtype=torch.int32, device="meta")
    with pytest.raises(gw.GewellInvalidArgument):
        gw.SequenceBatch(offsets, lengths, far, 2, 1)


def test_a_single_element_has_no_stride():
    """Views of one element of something wider are as good as any other."""
    import gewell_b200 as gw
    i32, wide = torch.int32, torch.arange(12, dtype=torch.int32).reshape(3, 4)
    offsets = torch.zeros(4, dtype=i32)
    held = gw.SequenceBatch(offsets, torch.ones(3, dtype=i32), wide[:, 1:2], 3, 1)._struct
    assert (held.page_table_stride, held.page_table_entries) == (4, 1)
    gw.SequenceBatch(offsets, torch.ones(3, dtype=i32), torch.empty_strided((3, 1), (1, 0), dtype=i32), 3, 1)
    gw.SequenceBatch(offsets[:2], torch.ones(8, dtype=i32)[::8], wide[:1], 1, 1)
    for bad in (wide.t(), wide[:, ::2]):
        with pytest.raises(gw.GewellInvalidArgument):
            gw.SequenceBatch(offsets, torch.ones(3, dtype=i32), bad[:3], 3, 1)
