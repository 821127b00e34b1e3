"""What the attention entry points refuse, before any CUDA call (no GPU: the pointers are never followed)."""
import ctypes

import pytest
import torch

from gewell_b200 import _lib

P = 1 << 20          # an aligned address


def lib():
    return _lib.load()


def heads(**changes):
    h = dict(input=P, input_stride=1024, output=2 * P, output_stride=1024, weight=0, heads=4, normalize=1)
    return _lib.HeadRows(**{**h, **changes})


def cache(**changes):
    c = dict(k_data=P, v_data=P, k_scales=P, v_scales=P, pages=8, kv_heads=4, page_tokens=16, head_dim=256)
    return _lib.KvCache(**{**c, **changes})


def batch(**changes):
    b = dict(row_offsets=P, context_lengths=P, page_table=P, page_table_stride=4, sequences=2, rows=6, max_rows=3)
    return _lib.Sequences(**{**b, **changes})


def refused(status, text):
    assert status == _lib.GW_INVALID_ARGUMENT
    assert text in lib().gw_last_error().decode(), lib().gw_last_error()


def norm(query, key=None, rows=3, width=256, positions=P, rotary=None, epsilon=1e-6):
    return lib().gw_qk_norm_rotary_bf16(query and ctypes.byref(query), key and ctypes.byref(key), rows, width, positions,
                                        rotary and ctypes.byref(rotary), epsilon, None)


def test_norm_rotary_refusals():
    assert norm(None, rows=0) == _lib.GW_OK
    refused(norm(None), "heads")
    for width in (0, 7, 12, 264, 520, 1024):
        refused(norm(heads(), width=width), "head width")
    for bad in (dict(input=0), dict(input=P + 2), dict(heads=0), dict(heads=2000), dict(weight=P + 4)):
        refused(norm(heads(**bad)), "aligned inputs")
    for bad in (dict(input_stride=1020), dict(input_stride=1016)):
        refused(norm(heads(**bad)), "row strides")
    for bad in (dict(output=0), dict(output=P + 8), dict(output_stride=1023), dict(output=P, output_stride=2048)):
        refused(norm(heads(**bad)), "output")
    refused(norm(heads(), heads(input_stride=8)), "row strides")
    turn = dict(inverse_frequencies=P, width=256, interleaved=0)
    for bad in (dict(inverse_frequencies=0), dict(width=258), dict(width=31)):
        refused(norm(heads(), rotary=_lib.Rotary(**{**turn, **bad})), "rotated width")
    refused(norm(heads(), positions=None, rotary=_lib.Rotary(**turn)), "positions")
    for epsilon in (-1.0, float("nan")):
        refused(norm(heads(), epsilon=epsilon), "epsilon")
    refused(norm(heads(), rows=1 << 25), "rows")


BAD_CACHES = [dict(k_data=0), dict(v_data=P + 8), dict(k_scales=0), dict(page_tokens=0), dict(page_tokens=48), dict(page_tokens=256),
              dict(head_dim=64), dict(head_dim=192), dict(pages=0), dict(kv_heads=0), dict(pages=1 << 27), dict(kv_heads=2048)]
BAD_BATCHES = [dict(row_offsets=0), dict(context_lengths=0), dict(page_table=0), dict(page_table_stride=0), dict(max_rows=0), dict(max_rows=7),
               dict(rows=1 << 25, max_rows=1), dict(sequences=1 << 21)]


def append(c=None, b=None, key=None, value=None, query=None, rotary=None, epsilon=1e-6):
    return lib().gw_kv_cache_append(ctypes.byref(c or cache()), ctypes.byref(b or batch()), ctypes.byref(key or heads()),
                                    ctypes.byref(value or heads()), query and ctypes.byref(query), None, rotary and ctypes.byref(rotary), epsilon, None)


def test_append_refusals():
    for bad in BAD_CACHES:
        assert append(c=cache(**bad)) == _lib.GW_INVALID_ARGUMENT, bad
    for bad in BAD_BATCHES:
        assert append(b=batch(**bad)) == _lib.GW_INVALID_ARGUMENT, bad
    assert append(b=batch(rows=0, max_rows=0)) == _lib.GW_OK and append(b=batch(sequences=0)) == _lib.GW_OK
    refused(append(key=heads(heads=3)), "heads")
    refused(append(value=heads(heads=2)), "heads")
    refused(append(key=heads(input=P + 2)), "aligned")
    refused(append(query=heads(output=0)), "output")
    refused(append(rotary=_lib.Rotary(P, 300, 0)), "rotated width")
    refused(append(epsilon=-1.0), "epsilon")


def attend(c=None, b=None, q=P, q_stride=2048, h=8, scale=0.1, y=P, y_stride=2048, scratch=P, capacity=1 << 40):
    return lib().gw_paged_attention_bf16(ctypes.byref(c or cache()), ctypes.byref(b or batch()), q, q_stride, h, scale, 0, y, y_stride, scratch,
                                         capacity, None)


def test_attention_refusals():
    for bad in BAD_CACHES:
        assert attend(c=cache(**bad)) == _lib.GW_INVALID_ARGUMENT, bad
    for bad in BAD_BATCHES:
        assert attend(b=batch(**bad)) == _lib.GW_INVALID_ARGUMENT, bad
    assert attend(b=batch(rows=0, max_rows=0)) == _lib.GW_OK
    for h in (0, 3, 6, 260):
        refused(attend(h=h), "query heads")
    for bad in (dict(q=0), dict(q=P + 2), dict(q_stride=2052), dict(q_stride=1024), dict(y=0), dict(y=P + 8), dict(y_stride=8)):
        refused(attend(**bad), "aligned")
    for scale in (float("nan"), float("inf")):
        refused(attend(scale=scale), "finite")
    needed = lib().gw_paged_attention_scratch_bytes(ctypes.byref(cache()), ctypes.byref(batch()), 8)
    assert needed >= 256
    for bad in (dict(scratch=0), dict(scratch=P + 16), dict(capacity=needed - 1)):
        refused(attend(**bad), "scratch")


def test_python_wrappers_refuse():
    import gewell_b200 as gw
    codes, scales = torch.zeros((2, 1, 16, 128), dtype=torch.uint8), torch.ones((2, 1))
    for bad in ((codes.float(), codes, scales, scales), (codes[:, :, ::2], codes, scales, scales), (codes, codes, scales.double(), scales),
                (codes, codes[:1], scales, scales[:1]), (codes, codes, scales[:1], scales)):
        with pytest.raises(gw.GewellInvalidArgument):
            gw.KvCache(*bad)
    i32 = torch.int32
    offsets, lengths, table = torch.tensor([0, 1], dtype=i32), torch.tensor([1], dtype=i32), torch.zeros((1, 4), dtype=i32)
    for bad in ((offsets.long(), lengths, table), (offsets[:1], lengths, table), (offsets, lengths, table[0]), (offsets, lengths, table.long())):
        with pytest.raises(gw.GewellInvalidArgument):
            gw.SequenceBatch(*bad, 1, 1)
    held, b = gw.KvCache(codes, codes.clone(), scales, scales.clone()), gw.SequenceBatch(offsets, lengths, table, 1, 1)
    x = torch.zeros((1, 1, 128), dtype=torch.bfloat16)
    if not torch.cuda.is_available():
        for call in (lambda: gw.kv_cache_append(held, b, x, x), lambda: gw.paged_attention(held, b, x, 1.0),
                     lambda: gw.qk_norm_rotary(x, None, None, None, torch.zeros(1, dtype=i32), None)):
            with pytest.raises((gw.GewellInvalidArgument, RuntimeError, AssertionError)):
                call()
