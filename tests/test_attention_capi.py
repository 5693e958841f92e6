"""Refusals of the attention operators' C entry points that are made before anything is launched: no GPU needed."""
import ctypes

import pytest

from mslk_amd import _lib

SOMEWHERE = 1 << 20   # a pointer that is not followed


def rows(d, stride):
    return ctypes.byref(_lib.Heads(SOMEWHERE, stride, d))


def decode(sequences, hq, hkv, d, table_width, page_size):
    strides = (ctypes.c_int64 * 3)(0, 0, 0)
    cache = _lib.PagedCache(SOMEWHERE, SOMEWHERE, None, None, strides, strides, strides, strides, 1, page_size, SOMEWHERE, table_width, 0, SOMEWHERE, 0)
    rc = _lib.lib().mslk_amd_attention_decode(rows(d, hq * d), 0, sequences, hq, hkv, d, ctypes.byref(cache), 1.0, SOMEWHERE, SOMEWHERE, None, 0, None)
    return rc, _lib.lib().mslk_amd_last_error().decode()


@pytest.mark.parametrize("sequences,hkv,table_width,page_size", [
    (1, 1, (1 << 20) + 1, 1 << 10), (1, 1, 3, 1 << 29),      # a key more than 2^30, keys beyond it were dropped
    (2048, 1, 1 << 29, 1 << 29), (65535, 8, 1 << 29, 1 << 29)])   # the number of tiles passes 2^64
def test_decode_refuses_more_room_than_keys_are_counted_for(sequences, hkv, table_width, page_size):
    rc, text = decode(sequences, hkv, hkv, 8, table_width, page_size)
    assert rc != 0 and "2^30 keys" in text
    assert _lib.lib().mslk_amd_attention_decode_workspace_bytes(sequences, hkv, hkv, 8, table_width, page_size) == 0


def test_decode_refuses_more_tiles_than_it_counts():
    rc, text = decode(65535, 64, 64, 8, 1 << 20, 1 << 10)
    assert rc != 0 and "2^31 tiles" in text


def test_decode_accepts_room_for_2_to_the_30_keys():
    rc, text = decode(1, 1, 1, 8, 1 << 20, 1 << 10)
    assert rc != 0 and "workspace" in text   # what it asks for next
