"""Refusals of pointers that are no addresses of their type: a kernel's access to one would be a misaligned address."""
import ctypes

import pytest

from test_products_cpu import BACK, CHECK, FFN, INT8, QUANT, refused


def at(address):
    return ctypes.c_void_p(address)  # never dereferenced: each call fails its checks first


WORK = 1 << 20  # bytes, enough for any copy of these sizes


@pytest.mark.parametrize("kind,place,address", [
    (0, 0, 258), (0, 0, 257), (1, 0, 257), (2, 0, 257), (2, 7, 258), (2, 7, 257),
])
def test_quantize_rows_refuses(kind, place, address, abft):
    args = list(QUANT)
    args[2] = kind
    args[place] = at(address)
    assert refused(abft, "abft_quantize_rows", *args)


@pytest.mark.parametrize("checksum,expect", [(258, 256), (257, 256), (256, 260), (256, 257)])
def test_quantize_rows_refuses_places_of_expected_sums(checksum, expect, abft):
    args = list(QUANT)
    args[8], args[9] = at(checksum), at(expect)
    assert refused(abft, "abft_quantize_rows", *args)


@pytest.mark.parametrize("address", [257, 258])
def test_column_checksum_refuses(address, abft):
    args = list(CHECK)
    args[4] = at(address)
    assert refused(abft, "abft_column_checksum", *args)


@pytest.mark.parametrize("kind,place,address", [(2, 2, 258), (2, 5, 257), (0, 9, 258), (1, 9, 257), (2, 9, 257)])
def test_int8_matmul_refuses(kind, place, address, abft):
    args = list(INT8)
    args[11] = kind
    args[place] = at(address)
    assert refused(abft, "abft_int8_matmul", *args)


@pytest.mark.parametrize("expect,rowdiff", [(260, 256), (256, 260), (256, 257)])
def test_int8_matmul_refuses_places_of_row_sums(expect, rowdiff, abft):
    args = list(INT8)
    args[12], args[13] = at(expect), at(rowdiff)
    assert refused(abft, "abft_int8_matmul", *args)


@pytest.mark.parametrize("place", [0, 2, 4, 11, 13, 15])
@pytest.mark.parametrize("kind", [1, 2])
def test_gated_ffn_refuses(place, kind, abft):
    args = list(FFN)
    args[9] = kind
    args[13], args[14], args[15], args[16] = at(256), 8, at(256), 8
    args[17], args[18] = at(256), WORK
    args[place] = at(257)
    assert refused(abft, "abft_gated_ffn", *args)


@pytest.mark.parametrize("place", [0, 2, 4, 6, 8, 10, 17, 19, 21])
@pytest.mark.parametrize("kind", [1, 2])
def test_gated_ffn_backward_refuses(place, kind, abft):
    args = list(BACK)
    args[15] = kind
    args[place] = at(257)
    assert refused(abft, "abft_gated_ffn_backward", *args)
