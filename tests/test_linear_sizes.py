"""What the 8-bit linear layer's calls say without a GPU: sizes of packed
weights and workspaces, and refusals of null arguments."""
import ctypes

import pytest

from vectorstorekit_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def weight(outputs, inputs):
    return ctypes.byref(_lib.vsk_int8_weight(None, None, None, outputs, inputs))


@pytest.mark.parametrize("rows,inputs,blocks", [(1, 1, 2), (32, 64, 2), (33, 64, 4), (32, 65, 4),
                                                (100, 131072, 4 * 4096),
                                                (2 ** 31 - 1, 131072, 2 ** 26 * 4096)])
def test_packed_bytes(lib, rows, inputs, blocks):
    """Blocks of 32 rows and 32 places, the places filled up to 64s, 1 KB each."""
    assert lib.vsk_int8_packed_bytes(rows, inputs) == 1024 * blocks


@pytest.mark.parametrize("rows,inputs", [(0, 5), (5, 0), (-1, 5), (5, -1), (5, 131073),
                                         (2 ** 31, 5)])
def test_no_packed_bytes(lib, rows, inputs):
    assert lib.vsk_int8_packed_bytes(rows, inputs) == 0


def test_workspace(lib):
    size = lambda tokens, outputs, inputs: lib.vsk_int8_linear_workspace(weight(outputs, inputs),
                                                                          tokens)
    # codes in blocks, and the scales before them
    assert size(100, 4096, 4096) == 1024 + 4 * 128 * 1024
    assert size(300, 4096, 100) == 2048 + 10 * 4 * 1024
    assert size(2 ** 31 - 1, 1, 131072) == 2 ** 33 + 2 ** 26 * 4096 * 1024
    # few tokens need none
    assert size(1, 4096, 4096) == size(4, 4096, 4096) == size(8, 4096, 2048) == 0
    assert size(8, 4096, 4096) > 0
    # nor do calls that are refused
    assert lib.vsk_int8_linear_workspace(None, 5) == 0
    for bad in ((0, 5, 5), (-1, 5, 5), (2 ** 31, 5, 5), (100, 5, 0), (100, 5, 131073)):
        assert size(*bad) == 0


def test_null_contexts(lib):
    rows = ctypes.byref(_lib.vsk_int8_rows())
    assert lib.vsk_int8_linear(None, None, weight(5, 5), rows) < 0
    assert lib.vsk_int8_pack(None, None, 0, None, 5, weight(5, 5)) < 0
