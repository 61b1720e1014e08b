"""Which of the lookup gradient's ways a call takes, by the workspace that it asks for (no GPU): none where one launch looks
through the tokens for every block of the table's gradient."""

import ctypes

import pytest

from fsctep_amd import _lib


def room(rows, width, table):
    n = ctypes.c_int64()
    assert _lib.load().fsc_embedding_workspace(rows, width, table, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("rows,width,table", [(2048, 12288, 4000), (2048, 12288, 1600), (1024, 12288, 1600), (256, 4096, 30000),
                                              (512, 12288, 4000), (2048, 4096, 1601)])
def test_wide_rows_of_many_blocks_are_sorted(rows, width, table):
    """Looking through the tokens for each block of columns again took up to three and a half times as long."""
    assert room(rows, width, table) > 0


@pytest.mark.parametrize("rows,width,table", [(0, 12288, 4000), (32, 16, 100), (2048, 640, 100), (1024, 640, 5000), (2048, 256, 4096),
                                              (2048, 1024, 4096), (512, 12288, 24), (256, 12288, 100), (2048, 4096, 400)])
def test_the_rest_stays_one_launch(rows, width, table):
    assert room(rows, width, table) == 0


def test_either_type_finds_its_room():
    """16-bit rows have half the blocks of columns: a call of either type fits the room that the sizes alone give."""
    assert room(2048, 2048, 4096) > 0                # fp32 sorts here, bfloat16 does not
    assert room(2048, 2048, 2048) == 0
