"""Which bytes of a table of scales a tile of the 8-bit product reads (ocr_amd/csrc/scale_window.h, compiled for the host)."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'ocr_amd', 'csrc')


@pytest.fixture(scope='module')
def window(tmp_path_factory):
    folder = tmp_path_factory.mktemp('scale_window')
    src, lib = str(folder / 'w.cpp'), str(folder / 'w.so')
    with open(src, 'w') as f:
        f.write('#include "scale_window.h"\n'
                'extern "C" int64_t window(int64_t tile, int64_t rows, int64_t first) { return ocrhip::scale_window(tile, rows, first); }\n')
    subprocess.run(['g++', '-std=c++17', '-O1', '-Wall', '-Werror', '-shared', '-fPIC', '-I', CSRC, '-o', lib, src], check=True)
    f = ctypes.CDLL(lib).window
    f.argtypes, f.restype = [ctypes.c_int64] * 3, ctypes.c_int64
    return f


@pytest.mark.parametrize('tile', [128, 256])
def test_a_tile_reads_its_rows_scales_and_nothing_behind_the_table(window, tile):
    """A table of `rows` scales as the last columns of a wider buffer: it starts on 16 bytes and the buffer's rows are a multiple
    of 16 long, so round_up(rows, 16) bytes from its start are there, in the last row too, and no more."""
    for rows in list(range(1, 600)) + [16384, 79873, (1 << 24) + 300, (1 << 31) - 1]:
        for first in sorted({0, rows // tile // 2 * tile, (rows - 1) // tile * tile}):
            n = window(tile, rows, first)
            assert n % 4 == 0 and min(tile, rows - first) <= n <= tile      # whole loads, every row that exists
            assert first + n <= -(-rows // 16) * 16


def test_the_last_columns_of_a_wider_table(window):
    """65 rows in the last 80 of 1024 columns: 128 bytes from the start would end 48 behind the buffer."""
    assert window(128, 65, 0) == 68
