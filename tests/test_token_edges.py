"""Rows that start between vector boundaries: which vectors the kernels of gn_rms.cu read as a whole, on the host.  The rule itself
is compiled from csrc/gn_rows.h; the vectors are those of Frame (gn_rms.cu): vector i of a row holds its elements i * VE - skew and on."""
import ctypes
import os
import subprocess

import pytest

from channels_last_groupnorm_b200 import build


@pytest.fixture(scope="module")
def edge_rows(tmp_path_factory):
    folder = tmp_path_factory.mktemp("rows")
    source, lib = folder / "rows.cpp", folder / "rows.so"
    source.write_text('#include "gn_rows.h"\nextern "C" int edge_rows(int w, int64_t s) { return gnb200::edge_rows(w, s); }\n')
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", build.CSRC, str(source), "-o", str(lib)])
    fn = ctypes.CDLL(os.fspath(lib)).edge_rows
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_int, ctypes.c_int64]
    return fn


def reads_outside(width, c, rows, stride, skew, edge):
    """(row, vector) pairs that are read as a whole although an element of theirs lies outside of the tensor"""
    first = min(0, (rows - 1) * stride)
    last = max(0, (rows - 1) * stride) + c  # one past
    found = []
    for row in range(rows):
        inner = edge <= row < rows - edge
        for i in range((c + skew + width - 1) // width):
            begin, end = i * width - skew, (i + 1) * width - skew
            if inner or (begin >= 0 and end <= c):
                if row * stride + begin < first or row * stride + end > last:
                    found.append((row, i))
    return found


@pytest.mark.parametrize("width", [4, 8])
def test_no_vector_reaches_out_of_the_tensor(edge_rows, width):
    some = 0
    for c in range(1, 2 * width + 2):
        for stride in {c + k * width for k in range(-3, 3)} - {0}:  # (rows at a distance of 0 go element by element)
            for rows in (1, 2, 3, 4, 9, 20):
                edge = edge_rows(width, stride)
                for skew in range(width):
                    assert not reads_outside(width, c, rows, stride, skew, edge), (c, stride, rows, skew)
                    some += bool(reads_outside(width, c, rows, stride, skew, 1))
    assert some  # (one row at either end alone does not do)


@pytest.mark.parametrize("width", [4, 8])
def test_longer_rows_have_one_edge_row(edge_rows, width):
    for stride in (width - 1, width, 999, 1 << 40, -999):
        assert edge_rows(width, stride) == 1
