"""The rule by which the native FP8 products take scales as rows (host/row_strides.h), on
the CPU: what it takes lies where its two strides say, and it takes all that can."""

from __future__ import annotations

import ctypes
import itertools
import os
import subprocess

import pytest
import torch

HOST = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "mxfp4-gfx936_amd", "host")
SOURCE = """
#include "row_strides.h"
extern "C" int row_strides(const int64_t* sizes, const int64_t* strides, int64_t dims,
                           int64_t* out) {
  mx::RowStrides r;
  if (!r.read(sizes, strides, dims)) return 0;
  out[0] = r.row, out[1] = r.block;
  return 1;
}
"""


@pytest.fixture(scope="module")
def read(tmp_path_factory):
    """(sizes, strides) -> (row, block) or None"""
    at = tmp_path_factory.mktemp("row_strides")
    (at / "rule.cpp").write_text(SOURCE)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-fPIC", "-shared", f"-I{HOST}",
                    str(at / "rule.cpp"), "-o", str(at / "rule.so")], check=True)
    rule = ctypes.CDLL(str(at / "rule.so")).row_strides

    def call(sizes, strides):
        array, out = ctypes.c_int64 * len(sizes), (ctypes.c_int64 * 2)()
        taken = rule(array(*sizes), array(*strides), ctypes.c_int64(len(sizes)), out)
        return tuple(out) if taken else None

    return call


def offsets(sizes, strides):
    """Where each element lies, as rows of the last dimension."""
    at = [sum(i * s for i, s in zip(index, strides))
          for index in itertools.product(*(range(n) for n in sizes))]
    return [at[i:i + sizes[-1]] for i in range(0, len(at), sizes[-1])]


def check(read, sizes, strides):
    got = read(sizes, strides)
    at = offsets(sizes, strides)
    if got is not None:
        row, block = got
        assert row >= 1 and block >= 1, (sizes, strides)
        assert at == [[i * row + b * block for b in range(sizes[-1])] for i in range(len(at))], (
            sizes, strides, got)
        return
    # a view as rows, and both strides positive: nothing else may be handed on
    t = torch.empty(1).as_strided((1,) * len(sizes), strides).set_(
        torch.empty(4096).untyped_storage(), 0, sizes, strides)
    try:
        v = t.view(-1, sizes[-1])
    except RuntimeError:
        return
    assert (len(at) > 1 and v.stride(0) < 1) or (sizes[-1] > 1 and v.stride(1) < 1), (sizes,
                                                                                      strides)


@pytest.mark.parametrize("dims", [1, 2, 3, 4])
def test_every_small_layout(read, dims):
    for sizes in itertools.product((1, 2, 3), repeat=dims):
        for strides in itertools.product((0, 1, 2, 3, 6), repeat=dims):
            check(read, sizes, strides)


def test_layouts_of_expanded_scales(read):
    # one scale row for all of an inner, a middle or an outer dimension
    for sizes, strides in (((4, 500, 3), (3, 0, 1)), ((500, 4, 3), (0, 3, 1)),
                           ((4, 5, 6, 3), (90, 0, 3, 1)), ((4, 5, 6, 3), (15, 3, 0, 1)),
                           ((4, 5, 6, 3), (0, 18, 3, 1)), ((4, 1, 6, 3), (3, 0, 0, 1)),
                           ((4, 6, 3), (0, 0, 1))):
        assert read(sizes, strides) is None
        check(read, sizes, strides)


def test_plain_layouts_are_taken(read):
    assert read((3,), (1,)) == (1, 1)
    assert read((500, 3), (3, 1)) == (3, 1)
    assert read((500, 3), (1, 500)) == (1, 500)  # the quantizers'
    assert read((4, 5, 3), (5, 1, 20)) == (1, 20)
    assert read((4, 1, 5, 3), (35, 0, 7, 1)) == (7, 1)  # a dimension of 1 has any stride
    assert read((1, 1, 3), (0, 0, 2)) == (1, 2) and read((7, 1), (2, 0)) == (2, 1)
