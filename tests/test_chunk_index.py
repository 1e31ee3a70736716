"""The chunk operators' index arithmetic at the limits of what they accept, on
the CPU (tests/cpp/chunk_index.cpp, compiled so that a sum or product that
leaves its type wraps, as it does on the GPU)."""
import ctypes as C
import itertools
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("index") / "chunk_index.so")
    subprocess.run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fwrapv", "-fPIC",
                    "-shared", "-I" + os.path.join(ROOT, "kyro_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "chunk_index.cpp"), "-o", so], check=True)
    return C.CDLL(so)


@pytest.mark.parametrize("group", [1, 2, 3, 7, 8, 16, 32, 63, 64, 65, 127, 128])
def test_hidden_columns(index, group):
    """A slot of the context hides no column, however far back it lies; one of
    the chunk hides those of the tokens before its own."""
    limit, tokens = (1 << 30) - 1, 128 // group
    for ctx in (0, 1, 1 << 23, (1 << 25) + 1, 1 << 28, limit - 5):
        for n in (1, 2, 5):
            for t in {0, 1, ctx // 2, max(0, ctx - 300), max(0, ctx - 1), ctx, ctx + n - 1}:
                # the steps that an item with slot t goes through
                step0 = max(0, t // 256 * 256 - ctx) // tokens
                for step in range(step0, -(-n // tokens)):
                    want = max(0, (t - ctx - step * tokens) * group)
                    assert index.hidden_cols(t - ctx, step * tokens, group) == want


LENGTHS = [0, 1, 63, 64, 65, (1 << 30) - 1, (1 << 31) - 1, 1 << 31, (1 << 32) + 20, 1 << 62,
           (1 << 63) - 4, (1 << 63) - 1]
LENGTHS += [-1 - x for x in LENGTHS]


def test_rows_of_a_chunk(index):
    """No length and no starts pass for a chunk that fits if they do not."""
    ends = [-(1 << 31), -1, 0, 3, 12, 13, (1 << 31) - 1]
    for s0, s1, ctx, T, most in itertools.product(ends, ends, LENGTHS, (0, 12, (1 << 31) - 1),
                                                  (1, 64, (1 << 30) - 1)):
        ok = 0 <= s0 <= s1 <= T and (s0 == s1 or 0 <= ctx <= most - (s1 - s0))
        assert index.chunk_rows(s0, s1, C.c_int64(ctx), T, most) == (s1 - s0 if ok else -1)


def test_lengths_that_can_be_cut(index):
    for n, more, table, width in itertools.product(LENGTHS, (0, 1, 1000), (16, 1 << 29),
                                                   (1, 64, 1 << 40)):
        assert (index.evict_fits(C.c_int64(n), more, C.c_int64(table), C.c_int64(width)) != 0) == (
            n + more <= table and n <= width)
