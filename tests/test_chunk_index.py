"""The chunk operators' index arithmetic at the limits of what they accept, on
the CPU (tests/cpp/chunk_index.cpp, compiled so that a sum or product that
leaves its type wraps, as it does on the GPU)."""
import ctypes as C
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
