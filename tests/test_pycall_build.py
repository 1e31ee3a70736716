"""The extension module of the chunk operators' Python calls is used by the
Python and the torch it was built with, and by no other: it reads tensors by
their layout in memory."""
import os

import pytest
import torch


@pytest.fixture(scope="module", autouse=True)
def built():
    from kyro_b200 import build
    build.build()


def _loaded(monkeypatch):
    """What a fresh process would load."""
    from kyro_b200 import _lib
    monkeypatch.setattr(_lib, "_calls", None)
    try:
        return _lib.calls()
    except ImportError:
        return None


def test_the_module_is_the_one_of_this_torch(monkeypatch):
    from kyro_b200 import build
    m = _loaded(monkeypatch)
    assert os.path.samefile(m.__file__, build.pycall_path(torch.__version__))
    assert m.chunk_attention


def test_a_module_of_another_torch_is_not_loaded(monkeypatch):
    monkeypatch.setattr(torch, "__version__", "2.12.1+cu999")
    assert _loaded(monkeypatch) is None


def test_a_module_of_another_python_is_not_loaded(monkeypatch):
    import sysconfig
    monkeypatch.setitem(sysconfig.get_config_vars(), "EXT_SUFFIX",
                        ".cpython-399-x86_64-linux-gnu.so")
    assert _loaded(monkeypatch) is None


def test_a_change_of_torch_builds_the_module_anew(monkeypatch, tmp_path):
    """(the compiler's stand-in writes the file it is asked for)"""
    from kyro_b200 import build
    fake = tmp_path / "cxx"
    fake.write_text("#!/bin/sh\nwhile [ \"$1\" != -o ]; do shift; done\necho built > \"$2\"\n")
    fake.chmod(0o755)
    monkeypatch.setenv("CXX", str(fake))
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    there = build.pycall_path(torch.__version__)
    build._build_pycall(False, False)
    assert set(os.listdir(tmp_path)) == {"cxx", os.path.basename(there)}
    stamp = os.stat(there).st_mtime_ns
    build._build_pycall(False, False)
    assert os.stat(there).st_mtime_ns == stamp  # up to date
    monkeypatch.setattr(build.runpy, "run_path", lambda path: {"__version__": "9.9"})
    build._build_pycall(False, False)
    assert os.path.exists(build.pycall_path("9.9"))


@pytest.mark.parametrize("cxx", ["/nonexistent/c++", "false"])
def test_the_library_builds_without_a_host_compiler(monkeypatch, tmp_path, capfd, cxx):
    from kyro_b200 import build
    monkeypatch.setenv("CXX", cxx)
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    old = build.pycall_path(torch.__version__)
    open(old, "w").close()
    os.utime(old, (0, 0))
    assert build.build() == build.LIB
    assert "ctypes" in capfd.readouterr().err
    assert not os.path.exists(old)  # no module rather than an old one


def test_calls_without_the_module(monkeypatch, tmp_path):
    from kyro_b200 import _lib, build
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(_lib, "_calls", None)
    with pytest.warns(RuntimeWarning, match="kyro_b200.build"):
        assert _lib.calls() is None
    with open(build.pycall_path(torch.__version__), "w") as f:
        f.write("not a module")
    with pytest.warns(RuntimeWarning, match="kyro_b200.build"):
        assert _lib.calls() is None


@pytest.mark.gpu
def test_a_context_without_the_module(monkeypatch, tmp_path):
    """The same results, and the framework's other operators as before."""
    import chunk_ref as R
    from kyro_b200 import _lib, build
    from kyro_b200.verify import (Context, chunk_attention, kv_evict, kv_scores_add,
                                  qk_norm_rope_kv_write, verify_attention)
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    monkeypatch.setattr(build, "HERE", str(tmp_path))

    def steps(ctx):
        x = R.Batch(ctx.device, [7, 7], [90, 40], 8, 2, 128, seed=3)
        x.k_cache.nan_to_num_()
        x.v_cache.nan_to_num_()
        q = qk_norm_rope_kv_write(ctx, x.q, x.k_new, x.v_new, x.chunk_starts, x.block_table,
                                  x.context_lens, x.k_cache, x.v_cache, 16)
        lse = torch.empty(x.T, x.hq, device=ctx.device)
        out = chunk_attention(ctx, q, x.k_cache, x.v_cache, x.chunk_starts, x.block_table,
                              x.context_lens, lse=lse)
        scores = torch.zeros(2, 2, x.block_table.shape[1] * 16, device=ctx.device)
        kv_scores_add(ctx, q, x.k_cache, lse, x.chunk_starts, x.block_table, x.context_lens,
                      scores)
        other = verify_attention(ctx, q.view(2, 7, 8, 128), x.k_cache, x.v_cache, x.block_table,
                                 x.context_lens)
        free = torch.zeros(x.nb, dtype=torch.int32, device=ctx.device)
        free[:x.nb - x.used] = torch.from_numpy(x.perm[x.used:]).int()
        top = torch.full((1,), x.nb - x.used, dtype=torch.int32, device=ctx.device)
        refs = torch.ones(x.nb, dtype=torch.int32, device=ctx.device)
        x.context_lens += 7
        gone = kv_evict(ctx, 32, 2, 8, [scores], [x.k_cache], [x.v_cache], x.block_table,
                        x.context_lens, free, top, refs, 16)
        assert ctx.device_status() == 0
        return [q, lse, out, scores, other, gone, x.k_cache, x.v_cache, x.block_table, free, top]

    want = steps(Context(0))
    monkeypatch.setattr(_lib, "_calls", None)
    with pytest.warns(RuntimeWarning):
        ctx = Context(0)
    assert ctx._calls is None
    for a, b in zip(want, steps(ctx)):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
