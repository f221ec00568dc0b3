"""The extension with the decoding operators' direct calls: built where it can be, done without where not (no GPU)."""
import subprocess
import sysconfig

import pytest
import torch

from quipsharp_b200 import _native as N
from quipsharp_b200 import attention
from quipsharp_b200 import build_native


def test_calls_go_by_ctypes_without_it(tmp_path, monkeypatch):
    N.lib()
    monkeypatch.setattr(N, "_fast", None)
    monkeypatch.setattr(N, "_LIB_PATH", str(tmp_path / "libquipsharp_b200.so"))
    q, k = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    table, n = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.warns(RuntimeWarning, match="build_native"), pytest.raises(RuntimeError, match="CUDA tensors only"):
        attention.decode_attention(q, k, k, table, n)
    for name in ("attend", "fork_pages", "compact_pages", "extend_pages", "write_kv", "beam_select"):
        assert getattr(N.fast(), name)(1, 2) is None


@pytest.mark.parametrize("gone", ["compiler", "headers"])
def test_the_library_is_built_without_what_it_needs(gone, tmp_path, monkeypatch, capsys):
    def run(*args, **kw):
        raise AssertionError("nothing to compile with")

    monkeypatch.setattr(subprocess, "run", run)
    monkeypatch.setattr(build_native, "LIBDIR", str(tmp_path))
    if gone == "compiler":
        monkeypatch.setenv("CXX", str(tmp_path / "none"))
    else:
        paths = sysconfig.get_paths()
        monkeypatch.setattr(sysconfig, "get_paths", lambda: {**paths, "include": str(tmp_path)})
    assert build_native.build_fast(False, True) is None
    assert "ctypes" in capsys.readouterr().err


def test_it_is_built_again_for_another_torch(tmp_path, monkeypatch):
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        (tmp_path / "_fast.so").write_bytes(b"")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(subprocess, "run", run)
    monkeypatch.setattr(build_native, "LIBDIR", str(tmp_path))
    monkeypatch.setattr(build_native, "BUILD", str(tmp_path))
    for version, builds in ((torch.__version__, 1), (torch.__version__, 1), ("99.0", 2), ("99.0", 2)):
        monkeypatch.setattr(torch, "__version__", version)
        assert build_native.build_fast(False, False) == str(tmp_path / "_fast.so")
        assert len(calls) == builds
