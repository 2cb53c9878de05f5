"""The torch binding is rebuilt for another torch or Python, and a binding that
cannot be loaded is reported with what to do about it."""
import importlib.metadata
import os
import shutil
import subprocess
import sys

import pytest

from qwen600_engine_b200 import build

HERE = os.path.dirname(os.path.abspath(build.__file__))


def test_binding_is_tied_to_its_torch(monkeypatch, tmp_path):
    so = tmp_path / "_torch.so"
    so.write_bytes(b"")
    monkeypatch.setattr(build, "BINDING", str(so))
    monkeypatch.setattr(build, "BINDING_MADE_FOR", str(tmp_path / "made_for"))
    made = []

    def compiled(cmd, **kw):
        made.append(cmd)
        so.write_bytes(b"")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", compiled)
    os.utime(so, (2 ** 32, 2 ** 32))  # newer than its sources, but made for nothing that is known
    for calls in (1, 1):
        build.build_binding()
        os.utime(so, (2 ** 32, 2 ** 32))
        assert len(made) == calls
    version = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0.1" if name == "torch" else version(name))
    for calls in (2, 2):
        build.build_binding()
        os.utime(so, (2 ** 32, 2 ** 32))
        assert len(made) == calls


@pytest.mark.parametrize("module", ["w4", "losses"])
def test_a_binding_that_does_not_load_is_reported(module, tmp_path):
    package = tmp_path / "qwen600_engine_b200"
    package.mkdir()
    for f in os.listdir(HERE):
        if f.endswith(".py"):
            shutil.copy(os.path.join(HERE, f), package)
    os.symlink(build.LIB, package / os.path.basename(build.LIB))
    (package / "_torch.so").write_bytes(b"not a library")
    r = subprocess.run([sys.executable, "-c", f"import qwen600_engine_b200.{module}"], cwd=tmp_path, capture_output=True, text=True)
    assert r.returncode != 0 and "python -m qwen600_engine_b200.build" in r.stderr, r.stderr
