"""When the compiled wrappers are rebuilt, and what a failed import of them says."""
import importlib.metadata
import importlib.util
import os
import subprocess
import sys
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("_build_under_test", os.path.join(ROOT, "hipkittensp_b200", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    b.OPS, b.OPS_STAMP, b.calls = str(tmp_path / "ops.so"), str(tmp_path / "stamp"), []

    def run(cmd, **kw):
        b.calls.append(cmd)
        open(b.OPS, "w").close()
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(b, "subprocess", types.SimpleNamespace(run=run))
    return b


def test_wrappers_follow_the_installed_torch(build):
    build.build_torch_ops()
    assert len(build.calls) == 1 and open(build.OPS_STAMP).read() == importlib.metadata.version("torch")
    build.build_torch_ops()
    assert len(build.calls) == 1                                   # up to date
    with open(build.OPS_STAMP, "w") as f:
        f.write("0.0")                                             # built against another torch
    build.build_torch_ops()
    assert len(build.calls) == 2
    os.remove(build.OPS_STAMP)                                     # ... or against one that is not known
    build.build_torch_ops()
    assert len(build.calls) == 3
    build.build_torch_ops(force=True)
    assert len(build.calls) == 4


def test_an_import_that_fails_names_the_build_that_helps():
    code = "import sys; sys.modules['hipkittensp_b200._torch_ops'] = None; import hipkittensp_b200"
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert res.returncode != 0 and "build.py --force" in res.stderr
