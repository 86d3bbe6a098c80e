"""The library and its ctypes binding without PyTorch, and the Python module that belongs to one PyTorch (no GPU)."""

import os
import subprocess
import sys

import pytest
import torch

from lorafusion_b200 import _native as nat
from lorafusion_b200.csrc import build

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

NO_TORCH = """
import sys
class Block:
    def find_spec(self, name, path=None, target=None):
        if name.split(".")[0] == "torch":
            raise ModuleNotFoundError("No module named 'torch'", name="torch")
sys.meta_path.insert(0, Block())
"""


def without_torch(code):
    return subprocess.run([sys.executable, "-c", NO_TORCH + code], cwd=REPO, capture_output=True, text=True, timeout=300)


def test_the_binding_needs_no_torch():
    res = without_torch("from lorafusion_b200 import _native, config, workloads\n"
                        "print(_native.lib().lf_version().decode())\n"
                        "print(len(_native.header_symbols()))")
    assert res.returncode == 0, res.stderr
    assert res.stdout.startswith("lorafusion_b200")


def test_the_library_builds_without_torch(tmp_path):
    """What a build does after the library is linked (nothing is compiled here)."""
    res = without_torch(f"from lorafusion_b200.csrc import build\nbuild.LIB_DIR = {str(tmp_path)!r}\n"
                        "build._build_glue(False, False)")
    assert res.returncode == 0, res.stderr
    assert "no PyTorch" in res.stderr and not os.listdir(tmp_path)


def test_the_python_module_belongs_to_one_torch(monkeypatch, tmp_path):
    """After another PyTorch is installed the old module is neither loaded nor taken for built."""
    here = nat.glue_path()
    assert torch.__version__ in here
    monkeypatch.setattr(torch, "__version__", "99.0+cu999")
    assert nat.glue_path() != here
    monkeypatch.setattr(nat, "_glue", None)
    with pytest.raises(RuntimeError, match="99.0"):
        nat.glue()

    class Stop(Exception):
        pass

    def compile_(cmd, **kw):
        assert os.path.basename(nat.glue_path()) in " ".join(cmd)
        raise Stop

    monkeypatch.setattr(build.subprocess, "run", compile_)
    with pytest.raises(Stop):
        build._build_glue(False, False)
    monkeypatch.undo()
    if os.path.exists(here):
        monkeypatch.setattr(build.subprocess, "run", compile_)
        build._build_glue(False, False)  # built for this one: nothing to do
