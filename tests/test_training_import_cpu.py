"""The package without the training operators' module (CPU): it imports, and
only their names fail; a module built against another torch is built again."""
import os
import subprocess
import sys

import pytest

from tinygnn_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(code):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_package_imports_without_the_training_module():
    run("import sys; sys.modules['tinygnn_b200._torch_ops'] = None\n"
        "import tinygnn_b200 as tg\n"
        "assert tg.version() and tg.spmm and tg.InvalidArgument\n"
        "for name in ('layer_norm', 'training'):\n"
        "    try:\n"
        "        getattr(tg, name)\n"
        "    except ImportError:\n"
        "        continue\n"
        "    raise SystemExit('no ImportError for ' + name)\n")


def test_training_names_are_there_on_first_use():
    run("import sys, tinygnn_b200 as tg\n"
        "assert 'tinygnn_b200._torch_ops' not in sys.modules\n"
        "assert 'layer_norm' in dir(tg) and not hasattr(tg, 'no_such_name')\n"
        "from tinygnn_b200 import typed_linear\n"
        "assert typed_linear is tg.training.typed_linear is tg.typed_linear\n"
        "scope = {}\n"
        "exec('from tinygnn_b200 import *', scope)\n"
        "assert scope['layer_norm'] is tg.layer_norm and scope['spmm'] is tg.spmm\n")


def test_module_built_against_another_torch_is_built_again(tmp_path, monkeypatch):
    stamp = tmp_path / "stamp"
    monkeypatch.setattr(build, "TORCH_STAMP", str(stamp))
    calls = []
    monkeypatch.setattr(build, "_make", lambda args, quiet: calls.append(args))
    build.ensure_built(torchops=True)  # nothing known of it: taken as it is
    assert not calls
    stamp.write_text(build._torch_version())
    build.ensure_built(torchops=True)
    assert not calls
    stamp.write_text("1.0.0")
    build.ensure_built()  # the rest of the package does not ask
    assert not calls
    build.ensure_built(torchops=True)
    assert any("torchops" in a and "-W" in a for a in calls)
    assert stamp.read_text() == build._torch_version()
    calls.clear()
    build.ensure_built(torchops=True)
    assert not calls


def test_no_compiler_is_said(tmp_path, monkeypatch):
    stamp = tmp_path / "stamp"
    stamp.write_text("1.0.0")
    monkeypatch.setattr(build, "TORCH_STAMP", str(stamp))
    monkeypatch.setattr(build, "NVCC", str(tmp_path / "none"))
    monkeypatch.setenv("PATH", str(tmp_path))
    with pytest.raises(ImportError, match="another torch"):
        build.ensure_built(torchops=True)
    assert build.ensure_built() == build.LIB_PATH
