"""Building and loading the native parts on machines of another kind than this one."""
import os
import shutil
import subprocess
import sys

import pytest

from conftest import PKG, ROOT


@pytest.fixture
def tree(tmp_path):
    """A copy of the package and its header, built as here but for the module that needs torch."""
    shutil.copytree(PKG, tmp_path / "pkg", ignore=shutil.ignore_patterns("arctic_tensors*", "__pycache__"))
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    return tmp_path


def python(tree, code: str, paths=()) -> subprocess.CompletedProcess:
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=tree,
                          env={**os.environ, "PYTHONPATH": os.pathsep.join([*map(str, paths), str(tree / "pkg")])})


def test_build_without_torch(tree):
    """The library needs none; only the calls on torch tensors are left out, and say so."""
    (tree / "without").mkdir()
    (tree / "without" / "torch.py").write_text("raise ImportError('no torch here')\n")
    r = python(tree, "from arctic_embed_s_int8 import _lib\n"
                     "import os\n"
                     "assert os.path.samefile(_lib.build(), _lib.LIB_PATH)\n"
                     "_lib.lib()\n"
                     "try:\n    _lib.tensors()\nexcept ImportError as e:\n    print(e)\n", [tree / "without"])
    assert r.returncode == 0, r.stderr[-800:]
    assert "no torch here" in r.stdout


def test_module_of_another_torch_is_not_used(tree):
    """A module is built for one torch and one interpreter: after a change of either, make builds another, and one that
    is not there is asked for rather than another loaded."""
    build = "from arctic_embed_s_int8 import _lib; _lib.build(); print(_lib.tensors().__file__)"
    first = python(tree, build)
    assert first.returncode == 0, first.stderr[-800:]
    # the same torch under another version's name
    (tree / "other").mkdir()
    (tree / "other" / "sitecustomize.py").write_text("import torch\ntorch.__version__ += '.other'\n")
    missing = python(tree, "from arctic_embed_s_int8 import _lib; _lib.tensors()", [tree / "other"])
    assert missing.returncode != 0 and "is missing" in missing.stderr
    second = python(tree, build, [tree / "other"])
    assert second.returncode == 0, second.stderr[-800:]
    assert second.stdout != first.stdout
    assert python(tree, build).stdout == first.stdout
