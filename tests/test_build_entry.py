"""build() in a tree without built files: the package is imported before its extension exists."""
import os
import shutil
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_build_in_a_clean_tree(tmp_path):
    """The compilers' part is taken by a copy of the files that are built here already."""
    skip = shutil.ignore_patterns("*.so", "*.o", "__pycache__")
    for name in ("fastgate_b200", "include"):
        shutil.copytree(os.path.join(ROOT, name), tmp_path / name, ignore=skip)
    os.makedirs(tmp_path / "oracle")
    (tmp_path / "oracle" / "__init__.py").write_text("")
    (tmp_path / "oracle" / "oracle.py").write_text("def build():\n    pass\n")
    (tmp_path / "oracle" / "build_ref.py").write_text("def reference_root():\n    return None\n")
    shutil.copy(os.path.join(ROOT, "__graft_entry__.py"), tmp_path)
    code = f"""
import shutil
from fastgate_b200 import build
def build_all(*a, **k):
    for name in ("libfastgate_b200.so", "_C.so"):
        shutil.copy({os.path.join(ROOT, "fastgate_b200")!r} + "/" + name, {str(tmp_path / "fastgate_b200")!r})
build.build_all = build_all
import __graft_entry__
__graft_entry__.build()
import fastgate_b200
assert fastgate_b200.add_rmsnorm and fastgate_b200.__file__.startswith({str(tmp_path)!r})
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=tmp_path, timeout=300)
