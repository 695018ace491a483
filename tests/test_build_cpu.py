"""The build of the Python helpers' extension module follows the torch that is installed, or skips it."""

import os
import stat
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "thunderkittens-sm7x_b200")


def executable(path, text):
    path.write_text(text)
    path.chmod(path.stat().st_mode | stat.S_IXUSR)
    return str(path)


@pytest.mark.parametrize("abi", [0, 1])
def test_extension_is_built_for_the_installed_torch(tmp_path, abi):
    """A torch of either C++ ABI: the compiler is told which (it only writes down its arguments here)."""
    (tmp_path / "torch").mkdir()
    (tmp_path / "torch" / "__init__.py").write_text(f"def compiled_with_cxx11_abi():\n    return {bool(abi)}\n")
    cxx = executable(tmp_path / "cxx", f'#!/bin/sh\nprintf "%s\\n" "$@" > {tmp_path}/args\n')
    out = str(tmp_path / "_ops.so")
    env = {**os.environ, "PYTHONPATH": str(tmp_path)}
    subprocess.run(["make", "-s", "-C", PKG, f"OPS={out}", f"CXX={cxx}", f"PYTHON={sys.executable}", "-o", os.path.join(PKG, "tk_b200", "libtk_b200.so"),
                    out], check=True, env=env)
    args = (tmp_path / "args").read_text().split("\n")
    assert f"-D_GLIBCXX_USE_CXX11_ABI={abi}" in args
    assert f"-I{tmp_path}/torch/include" in args


def test_build_without_torch():
    """The library alone is a build: nothing of it needs torch."""
    code = ("import subprocess, sys\n"
            "sys.modules['torch'] = None\n"
            "sys.path.insert(0, %r)\n"
            "import __graft_entry__ as g, oracle\n"
            "subprocess.run = lambda *a, **k: None\n"
            "g.build()\n" % ROOT)
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT)
