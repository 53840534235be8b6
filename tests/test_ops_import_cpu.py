"""The package without the operators' compiled calls, and when those are built again."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _package(to, calls):
    """A package of this one's files: without _calls.so, or with one that does not load."""
    here, there = os.path.join(ROOT, "nmt_gan_amd"), to / "nmt_gan_amd"
    there.mkdir()
    for name in os.listdir(here):
        if name.endswith(".py") or name == "libnmtgan_hip.so":
            os.symlink(os.path.join(here, name), there / name)
    if calls is not None:
        (there / "_calls.so").write_bytes(calls)


@pytest.mark.parametrize("calls", [None, b"built for another torch"])
def test_everything_else_works_without_the_compiled_calls(tmp_path, calls):
    _package(tmp_path, calls)
    code = """
import nmt_gan_amd
from nmt_gan_amd import *
from nmt_gan_amd import _lib, ops as again
assert nmt_gan_amd.__file__.startswith(%r)
assert Model is nmt_gan_amd.Model and DisCNN is nmt_gan_amd.DisCNN and ops is again
assert _lib.lib.nmtgan_version() == 1
assert ops.split_flat.__doc__
import torch
x = torch.zeros(4)
for call in (lambda: ops.global_norm([x]), lambda: ops.TensorList([x]), lambda: ops.linear_xent(x, x, x), lambda: ops.global_norm([x])):
    try:
        call()
    except ImportError as e:
        assert "_calls.so" in str(e)
    else:
        raise AssertionError("no error")
print("fine")
""" % str(tmp_path)
    got = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, env=dict(os.environ, PYTHONPATH=str(tmp_path)), capture_output=True, text=True)
    assert got.stdout.strip() == "fine", got.stderr


@pytest.mark.skipif(shutil.which("make") is None, reason="needs make")
def test_what_make_builds(tmp_path):
    """Another torch or Python: the calls are built again, the library is not.  No torch: the library alone."""
    csrc = tmp_path / "nmt_gan_amd" / "csrc"
    shutil.copytree(os.path.join(ROOT, "nmt_gan_amd", "csrc"), csrc, ignore=lambda d, names: [n for n in names if n.endswith((".o", ".env"))])
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    for name in os.listdir(csrc):
        if name.endswith(".hip"):
            (csrc / (name[:-4] + ".o")).touch()
    (csrc.parent / "libnmtgan_hip.so").touch()

    def python(name, version):
        """A python whose torch is of that version, or which has none."""
        path = tmp_path / name
        path.write_text("""#!%s
import sys
code = sys.argv[2]
if "find_spec" in code: print(%r)
elif "metadata" in code: print(%r)
else: print("/usr/include/python3")
""" % (sys.executable, "/opt/torch" if version else "", version))
        path.chmod(0o755)
        return str(path)

    def would(py, *goals):
        got = subprocess.run(["make", "-n", "-C", str(csrc), "PYTHON=" + py, *goals], check=True, capture_output=True, text=True).stdout
        return "calls.cpp" in got, ".hip" in got

    one, two, none = python("one", "2.1 on 3.10"), python("two", "2.2 on 3.10"), python("none", "")
    assert would(one) == (True, False)                              # not built yet
    (csrc.parent / "_calls.so").touch()
    assert would(one) == (False, False)
    assert would(two) == (True, False)
    os.utime(csrc.parent / "_calls.so", (2 ** 31, 2 ** 31))
    assert would(two) == (False, False)
    assert would(none) == (False, False)
    os.remove(csrc.parent / "_calls.so")
    assert would(none) == (False, False)
    assert would(one, "lib") == (False, False)
    os.remove(csrc / "gemm.o")
    assert would(none) == (False, True)
