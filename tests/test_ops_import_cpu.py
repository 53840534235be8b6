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
