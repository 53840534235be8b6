"""The argument structures of the operators in the ctypes binding and in the C header have the same layout."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from nmt_gan_amd import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PAIRS = [("nmtgan_span_args", L.SpanArgs), ("nmtgan_span_grads", L.SpanGrads), ("nmtgan_xent_args", L.XentArgs),
         ("nmtgan_grad_ref", L.GradRef)]


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_structures_match_the_header(tmp_path):
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "nmtgan.h"', "int main(void) {"]
    want = []
    for name, cls in PAIRS:
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        want.append(C.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (name, field))
            want.append(getattr(cls, field).offset)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    assert [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()] == want
