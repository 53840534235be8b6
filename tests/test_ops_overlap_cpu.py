"""Span attention and the cross entropy refuse outputs that lie over an input or another output, before any launch."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from nmt_gan_amd import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20                                                         # spaced addresses that nobody reads
AT = {n: P + (i << 16) for i, n in enumerate(("q", "k", "v", "lo", "hi", "pos", "slopes", "out", "lse", "dout", "dq", "dk", "dv", "ws"))}


def _refused(rc, *names):
    text = L.lib.nmtgan_last_error().decode()
    assert rc != 0 and "overlaps" in text and all(n in text for n in names), text


def _span(**kw):
    a = L.SpanArgs(dtype=L.NMTGAN_F32, M=4, N=4, heads=2, kv_heads=2, dh=64, ldq=128, ldk=128, ldv=128, scale=1.0, cap=0.0, ldo=128)
    for n in ("q", "k", "v", "lo", "hi", "pos", "slopes", "out", "lse"):
        setattr(a, n, kw.get(n, AT[n]))
    return a


@pytest.mark.parametrize("name", ["q", "k", "v", "lo", "hi", "pos", "slopes", "lse"])
@pytest.mark.parametrize("off", [0, 16, 3 * 512 + 496])             # the first row, inside it, the last row's last bytes
def test_out_over(name, off):
    a = _span(**{name: AT["out"] + off})
    _refused(L.lib.nmtgan_attn_span(C.byref(a), None), "out", name)
    need = L.lib.nmtgan_attn_span_step_workspace_bytes(4, 2, 2, 64, 5000)
    _refused(L.lib.nmtgan_attn_span_step(C.byref(a), 5000, AT["ws"], need, None), "out", name)
    _refused(L.lib.nmtgan_attn_span_step(C.byref(_span()), 5000, AT["out"] + off & ~15, need, None), "out", "workspace")


def test_lse_over():
    _refused(L.lib.nmtgan_attn_span(C.byref(_span(lse=AT["k"] + 2044)), None), "lse", "k")


@pytest.mark.parametrize("one,other", [("dq", "q"), ("dq", "dout"), ("dk", "k"), ("dv", "v"), ("dk", "dv"), ("dq", "dk"), ("dq", "out"), ("dv", "lse"),
                                       ("dk", "lo"), ("dv", "slopes"), ("dq", "ws")])
@pytest.mark.parametrize("off", [0, 3 * 512 + 496])
def test_gradients_over(one, other, off):
    at = dict(AT)
    if other == "ws":
        at[one] = at["ws"] + (off & 496)                            # (a workspace of a KiB)
    else:
        at[other] = at[one] + off
    a = _span(**{n: at[n] for n in ("q", "k", "v", "lo", "hi", "pos", "slopes", "out", "lse")})
    g = L.SpanGrads(dout=at["dout"], ld_dout=128, dq=at["dq"], ld_dq=128, dk=at["dk"], ld_dk=128, dv=at["dv"], ld_dv=128)
    need = L.lib.nmtgan_attn_span_grads_workspace_bytes(4, 2)
    _refused(L.lib.nmtgan_attn_span_grads(C.byref(a), C.byref(g), at["ws"], need, None), one, "workspace" if other == "ws" else other)


@pytest.mark.parametrize("one,other", [("loss", "lse"), ("loss", "h"), ("lse", "w"), ("loss", "labels"), ("lse", "workspace")])
def test_xent_over(one, other):
    at = {n: P + (i << 16) for i, n in enumerate(("h", "w", "labels", "loss", "lse"))}
    at["workspace"] = P + (1 << 20)
    at[other] = at[one] & ~255 if other == "workspace" else at[one]
    a = L.XentArgs(dtype=L.NMTGAN_F32, M=4, V=10, d=64, h=at["h"], ldh=64, w=at["w"], ldw=64, labels=at["labels"], smoothing=0.0)
    _refused(L.lib.nmtgan_linear_xent(C.byref(a), at["loss"], at["lse"], at["workspace"], 1 << 16, None), one, other)


@pytest.mark.parametrize("one,other", [("dh", "h"), ("dw", "w"), ("dh", "dw"), ("dw", "h"), ("dh", "labels"), ("dw", "lse"), ("dh", "grad_row"), ("dw", "workspace")])
def test_xent_gradients_over(one, other):
    at = {n: P + (i << 16) for i, n in enumerate(("h", "w", "labels", "lse", "grad_row", "dh", "dw"))}
    at["workspace"] = P + (1 << 20)
    at[other] = at[one]
    a = L.XentArgs(dtype=L.NMTGAN_F32, M=4, V=10, d=64, h=at["h"], ldh=64, w=at["w"], ldw=64, labels=at["labels"], smoothing=0.0)
    _refused(L.lib.nmtgan_linear_xent_grads(C.byref(a), at["lse"], at["grad_row"], at["dh"], 64, at["dw"], 64, at["workspace"], 1 << 30, None),
             one, other)


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_the_comparison_of_regions_against_every_byte(tmp_path):
    """regions_meet on small strided regions against marking their bytes."""
    src, exe = tmp_path / "r.cpp", tmp_path / "r"
    text = open(os.path.join(ROOT, "nmt_gan_amd", "csrc", "regions.h")).read().replace('#include "common.h"', "")
    src.write_text("""#include <stdint.h>
#include <stdio.h>
#include <vector>
#define NMTGAN_REQUIRE(c, ...) do { if (!(c)) return -2; } while (0)
""" + text.replace("#pragma once", "") + """
int main() {
  using namespace nmtgan;
  unsigned seed = 1;
  auto next = [&](int n) { seed = seed * 1664525u + 1013904223u; return (int)((seed >> 8) % n); };
  int met = 0;
  for (int t = 0; t < 200000; ++t) {
    const int wx = 1 + next(6), wy = 1 + next(6), lx = wx + next(9);
    const int ly = next(2) ? (lx >= wy ? lx : wy) : wy + next(9);
    const Region x("x", (void*)(uintptr_t)(100 + next(60)), next(6), lx, wx), y("y", (void*)(uintptr_t)(100 + next(60)), next(6), ly, wy);
    std::vector<int> mark(1000);
    bool meet = false;
    for (int i = 0; i < x.rows; ++i) for (int b = 0; b < wx; ++b) mark[x.at + i * lx + b] = 1;
    for (int i = 0; i < y.rows; ++i) for (int b = 0; b < wy; ++b) meet = meet || mark[y.at + i * ly + b];
    met += meet;
    if (regions_meet(x, y) != meet || regions_meet(y, x) != meet) return printf("case %d\\n", t), 1;
  }
  return met > 20000 && met < 180000 ? 0 : 2;
}
""")
    subprocess.run(["g++", "-std=c++17", "-o", str(exe), str(src)], check=True)
    subprocess.run([str(exe)], check=True)
