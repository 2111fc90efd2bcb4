"""csrc/kernel_table.h: what is asked of the runtime per kernel and device is
asked once, for however many kernels a process uses (no GPU: the table is host
code, compiled here with a counting stand-in for the runtime)."""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ethos_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "kernel_table.h"
int main() {
  ethos::KernelTable<int> table;
  static char kernels[500];
  int asked = 0, wrong = 0, got = 0;
  for (int pass = 0; pass < 3; ++pass)
    for (int dev = 0; dev < 64; dev += 21)
      for (int k = 0; k < 500; ++k) {
        if (!table.get(dev, kernels + k, &got, [&](int* v) { ++asked; *v = 1000 * dev + k; return true; })) ++wrong;
        if (got != 1000 * dev + k) ++wrong;
      }
  // a failure is not remembered, and a device outside the table is refused
  char other;
  if (table.get(0, &other, &got, [](int*) { return false; })) ++wrong;
  if (!table.get(0, &other, &got, [](int* v) { *v = 7; return true; }) || got != 7) ++wrong;
  if (table.get(64, &other, &got, [](int*) { return true; })) ++wrong;
  if (table.get(-1, &other, &got, [](int*) { return true; })) ++wrong;
  std::printf("%d %d\n", asked, wrong);
}
"""


def test_each_kernel_is_asked_for_once_per_device(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert out.split() == [str(4 * 500), "0"]


def test_the_library_keeps_its_queries_in_that_table():
    """Neither query of csrc/host.cuh has a table of its own."""
    text = open(os.path.join(CSRC, "host.cuh")).read()
    assert text.count("KernelTable<int> table") == 2 and "static const void* seen" not in text
