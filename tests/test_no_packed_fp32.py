"""The library holds no packed fp32 instruction: every source is compiled without them, and none is written by hand."""
import os
import re

from orca_amd import build

CSRC = build.CSRC


def test_the_flags():
  flags = " ".join(build.FLAGS)
  assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in flags


def test_the_sources():
  names = [f for f in os.listdir(CSRC) if f.endswith((".hip", ".h"))]
  assert set(build.SOURCES) <= set(names)
  for f in names:
    with open(os.path.join(CSRC, f)) as src:
      assert not re.search(r"v_pk_(add|mul|fma)_f32", src.read()), f
