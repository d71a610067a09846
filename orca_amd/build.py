"""Builds liborca_hip.so (the C-ABI library declared in include/orca_hip.h) in-tree with hipcc for
gfx950.  Needs no GPU (hipcc cross-compiles); the .so files lie beside the sources."""
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "liborca_hip.so")
HOST = os.path.join(HERE, "_host.so")      # csrc/bind.cpp: torch tensors -> C ABI for the calls where the host's time counts
SOURCES = ["csr.hip", "tgat.hip", "tgat_bwd.hip", "gru_bwd.hip", "gru.hip", "state.hip", "plan.hip", "plan_dev.hip", "engine.hip", "optim.hip", "clip.hip", "clip_adam.hip", "embedding.hip", "decoder.hip"]
FLAGS = ["-O3", "--offload-arch=gfx950", "-std=c++20", "-fPIC", "-fvisibility=hidden", "-Wall",
         "-Wno-unused-result", "-Wno-unused-function",
         # no packed fp32 instructions: some of their forms have given wrong results on gfx950, now and then and without an error
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _stale(target, deps):
  if not os.path.exists(target):
    return True
  t = os.path.getmtime(target)
  return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=False):
  hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
  # every header is a dependency of every object: the sampler and the split GRU live in headers
  inc = os.path.join(HERE, "..", "include")
  headers = sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")) + \
            sorted(os.path.join(inc, f) for f in os.listdir(inc) if f.endswith(".h"))
  objs, jobs = [], []
  os.makedirs(os.path.join(CSRC, "build"), exist_ok=True)
  for s in SOURCES:
    src = os.path.join(CSRC, s)
    obj = os.path.join(CSRC, "build", s.replace(".hip", ".o"))
    objs.append(obj)
    if force or _stale(obj, [src, os.path.abspath(__file__)] + headers):      # (this file: the flags)
      jobs.append([hipcc] + FLAGS + ["-c", src, "-o", obj])

  def run(cmd):
    if verbose:
      print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)

  bind = os.path.join(CSRC, "bind.cpp")
  host = []
  if force or _stale(HOST, [bind, os.path.join(inc, "orca_hip.h")]):
    import torch      # (headers and libraries of the torch that will load it)
    t = os.path.dirname(torch.__file__)
    host = [[os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall", "-D__HIP_PLATFORM_AMD__=1",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I" + os.path.join(t, "include"),
             "-I" + sysconfig.get_paths()["include"], "-I/opt/rocm/include", bind, "-o", HOST, "-L" + os.path.join(t, "lib"),
             "-ltorch_python", "-ltorch_cpu", "-lc10_hip", "-lc10"]]

  with ThreadPoolExecutor(max_workers=4) as ex:
    list(ex.map(run, host + jobs))
  if jobs or _stale(OUT, objs):
    run([hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", OUT] + objs)
  return OUT


if __name__ == "__main__":
  print(build(force="--force" in sys.argv, verbose=True))
