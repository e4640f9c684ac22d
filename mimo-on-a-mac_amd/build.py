"""Build libmimo_moe.so (gfx950) and the host module _calls.so in-tree, in mimo-on-a-mac_amd/mimo_stream/.

    python mimo-on-a-mac_amd/build.py

Each csrc/*.hip file is compiled in parallel with hipcc, then linked into one shared library.  Object files go
to mimo-on-a-mac_amd/_build/ (git-ignored).  csrc/calls.cpp is host code alone: g++, against the installed torch and Python.
"""
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "mimo_stream", "libmimo_moe.so")
SOURCES = ["codec.hip", "router.hip", "decode.hip", "prefill.hip", "layer.hip", "cache.hip", "attend.hip"]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# -fconstexpr-steps: the bf16 sigmoid table (csrc/sigmoid_table.h) is evaluated by the compiler, ~7M steps
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-fconstexpr-steps=100000000",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


CALLS = os.path.join(HERE, "mimo_stream", "_calls.so")


def _calls_command(out):
    import torch
    from torch.utils import cpp_extension
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    include = [f for path in cpp_extension.include_paths() for f in ("-isystem", path)]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            f"-I{sysconfig.get_paths()['include']}", *include, os.path.join(CSRC, "calls.cpp"), "-o", out, f"-L{lib}", "-ltorch_python",
            "-ltorch_cpu", "-lc10"]


def _run(cmd):
    p = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    out = "\n".join(l for l in p.stdout.splitlines() if "packed-fp32-ops" not in l)
    if p.returncode != 0:
        raise RuntimeError(f"command failed ({p.returncode}): {' '.join(cmd)}\n{out}")
    return out


def build(verbose=False):
    os.makedirs(OUT_DIR, exist_ok=True)
    objs = [os.path.join(OUT_DIR, s.replace(".hip", ".o")) for s in SOURCES]
    cmds = [[HIPCC, *FLAGS, "-c", os.path.join(CSRC, s), "-o", o] for s, o in zip(SOURCES, objs)]
    cmds.append(_calls_command(CALLS + ".tmp"))
    with ThreadPoolExecutor(max_workers=len(cmds)) as ex:
        outs = list(ex.map(_run, cmds))
    tmp = LIB + ".tmp"
    outs.append(_run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objs]))
    os.replace(tmp, LIB)
    os.replace(CALLS + ".tmp", CALLS)
    if verbose:
        for o in outs:
            if o.strip():
                print(o)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
