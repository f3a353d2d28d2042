"""Build libvits_amd.so (gfx950) in-tree with hipcc.  Run: python -m vits_amd.build"""
from __future__ import annotations

import os
import re
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libvits_amd.so")
BINDING = os.path.join(LIBDIR, "_vits_ops.so")      # torch tensors to the library's paged-cache operators (host code only)
CXX = os.environ.get("CXX", "g++")
SOURCES = ["kernels_conv.hip", "kernels_gl16.hip", "kernels_chain.hip", "kernels_misc.hip", "kernels_paged.hip",
           "model.hip"]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# no packed fp32 arithmetic (v_pk_add_f32 and its like, which -O3 makes of ordinary float code): some of its forms have
# given wrong results now and then.  The host pass does not know the feature and says so; that is harmless.
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fno-gpu-rdc", "-Wall", "-Wno-unused-function",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

# The paged attention keeps its accumulators in the registers that the vector unit reads too.  Left to choose, the compiler gives
# builds with much LDS the other kind, moves values there, and has been seen to move only those of the lanes that were on.
# Where a build needs more than 256 registers it takes those too, whatever the flag says: so the compiler reports what it used, and a
# build that has any, or scratch, is refused (the widest today: 252, none, none).
USAGE = "-Rpass-analysis=kernel-resource-usage"
SOURCE_FLAGS = {"kernels_paged.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form", USAGE]}
MOST = {"VGPRs": 256, "AGPRs": 0, "ScratchSize": 0, "VGPRs Spill": 0}


def _check_registers(source: str, report: str) -> str:
    """Refuses a build whose kernels use more than MOST; returns what else the compiler said."""
    kernel, seen, rest, quoted = "", set(), [], False
    for line in report.splitlines():
        if f"[{USAGE}]" not in line:
            quoted = quoted and re.match(r"\s*\d*\s+\|", line) is not None            # the source line that a remark is about
            if not quoted:
                rest.append(line)
            continue
        quoted = True
        name, _, value = line.split("remark: ")[1].replace(f"[{USAGE}]", "").strip().partition(": ")
        name = name.split(" [")[0]
        if name == "Function Name":
            kernel = value
        elif name in MOST:
            seen.add(name)
            if int(value) > MOST[name]:
                raise RuntimeError(f"{source}: {kernel} uses {value} {name}, at most {MOST[name]} allowed")
    if seen != set(MOST):
        raise RuntimeError(f"{source}: the compiler did not say which registers its kernels use")
    return "".join(x + "\n" for x in rest)


def _stale(target: str, deps, command: str) -> bool:
    """Whether a target is missing, older than what it is made of, or made by another command than this one."""
    try:
        with open(target + ".cmd") as f:
            if f.read() != command:
                return True
        t = os.path.getmtime(target)
    except OSError:
        return True
    return any(os.path.getmtime(d) > t for d in deps)


def _binding_command(source: str):
    """(BUILT_FOR does nothing but make another torch another command.)"""
    import torch
    at = os.path.dirname(torch.__file__)
    return [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            f'-DBUILT_FOR="{torch.__version__}"', "-isystem", sysconfig.get_paths()["include"], "-isystem", os.path.join(at, "include"), source,
            "-o", BINDING, "-L" + os.path.join(at, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10"]


def build(force: bool = False, verbose: bool = True) -> str:
    os.makedirs(LIBDIR, exist_ok=True)
    headers = [os.path.join(CSRC, "common.h"), os.path.join(os.path.dirname(HERE), "include", "vits_amd.h")]
    paged = [os.path.join(CSRC, "paged.h")] + headers[1:]
    deps = {"kernels_paged.hip": paged, "model.hip": headers + paged}
    bind = os.path.join(CSRC, "ops_binding.cpp")
    targets = [(BINDING, [bind, headers[1]], _binding_command(bind))]
    objs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(LIBDIR, src.replace(".hip", ".o"))
        objs.append(o)
        targets.append((o, [s] + deps.get(src, headers[:1]), [HIPCC, *FLAGS, *SOURCE_FLAGS.get(src, []), "-c", s, "-o", o]))

    def make(target) -> bool:
        path, made_of, cmd = target
        line = " ".join(cmd)
        if not force and not _stale(path, made_of, line):
            return False
        if verbose:
            print(line, flush=True)
        if os.path.exists(path + ".cmd"):            # (a build that fails leaves no target that passes for a built one)
            os.remove(path + ".cmd")
        if USAGE in cmd:
            done = subprocess.run(cmd, stderr=subprocess.PIPE, text=True)
            if done.returncode:
                sys.stderr.write(done.stderr)
                done.check_returncode()
            sys.stderr.write(_check_registers(os.path.basename(made_of[0]), done.stderr))
        else:
            subprocess.run(cmd, check=True)
        with open(path + ".cmd", "w") as f:
            f.write(line)
        return True
    with ThreadPoolExecutor(max_workers=4) as ex:
        list(ex.map(make, targets))
    make((LIB, objs, [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB, *objs]))
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB)
