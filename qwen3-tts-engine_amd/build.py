"""Build recipe for the q3attn HIP library (gfx950): ``python build.py`` or ``build()``.

Compiles every ``csrc/*.hip`` with hipcc for gfx950 and links ``q3attn/libq3attn.so`` in-tree, so
the built library travels with the source tree; ``binding/torch_ops.cpp``, the torch ops that are
registered from C++, becomes ``q3attn/libq3torch.so`` beside it (host code only, by the host compiler against
torch's headers).  Object files go to ``_build/`` (git-ignored).
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "q3attn", "libq3attn.so")
# HBM probes (measurement infrastructure for bench.py --workload probe), a library of their own
PROBE_SRC = os.path.join(HERE, "probe", "hbm_probe.hip")
PROBE_OUT = os.path.join(HERE, "q3attn", "libq3probe.so")
# torch ops over the C ABI, a library of their own that links libq3attn.so and torch
TORCH_SRC = os.path.join(HERE, "binding", "torch_ops.cpp")
TORCH_OUT = os.path.join(HERE, "q3attn", "libq3torch.so")
BUILD = os.path.join(HERE, "_build")
ARCH = os.environ.get("Q3A_OFFLOAD_ARCH", "gfx950")

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CXX = os.environ.get("CXX", "g++")
CFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-fPIC", "-std=c++17", "-mcode-object-version=5",
    "-Wall", "-Wno-unused-function",
    # no packed-fp32 instructions in generated code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA accumulators in VGPRs: loop-carried accumulators that VALU code also touches are otherwise
    # copied VGPR <-> AGPR around every MFMA block
    "-mllvm", "-amdgpu-mfma-vgpr-form=1",
]


def scratch_users(remarks: str) -> list[str]:
    """Kernels whose resource-usage remarks report scratch (private) memory per lane: a register array the
    compiler could not keep in VGPRs, which turns every access into a memory round trip."""
    users, name = [], None
    for ln in remarks.splitlines():
        m = re.search(r"remark: Function Name: (\S+)", ln)
        if m:
            name = m.group(1)
            continue
        m = re.search(r"remark:\s+ScratchSize \[bytes/lane\]: (\d+)", ln)
        if m and int(m.group(1)) > 0:
            users.append(f"{name} ({m.group(1)} B/lane)")
    return users


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, os.path.basename(os.path.dirname(src)) + "_" + os.path.basename(src) + ".o")
    cmd = [HIPCC, *CFLAGS, "-Rpass-analysis=kernel-resource-usage", "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    lines = [ln for ln in (r.stdout + r.stderr).splitlines() if "packed-fp32-ops" not in ln]
    # drop the remarks and the source excerpts the compiler prints under them
    msg = "\n".join(ln for ln in lines if "remark:" not in ln and not re.match(r"^\s*(\d+\s+)?\|", ln))
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{msg}")
    spills = scratch_users("\n".join(lines))
    if spills:
        raise RuntimeError(f"{src}: kernels using scratch memory: {', '.join(spills)}")
    if msg.strip():
        print(msg, file=sys.stderr)
    return obj


def _run(cmd, what: str) -> None:
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError(f"{what} failed: {e}") from e
    if r.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{r.stdout}{r.stderr}")


def _compile_torch_ops() -> str:
    import torch
    root = os.path.dirname(torch.__file__)
    obj = os.path.join(BUILD, "binding_torch_ops.cpp.o")
    _run([CXX, "-O2", "-fPIC", "-std=c++17", "-Wall", "-DUSE_ROCM=1", "-D__HIP_PLATFORM_AMD__=1",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-isystem", os.path.join(root, "include"),
          "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"), "-isystem", os.path.join(ROCM, "include"),
          "-c", TORCH_SRC, "-o", obj], f"compiling {TORCH_SRC}")
    return obj


def _link_torch_ops(obj: str) -> None:
    import torch
    _run([CXX, "-shared", obj, "-L" + os.path.dirname(OUT), "-lq3attn", "-L" + os.path.join(os.path.dirname(torch.__file__), "lib"),
          "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-Wl,-rpath,$ORIGIN", "-o", TORCH_OUT + ".tmp"], f"linking {TORCH_OUT}")
    os.replace(TORCH_OUT + ".tmp", TORCH_OUT)


def build(verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as ex:
        binding = ex.submit(_compile_torch_ops)
        objs = list(ex.map(_compile, srcs + [PROBE_SRC]))
    for out, parts in ((OUT, objs[:-1]), (PROBE_OUT, objs[-1:])):
        tmp = out + ".tmp"
        soname = ["-Wl,-soname," + os.path.basename(out)]
        _run([HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *soname, *parts, "-o", tmp], "link")
        os.replace(tmp, out)
        if verbose:
            print(f"built {out}")
    # Last, since it needs a host compiler and torch's headers and nothing needs it: where it fails, the HIP libraries are there all
    # the same, and no binding of an earlier build beside them.
    try:
        _link_torch_ops(binding.result())
    except (RuntimeError, ImportError) as e:
        if os.path.exists(TORCH_OUT):
            os.remove(TORCH_OUT)
        raise RuntimeError(f"{OUT} is built, but the torch ops of {TORCH_SRC} are not: {e}") from e
    if verbose:
        print(f"built {TORCH_OUT}")
    return OUT


if __name__ == "__main__":
    build(verbose=True)
