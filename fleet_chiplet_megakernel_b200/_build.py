"""Ahead-of-time build of the native library (no JIT at run time).

``python -m fleet_chiplet_megakernel_b200._build`` or ``build()`` compiles the
CUDA sources for sm_100a into ``libb200mk.so`` next to this file.  The built
library is what the package loads; there is no fallback when it is missing.
Beside it stands ``_serving_native.so``, the binding of the serving operators.
"""
import json
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libb200mk.so")
BINDING = os.path.join(HERE, "_serving_native.so")  # the serving operators as Python functions (serving.py)
BINDING_SOURCE = "mk_binding.cpp"
OBJDIR = os.path.join(HERE, "build")
REPORT = os.path.join(OBJDIR, "instances.json")  # what ptxas made of every kernel instance
# mk_kernel_tp.cu, mk_kernel_hier.cu and mk_kernel_moe.cu include mk_kernel.cu with other build switches (see its header); each
# is compiled once per linear path that its programs take (MK_NC, see mk_launch.cu)
SOURCES = {"mk_kernel.cu": (0, 8, 16, 32), "mk_kernel_tp.cu": (0, 8, 16, 32), "mk_kernel_hier.cu": (0, 8, 16, 32), "mk_kernel_moe.cu": (0,),
           "mk_launch.cu": None, "mk_runtime.cpp": None, "mk_noalloc.cu": None,
           "mk_step_plan.cu": None, "mk_rotate_append.cu": None, "mk_chunk_attention.cu": None, "mk_chunk_attention_tiles.cu": None, "mk_sample.cu": None}
HEADERS = ["mk_types.h", "mk_wide.cuh", "mk_serving.cuh", "mk_chunk_attention.cuh", os.path.join("..", "..", "include", "b200mk.h")]


def _nvcc():
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found: the native library cannot be built")


def needs_build():
    if not os.path.exists(LIB) or not os.path.exists(BINDING):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(BINDING))
    deps = [os.path.join(CSRC, s) for s in list(SOURCES) + HEADERS + [BINDING_SOURCE]]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def resources(ptxas):
    """Registers, stack and spills (bytes) a thread of the megakernel, from the output of ``ptxas -v``; None without one."""
    entry = re.search(r"Compiling entry function '\w*megakernel\w*'.*?(?=Compiling entry function|\Z)", ptxas, re.S)
    if entry is None:
        return None
    stack, stores, loads = map(int, re.search(r"(\d+) bytes stack frame, (\d+) bytes spill stores, (\d+) bytes spill loads", entry[0]).groups())
    return {"registers": int(re.search(r"Used (\d+) registers", entry[0])[1]), "stack": stack, "spill_stores": stores, "spill_loads": loads}


def check_registers(instances):
    """The warp roles share out kLaunchRegs registers a thread (mk_types.h): an instance with fewer would wait for them for good."""
    with open(os.path.join(CSRC, "mk_types.h")) as f:
        need = int(re.search(r"kLaunchRegs = (\d+)", f.read())[1])
    few = {name: r and r["registers"] for name, r in instances.items() if r is None or r["registers"] < need}  # (None: no kernel found)
    if few:
        raise RuntimeError(f"kernel instances with fewer than {need} registers a thread: {few}")


def binding_command():
    """The binding is compiled against the torch that runs it (its headers, its C++ ABI) and linked with torch alone.  The C++ runtime is
    named: it has to be the process's shared one.  Some installations of g++ link a static one where no other is named, and with two of them a C++ stream
    in the module (torch's macros format their errors through one) ends the process at the first number."""
    import torch
    root = os.path.dirname(torch.__file__)
    lib = os.path.join(root, "lib")
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"],
               os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")]
    return ([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"] +
            [f"-I{i}" for i in include] + [os.path.join(CSRC, BINDING_SOURCE), "-o", BINDING, f"-L{lib}"] +
            [f"-l{n}" for n in ("c10", "c10_cuda", "torch_cpu", "torch_cuda", "torch", "torch_python", ":libstdc++.so.6")])


def build(force=False, verbose=False):
    if not force and not needs_build():
        return LIB
    flags = ["-Xptxas", "-v", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC"]
    os.makedirs(OBJDIR, exist_ok=True)
    jobs = []
    for src, instances in SOURCES.items():
        stem = os.path.splitext(src)[0]
        for nc in instances or (None,):
            obj = os.path.join(OBJDIR, stem + ("" if nc is None else f"_{nc}") + ".o")
            define = [] if nc is None else [f"-DMK_NC={nc}"]
            jobs.append(([_nvcc()] + flags + define + ["-c", os.path.join(CSRC, src), "-o", obj], obj))
    jobs.append((binding_command(), None))
    # one nvcc per object, as many side by side as there are cores, then one link
    with ThreadPoolExecutor(max_workers=os.cpu_count() or 4) as pool:
        done = list(pool.map(lambda job: subprocess.run(job[0], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True), jobs))
    instances = {}
    for (cmd, obj), r in zip(jobs, done):
        if verbose or r.returncode != 0:
            sys.stdout.write(" ".join(cmd) + "\n" + r.stdout)
        if r.returncode != 0:
            raise subprocess.CalledProcessError(r.returncode, cmd)
        if obj is None:
            continue
        name = os.path.splitext(os.path.basename(obj))[0]
        if name.startswith("mk_kernel"):
            instances[name] = resources(r.stdout)
    check_registers(instances)
    with open(REPORT, "w") as f:
        json.dump(instances, f, indent=1)
    objs = [obj for _, obj in jobs if obj is not None]
    subprocess.check_call([_nvcc(), "-shared", "-o", LIB] + objs)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
