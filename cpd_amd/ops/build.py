"""Ahead-of-time build driver for the cpd_amd native extensions.

Two in-tree shared objects (the reference builds JIT-only via
torch.utils.cpp_extension.load, quant_function.py:10-17; we build AOT so the
.so travels with the repo snapshot and CI can check the build without a GPU):

  * ``_cpd_cpu.so``  — host C++ (g++), always available.
  * ``_cpd_hip.so``  — hand-written HIP/CDNA4 kernels, compiled by hipcc for
    gfx950 only (cross-compiles fine on a machine with no GPU).

Invoked by ``__graft_entry__.build()`` and usable directly:
``python -m cpd_amd.ops.build``.
"""
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_obj")  # intermediate objects (not shipped)

GFX_ARCH = os.environ.get("PYTORCH_ROCM_ARCH", "gfx950")


def _torch_paths():
    import torch
    from torch.utils import cpp_extension as ce

    incs = list(ce.include_paths()) + [sysconfig.get_paths()["include"]]
    libs = list(ce.library_paths())
    abi = "1" if torch.compiled_with_cxx11_abi() else "0"
    return incs, libs, abi


def _common_flags(ext_name, incs, abi):
    flags = [
        "-O3",
        "-std=c++17",
        "-fPIC",
        "-shared",
        f"-DTORCH_EXTENSION_NAME={ext_name}",
        "-DTORCH_API_INCLUDE_EXTENSION_H",
        f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
    ]
    flags += [f"-I{p}" for p in incs]
    flags += [f"-I{CSRC}"]
    return flags


def _link_flags(libs, hip=False):
    out = []
    for p in libs:
        out += [f"-L{p}", f"-Wl,-rpath,{p}"]
    out += ["-ltorch", "-ltorch_cpu", "-lc10", "-ltorch_python"]
    if hip:
        out += ["-ltorch_hip", "-lc10_hip", "-lamdhip64"]
    return out


def _run(cmd, verbose):
    if verbose:
        print("[cpd-build]", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


def _stale(target, sources):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC)
               if f.endswith(".h")]
    deps = list(sources) + headers + [__file__]
    return any(os.path.getmtime(s) > t for s in deps)


def _deps_of(obj):
    """What the compiler's dependency file says ``obj`` was made from, or
    None where there is none."""
    try:
        with open(obj[:-2] + ".d") as f:
            names = f.read().replace("\\\n", " ").split(":", 1)[1].split()
    except (OSError, IndexError):
        return None
    return [n for n in names if n.startswith(CSRC)]


def _made_by(obj):
    """The command that ``obj`` was finished by, or None."""
    try:
        with open(obj[:-2] + ".cmd") as f:
            return f.read()
    except OSError:
        return None


def _object_stale(obj, src, cmd):
    deps = _deps_of(obj)
    if deps is None or not os.path.exists(obj) or _made_by(obj) != cmd:
        return True
    t = os.path.getmtime(obj)
    return any(not os.path.exists(s) or os.path.getmtime(s) > t
               for s in deps + [src, __file__])


def build_cpu(force=False, verbose=True):
    target = os.path.join(HERE, "_cpd_cpu.so")
    srcs = [os.path.join(CSRC, "cpu_ops.cpp")]
    if not force and not _stale(target, srcs):
        return target
    incs, libs, abi = _torch_paths()
    cmd = (
        ["g++"]
        + _common_flags("_cpd_cpu", incs, abi)
        + ["-fopenmp", "-march=native"]
        + srcs
        + _link_flags(libs)
        + ["-o", target]
    )
    _run(cmd, verbose)
    return target


def build_hip(force=False, verbose=True):
    target = os.path.join(HERE, "_cpd_hip.so")
    srcs = sorted(
        os.path.join(CSRC, f)
        for f in os.listdir(CSRC)
        if f.endswith(".hip") or f == "hip_bindings.cpp"
    )
    if not srcs:
        return None
    if not force and not _stale(target, srcs):
        return target
    incs, libs, abi = _torch_paths()
    # one object per source, compiled side by side: the host pass over
    # torch's headers is most of a source's time
    compile_flags = (
        ["hipcc", f"--offload-arch={GFX_ARCH}"]
        + [f for f in _common_flags("_cpd_hip", incs, abi) if f != "-shared"]
        + [
            "-D__HIP_PLATFORM_AMD__=1",
            "-DUSE_ROCM=1",
            "-DHIPBLAS_V2",
            "-fno-gpu-rdc",
            "-Wno-unused-result",
            # hipcc -O3 turns pairs of float operations into packed FP32
            # instructions by itself; some of their forms give wrong results
            # on gfx950, so the feature is off for all device code.  (The
            # host pass warns that it does not know it: harmless.)
            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        ]
    )
    os.makedirs(OBJ, exist_ok=True)
    objs = [os.path.join(OBJ, os.path.basename(s) + ".o") for s in srcs]
    # An object is taken again only if this very command (its architecture and
    # flags) made it, and came to its end.
    jobs = [(s, o, compile_flags + ["-MMD", "-MF", o[:-2] + ".d", "-c", s,
                                    "-o", o]) for s, o in zip(srcs, objs)]
    todo = [j for j in jobs
            if force or _object_stale(j[1], j[0], " ".join(j[2]))]

    def compile_one(job):
        _, obj, cmd = job
        said = obj[:-2] + ".cmd"
        if os.path.exists(said):
            os.remove(said)
        _run(cmd, verbose)
        with open(said, "w") as f:
            f.write(" ".join(cmd))

    workers = max(1, min(int(os.environ.get("MAX_JOBS", "8")), len(todo)))
    with ThreadPoolExecutor(max_workers=workers) as pool:
        list(pool.map(compile_one, todo))
    _run(["hipcc", f"--offload-arch={GFX_ARCH}", "-shared", "-fPIC",
          "-fno-gpu-rdc"] + objs + _link_flags(libs, hip=True)
         + ["-o", target], verbose)
    return target


def build_all(force=False, verbose=True):
    cpu = build_cpu(force=force, verbose=verbose)
    hip = build_hip(force=force, verbose=verbose)
    return cpu, hip


if __name__ == "__main__":
    force = "--force" in sys.argv
    cpu, hip = build_all(force=force)
    print("built:", cpu, hip)
