"""In-tree build of the native extensions ``distributed_pytorch_amd/_C*.so`` and ``_T*.so``.

``python -m distributed_pytorch_amd.build`` compiles every ``csrc/**/*.hip`` for gfx950 with
hipcc (cross-compiles without a GPU), the C++ runtime / bindings, and links two pybind11 modules that
sit next to the package so they travel to the GPU box with the tree: ``_C``, and ``_T`` (``csrc/transformer``:
operators with autograd nodes in C++, the only part built against torch's headers).  Objects are cached under
``build/`` and rebuilt only when a source (or a header that it includes) is newer or the command that makes them changed.
"""
from __future__ import annotations

import os
import re
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
HIPCC = os.path.join(ROCM, "bin", "hipcc")
ARCH = "gfx950"
# scalar fp32 VALU forms only: some packed fp32 forms that -O3 makes from ordinary float code have given wrong results
# now and then on this hardware.  (The host pass warns that it does not know the feature; harmless.)
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _sources():
    """{module: sources}: ``_C`` (no torch headers) and ``_T`` (``csrc/transformer``, built against torch's)."""
    out = {"_C": [], "_T": []}
    for root, _, files in os.walk(CSRC):
        for f in sorted(files):
            if f.endswith((".hip", ".cpp")):
                out["_T" if os.path.basename(root) == "transformer" else "_C"].append(os.path.join(root, f))
    return out


def _mtime_with_headers(path: str, seen=None) -> float:
    """Newest modification time of a source and of the package's own headers that it includes."""
    seen = set() if seen is None else seen
    path = os.path.normpath(path)
    if path in seen or not os.path.isfile(path):
        return 0.0
    seen.add(path)
    newest = os.path.getmtime(path)
    with open(path) as f:
        for name in re.findall(r'^\s*#include\s+"([^"]+)"', f.read(), re.M):
            for base in (os.path.dirname(path), CSRC):
                newest = max(newest, _mtime_with_headers(os.path.join(base, name), seen))
    return newest


def target_path(module: str = "_C") -> str:
    return os.path.join(HERE, module + sysconfig.get_config_var("EXT_SUFFIX"))


def _torch_flags():
    """(compiler flags, linker flags) of a host source that includes torch's headers."""
    import torch

    root = os.path.dirname(torch.__file__)
    inc = ["-I" + os.path.join(root, "include"), "-I" + os.path.join(root, "include", "torch", "csrc", "api", "include")]
    libs = ["-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10", "-lc10_hip"]
    return ["-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM"] + inc, libs


def _stale(out: str, stamp: str, cmd, newest: float) -> bool:
    """Whether ``out`` has to be made again: it is not there, older than what it is made of, or made by another command."""
    if not os.path.exists(out) or os.path.getmtime(out) < newest or not os.path.exists(stamp):
        return True
    with open(stamp) as f:
        return f.read() != " ".join(cmd)


def _make(out: str, stamp: str, cmd, verbose: bool, what: str) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    if os.path.exists(stamp):
        os.remove(stamp)                  # (what an interrupted command leaves is made again)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("%s\n%s" % (what, r.stderr[-4000:]))
    with open(stamp, "w") as f:
        f.write(" ".join(cmd))


def build(verbose: bool = False, force: bool = False, jobs: int = 0) -> str:
    import pybind11

    objdir = os.path.join(os.path.dirname(HERE), "build", "obj")
    os.makedirs(objdir, exist_ok=True)
    inc = ["-I" + pybind11.get_include(), "-I" + sysconfig.get_paths()["include"], "-I" + CSRC,
           "-I" + os.path.join(ROCM, "include")]
    common = [HIPCC, "--offload-arch=" + ARCH, "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden",
              "-Wno-unused-result"] + NO_PACKED_FP32 + inc + os.environ.get("DPA_BUILD_DEFS", "").split()
    torch_cc, torch_ld = _torch_flags()
    host = ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden"] + torch_cc + inc[1:]
    todo, objs = [], {}
    for module, sources in _sources().items():
        objs[module] = []
        for src in sources:
            obj = os.path.join(objdir, os.path.relpath(src, CSRC).replace(os.sep, "_") + ".o")
            objs[module].append(obj)
            cmd = (host if module == "_T" and src.endswith(".cpp") else common) + ["-c", src, "-o", obj]
            if force or _stale(obj, obj + ".cmd", cmd, _mtime_with_headers(src)):
                todo.append((src, obj, cmd))

    def compile_one(job):
        src, obj, cmd = job
        _make(obj, obj + ".cmd", cmd, verbose, "compile failed: " + src)

    jobs = jobs or min(8, int(os.environ.get("MAX_JOBS", "8")), max(1, len(todo)))
    if todo:
        with ThreadPoolExecutor(max_workers=jobs) as ex:
            list(ex.map(compile_one, todo))
    for module, files in objs.items():
        tgt, stamp = target_path(module), os.path.join(objdir, module + ".cmd")
        # no rpath: at run time libamdhip64.so.7 (and torch's libraries) resolve to the copies torch loaded first
        cmd = [HIPCC, "--offload-arch=" + ARCH, "-shared", "-fPIC", "-o", tgt] + files + ["-ldl"] + (torch_ld if module == "_T" else [])
        if _stale(tgt, stamp, cmd, max(os.path.getmtime(f) for f in files)):
            _make(tgt, stamp, cmd, verbose, "link failed:")
    return target_path()


if __name__ == "__main__":
    path = build(verbose="-v" in sys.argv, force="-f" in sys.argv)
    print("built", path)
