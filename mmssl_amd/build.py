"""Builds libmmssl_hip.so in-tree with hipcc for gfx950 (cross-compiles without a GPU).

    python -m mmssl_amd.build [--force]

Each csrc/*.hip is compiled to an object (in parallel) and linked into mmssl_amd/libmmssl_hip.so; beside them
csrc/torch_binding.cpp is compiled against this torch's headers into mmssl_amd/_torch_binding.so (host code only: argument
checks and autograd nodes around the library's C entry points). Both are git-ignored.
"""
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_obj")
LIB = os.path.join(HERE, "libmmssl_hip.so")
BINDING = os.path.join(HERE, "_torch_binding.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# built without packed fp32 instructions (v_pk_add / mul / fma_f32), as a precaution; the default bench takes
# no longer without them. The host pass does not know the feature and says so once per unit, which means nothing
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function",
         "-munsafe-fp-atomics", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))


def _deps_mtime():
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".hpp", ".h"))]
    hdrs.append(os.path.join(HERE, "..", "include", "mmssl_hip.h"))
    hdrs.append(os.path.abspath(__file__))            # the flags
    return max(os.path.getmtime(h) for h in hdrs)


def _compile(src, force, hdr_m):
    obj = os.path.join(OBJ, src[:-4] + ".o")
    s = os.path.join(CSRC, src)
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(s), hdr_m):
        return obj, False
    cmd = [HIPCC] + FLAGS + ["-c", s, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("hipcc failed for %s:\n%s\n%s" % (src, r.stdout, r.stderr))
    if r.stderr.strip():
        sys.stderr.write(r.stderr)
    return obj, True


def _compile_binding(force, hdr_m):
    """True if _torch_binding.so was made anew."""
    import torch
    src = os.path.join(CSRC, "torch_binding.cpp")
    tdir = os.path.dirname(torch.__file__)
    newest = max(os.path.getmtime(src), hdr_m, os.path.getmtime(os.path.join(tdir, "version.py")))
    if not force and os.path.exists(BINDING) and os.path.getmtime(BINDING) >= newest:
        return False
    tmp = BINDING + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__",
           "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI, "-DTORCH_EXTENSION_NAME=_torch_binding",
           "-I/opt/rocm/include", "-I" + os.path.join(tdir, "include"),
           "-I" + os.path.join(tdir, "include", "torch", "csrc", "api", "include"), "-I" + sysconfig.get_paths()["include"],
           src, "-o", tmp, "-L" + os.path.join(tdir, "lib"), "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip",
           "-ldl"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("%s failed for torch_binding.cpp:\n%s\n%s" % (cmd[0], r.stdout, r.stderr))
    os.replace(tmp, BINDING)
    return True


def build(force=False, verbose=True):
    os.makedirs(OBJ, exist_ok=True)
    hdr_m = _deps_mtime()
    with ThreadPoolExecutor(max_workers=8) as ex:
        binding = ex.submit(_compile_binding, force, hdr_m)
        res = list(ex.map(lambda s: _compile(s, force, hdr_m), _sources()))
        new_binding = binding.result()
    objs = [o for o, _ in res]
    build.last = {"compiled": [os.path.basename(o) for o, c in res if c] + (["_torch_binding.so"] if new_binding else []),
                  "reused": [os.path.basename(o) for o, c in res if not c], "linked": False}
    if force or any(c for _, c in res) or not os.path.exists(LIB):
        cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("link failed:\n%s\n%s" % (r.stdout, r.stderr))
        build.last["linked"] = True
        if verbose:
            print("built %s: %d unit(s) compiled for gfx950, %d object(s) reused" % (
                LIB, sum(c for _, c in res), len(build.last["reused"])))
    elif verbose:
        print("up to date: %s (%d objects newer than their sources and headers; --force recompiles)" % (LIB, len(objs)))
    return LIB


build.last = None


if __name__ == "__main__":
    build(force="--force" in sys.argv)
