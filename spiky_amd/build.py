"""Build libspiky_lut.so (the HIP kernels + C ABI) in-tree for gfx950.

Run as ``python -m spiky_amd.build`` or through ``__graft_entry__.build()``; without torch, a host
compiler or Python's headers, for hosts in C or C++, as ``python spiky_amd/build.py --library``.
The library lands next to this file so that it travels with the source tree.
"""
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libspiky_lut.so")
SOURCES = ["lut_fc.hip", "lut_tm.hip", "lut_seq.hip", "lut_sparse.hip", "lut_densify.hip", "lut_product.hip", "lut_seq_sparse.hip",
           "lut_builder.hip", "lut_capi.hip", "lm/lm_dropout.hip", "lm/lm_residual.hip", "lm/lm_logits.hip",
           "lm/lm_capi.hip"]
ARCH = os.environ.get("SPIKY_OFFLOAD_ARCH", "gfx950")

HIPCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-fPIC",
    f"--offload-arch={ARCH}",
    # packed fp32 VALU forms are kept out of every kernel on this target
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-munsafe-fp-atomics",
    "-Wall",
    "-Wno-unused-result",
]


# The operators on torch tensors: host code, which calls the library.
BINDING = os.path.join(HERE, "_lm_torch.so")
BINDING_SOURCE = os.path.join("lm", "lm_torch.cpp")


def _hipcc():
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    raise RuntimeError("hipcc not found")


def build_binding(verbose=False):
    """Compile the torch binding against the library, which must be there."""
    found = importlib.util.find_spec("torch")
    if found is None:
        raise RuntimeError("the torch binding needs torch, which is not found")
    torch = os.path.dirname(found.origin)
    tmp = BINDING + ".tmp"
    include = [os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"),
               "/opt/rocm/include", sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__",
           "-DUSE_ROCM", *(f for i in include for f in ("-isystem", i)), os.path.join(CSRC, BINDING_SOURCE), "-o", tmp,
           "-L" + os.path.join(torch, "lib"), "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python", "-L" + HERE,
           "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    os.replace(tmp, BINDING)
    return BINDING


def build(verbose=False, binding=None):
    """Compile every source to an object, link the shared library, then build the torch binding:
    where torch is found, or always (binding=True) or never (False).  The library needs hipcc alone."""
    hipcc = _hipcc()
    objs = []
    os.makedirs(os.path.join(HERE, "_build"), exist_ok=True)
    for src in SOURCES:
        path = os.path.join(CSRC, src)
        if not os.path.exists(path):
            continue
        obj = os.path.join(HERE, "_build", os.path.basename(src).replace(".hip", ".o"))
        cmd = [hipcc, *HIPCC_FLAGS, "-c", path, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
        objs.append(obj)
    tmp = LIB + ".tmp"
    cmd = [hipcc, "-shared", f"--offload-arch={ARCH}", "-fPIC", *objs, "-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    os.replace(tmp, LIB)
    if binding is None:
        binding = importlib.util.find_spec("torch") is not None
        if not binding:
            print("torch not found: built without the torch binding", file=sys.stderr)
    if binding:
        build_binding(verbose)
    return LIB


if __name__ == "__main__":
    build(verbose="-v" in sys.argv, binding=False if "--library" in sys.argv else None)
    print(LIB)
