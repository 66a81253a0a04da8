"""Compile libhnsw_amd.so (host index + HIP kernels for gfx950 + C ABI) and _tensors.so (its token cache on torch tensors) in-tree."""
from __future__ import annotations

import importlib.util
import os
import subprocess
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "libhnsw_amd.so")


def tensors(out=None) -> None:
    """_tensors.so: the token cache's calls on torch tensors (host code).  Without a torch install there is no such module, and the rest
    of the package does not need it."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.origin:
        return
    root = os.path.dirname(spec.origin)
    subprocess.check_call(["make", "-C", os.path.join(HERE, "csrc"), "tensors", f"TORCH={root}", f"PYINC={sysconfig.get_paths()['include']}"], stdout=out)


def build(verbose: bool = False) -> str:
    out = None if verbose else subprocess.DEVNULL
    # `checks`: the same library with the visited sets' invariants re-read and counted, for one GPU test (never loaded otherwise)
    subprocess.check_call(["make", "-C", os.path.join(HERE, "csrc"), f"-j{min(8, os.cpu_count() or 1)}", "all", "checks"], stdout=out)
    tensors(out)
    if not os.path.exists(LIB):
        raise RuntimeError("libhnsw_amd.so was not produced")
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
