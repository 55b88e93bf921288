"""Build libshard_hip.so (gfx950) in-tree with hipcc.

    python -m shard_amd.build            # or shard_amd.build.build()

Each ``csrc/*.hip`` is compiled to an object with its own flags (the integer
chains in quant.hip with -ffp-contract=off so no multiply-add is fused), then
all objects are linked into ``shard_amd/libshard_hip.so``.  ``csrc/dispatch.cpp``,
host code against torch's headers, becomes ``shard_amd/_dispatch.so``.
"""
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libshard_hip.so")
DISPATCH = os.path.join(HERE, "_dispatch.so")
ARCH = os.environ.get("SHARD_OFFLOAD_ARCH", "gfx950")

COMMON = [
    f"--offload-arch={ARCH}", "-O3", "-fPIC", "-std=c++17",
    # packed fp32 arithmetic stays off in all device code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-result",
]
PER_FILE = {
    "quant.hip": ["-ffp-contract=off"],
    "decode_attn.hip": [],
    "pca.hip": ["-ffp-contract=off"],  # the fused undo-RoPE rounds as k_prepare does
    "reconstruct.hip": ["-ffp-contract=off"],
    "abi.hip": [],
    "fp16_decode.hip": [],
}


def hipcc() -> str:
    p = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(p):
        raise RuntimeError("hipcc not found; libshard_hip.so cannot be built")
    return p


def sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))


def dispatch_command(out: str):
    import torch
    root = os.path.dirname(torch.__file__)
    return [shutil.which("g++") or "c++", "-O2", "-fPIC", "-shared", "-std=c++17",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            "-isystem", os.path.join(root, "include"),
            "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
            "-isystem", sysconfig.get_paths()["include"], os.path.join(CSRC, "dispatch.cpp"), "-o", out,
            "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10"]


def build(verbose: bool = False, jobs: int = 4) -> str:
    """Compile every csrc/*.hip for gfx950 and link libshard_hip.so. Returns its path.

    _dispatch.so, which only makes eager calls cheaper, may fail to build (no
    g++, no headers): a warning says so, and the one of an earlier build, which
    may not fit the new library, is removed.  Where the library does not build,
    both files stay as they were."""
    cc = hipcc()
    objdir = tempfile.mkdtemp(prefix="shard_build_")
    procs, dispatch = [], None
    try:
        new_lib, new_dispatch = os.path.join(objdir, "lib.so"), os.path.join(objdir, "dispatch.so")
        try:
            dispatch = _start(dispatch_command(new_dispatch), verbose)
        except Exception as exc:  # no compiler, no torch to build against
            no_dispatch = repr(exc)
        objs = []
        for src in sources():
            obj = os.path.join(objdir, src.replace(".hip", ".o"))
            procs.append((src, _start([cc, *COMMON, *PER_FILE.get(src, []), "-c", os.path.join(CSRC, src), "-o", obj], verbose)))
            objs.append(obj)
            if len(procs) >= jobs:
                _drain(procs)
        _drain(procs)
        procs.append(("the library", _start([cc, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", new_lib], verbose)))
        _drain(procs)
        if dispatch is not None:
            out, _ = dispatch.communicate()
            no_dispatch = out if dispatch.returncode else None
        if os.path.exists(DISPATCH):  # never an old one beside a new library
            os.remove(DISPATCH)
        _put(new_lib, LIB)
        if no_dispatch is None:
            _put(new_dispatch, DISPATCH)
        else:
            sys.stderr.write(f"warning: _dispatch.so not built, eager calls go through Python:\n{no_dispatch}\n")
    finally:
        for p in [p for _, p in procs] + [dispatch]:  # what a failure left running
            if p is not None and p.poll() is None:
                p.kill()
                p.wait()
        shutil.rmtree(objdir, ignore_errors=True)
    return LIB


def _start(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def _put(src, dst):
    """In one step, as a process may have the old file open."""
    shutil.copy(src, dst + ".tmp")
    os.replace(dst + ".tmp", dst)


def _drain(procs):
    while procs:
        src, p = procs[0]
        out, _ = p.communicate()
        procs.pop(0)
        if p.returncode != 0:
            raise RuntimeError(f"hipcc failed on {src}:\n{out}")
        warn = [ln for ln in out.splitlines() if "warning" in ln and "packed-fp32-ops" not in ln]
        if warn:
            sys.stderr.write(f"[{src}]\n" + "\n".join(warn[:20]) + "\n")


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
