"""Build libsigcomp_b200.so (nvcc, sm_100a) and its torch binding _int8.so (g++) in-tree."""

import os
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB = PKG / "libsigcomp_b200.so"
BINDING = PKG / "_int8.so"
BINDING_SOURCE = CSRC / "sc_torch.cpp"
BINDING_STAMP = PKG / "_build" / "_int8.built_for"
SOURCES = ["sc_capi.cu", "sc_codec.cu", "sc_frames.cu", "sc_int8.cu", "sc_mlp_simple.cu", "sc_mlp_tc.cu", "sc_signal.cu"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr",
    "-ccbin", "/usr/bin/g++",
]


# Kernels whose tcgen05.ld results land in registers asynchronously (until tcgen05.wait::ld):
# a register spill placed between a load and its wait would store values not yet written, so the
# build refuses any spill in them.  ptxas -v reports stack and spills per entry function.
NO_SPILL_KERNELS = ("k_fused2", "k_small_decode", "k_pair", "k_few")
NO_SPILL_SOURCES = ("sc_mlp_tc.cu", "sc_int8.cu")


def spilling_kernels(ptxas_log, names=NO_SPILL_KERNELS):
    """[(mangled name, spill store bytes, spill load bytes)] of the entry functions in a
    `ptxas -v` log whose name contains one of `names` and that spill."""
    bad, current = [], None
    for line in ptxas_log.splitlines():
        if "Function properties for" in line:
            current = line.split("Function properties for", 1)[1].strip()
        elif current is not None and "spill stores" in line:
            parts = line.replace(",", "").split()
            stores = int(parts[parts.index("spill") - 2])
            loads = int(parts[parts.index("loads") - 3])
            if any(n in current for n in names) and (stores or loads):
                bad.append((current, stores, loads))
            current = None
    return bad


def _stale():
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    deps = [CSRC / s for s in SOURCES] + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + \
        [PKG.parent / "include" / "sigcomp_b200.h", Path(__file__)]
    return any(d.stat().st_mtime > t for d in deps if d.exists())


def _built_for():
    """What the binding is compiled against, beside its own sources."""
    import torch
    return f"torch {torch.__version__}, python {sys.version_info.major}.{sys.version_info.minor}"


def _binding_stale():
    if not BINDING.exists() or not BINDING_STAMP.exists() or BINDING_STAMP.read_text() != _built_for():
        return True
    header = PKG.parent / "include" / "sigcomp_b200.h"
    return BINDING.stat().st_mtime <= max(f.stat().st_mtime for f in (BINDING_SOURCE, header, Path(__file__)))


def build_binding(force=False, verbose=False):
    """The torch binding of the int8 operators, linked against libsigcomp_b200.so beside it."""
    if not force and not _binding_stale():
        return BINDING
    import torch
    from torch.utils.cpp_extension import include_paths
    libs = Path(torch.__file__).resolve().parent / "lib"
    tmp = BINDING.with_suffix(".so.tmp")
    includes = [sysconfig.get_paths()["include"], *include_paths(), "/usr/local/cuda/include"]
    cmd = ["/usr/bin/g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f'-DSC_TORCH_VERSION="{torch.__version__}"',
           *(a for d in includes for a in ("-isystem", str(d))), str(BINDING_SOURCE), "-o", str(tmp), f"-L{PKG}",
           f"-l:{LIB.name}", f"-L{libs}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
           "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    os.replace(tmp, BINDING)
    BINDING_STAMP.parent.mkdir(exist_ok=True)
    BINDING_STAMP.write_text(_built_for())
    return BINDING


def build(force=False, verbose=False, jobs=4):
    if not force and not _stale():
        build_binding(force, verbose)
        return LIB
    objs = []
    build_dir = PKG / "_build"
    build_dir.mkdir(exist_ok=True)
    procs = []
    for src in SOURCES:
        obj = build_dir / (src + ".o")
        extra = ["-Xptxas", "-v"] if src in NO_SPILL_SOURCES else []
        cmd = [NVCC, *FLAGS, *extra, "-c", str(CSRC / src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd))
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(str(obj))
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed.append((src, out.decode()))
            continue
        if src in NO_SPILL_SOURCES:
            spills = spilling_kernels(out.decode())
            if spills:
                failed.append((src, "register spills in kernels that must not spill: " + "; ".join(
                    f"{name}: {st} B stored, {ld} B loaded" for name, st, ld in spills)))
                continue
        if verbose and out:
            print(out.decode())
    if failed:
        for src, out in failed:
            sys.stderr.write(f"--- {src}\n{out}\n")
        raise RuntimeError("nvcc failed for " + ", ".join(s for s, _ in failed))
    tmp = LIB.with_suffix(".so.tmp")
    subprocess.run([NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-ccbin", "/usr/bin/g++",
                    *objs, "-o", str(tmp), "-lcudart"], check=True)
    os.replace(tmp, LIB)
    build_binding(force, verbose)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
