"""Build libartemis_synth.so and libartemis_ops.so for gfx950 with hipcc (in-tree; cross-compiles without a
GPU)."""
from __future__ import annotations

import os
import subprocess

_PKG = os.path.dirname(os.path.abspath(__file__))
_ROOT = os.path.dirname(_PKG)
CSRC = os.path.join(_PKG, "csrc")
SRC = os.path.join(CSRC, "synth_kernels.hip")        # C ABI, host logic, direct kernels
TILES_SRC = os.path.join(CSRC, "synth_tiles.hip")     # LDS-staged kernels, one object per radius
DEVICE_HDR = os.path.join(CSRC, "synth_device.hpp")
TILE_RADII = (2, 4, 8, 14, 24)
BF16_RADII = (8, 14, 24)       # bf16 frames: smaller requests run the radius-8 kernels
INCLUDE = os.path.join(_ROOT, "include")
LIB_DIR = os.path.join(_PKG, "lib")
OBJ_DIR = os.path.join(LIB_DIR, "obj")
LIB_PATH = os.path.join(LIB_DIR, "libartemis_synth.so")
OPS_LIB_PATH = os.path.join(LIB_DIR, "libartemis_ops.so")
OPS_HOST_PATH = os.path.join(LIB_DIR, "_artemis_ops.so")   # ops_torch.cpp: the operators on torch tensors
OPS_TYPES = ("float", "__bf16", "_Float16")   # ops_attention_type.hip: one object per element type

HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-fPIC",
    "-munsafe-fp-atomics",  # fp32 atomicAdd -> one global_atomic_add_f32, no CAS loop
    # contract a*b+c only where one source expression spells it (not wherever the backend finds
    # a chance): every unrolled copy of the per-row arithmetic then rounds identically, so a pixel's
    # bits do not depend on which row slot of a tile computed it
    "-ffp-contract=on",
    "-Wall",
    # no packed fp32 instructions (v_pk_add_f32 and its like), which -O3 makes of ordinary float code: a precaution, since forms
    # of them are said to go wrong at times; nothing here shows it, and nothing is lost (1493 Mpix/s without, 1490 with)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]
OPS_FLAGS = HIPCC_FLAGS + ["-std=c++17"]


def _stale(path, prefix, header) -> bool:
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.startswith(prefix)] + [os.path.join(INCLUDE, header)]
    return any(os.path.getmtime(d) > t for d in deps)


def needs_build() -> bool:
    return _stale(LIB_PATH, "synth_", "artemis_synth.h")


def ops_need_build() -> bool:
    return _stale(OPS_LIB_PATH, "ops_", "artemis_ops.h") or _stale(OPS_HOST_PATH, "ops_torch", "artemis_ops.h")


def build(force: bool = False, verbose: bool = False, extra_flags=()) -> str:
    """Compile the HIP kernels + C ABI into artemis_amd/lib/libartemis_synth.so: the host
    translation unit and one object per tile radius in parallel, then one link."""
    if not force and not needs_build():
        return LIB_PATH
    jobs = [(SRC, os.path.join(OBJ_DIR, "synth_kernels.o"), [])]
    jobs += [(TILES_SRC, os.path.join(OBJ_DIR, f"synth_tiles_r{r}.o"), [f"-DSYNTH_TILE_R={r}"])
             for r in TILE_RADII]
    jobs += [(TILES_SRC, os.path.join(OBJ_DIR, f"synth_tiles_r{r}_bf16.o"),
              [f"-DSYNTH_TILE_R={r}", "-DSYNTH_TILE_BF16=1"]) for r in BF16_RADII]
    return _compile_and_link(jobs, HIPCC_FLAGS, extra_flags, LIB_PATH, verbose)


def build_ops(force: bool = False, verbose: bool = False, extra_flags=()) -> str:
    """The same for artemis_amd/lib/libartemis_ops.so: layer norm, windowed attention (one object per
    element type), AdamW; and the extension module around it."""
    if not force and not ops_need_build():
        return OPS_LIB_PATH
    from concurrent.futures import ThreadPoolExecutor
    with ThreadPoolExecutor(1) as pool:      # (the module's 45 s of torch headers beside the kernels)
        module = pool.submit(_compile_ops_host, OPS_HOST_PATH + ".o", verbose)
        _build_ops_lib(verbose, extra_flags)
        module.result()
    _run(["g++", "-shared", "-o", OPS_HOST_PATH, OPS_HOST_PATH + ".o", "-L" + LIB_DIR, "-lartemis_ops",
          *[f"-L{p}" for p in _torch_paths()[1]], "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10", "-lc10_hip",
          "-ltorch_python", "-Wl,-rpath,$ORIGIN"], verbose)
    os.remove(OPS_HOST_PATH + ".o")
    return OPS_LIB_PATH


def _torch_paths():
    from torch.utils import cpp_extension
    return cpp_extension.include_paths("cuda"), cpp_extension.library_paths("cuda")


def _compile_ops_host(obj, verbose):
    import sysconfig
    os.makedirs(LIB_DIR, exist_ok=True)
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-I" + INCLUDE,
          *[f"-I{p}" for p in (*_torch_paths()[0], sysconfig.get_paths()["include"])], "-c", "-o", obj,
          os.path.join(CSRC, "ops_torch.cpp")], verbose)


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("failed: " + " ".join(cmd) + "\n" + r.stderr)


def _build_ops_lib(verbose, extra_flags) -> str:
    jobs = [(os.path.join(CSRC, f"ops_{n}.hip"), os.path.join(OBJ_DIR, f"ops_{n}.o"), [])
            for n in ("host", "norm", "adamw", "attention")]
    jobs += [(os.path.join(CSRC, "ops_attention_type.hip"), os.path.join(OBJ_DIR, f"ops_attention_{t}.o"),
              [f"-DOPS_TYPE={t}"]) for t in OPS_TYPES]
    return _compile_and_link(jobs, OPS_FLAGS, extra_flags, OPS_LIB_PATH, verbose)


def _compile_and_link(jobs, flags, extra_flags, lib_path, verbose) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    hipcc = os.environ.get("HIPCC", "hipcc")
    workers = max(1, min(len(jobs), int(os.environ.get("MAX_JOBS", os.cpu_count() or 1))))

    def compile_one(job):
        src, obj, defs = job
        _run([hipcc, *flags, *extra_flags, *defs, "-I" + INCLUDE, "-c", "-o", obj, src], verbose)

    from concurrent.futures import ThreadPoolExecutor
    with ThreadPoolExecutor(workers) as pool:
        list(pool.map(compile_one, jobs))
    _run([hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", lib_path] + [j[1] for j in jobs], verbose)
    return lib_path


if __name__ == "__main__":
    print(build_ops(force=True, verbose=True))
    print(build(force=True, verbose=True))
