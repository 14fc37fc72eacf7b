"""Build and load ``libmegacute_b200.so`` (the CUDA kernel + C ABI of include/megacute_b200.h).

The library is compiled in-tree with nvcc for sm_100a only.  There is no fallback: if the library
is missing or does not load, every entry point of the runtime raises.
"""

from __future__ import annotations

import ctypes
import os
import pathlib
import shutil
import subprocess
import tempfile
import warnings

PKG = pathlib.Path(__file__).resolve().parent
CSRC = PKG / "csrc"
# MEGACUTE_B200_CHECK=1 selects the self-checking build (-DMK_CHECK: the kernel verifies the state of its shared-memory
# barriers before it arms or releases them and reports instead of going on; csrc/mk_device.cuh check_phase), a library
# file of its own beside the normal one.
CHECK_BUILD = os.environ.get("MEGACUTE_B200_CHECK") == "1"
LIB_PATH = pathlib.Path(os.environ.get("MEGACUTE_B200_LIB", PKG / ("libmegacute_b200_check.so" if CHECK_BUILD else "libmegacute_b200.so")))
# Relocatable device code: each op body is its own translation unit so that ptxas allocates its
# registers independently (csrc/ops.cuh says why).  -maxrregcount is the cap of a 12-warp CTA
# (three warps share one SM sub-partition's 16 K registers); callees in other translation units do
# not see the kernel's __launch_bounds__.
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-rdc=true",
              "-maxrregcount=168", "-shared", "-Xcompiler", "-fPIC"]
# Sources of kernels of their own, compiled as whole programs: in relocatable device code their functions would get the registers of a
# separate call, under the cap above.
WHOLE_PROGRAM = ("rotary.cu", "paged_attention.cu", "paged_attention_few.cu", "paged_attention_chunk.cu")
WHOLE_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-c"]

ST_WORDS = 16
MAX_PTRS = 12


class OpDesc(ctypes.Structure):
    """mk_op_desc (256 bytes)."""
    _fields_ = [("kind", ctypes.c_int32), ("flags", ctypes.c_int32), ("i", ctypes.c_int32 * 22),
                ("f", ctypes.c_float * 4), ("ptr", ctypes.c_uint64 * MAX_PTRS), ("ld", ctypes.c_int32 * MAX_PTRS)]


class Caps(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("sm_count", "cc_major", "cc_minor", "max_smem_optin", "kernel_smem",
                                              "kernel_threads", "kernel_regs", "reserved")]


class Batch(ctypes.Structure):
    """mk_batch"""
    _fields_ = [("pos", ctypes.c_void_p), ("starts", ctypes.c_void_p), ("pos_ld", ctypes.c_int64), ("rows", ctypes.c_int32),
                ("seqs", ctypes.c_int32)]


class Rotation(ctypes.Structure):
    """mk_rotation"""
    _fields_ = [("cos", ctypes.c_void_p), ("sin", ctypes.c_void_p), ("ld_cos", ctypes.c_int64), ("ld_sin", ctypes.c_int64),
                ("rows", ctypes.c_int32), ("columns", ctypes.c_int32), ("dtype", ctypes.c_int32), ("interleaved", ctypes.c_int32)]


class PagedCache(ctypes.Structure):
    """mk_paged_cache"""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("table", ctypes.c_void_p), ("ld_k", ctypes.c_int64),
                ("ld_v", ctypes.c_int64), ("table_ld", ctypes.c_int64), ("pages", ctypes.c_int32), ("page_size", ctypes.c_int32),
                ("table_cols", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("dtype", ctypes.c_int32)]


assert ctypes.sizeof(OpDesc) == 256
assert (ctypes.sizeof(Batch), ctypes.sizeof(Rotation), ctypes.sizeof(PagedCache)) == (32, 48, 72)

# name -> (restype, argtypes); every symbol include/megacute_b200.h declares
_P = ctypes.c_void_p
_I32P = ctypes.POINTER(ctypes.c_int32)
_BATCH, _ROTATION, _CACHE = ctypes.POINTER(Batch), ctypes.POINTER(Rotation), ctypes.POINTER(PagedCache)
SYMBOLS = {
    "mk_strerror": (ctypes.c_char_p, [ctypes.c_int]),
    "mk_last_cuda_error": (ctypes.c_char_p, []),
    "mk_query": (ctypes.c_int, [ctypes.c_int, ctypes.POINTER(Caps)]),
    "mk_program_create": (ctypes.c_int, [ctypes.c_int, _P, ctypes.c_int, _P, ctypes.c_int, _P, ctypes.c_int,
                                         ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.POINTER(_P)]),
    "mk_program_set_ops": (ctypes.c_int, [_P, _P, ctypes.c_int, _P]),
    "mk_program_set_direct": (ctypes.c_int, [_P, _P, ctypes.c_size_t, _P]),
    "mk_launch": (ctypes.c_int, [_P, _P]),
    "mk_program_set_timeout": (ctypes.c_int, [_P, ctypes.c_uint64]),
    "mk_program_status": (ctypes.c_int, [_P, _P, _I32P]),
    "mk_program_reset": (ctypes.c_int, [_P, _P]),
    "mk_program_epoch": (ctypes.c_int, [_P]),
    "mk_program_tcgen05_ops": (ctypes.c_int, [_P]),
    "mk_program_tcgen05_attention_ops": (ctypes.c_int, [_P]),
    "mk_program_packed_bytes": (ctypes.c_longlong, [_P]),
    "mk_program_refresh_weights": (ctypes.c_int, [_P, ctypes.c_void_p]),
    "mk_program_read_counters": (ctypes.c_int, [_P, _I32P, ctypes.c_int]),
    "mk_program_read_trace": (ctypes.c_int, [_P, _P, ctypes.c_size_t]),
    "mk_program_clear_trace": (ctypes.c_int, [_P, _P]),
    "mk_program_poke_wait": (ctypes.c_int, [_P, ctypes.c_int, ctypes.c_int, ctypes.c_int]),
    "mk_program_destroy": (None, [_P]),
    "mk_launch_noalloc": (ctypes.c_int, [ctypes.c_int, _P, ctypes.c_int, _P, ctypes.c_int, _P, ctypes.c_int, _P, ctypes.c_int,
                                         ctypes.c_int, ctypes.c_int, _P, _I32P]),
    "mk_noalloc_status": (ctypes.c_int, [ctypes.c_int, _P, _I32P]),
    "mk_rotary": (ctypes.c_int, [ctypes.c_int, _BATCH, _ROTATION, _P, ctypes.c_int64, _P, ctypes.c_int64, ctypes.c_int, ctypes.c_int,
                                 ctypes.c_int, _P]),
    "mk_paged_append": (ctypes.c_int, [ctypes.c_int, _BATCH, _ROTATION, _CACHE, _P, ctypes.c_int64, _P, ctypes.c_int64, ctypes.c_int, _P]),
    "mk_paged_attention_workspace": (ctypes.c_longlong, [ctypes.c_int] * 5),
    "mk_paged_attention": (ctypes.c_int, [ctypes.c_int, _BATCH, _CACHE, _P, ctypes.c_int64, _P, ctypes.c_int64, ctypes.c_int, ctypes.c_float,
                                          ctypes.c_int, ctypes.c_int, _P, ctypes.c_size_t, _P]),
    "mk_paged_attention_status": (ctypes.c_int, [ctypes.c_int, _P]),
    "mk_paged_attention_failures": (ctypes.c_int, [ctypes.c_int, _P, ctypes.POINTER(ctypes.c_uint32)]),
    "mk_argmax": (ctypes.c_int, [_P, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_longlong, _P, _P]),
}


def sources():
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + [PKG.parent / "include" / "megacute_b200.h"]


def needs_build() -> bool:
    return needs_build_of(LIB_PATH)


def needs_build_of(path: pathlib.Path) -> bool:
    return not path.exists() or any(s.stat().st_mtime > path.stat().st_mtime for s in sources())


def build(force: bool = False, verbose: bool = False, check: bool | None = None) -> pathlib.Path:
    """Compile the library with nvcc (cross-compiles without a GPU), and the Python module beside it, without which calls go through
    ctypes: where that does not compile there is a warning.  `check`: the -DMK_CHECK build (default: the one this process loads)."""
    check = CHECK_BUILD if check is None else check
    out = LIB_PATH if check == CHECK_BUILD else PKG / ("libmegacute_b200_check.so" if check else "libmegacute_b200.so")
    if force or needs_build_of(out):
        _build_library(out, check, verbose)
    try:
        build_binding(force)
    except (RuntimeError, OSError) as e:
        warnings.warn(f"{BINDING_PATH.name} was not built, its calls go through ctypes: {e}", RuntimeWarning, stacklevel=2)
    return out


def _build_library(out: pathlib.Path, check: bool, verbose: bool):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    define, loud = ["-DMK_CHECK"] if check else [], ["-Xptxas", "-v"] if verbose else []
    with tempfile.TemporaryDirectory() as tmp:
        objects = [pathlib.Path(tmp) / f"{name}.o" for name in WHOLE_PROGRAM]
        cmds = [[nvcc, *loud, *WHOLE_FLAGS, *define, "-o", str(o), str(CSRC / name)] for o, name in zip(objects, WHOLE_PROGRAM)]
        rest = [str(f) for f in sorted(CSRC.glob("*.cu")) if f.name not in WHOLE_PROGRAM]
        link = [nvcc, *loud, *NVCC_FLAGS, *define, "-o", str(out), *rest, *[str(o) for o in objects]]
        running = [subprocess.Popen(c, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True) for c in cmds]
        done = [(c, *r.communicate(), r.returncode) for c, r in zip(cmds, running)]
        if all(rc == 0 for *_, rc in done):
            r = subprocess.run(link, capture_output=True, text=True)
            done.append((link, r.stdout, r.stderr, r.returncode))
    for cmd, stdout, stderr, rc in done:
        if rc != 0:
            raise RuntimeError(f"nvcc failed:\n{' '.join(cmd)}\n{stdout}\n{stderr}")
        if verbose:
            print(stderr)


BINDING_PATH = PKG / "_binding.so"


def build_binding(force: bool = False) -> pathlib.Path:
    """Compile csrc/binding.cpp, the Python module through which paged.py calls the library, against this interpreter and its torch.  Raises
    if that fails, and leaves no module of older sources behind."""
    import sysconfig

    import torch
    source, header = CSRC / "binding.cpp", PKG.parent / "include" / "megacute_b200.h"
    built_for = f"{torch.__version__} {sysconfig.get_config_var('SOABI')}"
    stamp = BINDING_PATH.with_suffix(".built_for")
    if not force and BINDING_PATH.exists() and stamp.exists() and stamp.read_text() == built_for and \
            all(f.stat().st_mtime <= BINDING_PATH.stat().st_mtime for f in (source, header)):
        return BINDING_PATH
    for f in (stamp, BINDING_PATH):
        f.unlink(missing_ok=True)
    home = pathlib.Path(torch.__file__).resolve().parent
    nvcc = pathlib.Path(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc").resolve()
    includes = [header.parent, home / "include", home / "include" / "torch" / "csrc" / "api" / "include", nvcc.parent.parent / "include",
                sysconfig.get_paths()["include"]]
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f'-DMK_TORCH_VERSION="{torch.__version__}"',
           *[f"-I{i}" for i in includes], "-o", str(BINDING_PATH), str(source), f"-L{home / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    stamp.write_text(built_for)
    return BINDING_PATH


_lib = None


def load():
    """The loaded library.  Raises if it has not been built (no CPU fallback exists)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            if os.environ.get("MEGACUTE_B200_AUTOBUILD", "1") == "1" and (CSRC / "megakernel.cu").exists():
                build()
            else:
                raise RuntimeError(f"{LIB_PATH} is missing: run `python -c 'import __graft_entry__ as e; e.build()'`")
        lib = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in SYMBOLS.items():
            fn = getattr(lib, name)          # AttributeError if the library lacks a declared symbol
            fn.restype, fn.argtypes = res, args
        _lib = lib
    return _lib


class MegakernelError(RuntimeError):
    pass


class MegakernelTimeout(MegakernelError):
    """A device-side wait exceeded its limit; the launch ended with an error status."""


def check(rc: int, what: str = ""):
    if rc == 0:
        return
    lib = load()
    msg = lib.mk_strerror(rc).decode()
    if rc in (-1, -2):                   # CUDA errors and argument errors carry a detail message
        detail = lib.mk_last_cuda_error().decode()
        if detail:
            msg += ": " + detail
    raise MegakernelError(f"{what}: {msg}" if what else msg)
