"""Host-side binding of the gfx950 attention forward (``libfav4_bshd.so``).

Mirrors the reference harness's ctypes binding, ``benchmarks/bshd.py:18-20``
(``Args``) and ``:56-74`` (``Runner.call``): the same argument structure, the
same argument checks, the stream taken from torch's current stream, the scale
1/sqrt(128) by default, and a ``RuntimeError`` carrying the HIP status when the
C ABI returns non-zero.  The library is the product; this module only moves
pointers.  There is no fallback: if the library is missing, loading raises.
"""
from __future__ import annotations

import ctypes as C
import math
import os
import struct
import subprocess
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
LIB_PATH = ROOT / "build" / "libfav4_bshd.so"
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
D = 128
SCALE = 1 / math.sqrt(D)

HIPCC_FLAGS = [
    "-O3", "-std=c++17", "--offload-arch=gfx950", "-fPIC", "-shared", "-fvisibility=hidden",
    f"-I{INCLUDE}", f"-I{CSRC}",
    "-fgpu-flush-denormals-to-zero",
    # keep the compiler from emitting packed-FP32 VALU ops (v_pk_fma_f32 & co.)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # per-kernel VGPR / AGPR / SGPR counts, spills, LDS and occupancy, as
    # compiler remarks (the reference's scripts/build.sh:14-17 keeps the same)
    "-Rpass-analysis=kernel-resource-usage",
]
KAT_LIB_PATH = ROOT / "build" / "libfav4_loader_kat.so"
CEILING_LIB_PATH = ROOT / "build" / "libfav4_mfma_ceiling.so"
SERVING_LIB_PATH = ROOT / "build" / "libfav4_serving.so"
MX4_LIB_PATH = ROOT / "build" / "libfav4_mx4.so"
MX4_BLOCKS_PATH = ROOT / "build" / "fav4_mx4_blocks.so"
RESOURCE_LOG = ROOT / "build" / "resource-usage.txt"
MANIFEST = ROOT / "build" / "build-manifest.json"

class Args(C.Structure):
    """``struct Fav4Args`` (include/fav4_bshd.h): 5 pointers, 4 ints, 1 float."""
    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v", "o", "lse")] + [
        (n, C.c_int) for n in ("batch", "heads", "sq", "sk")] + [("scale", C.c_float)]


class VarlenArgs(C.Structure):
    """``struct Fav4VarlenArgs`` (include/fav4_bshd.h): 7 pointers, 7 ints, 1 float."""
    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v", "o", "lse", "cu_seqlens_q", "cu_seqlens_k")] + [
        (n, C.c_int) for n in ("batch", "heads", "kv_heads", "max_seqlen_q", "max_seqlen_k", "total_q",
                               "total_k")] + [("scale", C.c_float)]


class PagedArgs(C.Structure):
    """``struct Fav4PagedArgs`` (include/fav4_bshd.h): 8 pointers, 10 ints, 1 float."""
    _fields_ = [(n, C.c_void_p) for n in ("q", "k_cache", "v_cache", "o", "lse", "cu_seqlens_q", "seqlens_k",
                                          "block_table")] + [
        (n, C.c_int) for n in ("batch", "heads", "kv_heads", "max_seqlen_q", "max_seqlen_k", "total_q", "total_k",
                               "num_pages", "page_size", "max_pages_per_seq")] + [("scale", C.c_float)]


class AppendArgs(C.Structure):
    """``struct Fav4AppendArgs`` (include/fav4_serving.h): 12 pointers, 4 long longs, 10 ints."""
    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v", "q_out", "k_cache", "v_cache", "cos", "sin", "cu_seqlens_q",
                                          "seqlens_k", "block_table", "positions")] + [
        (n, C.c_longlong) for n in ("q_stride", "k_stride", "v_stride", "q_out_stride")] + [
        (n, C.c_int) for n in ("batch", "heads", "kv_heads", "total_q", "num_pages", "page_size", "max_pages_per_seq",
                               "rotary_dim", "rotary_rows", "interleaved")]


class PrefixArgs(C.Structure):
    """``struct Fav4PrefixArgs`` (include/fav4_serving.h): PagedArgs, 3 pointers, 2 ints."""
    _fields_ = [("paged", PagedArgs)] + [(n, C.c_void_p) for n in ("prefix_table", "prefix_lens",
                                                                   "cu_prefix_seqs")] + [
        (n, C.c_int) for n in ("num_prefixes", "max_pages_per_prefix")]


# The same two structs, for packing in one step.
_APPEND = struct.Struct("@12P4q10i")
_PREFIX = struct.Struct("@8P10if3P2i0P")


class Mx4AppendArgs(C.Structure):
    """``struct Fav4Mx4AppendArgs`` (include/fav4_mx4.h): AppendArgs, 2 pointers."""
    _fields_ = [("append", AppendArgs)] + [(n, C.c_void_p) for n in ("k_scales", "v_scales")]


class Mx4GatherArgs(C.Structure):
    """``struct Fav4Mx4GatherArgs`` (include/fav4_mx4.h): 9 pointers, 2 long longs, 6 ints."""
    _fields_ = [(n, C.c_void_p) for n in ("k_cache", "k_scales", "v_cache", "v_scales", "k", "v", "cu_seqlens_k",
                                          "starts", "block_table")] + [
        (n, C.c_longlong) for n in ("k_stride", "v_stride")] + [
        (n, C.c_int) for n in ("batch", "kv_heads", "total_k", "num_pages", "page_size", "max_pages_per_seq")]


class Mx4PagedArgs(C.Structure):
    """``struct Fav4Mx4PagedArgs`` (include/fav4_mx4.h): PagedArgs, 2 pointers."""
    _fields_ = [("paged", PagedArgs)] + [(n, C.c_void_p) for n in ("k_scales", "v_scales")]


class Strides(C.Structure):
    """``struct Fav4Strides`` (include/fav4_bshd.h): element strides of a [B, S, H, 128] view."""
    _fields_ = [(n, C.c_longlong) for n in ("batch", "seq", "head")]


def parse_resource_usage(text: str) -> dict:
    """Per-kernel fields of hipcc's kernel-resource-usage remarks."""
    table, name = {}, None
    for line in text.splitlines():
        if "remark:" not in line or "kernel-resource-usage" not in line:
            continue
        body = line.split("remark:", 1)[1].rsplit("[-Rpass-analysis", 1)[0].strip()
        key, _, val = body.partition(":")
        key, val = key.strip(), val.strip()
        if key == "Function Name":
            name = val
            table[name] = {}
        elif name is not None:
            table[name][key] = int(val) if val.lstrip("-").isdigit() else val
    return table


def _extension_command(src: Path) -> list:
    """The host compiler's command for a Python extension that reads torch tensors (ImportError or FileNotFoundError,
    naming what is missing, where it cannot be built)."""
    import shutil
    import sysconfig
    import torch
    home, python = Path(torch.__file__).parent, Path(sysconfig.get_paths()["include"])
    compiler = os.environ.get("CXX", "g++")
    if shutil.which(compiler) is None:
        raise FileNotFoundError(f"no compiler {compiler}")
    for header in (home / "include/torch/csrc/autograd/python_variable.h", python / "Python.h"):
        if not header.exists():
            raise FileNotFoundError(f"no header {header}")
    system = ["/opt/rocm/include", home / "include", home / "include/torch/csrc/api/include", python]
    return [compiler, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            "-D__HIP_PLATFORM_AMD__", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            f'-DFAV4_TORCH="{torch.__version__}"', f"-I{INCLUDE}",
            *(x for d in system for x in ("-isystem", str(d))), str(src), f"-L{home / 'lib'}", "-ltorch_python",
            "-ltorch_cpu", "-lc10"]


def build_library(out: Path = LIB_PATH, verbose: bool = False) -> Path:
    """Compile ``csrc/bshd.hip`` for gfx950 into ``build/libfav4_bshd.so``, the
    serving operators ``csrc/serving.hip`` into ``build/libfav4_serving.so``, those of
    4-bit caches ``csrc/mx4.hip`` into ``build/libfav4_mx4.so`` and their binding's argument
    blocks ``csrc/mx4_blocks.cpp`` into ``build/fav4_mx4_blocks.so``, the loader probe
    ``csrc/loader_kat.hip`` into ``build/libfav4_loader_kat.so`` (a test library) and the
    MFMA-only probe ``csrc/mfma_ceiling.hip`` into
    ``build/libfav4_mfma_ceiling.so`` (a measurement library, read by
    ``bench.py --mfma-ceiling``), keep the compiler's kernel-resource-usage remarks in
    ``build/resource-usage.txt`` and write ``build/build-manifest.json``
    (toolchain, flags, source and library sha256, per-kernel resources).

    The extension alone needs torch, its headers and a host compiler.  Where one of them is
    missing it is left out, with a warning, and loading it says why."""
    import hashlib
    import json
    import platform
    import time
    import warnings
    out.parent.mkdir(parents=True, exist_ok=True)
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    jobs = {out: CSRC / "bshd.hip", SERVING_LIB_PATH: CSRC / "serving.hip", MX4_LIB_PATH: CSRC / "mx4.hip",
            KAT_LIB_PATH: CSRC / "loader_kat.hip", CEILING_LIB_PATH: CSRC / "mfma_ceiling.hip"}
    commands = {lib: [hipcc, *HIPCC_FLAGS, str(src)] for lib, src in jobs.items()}
    left_out, extension_build = {}, None
    extension = CSRC / "mx4_blocks.cpp"
    MX4_BLOCKS_PATH.unlink(missing_ok=True)       # an earlier build's may pack other argument blocks
    try:
        commands[MX4_BLOCKS_PATH] = _extension_command(extension)
        import torch
        jobs[MX4_BLOCKS_PATH] = extension
        extension_build = {"command": commands[MX4_BLOCKS_PATH], "torch": torch.__version__}
    except (ImportError, FileNotFoundError) as e:
        left_out[MX4_BLOCKS_PATH.name] = str(e)
        warnings.warn(f"{MX4_BLOCKS_PATH.name} is left out: {e}")
    procs = {}
    for lib, command in commands.items():
        tmp = lib.with_suffix(".so.tmp")
        procs[lib] = (tmp, subprocess.Popen([*command, "-o", str(tmp)],
                                            stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True))
    remarks = []
    for lib, (tmp, proc) in procs.items():        # the extension last: the libraries are in place if it fails
        _, err = proc.communicate()
        if proc.returncode != 0:
            raise RuntimeError(f"{Path(commands[lib][0]).name} failed ({proc.returncode}) on {jobs[lib].name}:\n{err[-4000:]}")
        if verbose and err:
            print(err)
        remarks.append(err)
        os.replace(tmp, lib)
    text = "\n".join(remarks)
    RESOURCE_LOG.write_text(text)
    sha = lambda p: hashlib.sha256(Path(p).read_bytes()).hexdigest()
    version = subprocess.run([hipcc, "--version"], capture_output=True, text=True).stdout
    sources = sorted(p for ext in ("hip", "hpp", "cpp") for p in CSRC.glob(f"*.{ext}")) + sorted(INCLUDE.glob("*.h"))
    manifest = {
        "built_at": time.strftime("%Y-%m-%dT%H:%M:%SZ", time.gmtime()),
        "host": platform.node(),
        "hipcc": hipcc, "hipcc_version": [ln for ln in version.splitlines() if ln.strip()][:3],
        "flags": HIPCC_FLAGS,
        "sources": {str(p.relative_to(ROOT)): sha(p) for p in sources},
        "libraries": {lib.name: {"sha256": sha(lib), "bytes": lib.stat().st_size, "source": jobs[lib].name}
                      for lib in jobs},
        "left_out": left_out,
        "extension": extension_build,
        "kernel_resources": parse_resource_usage(text),
    }
    MANIFEST.write_text(json.dumps(manifest, indent=1))
    return out


_LIB = None


def load_library(path: Path = LIB_PATH) -> C.CDLL:
    """Load the built library (raises OSError if it is missing).

    PyTorch-ROCm wheels bundle their own HIP and HSA runtimes. Torch is
    therefore imported first when it is installed. The library's
    libamdhip64.so.7 dependency then binds to the runtime already in the
    process, and torch's streams and the library share one runtime.
    Loaded the other way round, the process holds two HIP runtimes, and
    the library's launches fail with hipErrorNoDevice (100)."""
    global _LIB
    if _LIB is None or Path(_LIB._name) != Path(path):
        if not Path(path).exists():
            raise OSError(f"{path} not built; run __graft_entry__.build() first")
        try:
            import torch  # noqa: F401  (binds the library to torch's HIP runtime)
        except ImportError:
            pass
        lib = C.CDLL(str(path))
        lib.fav4_bshd_forward.argtypes = [C.POINTER(Args), C.c_int, C.c_int, C.c_void_p]
        lib.fav4_bshd_forward.restype = C.c_int
        lib.fav4_bshd_select_config.argtypes = [C.POINTER(Args)]
        lib.fav4_bshd_select_config.restype = C.c_int
        lib.fav4_bshd_select_config_masked.argtypes = [C.POINTER(Args), C.c_int]
        lib.fav4_bshd_select_config_masked.restype = C.c_int
        lib.fav4_bshd_forward_splitkv.argtypes = [C.POINTER(Args), C.c_int, C.c_int, C.c_void_p, C.c_size_t,
                                                  C.c_void_p]
        lib.fav4_bshd_forward_splitkv.restype = C.c_int
        lib.fav4_bshd_splitkv_workspace_size.argtypes = [C.POINTER(Args), C.c_int, C.c_int]
        lib.fav4_bshd_splitkv_workspace_size.restype = C.c_longlong
        lib.fav4_bshd_splitkv_select.argtypes = [C.POINTER(Args), C.c_int]
        lib.fav4_bshd_splitkv_select.restype = C.c_int
        lib.fav4_bshd_forward_splitkv_gqa.argtypes = [C.POINTER(Args), C.c_int, C.c_int, C.c_int, C.c_void_p,
                                                      C.c_size_t, C.c_void_p]
        lib.fav4_bshd_forward_splitkv_gqa.restype = C.c_int
        lib.fav4_bshd_splitkv_gqa_workspace_size.argtypes = [C.POINTER(Args), C.c_int, C.c_int, C.c_int]
        lib.fav4_bshd_splitkv_gqa_workspace_size.restype = C.c_longlong
        lib.fav4_bshd_splitkv_gqa_select.argtypes = [C.POINTER(Args), C.c_int, C.c_int]
        lib.fav4_bshd_splitkv_gqa_select.restype = C.c_int
        lib.fav4_bshd_forward_splitkv_gqa_noalloc.argtypes = [C.POINTER(Args), C.c_int, C.c_int, C.c_int,
                                                              C.c_void_p]
        lib.fav4_bshd_forward_splitkv_gqa_noalloc.restype = C.c_int
        lib.fav4_bshd_forward_gqa.argtypes = [C.POINTER(Args), C.c_int, C.c_int, C.c_int, C.c_void_p]
        lib.fav4_bshd_forward_gqa.restype = C.c_int
        lib.fav4_bshd_forward_strided.argtypes = [C.POINTER(Args), C.c_int] + [C.POINTER(Strides)] * 4 + [
            C.c_int, C.c_int, C.c_void_p]
        lib.fav4_bshd_forward_strided.restype = C.c_int
        lib.fav4_bshd_forward_varlen.argtypes = [C.POINTER(VarlenArgs), C.c_int, C.c_void_p]
        lib.fav4_bshd_forward_varlen.restype = C.c_int
        lib.fav4_bshd_forward_splitkv_varlen.argtypes = [C.POINTER(VarlenArgs), C.c_int, C.c_int, C.c_void_p,
                                                         C.c_size_t, C.c_void_p]
        lib.fav4_bshd_forward_splitkv_varlen.restype = C.c_int
        lib.fav4_bshd_splitkv_varlen_workspace_size.argtypes = [C.POINTER(VarlenArgs), C.c_int, C.c_int]
        lib.fav4_bshd_splitkv_varlen_workspace_size.restype = C.c_longlong
        lib.fav4_bshd_splitkv_varlen_select.argtypes = [C.POINTER(VarlenArgs), C.c_int]
        lib.fav4_bshd_splitkv_varlen_select.restype = C.c_int
        lib.fav4_bshd_forward_splitkv_paged.argtypes = [C.POINTER(PagedArgs), C.c_int, C.c_int, C.c_void_p,
                                                        C.c_size_t, C.c_void_p]
        lib.fav4_bshd_forward_splitkv_paged.restype = C.c_int
        lib.fav4_bshd_splitkv_paged_workspace_size.argtypes = [C.POINTER(PagedArgs), C.c_int, C.c_int]
        lib.fav4_bshd_splitkv_paged_workspace_size.restype = C.c_longlong
        lib.fav4_bshd_splitkv_paged_select.argtypes = [C.POINTER(PagedArgs), C.c_int]
        lib.fav4_bshd_splitkv_paged_select.restype = C.c_int
        _LIB = lib
    return _LIB


_SERVING = None


def load_serving_library(path: Path = SERVING_LIB_PATH) -> C.CDLL:
    """Load the serving operators' library (raises OSError if it is missing); torch first, as load_library says."""
    global _SERVING
    if _SERVING is None or Path(_SERVING._name) != Path(path):
        if not Path(path).exists():
            raise OSError(f"{path} not built; run __graft_entry__.build() first")
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        lib = C.CDLL(str(path))
        # The argument blocks are passed as packed bytes or by reference.
        lib.fav4_bshd_append_paged.argtypes = [C.c_void_p, C.c_void_p]
        lib.fav4_bshd_append_paged.restype = C.c_int
        lib.fav4_bshd_forward_prefix_paged.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_size_t, C.c_void_p]
        lib.fav4_bshd_forward_prefix_paged.restype = C.c_int
        lib.fav4_bshd_prefix_paged_workspace_size.argtypes = [C.c_void_p, C.c_int]
        lib.fav4_bshd_prefix_paged_workspace_size.restype = C.c_longlong
        _SERVING = lib
    return _SERVING


_MX4 = None


def load_mx4_library(path: Path = MX4_LIB_PATH) -> C.CDLL:
    """Load the library of the 4-bit caches' operators (raises OSError if it is missing); torch first, as load_library
    says."""
    global _MX4
    if _MX4 is None or Path(_MX4._name) != Path(path):
        if not Path(path).exists():
            raise OSError(f"{path} not built; run __graft_entry__.build() first")
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        lib = C.CDLL(str(path))
        # The argument blocks are passed as packed bytes or by reference.
        lib.fav4_bshd_append_paged_mx4.argtypes = [C.c_void_p, C.c_void_p]
        lib.fav4_bshd_append_paged_mx4.restype = C.c_int
        lib.fav4_bshd_gather_paged_mx4.argtypes = [C.c_void_p, C.c_void_p]
        lib.fav4_bshd_gather_paged_mx4.restype = C.c_int
        lib.fav4_bshd_forward_paged_mx4.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_size_t, C.c_void_p]
        lib.fav4_bshd_forward_paged_mx4.restype = C.c_int
        lib.fav4_bshd_paged_mx4_workspace_size.argtypes = [C.c_void_p, C.c_int]
        lib.fav4_bshd_paged_mx4_workspace_size.restype = C.c_longlong
        _MX4 = lib
    return _MX4


_MX4_BLOCKS = None


def _left_out(path: Path) -> str:
    """Why the last build left a library out (empty: it did not)."""
    import json
    try:
        why = json.loads(MANIFEST.read_text()).get("left_out", {}).get(Path(path).name)
    except (OSError, ValueError):
        why = None
    return f" ({why})" if why else ""


def load_mx4_blocks(path: Path = MX4_BLOCKS_PATH):
    """The module that checks torch tensors and packs them into the argument blocks of the 4-bit caches' calls (raises
    OSError if it is missing, or was built against another torch than the one in the process)."""
    global _MX4_BLOCKS
    if _MX4_BLOCKS is None:
        if not Path(path).exists():
            raise OSError(f"{path} not built{_left_out(path)}; run __graft_entry__.build() first")
        import importlib.machinery
        import importlib.util
        import torch
        loader = importlib.machinery.ExtensionFileLoader("fav4_mx4_blocks", str(path))
        try:
            module = importlib.util.module_from_spec(importlib.util.spec_from_loader("fav4_mx4_blocks", loader))
            loader.exec_module(module)
        except ImportError as e:
            raise OSError(f"{path} does not load with torch {torch.__version__} ({e}); run __graft_entry__.build() again") from e
        if module.torch_version != torch.__version__:
            raise OSError(f"{path} was built against torch {module.torch_version}, not {torch.__version__}; run "
                          "__graft_entry__.build() again")
        _MX4_BLOCKS = module
    return _MX4_BLOCKS


class Runner:
    """ctypes runner with the reference harness's call signature (bshd.py:56-74)."""

    def __init__(self, path: Path = LIB_PATH):
        self.hip = load_library(path)

    def args(self, q, k, v, o, lse, scale=None, kv_heads=None) -> Args:
        import torch
        assert all(x.dtype == torch.bfloat16 and x.is_cuda and x.is_contiguous() for x in (q, k, v, o))
        b, sq, h, d = q.shape
        kvh = h if kv_heads is None else kv_heads
        assert d == D and k.shape == v.shape and k.shape[0] == b and tuple(k.shape[2:]) == (kvh, d)
        assert o.shape == q.shape
        assert lse is None or (tuple(lse.shape) == (b, h, sq) and lse.is_contiguous()
                               and lse.dtype == torch.float32)
        return Args(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                    lse.data_ptr() if lse is not None else None,
                    b, h, sq, k.shape[1], 1 / math.sqrt(d) if scale is None else scale)

    def call(self, q, k, v, o, lse, causal, config=0, scale=None, stream=None):
        import torch
        a = self.args(q, k, v, o, lse, scale)
        if stream is None:
            stream = torch.cuda.current_stream().cuda_stream
        status = self.hip.fav4_bshd_forward(C.byref(a), int(causal), int(config), stream)
        if status:
            raise RuntimeError(f"config {config}: HIP status {status}")

    def call_gqa(self, q, k, v, o, lse, causal, config=0, scale=None, stream=None):
        """fav4_bshd_forward_gqa: K/V heads = k.shape[2] (must divide q's heads)."""
        import torch
        a = self.args(q, k, v, o, lse, scale, kv_heads=k.shape[2])
        if stream is None:
            stream = torch.cuda.current_stream().cuda_stream
        status = self.hip.fav4_bshd_forward_gqa(C.byref(a), int(k.shape[2]), int(causal), int(config), stream)
        if status:
            raise RuntimeError(f"gqa config {config}: HIP status {status}")

    def select_config(self, q, k, causal=None) -> int:
        """Config ID that config 0 resolves to: the reference's dense query
        when `causal` is None, else fav4_bshd_select_config_masked."""
        b, sq, h, _ = q.shape
        a = Args(None, None, None, None, None, b, h, sq, k.shape[1], 1 / math.sqrt(D))
        if causal is None:
            return self.hip.fav4_bshd_select_config(C.byref(a))
        return self.hip.fav4_bshd_select_config_masked(C.byref(a), int(causal))

    # ---- split-KV (fav4_bshd_forward_splitkv; no reference counterpart) ----
    @staticmethod
    def shape_args(batch, heads, sq, sk) -> Args:
        return Args(None, None, None, None, None, batch, heads, sq, sk, 1 / math.sqrt(D))

    def splitkv_select(self, batch, heads, sq, sk, causal, kv_heads=None) -> int:
        a = self.shape_args(batch, heads, sq, sk)
        if kv_heads is None:
            return self.hip.fav4_bshd_splitkv_select(C.byref(a), int(causal))
        return self.hip.fav4_bshd_splitkv_gqa_select(C.byref(a), int(kv_heads), int(causal))

    def splitkv_workspace_size(self, batch, heads, sq, sk, causal, splits=0, kv_heads=None) -> int:
        a = self.shape_args(batch, heads, sq, sk)
        if kv_heads is None:
            return self.hip.fav4_bshd_splitkv_workspace_size(C.byref(a), int(causal), int(splits))
        return self.hip.fav4_bshd_splitkv_gqa_workspace_size(C.byref(a), int(kv_heads), int(causal), int(splits))

    def call_splitkv(self, q, k, v, o, lse, causal, splits=0, workspace=None, scale=None, stream=None):
        """Split-KV forward; K/V heads = k.shape[2] (fewer than q's: the GQA
        entry point).  `workspace` is a CUDA tensor (any dtype, 256-byte
        aligned); None allocates one of the required size here (the library
        never allocates)."""
        import torch
        kvh = k.shape[2]
        gqa = kvh != q.shape[2]
        a = self.args(q, k, v, o, lse, scale, kv_heads=kvh)
        if workspace is None:
            if gqa:
                need = self.hip.fav4_bshd_splitkv_gqa_workspace_size(C.byref(a), int(kvh), int(causal), int(splits))
            else:
                need = self.hip.fav4_bshd_splitkv_workspace_size(C.byref(a), int(causal), int(splits))
            if need < 0:
                raise RuntimeError(f"splits {splits}: arguments rejected")
            workspace = torch.empty(max(need, 1), device=q.device, dtype=torch.uint8)
        nbytes = workspace.numel() * workspace.element_size()
        if stream is None:
            stream = torch.cuda.current_stream().cuda_stream
        if gqa:
            status = self.hip.fav4_bshd_forward_splitkv_gqa(C.byref(a), int(kvh), int(causal), int(splits),
                                                             workspace.data_ptr(), nbytes, stream)
        else:
            status = self.hip.fav4_bshd_forward_splitkv(C.byref(a), int(causal), int(splits), workspace.data_ptr(),
                                                         nbytes, stream)
        if status:
            raise RuntimeError(f"splitkv splits {splits}: HIP status {status}")
        return workspace

    def call_splitkv_noalloc(self, q, k, v, o, lse, causal, splits=0, scale=None, stream=None):
        """fav4_bshd_forward_splitkv_gqa_noalloc: split-KV with the library's own
        64 MiB per-device partials array (no workspace); K/V heads = k.shape[2]."""
        import torch
        kvh = k.shape[2]
        a = self.args(q, k, v, o, lse, scale, kv_heads=kvh)
        if stream is None:
            stream = torch.cuda.current_stream().cuda_stream
        status = self.hip.fav4_bshd_forward_splitkv_gqa_noalloc(C.byref(a), int(kvh), int(causal), int(splits),
                                                                 stream)
        if status:
            raise RuntimeError(f"splitkv noalloc splits {splits}: HIP status {status}")

    # ---- arbitrary strides (fav4_bshd_forward_strided; no reference counterpart) ----
    def call_strided(self, q, k, v, o, lse, causal, config=0, scale=None, stream=None):
        """q/o: [B, Sq, H, 128] and k/v: [B, Sk, KVH, 128] views with any strides whose last
        dimension is contiguous (e.g. ``x_bhsd.transpose(1, 2)``, ``qkv[:, :, 0]``);
        lse: FP32 [B, H, Sq] contiguous or None."""
        import torch
        for x in (q, k, v, o):
            assert x.dtype == torch.bfloat16 and x.is_cuda and x.dim() == 4 and x.shape[3] == D and x.stride(3) == 1
        b, sq, h, _ = q.shape
        assert o.shape == q.shape and k.shape == v.shape and k.shape[0] == b
        assert lse is None or (tuple(lse.shape) == (b, h, sq) and lse.is_contiguous() and lse.dtype == torch.float32)
        a = Args(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                 lse.data_ptr() if lse is not None else None, b, h, sq, k.shape[1],
                 1 / math.sqrt(D) if scale is None else scale)
        st = [Strides(x.stride(0), x.stride(1), x.stride(2)) for x in (q, k, v, o)]
        if stream is None:
            stream = torch.cuda.current_stream().cuda_stream
        status = self.hip.fav4_bshd_forward_strided(C.byref(a), int(k.shape[2]), *[C.byref(x) for x in st],
                                                    int(causal), int(config), stream)
        if status:
            raise RuntimeError(f"strided config {config}: HIP status {status}")

    # ---- packed variable-length sequences (fav4_bshd_forward_varlen; no reference counterpart) ----
    def varlen_args(self, q, k, v, o, lse, cu_q, cu_k, max_q, max_k, scale=None) -> VarlenArgs:
        """q/o: [total_q, heads, 128]; k/v: [total_k, kv_heads, 128] (BF16, contiguous);
        cu_q/cu_k: int32 [batch+1] on the device; lse: FP32 [heads, total_q] or None."""
        import torch
        assert all(x.dtype == torch.bfloat16 and x.is_cuda and x.is_contiguous() for x in (q, k, v, o))
        assert q.dim() == 3 and q.shape[2] == D and o.shape == q.shape and k.shape == v.shape and k.dim() == 3
        assert all(c.dtype == torch.int32 and c.is_cuda and c.is_contiguous() and c.dim() == 1 for c in (cu_q, cu_k))
        assert cu_q.numel() == cu_k.numel() >= 2
        tq, h, _ = q.shape
        assert lse is None or (tuple(lse.shape) == (h, tq) and lse.is_contiguous() and lse.dtype == torch.float32)
        return VarlenArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                          lse.data_ptr() if lse is not None else None, cu_q.data_ptr(), cu_k.data_ptr(),
                          cu_q.numel() - 1, h, k.shape[1], int(max_q), int(max_k), tq, k.shape[0],
                          1 / math.sqrt(D) if scale is None else scale)

    def call_varlen(self, q, k, v, o, lse, cu_q, cu_k, max_q, max_k, causal, scale=None, stream=None):
        import torch
        a = self.varlen_args(q, k, v, o, lse, cu_q, cu_k, max_q, max_k, scale)
        if stream is None:
            stream = torch.cuda.current_stream().cuda_stream
        status = self.hip.fav4_bshd_forward_varlen(C.byref(a), int(causal), stream)
        if status:
            raise RuntimeError(f"varlen: HIP status {status}")

    # ---- split-KV of packed batches (fav4_bshd_forward_splitkv_varlen; no reference counterpart) ----
    @staticmethod
    def varlen_shape_args(batch, heads, kv_heads, max_q, max_k, total_q, total_k) -> VarlenArgs:
        """Shape-only arguments for the select / workspace queries (no buffers)."""
        return VarlenArgs(None, None, None, None, None, None, None, batch, heads, kv_heads, max_q, max_k,
                          total_q, total_k, 1 / math.sqrt(D))

    def splitkv_varlen_select(self, batch, heads, kv_heads, max_q, max_k, total_q, total_k, causal) -> int:
        a = self.varlen_shape_args(batch, heads, kv_heads, max_q, max_k, total_q, total_k)
        return self.hip.fav4_bshd_splitkv_varlen_select(C.byref(a), int(causal))

    def splitkv_varlen_workspace_size(self, batch, heads, kv_heads, max_q, max_k, total_q, total_k, causal,
                                      splits=0) -> int:
        a = self.varlen_shape_args(batch, heads, kv_heads, max_q, max_k, total_q, total_k)
        return self.hip.fav4_bshd_splitkv_varlen_workspace_size(C.byref(a), int(causal), int(splits))

    def call_splitkv_varlen(self, q, k, v, o, lse, cu_q, cu_k, max_q, max_k, causal, splits=0, workspace=None,
                            scale=None, stream=None):
        """Split-KV over packed sequences; tensors as for call_varlen.  `workspace`
        as for call_splitkv (None: allocated here)."""
        import torch
        a = self.varlen_args(q, k, v, o, lse, cu_q, cu_k, max_q, max_k, scale)
        if workspace is None:
            need = self.hip.fav4_bshd_splitkv_varlen_workspace_size(C.byref(a), int(causal), int(splits))
            if need < 0:
                raise RuntimeError(f"splitkv varlen splits {splits}: arguments rejected")
            workspace = torch.empty(max(need, 1), device=q.device, dtype=torch.uint8)
        nbytes = workspace.numel() * workspace.element_size()
        if stream is None:
            stream = torch.cuda.current_stream().cuda_stream
        status = self.hip.fav4_bshd_forward_splitkv_varlen(C.byref(a), int(causal), int(splits),
                                                            workspace.data_ptr(), nbytes, stream)
        if status:
            raise RuntimeError(f"splitkv varlen splits {splits}: HIP status {status}")
        return workspace


    # ---- split-KV decode over paged K/V caches (no reference counterpart) ----
    def paged_args(self, q, k_cache, v_cache, o, lse, cu_q, seqlens_k, block_table, max_q, max_k, total_k=None,
                   scale=None) -> PagedArgs:
        """q/o: [total_q, heads, 128]; k_cache/v_cache: [num_pages, page_size, kv_heads, 128] (BF16,
        contiguous); cu_q: int32 [batch+1]; seqlens_k: int32 [batch]; block_table: int32
        [batch, max_pages_per_seq] (device tensors); lse: FP32 [heads, total_q] or None.  total_k
        (cached keys over the batch) only steers Auto: max_k * batch says that every sequence has
        max_k keys; None (not known) passes one less than that for two sequences or more."""
        import torch
        assert all(x.dtype == torch.bfloat16 and x.is_cuda and x.is_contiguous() for x in (q, k_cache, v_cache, o))
        assert q.dim() == 3 and q.shape[2] == D and o.shape == q.shape
        assert k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.shape[3] == D
        assert all(c.dtype == torch.int32 and c.is_cuda and c.is_contiguous() for c in (cu_q, seqlens_k, block_table))
        assert block_table.dim() == 2 and cu_q.numel() == seqlens_k.numel() + 1 == block_table.shape[0] + 1
        tq, h, _ = q.shape
        assert lse is None or (tuple(lse.shape) == (h, tq) and lse.is_contiguous() and lse.dtype == torch.float32)
        b = seqlens_k.numel()
        if total_k is None:
            total_k = int(max_k) * b - (b > 1)
        return PagedArgs(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(),
                         lse.data_ptr() if lse is not None else None, cu_q.data_ptr(), seqlens_k.data_ptr(),
                         block_table.data_ptr(), b, h, k_cache.shape[2], int(max_q), int(max_k), tq,
                         int(total_k), k_cache.shape[0], k_cache.shape[1],
                         block_table.shape[1], 1 / math.sqrt(D) if scale is None else scale)

    @staticmethod
    def paged_shape_args(batch, heads, kv_heads, max_q, max_k, total_q, total_k, page_size, max_pages,
                         num_pages) -> PagedArgs:
        """Shape-only arguments for the select / workspace queries (no buffers)."""
        return PagedArgs(None, None, None, None, None, None, None, None, batch, heads, kv_heads, max_q, max_k, total_q,
                         total_k, num_pages, page_size, max_pages, 1 / math.sqrt(D))

    def splitkv_paged_select(self, batch, heads, kv_heads, max_q, max_k, total_q, total_k, page_size, max_pages,
                             num_pages, causal=0) -> int:
        """Auto chunk count for call_splitkv_paged with the same mask (0 dense, 2 bottom-right)."""
        a = self.paged_shape_args(batch, heads, kv_heads, max_q, max_k, total_q, total_k, page_size, max_pages,
                                  num_pages)
        return self.hip.fav4_bshd_splitkv_paged_select(C.byref(a), int(causal))

    def splitkv_paged_workspace_size(self, batch, heads, kv_heads, max_q, max_k, total_q, total_k, page_size,
                                     max_pages, num_pages, splits=0, causal=0) -> int:
        """Workspace bytes of call_splitkv_paged with the same mask (0 dense, 2 bottom-right):
        the chunk plan, and so the size, depends on it."""
        a = self.paged_shape_args(batch, heads, kv_heads, max_q, max_k, total_q, total_k, page_size, max_pages,
                                  num_pages)
        return self.hip.fav4_bshd_splitkv_paged_workspace_size(C.byref(a), int(causal), int(splits))

    def call_splitkv_paged(self, q, k_cache, v_cache, o, lse, cu_q, seqlens_k, block_table, max_q, max_k,
                           splits=0, workspace=None, total_k=None, scale=None, stream=None, causal=0):
        """Decode over paged caches (causal 0 = dense, 2 = bottom-right); `workspace` as for
        call_splitkv (None: allocated here)."""
        import torch
        a = self.paged_args(q, k_cache, v_cache, o, lse, cu_q, seqlens_k, block_table, max_q, max_k, total_k, scale)
        if workspace is None:
            need = self.hip.fav4_bshd_splitkv_paged_workspace_size(C.byref(a), int(causal), int(splits))
            if need < 0:
                raise RuntimeError(f"splitkv paged splits {splits}: arguments rejected")
            workspace = torch.empty(max(need, 1), device=q.device, dtype=torch.uint8)
        nbytes = workspace.numel() * workspace.element_size()
        if stream is None:
            stream = torch.cuda.current_stream().cuda_stream
        status = self.hip.fav4_bshd_forward_splitkv_paged(C.byref(a), int(causal), int(splits), workspace.data_ptr(),
                                                           nbytes, stream)
        if status:
            raise RuntimeError(f"splitkv paged splits {splits}: HIP status {status}")
        return workspace

    # ---- serving operators on paged K/V caches (include/fav4_serving.h; no reference counterpart) ----
    # A decode step is a few microseconds of GPU time, so these calls keep the host's part short: the argument blocks
    # are packed in one step, and every tensor's properties are read once.
    @property
    def serving(self) -> C.CDLL:
        lib = self.__dict__.get("_serving")
        if lib is None:
            lib = self._serving = load_serving_library()
        return lib

    @staticmethod
    def _stream(torch, device, stream):
        """The stream to launch on (None: torch's current one), with `device`, the tensors', current."""
        if device < 0:
            raise ValueError("tensors on the host: the library works on GPU memory")
        if device != torch.cuda.current_device():
            raise ValueError(f"tensors on cuda:{device}, current device cuda:{torch.cuda.current_device()}")
        if stream is not None:
            return stream
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)       # without a Stream object
        return raw(device) if raw is not None else torch.cuda.current_stream().cuda_stream

    @staticmethod
    def _allocation_stream(torch, stream):
        """torch's stream for a raw handle (None: its current one), to allocate on; 0 is the default stream, for which
        ExternalStream would make a stream of its own."""
        if stream is None:
            return None
        return torch.cuda.ExternalStream(stream) if stream else torch.cuda.default_stream()

    @staticmethod
    def _append_block(torch, q, k, v, q_out, k_cache, v_cache, cu_q, seqlens_k, block_table, cos, sin, interleaved,
                      positions) -> bytes:
        bf16, i32, dev = torch.bfloat16, torch.int32, k.get_device()
        num_pages, page_size, kv_heads, d = caches = k_cache.shape
        assert d == D and v_cache.shape == caches and k_cache.dtype is bf16 and v_cache.dtype is bf16
        assert k_cache.is_contiguous() and v_cache.is_contiguous()
        batch, pages = block_table.shape
        assert cu_q.dtype is i32 and seqlens_k.dtype is i32 and block_table.dtype is i32
        assert cu_q.shape == (batch + 1,) and seqlens_k.shape == (batch,)
        assert cu_q.is_contiguous() and seqlens_k.is_contiguous() and block_table.is_contiguous()
        assert dev == k_cache.get_device() == v_cache.get_device() == v.get_device() == cu_q.get_device() \
            == seqlens_k.get_device() == block_table.get_device(), "all tensors on one device"
        # Rows: any stride between tokens (a single token has none that counts), heads and dims contiguous.
        tokens = k.shape[0]
        assert k.shape == v.shape == (tokens, kv_heads, D) and k.dtype is bf16 and v.dtype is bf16
        k_stride, k1, k2 = k.stride()
        v_stride, v1, v2 = v.stride()
        assert k2 == v2 == 1 and (kv_heads == 1 or k1 == v1 == D)
        heads, q_stride, o_stride, q_ptr, o_ptr = 1, 0, 0, 0, 0
        assert (q is None) == (q_out is None)
        if q is not None:
            heads = q.shape[1]
            assert q.shape == q_out.shape == (tokens, heads, D) and q.dtype is bf16 and q_out.dtype is bf16
            assert q.get_device() == q_out.get_device() == dev, "all tensors on one device"
            q_stride, q1, q2 = q.stride()
            o_stride, o1, o2 = q_out.stride()
            assert q2 == o2 == 1 and (heads == 1 or q1 == o1 == D)
            q_ptr, o_ptr = q.data_ptr(), q_out.data_ptr()
        if tokens == 1:
            k_stride = v_stride = kv_heads * D
            q_stride = o_stride = heads * D
        rows = half = c_ptr = s_ptr = p_ptr = 0
        assert (cos is None) == (sin is None)
        if cos is not None:
            rows, half = cos.shape
            assert sin.shape == cos.shape and cos.dtype is sin.dtype is torch.float32
            assert cos.is_contiguous() and sin.is_contiguous() and cos.get_device() == sin.get_device() == dev
            c_ptr, s_ptr = cos.data_ptr(), sin.data_ptr()
        if positions is not None:
            assert positions.dtype is i32 and positions.shape == (tokens,) and positions.is_contiguous()
            assert positions.get_device() == dev, "all tensors on one device"
            p_ptr = positions.data_ptr()
        return _APPEND.pack(q_ptr, k.data_ptr(), v.data_ptr(), o_ptr, k_cache.data_ptr(), v_cache.data_ptr(), c_ptr,
                            s_ptr, cu_q.data_ptr(), seqlens_k.data_ptr(), block_table.data_ptr(), p_ptr, q_stride,
                            k_stride, v_stride, o_stride, batch, heads, kv_heads, tokens, num_pages, page_size, pages,
                            2 * half, rows, 1 if interleaved else 0)

    def call_append_paged(self, q, k, v, q_out, k_cache, v_cache, cu_q, seqlens_k, block_table, cos=None, sin=None,
                          interleaved=False, positions=None, stream=None):
        """fav4_bshd_append_paged: store the new tokens' K and V in the caches, K and Q rotated by position on the way.
        q/q_out: [total_q, heads, 128] or both None; k/v: [total_q, kv_heads, 128] (BF16; any stride between tokens);
        k_cache/v_cache: [num_pages, page_size, kv_heads, 128] (BF16, contiguous); cu_q: int32 [batch+1]; seqlens_k:
        int32 [batch], new tokens included; block_table: int32 [batch, max_pages]; cos/sin: FP32 [rows, rotary_dim / 2]
        or None (no rotation); positions: int32 [total_q] or None (a token's slot).  q_out may be q: in place."""
        import torch
        block = self._append_block(torch, q, k, v, q_out, k_cache, v_cache, cu_q, seqlens_k, block_table, cos, sin,
                                   interleaved, positions)
        status = self.serving.fav4_bshd_append_paged(block, self._stream(torch, k.get_device(), stream))
        if status:
            raise RuntimeError(f"append paged: HIP status {status}")

    @staticmethod
    def _prefix_block(torch, q, k_cache, v_cache, o, lse, cu_q, seqlens_k, block_table, prefix_table, prefix_lens,
                      cu_prefix_seqs, max_q, max_k, total_k, scale) -> bytes:
        bf16, i32, dev = torch.bfloat16, torch.int32, q.get_device()
        num_pages, page_size, kv_heads, d = caches = k_cache.shape
        assert d == D and v_cache.shape == caches and k_cache.dtype is bf16 and v_cache.dtype is bf16
        assert k_cache.is_contiguous() and v_cache.is_contiguous()
        batch, pages = block_table.shape
        prefixes, prefix_pages = prefix_table.shape
        assert cu_q.shape == (batch + 1,) and seqlens_k.shape == (batch,)
        assert prefix_lens.shape == (prefixes,) and cu_prefix_seqs.shape == (prefixes + 1,)
        for x in (cu_q, seqlens_k, block_table, prefix_table, prefix_lens, cu_prefix_seqs):
            assert x.dtype is i32 and x.is_contiguous() and x.get_device() == dev, "int32, contiguous, on one device"
        tokens, heads, d = q.shape
        assert d == D and o.shape == q.shape and q.dtype is bf16 and o.dtype is bf16
        assert q.is_contiguous() and o.is_contiguous()
        assert dev == k_cache.get_device() == v_cache.get_device() == o.get_device(), "all tensors on one device"
        lse_ptr = 0
        if lse is not None:
            assert lse.shape == (heads, tokens) and lse.is_contiguous() and lse.dtype is torch.float32
            assert lse.get_device() == dev, "all tensors on one device"
            lse_ptr = lse.data_ptr()
        return _PREFIX.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(), lse_ptr,
                            cu_q.data_ptr(), seqlens_k.data_ptr(), block_table.data_ptr(), batch, heads, kv_heads,
                            int(max_q), int(max_k), tokens, 0 if total_k is None else int(total_k), num_pages,
                            page_size, pages, SCALE if scale is None else scale, prefix_table.data_ptr(),
                            prefix_lens.data_ptr(), cu_prefix_seqs.data_ptr(), prefixes, prefix_pages)

    def prefix_paged_workspace_size(self, batch, heads, kv_heads, max_q, max_k, total_q, page_size, max_pages,
                                    num_pages, num_prefixes, max_prefix_pages, causal=0) -> int:
        """Workspace bytes of call_prefix_paged for a batch of this shape (-1: rejected)."""
        a = PrefixArgs(self.paged_shape_args(batch, heads, kv_heads, max_q, max_k, total_q, 0, page_size, max_pages,
                                             num_pages), None, None, None, num_prefixes, max_prefix_pages)
        return self.serving.fav4_bshd_prefix_paged_workspace_size(C.byref(a), int(causal))

    def call_prefix_paged(self, q, k_cache, v_cache, o, lse, cu_q, seqlens_k, block_table, prefix_table, prefix_lens,
                          cu_prefix_seqs, max_q, max_k, workspace=None, total_k=None, scale=None, stream=None,
                          causal=0):
        """fav4_bshd_forward_prefix_paged: call_splitkv_paged for sequences that share leading pages.  Tensors as for
        paged_args, and prefix_table: int32 [num_prefixes, max_pages]; prefix_lens: int32 [num_prefixes];
        cu_prefix_seqs: int32 [num_prefixes + 1].  causal 0 dense, 2 bottom-right.  `workspace` as for call_splitkv
        (None: allocated here); returned for the next call."""
        import torch
        block = self._prefix_block(torch, q, k_cache, v_cache, o, lse, cu_q, seqlens_k, block_table, prefix_table,
                                   prefix_lens, cu_prefix_seqs, max_q, max_k, total_k, scale)
        raw = self._stream(torch, q.get_device(), stream)
        causal = int(causal)
        if workspace is None:
            need = self.serving.fav4_bshd_prefix_paged_workspace_size(block, causal)
            if need < 0:
                raise RuntimeError("prefix paged: arguments rejected")
            # Allocated for the stream that uses it, which then orders its reuse.
            with torch.cuda.stream(self._allocation_stream(torch, stream)):
                workspace = torch.empty(need, device=q.device, dtype=torch.uint8)
        assert workspace.get_device() == q.get_device() and workspace.is_contiguous()
        status = self.serving.fav4_bshd_forward_prefix_paged(block, causal, workspace.data_ptr(), workspace.nbytes, raw)
        if status:
            raise RuntimeError(f"prefix paged: HIP status {status}")
        return workspace

    # ---- 4-bit paged K/V caches (include/fav4_mx4.h; no reference counterpart) ----
    # Caches as pairs of uint8 tensors, contiguous: codes [num_pages, kv_heads, page_size, 64] and scales
    # [num_pages, kv_heads, page_size, 4].
    @property
    def mx4(self) -> C.CDLL:
        lib = self.__dict__.get("_mx4")
        if lib is None:
            lib = self._mx4 = load_mx4_library()
        return lib

    @property
    def mx4_blocks(self):
        blocks = self.__dict__.get("_mx4_blocks")
        if blocks is None:
            blocks = self._mx4_blocks = load_mx4_blocks()
        return blocks

    @staticmethod
    def mx4_caches(num_pages, kv_heads, page_size, device="cuda"):
        """(k_cache, k_scales, v_cache, v_scales) of zeros."""
        import torch
        shape = (num_pages, kv_heads, page_size)
        return tuple(torch.zeros((*shape, n), dtype=torch.uint8, device=device)
                     for n in (D // 2, D // 32, D // 2, D // 32))

    def call_append_paged_mx4(self, q, k, v, q_out, k_cache, k_scales, v_cache, v_scales, cu_q, seqlens_k, block_table,
                              cos=None, sin=None, interleaved=False, positions=None, stream=None):
        """fav4_bshd_append_paged_mx4: call_append_paged into 4-bit caches (see mx4_caches); the other tensors as
        there."""
        import torch
        block = self.mx4_blocks.append(q, k, v, q_out, k_cache, k_scales, v_cache, v_scales, cu_q, seqlens_k, block_table,
                                       cos, sin, interleaved, positions)
        status = self.mx4.fav4_bshd_append_paged_mx4(block, self._stream(torch, k.get_device(), stream))
        if status:
            raise RuntimeError(f"append paged mx4: HIP status {status}")

    def call_gather_paged_mx4(self, k_cache, k_scales, v_cache, v_scales, k, v, cu_k, block_table, starts=None,
                              stream=None):
        """fav4_bshd_gather_paged_mx4: the numbers that 4-bit caches (see mx4_caches) hold, as BF16 rows.  k/v:
        [total_k, kv_heads, 128] (any stride between rows), of which [cu_k[b], cu_k[b + 1]) get keys starts[b], ... of
        sequence b; cu_k: int32 [batch+1]; block_table: int32 [batch, max_pages]; starts: int32 [batch] or None (0)."""
        import torch
        block = self.mx4_blocks.gather(k_cache, k_scales, v_cache, v_scales, k, v, cu_k, block_table, starts)
        status = self.mx4.fav4_bshd_gather_paged_mx4(block, self._stream(torch, k.get_device(), stream))
        if status:
            raise RuntimeError(f"gather paged mx4: HIP status {status}")

    def paged_mx4_workspace_size(self, batch, heads, kv_heads, max_q, max_k, total_q, page_size, max_pages, num_pages,
                                 causal=0) -> int:
        """Workspace bytes of call_paged_mx4 for a batch of this shape (-1: rejected)."""
        a = Mx4PagedArgs(self.paged_shape_args(batch, heads, kv_heads, max_q, max_k, total_q, 0, page_size, max_pages,
                                               num_pages), None, None)
        return self.mx4.fav4_bshd_paged_mx4_workspace_size(C.byref(a), int(causal))

    def call_paged_mx4(self, q, k_cache, k_scales, v_cache, v_scales, o, lse, cu_q, seqlens_k, block_table, max_q,
                       max_k, workspace=None, total_k=None, scale=None, stream=None, causal=0):
        """fav4_bshd_forward_paged_mx4: attention over 4-bit caches (see mx4_caches); the other tensors as for
        paged_args, but for total_k: the sum of seqlens_k, which steers the cut alone; None (0) takes every sequence
        for max_k long.  causal 0 dense, 2 bottom-right.  `workspace` as for call_splitkv (None: allocated here);
        returned for the next call."""
        import torch
        block = self.mx4_blocks.paged(q, k_cache, k_scales, v_cache, v_scales, o, lse, cu_q, seqlens_k, block_table,
                                      max_q, max_k, total_k, scale)
        raw = self._stream(torch, q.get_device(), stream)
        causal = int(causal)
        if workspace is None:
            need = self.mx4.fav4_bshd_paged_mx4_workspace_size(block, causal)
            if need < 0:
                raise RuntimeError("paged mx4: arguments rejected")
            # Allocated for the stream that uses it, which then orders its reuse.
            with torch.cuda.stream(self._allocation_stream(torch, stream)):
                workspace = torch.empty(need, device=q.device, dtype=torch.uint8)
        assert workspace.get_device() == q.get_device() and workspace.is_contiguous()
        status = self.mx4.fav4_bshd_forward_paged_mx4(block, causal, workspace.data_ptr(), workspace.nbytes, raw)
        if status:
            raise RuntimeError(f"paged mx4: HIP status {status}")
        return workspace


def forward(q, k, v, causal=False, with_lse=False, config=0, scale=None):
    """Allocate O (and LSE) and run the forward; returns (o, lse or None)."""
    import torch
    o = torch.empty_like(q)
    lse = (torch.empty((q.shape[0], q.shape[2], q.shape[1]), device=q.device, dtype=torch.float32)
           if with_lse else None)
    Runner().call(q, k, v, o, lse, causal, config, scale)
    return o, lse
