"""Which kernels a call of the 4-bit caches' library launches, without a GPU: the host part of csrc/mx4.hip, built behind
a HIP runtime of stand-ins that write launches down.  Addresses are never read."""
import ctypes as C
import math
import os
import subprocess
from pathlib import Path

from tests.conftest import ROOT, load_package

RUNTIME = r"""
#include <hip/hip_runtime.h>
#include <map>
#include <string>

namespace {
std::map<const void*, std::string>& names() {
    static std::map<const void*, std::string> table;
    return table;
}
std::string launched;
dim3 grid, block;
size_t shared;
hipStream_t on;
}  // namespace

extern "C" {
char FATBIN[1];
void** __hipRegisterFatBinary(const void*) { return nullptr; }
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
    names()[host] = name;
}
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t s, hipStream_t q) {
    grid = g, block = b, shared = s, on = q;
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* s, hipStream_t* q) {
    *g = grid, *b = block, *s = shared, *q = on;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void* f, dim3 g, dim3 b, void**, size_t, hipStream_t) {
    launched += names()[f] + " " + std::to_string(g.x) + " " + std::to_string(b.x) + "\n";
    return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipGetDevice(int* device) {
    *device = 0;
    return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int* value, hipDeviceAttribute_t, int) {
    *value = 256;                     // CUs of an MI355X
    return hipSuccess;
}
__attribute__((visibility("default"))) const char* launches() {
    static std::string last;
    last.swap(launched);
    launched.clear();
    return last.c_str();
}
}
"""


def build(folder: Path) -> C.CDLL:
    """The library, in `folder`."""
    pkg = load_package().fav4_bshd
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    host, lib = folder / "mx4.o", folder / "mx4_launches.so"
    subprocess.run([hipcc, "--offload-host-only", "-std=c++17", "-O1", "-fPIC", "-fvisibility=hidden", "-c",
                    f"-I{pkg.INCLUDE}", f"-I{pkg.CSRC}", str(pkg.CSRC / "mx4.hip"), "-o", str(host)], check=True)
    symbols = subprocess.run(["nm", "-u", str(host)], capture_output=True, text=True, check=True).stdout.split()
    fatbin, = [s for s in symbols if s.startswith("__hip_fatbin")]
    source = folder / "runtime.cpp"
    source.write_text(RUNTIME.replace("FATBIN", fatbin))
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    str(source), str(host), "-Wl,-Bsymbolic", "-Wl,--no-undefined", "-o", str(lib)], check=True)
    out = C.CDLL(str(lib))
    out.launches.restype = C.c_char_p
    out.fav4_bshd_forward_paged_mx4.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_size_t, C.c_void_p]
    return out


def attention(lib, heads, kv_heads, page, lens, causal, lse=True, total_k=0, max_q=None, max_k=None, tail=0):
    """The attention's launches for a batch of (queries, keys): [(kernel, workgroups, threads)], with the template's
    arguments as they stand in the mangled name ("mx4_decode_kernelILi1ELi4E...")."""
    pkg = load_package()
    sq, sk = zip(*lens)
    max_q, max_k = max_q or max(max(sq), 1), max_k or max(max(sk), 1)
    width, pages = -(-max_k // page), sum(-(-k // page) for k in sk) + 3
    a = pkg.Mx4PagedArgs(pkg.PagedArgs(
        q=0x10000, k_cache=0x20000, v_cache=0x30000, o=0x40000, lse=0xa0000 if lse else None, cu_seqlens_q=0x50000,
        seqlens_k=0x60000, block_table=0x70000, batch=len(lens), heads=heads, kv_heads=kv_heads, max_seqlen_q=max_q,
        max_seqlen_k=max_k, total_q=max(sum(sq), 1) + tail, total_k=total_k, num_pages=pages, page_size=page,
        max_pages_per_seq=width, scale=1 / math.sqrt(128)), 0x80000, 0x90000)
    lib.launches()
    status = lib.fav4_bshd_forward_paged_mx4(C.byref(a), causal, 0x1000000, 1 << 40, None)
    assert status == 0, status
    out = []
    for line in lib.launches().decode().splitlines():
        name, grid, threads = line.split()
        out.append((name[name.index("mx4_"):], int(grid), int(threads)))
    return out


def kind(launched):
    """("decode" or "prefill", "whole" or "line", rows of a row tile) of attention()'s launches."""
    name, line = launched[0][0], len(launched) == 2
    assert line == any("mx4_merge_kernel" in n for n, *_ in launched) and len(launched) <= 2
    if name.startswith("mx4_decode_kernelILi"):
        return "decode", "line" if line else "whole", 16 * int(name[len("mx4_decode_kernelILi")])
    assert name.startswith("mx4_prefill_line_kernelILi" if line else "mx4_prefill_kernelILi"), name
    return "prefill", "line" if line else "whole", 32 * int(name.split("ILi")[1][0])
