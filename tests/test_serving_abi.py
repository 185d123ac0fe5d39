"""Host-only checks of the serving operators' C ABI (include/fav4_serving.h): exports, struct layouts, refusals
before any HIP call, and workspace sizes."""
import ctypes as C
import math
import subprocess

import pytest

from tests.conftest import ROOT, load_package

INVALID = 1


@pytest.fixture(scope="module")
def pkg():
    p = load_package()
    if not p.SERVING_LIB_PATH.exists():
        p.build_library()
    return p


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.load_serving_library()


def append_args(pkg, **over):
    """A call that would be accepted (addresses are never read on the host)."""
    a = dict(q=0x10000, k=0x20000, v=0x30000, q_out=0x40000, k_cache=0x50000, v_cache=0x60000, cos=0x70000,
             sin=0x80000, cu_seqlens_q=0x90000, seqlens_k=0xa0000, block_table=0xb0000, positions=None,
             q_stride=4096, k_stride=1024, v_stride=1024, q_out_stride=4096, batch=2, heads=32, kv_heads=8, total_q=2,
             num_pages=10, page_size=64, max_pages_per_seq=4, rotary_dim=128, rotary_rows=300, interleaved=0)
    a.update(over)
    return pkg.AppendArgs(**a)


def prefix_args(pkg, **over):
    paged = dict(q=0x10000, k_cache=0x20000, v_cache=0x30000, o=0x40000, lse=None, cu_seqlens_q=0x50000,
                 seqlens_k=0x60000, block_table=0x70000, batch=4, heads=32, kv_heads=8, max_seqlen_q=1,
                 max_seqlen_k=1000, total_q=4, total_k=4000, num_pages=100, page_size=64, max_pages_per_seq=16,
                 scale=1 / math.sqrt(128))
    own = dict(prefix_table=0x80000, prefix_lens=0x90000, cu_prefix_seqs=0xa0000, num_prefixes=1,
               max_pages_per_prefix=8)
    for k, v in over.items():
        (own if k in own else paged)[k] = v
    return pkg.PrefixArgs(pkg.PagedArgs(**paged), **own)


def test_exports(pkg):
    out = subprocess.run(["nm", "-D", "--defined-only", str(pkg.SERVING_LIB_PATH)], capture_output=True, text=True,
                         check=True).stdout
    names = {line.split()[-1] for line in out.splitlines() if line.strip()}
    assert {n for n in names if not n.startswith("_")} == {
        "fav4_bshd_append_paged", "fav4_bshd_forward_prefix_paged", "fav4_bshd_prefix_paged_workspace_size"}


@pytest.mark.parametrize("name", ["Append", "Prefix"])
def test_ctypes_layout_matches_the_header(pkg, name, tmp_path):
    cls = getattr(pkg, f"{name}Args")
    fields = [f[0] for f in cls._fields_]
    src = tmp_path / "layout.cpp"
    src.write_text('#include <cstddef>\n#include <cstdio>\n#include "fav4_serving.h"\nint main() {\n'
                   f'  std::printf("%zu", sizeof(Fav4{name}Args));\n'
                   + "".join(f'  std::printf(" %zu", offsetof(Fav4{name}Args, {f}));\n' for f in fields) + "}\n")
    exe = tmp_path / "layout"
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-Wno-invalid-offsetof", f"-I{ROOT / 'include'}",
                    "-I/opt/rocm/include", str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [C.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def test_packed_blocks_match_the_structs(pkg):
    """The blocks that Runner packs in one step lie as the ctypes structs do."""
    b = pkg.fav4_bshd
    for packer, block in ((b._APPEND, append_args(pkg, positions=0xc0000)), (b._PREFIX, prefix_args(pkg, lse=0xb0000))):
        assert packer.size == C.sizeof(block)
        flat = []
        for name, *_ in block._fields_:
            value = getattr(block, name)
            flat += [getattr(value, n) for n, *_ in value._fields_] if isinstance(value, C.Structure) else [value]
        assert packer.pack(*flat) == bytes(block)


APPEND_BAD = [{n: None} for n in ("k", "v", "q", "q_out", "k_cache", "v_cache", "cos", "sin", "cu_seqlens_q",
                                  "seqlens_k", "block_table")]
APPEND_BAD += [{n: 0x10008} for n in ("q", "k", "v", "q_out", "k_cache", "v_cache", "cos", "sin")]
APPEND_BAD += [{n: 0x10002} for n in ("cu_seqlens_q", "seqlens_k", "block_table", "positions")]
APPEND_BAD += [{n: v} for n in ("batch", "heads", "kv_heads", "total_q", "num_pages", "page_size", "max_pages_per_seq",
                                "rotary_rows") for v in (0, -1)]
APPEND_BAD += [dict(rotary_dim=v) for v in (-16, 8, 24, 144, 1)] + [dict(interleaved=v) for v in (-1, 2)]
APPEND_BAD += [dict(q_stride=4088), dict(q_stride=4100), dict(k_stride=1016), dict(v_stride=-1024), dict(v_stride=0),
               dict(q_out_stride=2048), dict(q_out=0x10000, q_out_stride=8192),
               dict(rotary_dim=0), dict(rotary_dim=0, cos=None), dict(total_q=1 << 27),
               dict(k_stride=1 << 50), dict(num_pages=1 << 30, page_size=1 << 20),
               dict(kv_heads=1 << 30), dict(heads=(1 << 31) - 1),
               dict(heads=(1 << 31) - 1, kv_heads=(1 << 31) - 1, total_q=(1 << 31) - 1)]


@pytest.mark.parametrize("over", APPEND_BAD, ids=str)
def test_append_refusals(pkg, lib, over):
    assert lib.fav4_bshd_append_paged(C.byref(append_args(pkg, **over)), None) == INVALID


def test_append_refuses_null(lib):
    assert lib.fav4_bshd_append_paged(None, None) == INVALID


PREFIX_SHAPES_BAD = [{n: v} for n in ("batch", "heads", "kv_heads", "max_seqlen_q", "max_seqlen_k", "total_q",
                                      "num_pages", "page_size", "max_pages_per_seq", "num_prefixes",
                                      "max_pages_per_prefix") for v in (0, -1)]
PREFIX_SHAPES_BAD += [dict(total_k=-1), dict(kv_heads=5), dict(kv_heads=64), dict(scale=0.0), dict(scale=-1.0),
                      dict(scale=float("nan")), dict(scale=float("inf")), dict(page_size=16), dict(page_size=33),
                      dict(max_seqlen_k=1025), dict(total_q=1 << 27), dict(heads=1 << 25, kv_heads=1), dict(heads=(1 << 15) + 8),
                      dict(num_pages=1 << 30, page_size=1 << 20),
                      dict(batch=1 << 20, max_seqlen_k=1 << 20, max_pages_per_seq=1 << 20),
                      dict(batch=(1 << 31) - 1, num_prefixes=(1 << 31) - 1, max_seqlen_q=(1 << 31) - 1,
                           heads=1 << 15, kv_heads=1 << 15, total_q=65535)]


@pytest.mark.parametrize("over", PREFIX_SHAPES_BAD, ids=str)
def test_prefix_shape_refusals(pkg, lib, over):
    a = prefix_args(pkg, **over)
    assert lib.fav4_bshd_prefix_paged_workspace_size(C.byref(a), 0) == -1
    assert lib.fav4_bshd_forward_prefix_paged(C.byref(a), 0, 0x1000000, 1 << 40, None) == INVALID


@pytest.mark.parametrize("over", [{n: None} for n in ("q", "k_cache", "v_cache", "o", "cu_seqlens_q", "seqlens_k",
                                                      "block_table", "prefix_table", "prefix_lens", "cu_prefix_seqs")]
                         + [{n: 0x10008} for n in ("q", "k_cache", "v_cache", "o")]
                         + [{n: 0x10002} for n in ("lse", "cu_seqlens_q", "seqlens_k", "block_table", "prefix_table",
                                                   "prefix_lens", "cu_prefix_seqs")], ids=str)
def test_prefix_pointer_refusals(pkg, lib, over):
    a = prefix_args(pkg, **over)
    assert lib.fav4_bshd_forward_prefix_paged(C.byref(a), 0, 0x1000000, 1 << 40, None) == INVALID


def test_prefix_refuses_masks_and_workspaces(pkg, lib):
    a = prefix_args(pkg)
    for causal in (-1, 1, 3):
        assert lib.fav4_bshd_prefix_paged_workspace_size(C.byref(a), causal) == -1
        assert lib.fav4_bshd_forward_prefix_paged(C.byref(a), causal, 0x1000000, 1 << 40, None) == INVALID
    need = lib.fav4_bshd_prefix_paged_workspace_size(C.byref(a), 0)
    assert need > 0
    for ws, size in ((None, need), (0x1000000, need - 1), (0x1000080, need)):
        assert lib.fav4_bshd_forward_prefix_paged(C.byref(a), 0, ws, size, None) == INVALID
    assert lib.fav4_bshd_forward_prefix_paged(None, 0, 0x1000000, need, None) == INVALID
    assert lib.fav4_bshd_prefix_paged_workspace_size(None, 0) == -1


def test_prefix_workspace_grows_with_the_batch(pkg, lib):
    """One workspace, sized for a serving loop's largest batch, serves the smaller ones, whatever way they are cut."""
    size = lambda **over: lib.fav4_bshd_prefix_paged_workspace_size(C.byref(prefix_args(pkg, **over)), 2)
    base = size()
    assert base > 0
    for kvh in (1, 2, 8, 32, 128):
        heads = max(32, kvh)
        last = 0
        for batch, q, prefixes in ((1, 1, 1), (2, 1, 1), (40, 1, 1), (40, 1, 20), (100, 1, 20), (100, 4, 20),
                                   (100, 30, 20), (300, 200, 64), (2000, 200, 64), (2000, 300, 300)):
            for keys in (64, 1000):
                n = size(batch=batch, max_seqlen_q=q, total_q=batch * q, num_prefixes=prefixes, max_seqlen_k=keys,
                         heads=heads, kv_heads=kvh)
                assert n >= last, (kvh, batch, q, prefixes, keys)
            last = n
    # Keys do not count: the partials are as many as the ranges and the row tiles.
    assert size(max_seqlen_k=64) == base == size(max_pages_per_prefix=100)


def test_runner_refuses_host_tensors(pkg):
    import torch
    r = pkg.Runner()
    bf16 = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    kc, vc, table = bf16(2, 64, 1, 128), bf16(2, 64, 1, 128), torch.zeros((1, 2), dtype=torch.int32)
    with pytest.raises(ValueError):
        r.call_append_paged(bf16(1, 2, 128), bf16(1, 1, 128), bf16(1, 1, 128), bf16(1, 2, 128), kc, vc, i32(0, 1),
                            i32(1), table)
    with pytest.raises(ValueError):
        r.call_prefix_paged(bf16(1, 2, 128), kc, vc, bf16(1, 2, 128), None, i32(0, 1), i32(1), table, table, i32(0),
                            i32(0, 1), 1, 64)


@pytest.mark.parametrize("wrong", ["dtype", "shape", "heads", "stride", "lens", "table", "angles", "q_out"])
def test_runner_checks_append_tensors(pkg, wrong):
    import torch
    bf16 = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    x = dict(q=bf16(3, 4, 128), k=bf16(3, 2, 128), v=bf16(3, 2, 128), q_out=bf16(3, 4, 128), k_cache=bf16(2, 64, 2, 128),
             v_cache=bf16(2, 64, 2, 128), cu_q=i32(0, 1, 3), seqlens_k=i32(1, 2),
             block_table=torch.zeros((2, 1), dtype=torch.int32), cos=torch.zeros(9, 64), sin=torch.zeros(9, 64))
    x.update(dict(dtype=dict(k=torch.zeros(3, 2, 128)), shape=dict(v=bf16(2, 2, 128)), heads=dict(k=bf16(3, 1, 128)),
                  stride=dict(k=bf16(3, 128, 2).transpose(1, 2)), lens=dict(seqlens_k=i32(1)),
                  table=dict(block_table=torch.zeros((2, 2), dtype=torch.int32).t()), angles=dict(sin=torch.zeros(9, 32)),
                  q_out=dict(q_out=None))[wrong])
    with pytest.raises((AssertionError, ValueError)) as e:
        pkg.Runner().call_append_paged(**x)
    assert "host" not in str(e.value)
