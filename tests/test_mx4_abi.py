"""Host-only checks of the 4-bit caches' C ABI (include/fav4_mx4.h): exports, struct layouts, refusals before any HIP
call, and workspace sizes."""
import ctypes as C
import math
import subprocess

import numpy as np
import pytest

from tests.conftest import ROOT, load_package
from tests.mx4 import GRID, quantise, values

INVALID = 1
TOP = (1 << 31) - 1


@pytest.fixture(scope="module")
def pkg():
    p = load_package()
    if not p.MX4_LIB_PATH.exists():
        p.build_library()
    return p


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.load_mx4_library()


def append_args(pkg, **over):
    """A call that would be accepted (addresses are never read on the host)."""
    inner = dict(q=0x10000, k=0x20000, v=0x30000, q_out=0x40000, k_cache=0x50000, v_cache=0x60000, cos=0x70000,
                 sin=0x80000, cu_seqlens_q=0x90000, seqlens_k=0xa0000, block_table=0xb0000, positions=None,
                 q_stride=4096, k_stride=1024, v_stride=1024, q_out_stride=4096, batch=2, heads=32, kv_heads=8,
                 total_q=2, num_pages=10, page_size=64, max_pages_per_seq=4, rotary_dim=128, rotary_rows=300,
                 interleaved=0)
    own = dict(k_scales=0xc0000, v_scales=0xd0000)
    for k, v in over.items():
        (own if k in own else inner)[k] = v
    return pkg.Mx4AppendArgs(pkg.AppendArgs(**inner), **own)


def gather_args(pkg, **over):
    a = dict(k_cache=0x10000, k_scales=0x20000, v_cache=0x30000, v_scales=0x40000, k=0x50000, v=0x60000,
             cu_seqlens_k=0x70000, starts=None, block_table=0x80000, k_stride=1024, v_stride=1024, batch=2, kv_heads=8,
             total_k=100, num_pages=10, page_size=64, max_pages_per_seq=4)
    a.update(over)
    return pkg.Mx4GatherArgs(**a)


def paged_args(pkg, **over):
    inner = dict(q=0x10000, k_cache=0x20000, v_cache=0x30000, o=0x40000, lse=None, cu_seqlens_q=0x50000,
                 seqlens_k=0x60000, block_table=0x70000, batch=4, heads=32, kv_heads=8, max_seqlen_q=1,
                 max_seqlen_k=1000, total_q=4, total_k=4000, num_pages=100, page_size=64, max_pages_per_seq=16,
                 scale=1 / math.sqrt(128))
    own = dict(k_scales=0x80000, v_scales=0x90000)
    for k, v in over.items():
        (own if k in own else inner)[k] = v
    return pkg.Mx4PagedArgs(pkg.PagedArgs(**inner), **own)


def test_exports(pkg):
    out = subprocess.run(["nm", "-D", "--defined-only", str(pkg.MX4_LIB_PATH)], capture_output=True, text=True,
                         check=True).stdout
    names = {line.split()[-1] for line in out.splitlines() if line.strip()}
    assert {n for n in names if not n.startswith("_")} == {
        "fav4_bshd_append_paged_mx4", "fav4_bshd_gather_paged_mx4", "fav4_bshd_forward_paged_mx4",
        "fav4_bshd_paged_mx4_workspace_size"}


@pytest.mark.parametrize("name", ["Append", "Gather", "Paged"])
def test_ctypes_layout_matches_the_header(pkg, name, tmp_path):
    cls = getattr(pkg, f"Mx4{name}Args")
    fields = [f[0] for f in cls._fields_]
    src = tmp_path / "layout.cpp"
    src.write_text('#include <cstddef>\n#include <cstdio>\n#include "fav4_mx4.h"\nint main() {\n'
                   f'  std::printf("%zu", sizeof(Fav4Mx4{name}Args));\n'
                   + "".join(f'  std::printf(" %zu", offsetof(Fav4Mx4{name}Args, {f}));\n' for f in fields) + "}\n")
    exe = tmp_path / "layout"
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-Wno-invalid-offsetof", f"-I{ROOT / 'include'}",
                    "-I/opt/rocm/include", str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [C.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def test_packed_blocks_match_the_structs(pkg):
    """The blocks that the binding packs, field by field."""
    import torch
    blocks = pkg.fav4_bshd.load_mx4_blocks()
    bf16 = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    caches = pkg.Runner.mx4_caches(7, 2, 48, device="cpu")
    qkv, q_out = bf16(5, 6 + 4, 128), bf16(5, 6, 128)
    q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
    cu, seqlens, table, positions, starts = i32(4), i32(3), i32(3, 9), i32(5), i32(3)
    cos, sin = torch.zeros(300, 32), torch.zeros(300, 32)
    ptrs = {n: x.data_ptr() for n, x in zip(("k_cache", "k_scales", "v_cache", "v_scales"), caches)}
    sizes = dict(batch=3, kv_heads=2, num_pages=7, page_size=48, max_pages_per_seq=9, block_table=table.data_ptr())

    def check(cls, block, **want):
        assert len(block) == C.sizeof(cls)
        got, a = {}, cls.from_buffer_copy(block)
        for name, *_ in a._fields_:
            value = getattr(a, name)
            got.update({n: getattr(value, n) for n, *_ in value._fields_} if isinstance(value, C.Structure)
                       else {name: value})
        assert got == want

    new = dict(cu_seqlens_q=cu.data_ptr(), seqlens_k=seqlens.data_ptr(), **sizes)
    check(pkg.Mx4AppendArgs, blocks.append(q, k, v, q_out, *caches, cu, seqlens, table, cos, sin, True, positions),
          q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_out=q_out.data_ptr(), cos=cos.data_ptr(), sin=sin.data_ptr(),
          positions=positions.data_ptr(), q_stride=1280, k_stride=1280, v_stride=1280, q_out_stride=768, heads=6,
          total_q=5, rotary_dim=64, rotary_rows=300, interleaved=1, **ptrs, **new)
    check(pkg.Mx4AppendArgs, blocks.append(None, k[:1], v[:1], None, *caches, cu, seqlens, table, None, None, False, None),
          q=None, k=k.data_ptr(), v=v.data_ptr(), q_out=None, cos=None, sin=None, positions=None, q_stride=0, k_stride=256,
          v_stride=256, q_out_stride=0, heads=1, total_q=1, rotary_dim=0, rotary_rows=0, interleaved=0, **ptrs, **new)
    for given in (starts, None):
        check(pkg.Mx4GatherArgs, blocks.gather(*caches, k, v, cu, table, given), k=k.data_ptr(), v=v.data_ptr(),
              cu_seqlens_k=cu.data_ptr(), starts=None if given is None else starts.data_ptr(), k_stride=1280,
              v_stride=1280, total_k=5, **ptrs, **sizes)
    lse = torch.zeros(6, 5)
    for given, total, scale, want in ((lse, None, None, 128 ** -0.5), (None, 77, 0.25, 0.25)):
        check(pkg.Mx4PagedArgs, blocks.paged(q_out, *caches, q_out, given, cu, seqlens, table, 2, 400, total, scale),
              q=q_out.data_ptr(), o=q_out.data_ptr(), lse=None if given is None else lse.data_ptr(), heads=6,
              max_seqlen_q=2, max_seqlen_k=400, total_q=5, total_k=total or 0, scale=C.c_float(want).value, **ptrs, **new)


def test_blocks_refuse_wrong_tensors(pkg):
    """Every tensor with another type, shape or layout, and numbers that do not fit."""
    import torch
    blocks = pkg.fav4_bshd.load_mx4_blocks()
    bf16 = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    caches = pkg.Runner.mx4_caches(7, 2, 48, device="cpu")
    q, k, v, cu, seqlens, table = bf16(5, 6, 128), bf16(5, 2, 128), bf16(5, 2, 128), i32(4), i32(3), i32(3, 9)
    cos, sin = torch.zeros(300, 32), torch.zeros(300, 32)
    calls = {blocks.append: [q, k, v, bf16(5, 6, 128), *caches, cu, seqlens, table, cos, sin, False, i32(5)],
             blocks.gather: [*caches, k, v, cu, table, i32(3)],
             blocks.paged: [q, *caches, bf16(5, 6, 128), torch.zeros(6, 5), cu, seqlens, table, 1, 99, None, None]}
    wrong = (lambda x: x.double(), lambda x: x[:-1], lambda x: x.unsqueeze(0), lambda x: torch.stack((x, x), -1)[..., 0])
    for call, args in calls.items():
        call(*args)
        for i, x in enumerate(args):
            if not isinstance(x, torch.Tensor):
                continue
            for change in wrong:
                with pytest.raises(AssertionError):
                    call(*args[:i], change(x), *args[i + 1:])
            with pytest.raises(TypeError):
                call(*args[:i], 5, *args[i + 1:])
        with pytest.raises(TypeError):
            call(*args[:-1])
    append, paged = calls[blocks.append], calls[blocks.paged]
    for i in (0, 3, 11, 12):
        with pytest.raises(AssertionError):
            blocks.append(*append[:i], None, *append[i + 1:])
    for i in (10, 11, 12):
        for bad, error in ((1 << 31, OverflowError), (1 << 80, OverflowError), ("x", ValueError), ([], TypeError)):
            with pytest.raises(error):
                blocks.paged(*paged[:i], bad, *paged[i + 1:])
    with pytest.raises(TypeError):
        blocks.paged(*paged[:13], "1")


APPEND_BAD = [{n: None} for n in ("k", "v", "q", "q_out", "k_cache", "v_cache", "cos", "sin", "cu_seqlens_q",
                                  "seqlens_k", "block_table", "k_scales", "v_scales")]
APPEND_BAD += [{n: 0x10008} for n in ("q", "k", "v", "q_out", "k_cache", "v_cache", "cos", "sin", "k_scales", "v_scales")]
APPEND_BAD += [{n: 0x10002} for n in ("cu_seqlens_q", "seqlens_k", "block_table", "positions")]
APPEND_BAD += [{n: v} for n in ("batch", "heads", "kv_heads", "total_q", "num_pages", "page_size", "max_pages_per_seq",
                                "rotary_rows") for v in (0, -1)]
APPEND_BAD += [dict(rotary_dim=v) for v in (-16, 8, 24, 144, 1)] + [dict(interleaved=v) for v in (-1, 2)]
APPEND_BAD += [dict(q_stride=4088), dict(q_stride=4100), dict(k_stride=1016), dict(v_stride=-1024), dict(v_stride=0),
               dict(q_out_stride=2048), dict(q_out=0x10000, q_out_stride=8192),
               dict(rotary_dim=0), dict(rotary_dim=0, cos=None), dict(total_q=1 << 27),
               dict(k_stride=1 << 50), dict(num_pages=1 << 30, page_size=1 << 20),
               dict(kv_heads=1 << 30), dict(heads=TOP), dict(heads=TOP, kv_heads=TOP, total_q=TOP),
               dict(batch=TOP), dict(batch=TOP - 62)]


@pytest.mark.parametrize("over", APPEND_BAD, ids=str)
def test_append_refusals(pkg, lib, over):
    assert lib.fav4_bshd_append_paged_mx4(C.byref(append_args(pkg, **over)), None) == INVALID


GATHER_BAD = [{n: None} for n in ("k_cache", "k_scales", "v_cache", "v_scales", "k", "v", "cu_seqlens_k", "block_table")]
GATHER_BAD += [{n: 0x10008} for n in ("k_cache", "k_scales", "v_cache", "v_scales", "k", "v")]
GATHER_BAD += [{n: 0x10002} for n in ("cu_seqlens_k", "starts", "block_table")]
GATHER_BAD += [{n: v} for n in ("batch", "kv_heads", "total_k", "num_pages", "page_size", "max_pages_per_seq")
               for v in (0, -1)]
GATHER_BAD += [dict(k_stride=1016), dict(v_stride=1028), dict(k_stride=0), dict(v_stride=-1024), dict(k_stride=1 << 50),
               dict(total_k=1 << 27), dict(kv_heads=TOP, total_k=TOP), dict(num_pages=1 << 30, page_size=1 << 20),
               dict(batch=TOP), dict(batch=TOP - 62)]


@pytest.mark.parametrize("over", GATHER_BAD, ids=str)
def test_gather_refusals(pkg, lib, over):
    assert lib.fav4_bshd_gather_paged_mx4(C.byref(gather_args(pkg, **over)), None) == INVALID


PAGED_SHAPES_BAD = [{n: v} for n in ("batch", "heads", "kv_heads", "max_seqlen_q", "max_seqlen_k", "total_q",
                                     "num_pages", "page_size", "max_pages_per_seq") for v in (0, -1)]
PAGED_SHAPES_BAD += [dict(total_k=-1), dict(kv_heads=5), dict(kv_heads=64), dict(scale=0.0), dict(scale=-1.0),
                     dict(scale=float("nan")), dict(scale=float("inf")), dict(page_size=8), dict(page_size=24),
                     dict(max_seqlen_k=1025), dict(total_q=1 << 27), dict(heads=1 << 25, kv_heads=1),
                     dict(heads=(1 << 15) + 8), dict(num_pages=1 << 30, page_size=1 << 20),
                     dict(batch=1 << 20, max_seqlen_k=1 << 20, max_pages_per_seq=1 << 20),
                     dict(batch=TOP, max_seqlen_q=TOP, heads=1 << 15, kv_heads=1 << 15, total_q=65535),
                     dict(max_seqlen_k=TOP - 62, max_pages_per_seq=1 << 30)]


@pytest.mark.parametrize("over", PAGED_SHAPES_BAD, ids=str)
def test_paged_shape_refusals(pkg, lib, over):
    a = paged_args(pkg, **over)
    assert lib.fav4_bshd_paged_mx4_workspace_size(C.byref(a), 0) == -1
    assert lib.fav4_bshd_forward_paged_mx4(C.byref(a), 0, 0x1000000, 1 << 40, None) == INVALID


@pytest.mark.parametrize("over", [{n: None} for n in ("q", "k_cache", "v_cache", "o", "cu_seqlens_q", "seqlens_k",
                                                      "block_table", "k_scales", "v_scales")]
                         + [{n: 0x10008} for n in ("q", "k_cache", "v_cache", "o", "k_scales", "v_scales")]
                         + [{n: 0x10002} for n in ("lse", "cu_seqlens_q", "seqlens_k", "block_table")], ids=str)
def test_paged_pointer_refusals(pkg, lib, over):
    a = paged_args(pkg, **over)
    assert lib.fav4_bshd_forward_paged_mx4(C.byref(a), 0, 0x1000000, 1 << 40, None) == INVALID


def test_refusals_of_null_masks_and_workspaces(pkg, lib):
    assert lib.fav4_bshd_append_paged_mx4(None, None) == INVALID
    assert lib.fav4_bshd_gather_paged_mx4(None, None) == INVALID
    a = paged_args(pkg)
    for causal in (-1, 1, 3):
        assert lib.fav4_bshd_paged_mx4_workspace_size(C.byref(a), causal) == -1
        assert lib.fav4_bshd_forward_paged_mx4(C.byref(a), causal, 0x1000000, 1 << 40, None) == INVALID
    need = lib.fav4_bshd_paged_mx4_workspace_size(C.byref(a), 0)
    assert need > 0
    for ws, size in ((None, need), (0x1000000, need - 1), (0x1000080, need)):
        assert lib.fav4_bshd_forward_paged_mx4(C.byref(a), 0, ws, size, None) == INVALID
    assert lib.fav4_bshd_forward_paged_mx4(None, 0, 0x1000000, need, None) == INVALID
    assert lib.fav4_bshd_paged_mx4_workspace_size(None, 0) == -1


def test_workspace_grows_with_the_batch(pkg, lib):
    """One workspace, sized for a serving loop's largest batch, serves the smaller ones, however they are cut."""
    size = lambda **over: lib.fav4_bshd_paged_mx4_workspace_size(C.byref(paged_args(pkg, **over)), 2)
    for kvh in (1, 2, 8, 32, 128):
        last = 0
        for batch, q, total in ((1, 1, 1), (2, 1, 2), (40, 1, 40), (100, 1, 100), (100, 4, 100), (100, 4, 400),
                                (100, 16, 400), (100, 16, 1600), (100, 30, 1600), (300, 200, 1600), (2000, 200, 5000),
                                (2000, 300, 60000), (2000, 300, 600000)):
            for keys in (64, 1000):
                n = size(batch=batch, max_seqlen_q=q, total_q=total, max_seqlen_k=keys, heads=max(32, kvh), kv_heads=kvh)
                assert n >= last > -1, (kvh, batch, q, total, keys)
            last = n
        assert size(kv_heads=kvh, heads=max(32, kvh), max_seqlen_k=64) == size(kv_heads=kvh, heads=max(32, kvh))


@pytest.mark.parametrize("kv_heads", [1, 8, 200, 257, 300, 512, 513, 2000, 1 << 15])
def test_workspace_holds_both_parts_of_a_row_tile(pkg, lib, kv_heads):
    """Every K/V head has a range of its own at least, with two partial blocks of up to 256 rows (32 with few rows): 128
    numbers of 4 bytes and two sums a row."""
    for q, rows in ((1, 32), (32, 32), (300, 256)):
        a = paged_args(pkg, heads=kv_heads, kv_heads=kv_heads, max_seqlen_q=q, total_q=q, batch=1)
        assert lib.fav4_bshd_paged_mx4_workspace_size(C.byref(a), 2) >= kv_heads * 2 * rows * (128 * 4 + 8) + 16


def test_grids_stay_below_the_most_threads(pkg, lib):
    """2^22 row tiles are too many over 8 K/V heads, not over one."""
    size = lambda kvh, total: lib.fav4_bshd_paged_mx4_workspace_size(C.byref(paged_args(
        pkg, batch=1, heads=8, kv_heads=kvh, max_seqlen_q=total, total_q=total, max_seqlen_k=64)), 2)
    assert size(1, 1 << 23) > 0 and size(8, 1 << 25) > 0
    many = lambda kvh: lib.fav4_bshd_paged_mx4_workspace_size(C.byref(paged_args(
        pkg, batch=1 << 21, heads=64, kv_heads=kvh, max_seqlen_q=100, total_q=1 << 24, max_seqlen_k=64)), 2)
    assert many(64) == -1


def test_runner_refuses_host_tensors_and_wrong_ones(pkg):
    import torch
    r = pkg.Runner()
    bf16 = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    caches, table = r.mx4_caches(2, 1, 64, device="cpu"), torch.zeros((1, 2), dtype=torch.int32)
    assert [tuple(x.shape) for x in caches] == [(2, 1, 64, 64), (2, 1, 64, 4)] * 2
    append = lambda c, **o: r.call_append_paged_mx4(bf16(1, 2, 128), o.get("k", bf16(1, 1, 128)), bf16(1, 1, 128),
                                                    bf16(1, 2, 128), *c, i32(0, 1), i32(1), table)
    gather = lambda c, **o: r.call_gather_paged_mx4(*c, o.get("k", bf16(1, 1, 128)), bf16(1, 1, 128), i32(0, 1), table,
                                                    starts=o.get("starts"))
    attend = lambda c, **o: r.call_paged_mx4(bf16(1, 2, 128), *c, o.get("o", bf16(1, 2, 128)), o.get("lse"), i32(0, 1),
                                             i32(1), table, 1, 64)
    for call in (append, gather, attend):
        with pytest.raises(ValueError, match="host"):
            call(caches)
        for i, wrong in enumerate((lambda x: x.int(), lambda x: x[:1], lambda x: x.transpose(0, 2), lambda x: x[..., :2])):
            bad = list(caches)
            bad[i % 4] = wrong(bad[i % 4])
            with pytest.raises(AssertionError):
                call(bad)
    with pytest.raises(AssertionError):
        append(caches, k=torch.zeros(1, 1, 128))
    with pytest.raises(AssertionError):
        gather(caches, k=bf16(1, 2, 128))
    with pytest.raises(AssertionError):
        gather(caches, starts=i32(1, 2))
    with pytest.raises(AssertionError):
        attend(caches, o=bf16(1, 1, 128))
    with pytest.raises(AssertionError):
        attend(caches, lse=torch.zeros(1, 2))


def test_the_reference_rounds_to_the_nearest():
    """The tests' own quantiser against a search over the grid, ties and the choice of scales included."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 128)).astype(np.float32)
    x[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0]
    x[0, 8:32] = 0
    codes, scales = quantise(x)
    got = values(codes, scales)
    assert got[0, :8].tolist() == [0, 1, 1, 2, 2, 4, 4, 6]
    power = np.exp2(scales.astype(np.float64) - 127).repeat(32, -1)
    assert (np.abs(x) <= 7 * power).all()
    most = np.abs(x).reshape(50, 4, 32).max(-1).repeat(32, -1)
    assert (most > 3.5 * power).all()
    near = np.abs(np.abs(x)[..., None] - GRID * power[..., None]).min(-1)
    assert (np.abs(np.abs(x) - np.abs(got)) == near).all()
