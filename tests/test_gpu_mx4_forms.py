"""Each form of the 4-bit caches' attention kernels (row tiles of 16, 32, 128 and 256 rows, whole and on a line), over
large pages, caches past 4 GiB, keys and queries that are no numbers, and again.  tests/test_mx4_launches.py holds every
batch to the form that it is here for."""
import numpy as np
import pytest
import torch

from tests.mx4 import Cache4, assert_guard_rows_untouched

pytestmark = pytest.mark.gpu

# Form: (kernel, whole or line, rows of a row tile, threads), and a batch that gets it: heads, K/V heads, (queries, keys).
FORMS = {
    "few": (("decode", "whole", 16, 512), 16, 8, [(1, 300), (1, 77), (1, 640)]),
    "few_long": (("decode", "whole", 16, 768), 16, 8, [(4, 2100), (3, 1500), (4, 900), (1, 2099)] * 4),
    "few_line": (("decode", "line", 16, 256), 16, 8, [(1, 5000), (1, 300), (1, 2100)] * 3),
    "drafts": (("decode", "whole", 32, 512), 16, 8, [(9, 400), (9, 90)]),
    "drafts_line": (("decode", "line", 32, 256), 16, 8, [(9, 6000), (9, 90), (6, 3500)]),
    "many_128": (("prefill", "whole", 128, 256), 16, 8, [(150, 150), (200, 333)] * 4),
    "many_256": (("prefill", "whole", 256, 512), 32, 8, [(512, 2000)] * 3 + [(512, 1777)]),
    "many_line_128": (("prefill", "line", 128, 256), 16, 8, [(100, 4000), (40, 1500), (70, 70)] * 2),
    "many_line_256": (("prefill", "line", 256, 512), 16, 8, [(300, 9000), (250, 2000)]),
}
PAGES = [64, 128, 192, 1024]


def batch_of(form, page, **more):
    _, heads, kv_heads, lens = FORMS[form]
    return Cache4(heads, kv_heads, page, lens, **more)


@pytest.mark.parametrize("causal", [0, 2])
@pytest.mark.parametrize("page", PAGES[1:])
@pytest.mark.parametrize("form", FORMS)
def test_pages_of_more_than_a_tile(gpu_runner, form, page, causal):
    batch = batch_of(form, page)
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, causal)
    batch.check(o, lse, causal)
    assert_guard_rows_untouched(batch)


@pytest.fixture(scope="module")
def room():
    """Codes of K and V of a little more than 2^32 bytes each, and their scales."""
    extra = 1 << 26
    return [torch.zeros(((1 << 32) + extra) * n // 64, dtype=torch.uint8, device="cuda:0") for n in (64, 4, 64, 4)]


@pytest.mark.parametrize("page", [64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_pages_on_both_sides_of_4_gib(gpu_runner, room, form, page):
    """Half of the pool's pages in use begin below 2^32 bytes of codes and half above."""
    batch = batch_of(form, page)
    kv_heads, pool = batch.kv_heads, batch.caches[0].shape[0]
    border = (1 << 32) // (page * kv_heads * 64)
    first = border - pool // 2
    caches = []
    for x, own, width in zip(room, batch.caches, (64, 4, 64, 4)):
        n = x.numel() // (page * kv_heads * width)
        whole = x[:n * page * kv_heads * width].view(n, kv_heads, page, width)
        whole[first:first + pool] = own
        caches.append(whole)
    assert first + pool <= caches[0].shape[0]
    used = np.zeros(batch.table.shape, dtype=bool)
    for b, pages in enumerate(batch.pages):
        used[b, :len(pages)] = True
    batch.table[used] += first
    batch.pages = [p + first for p in batch.pages]
    assert (batch.table[used] < border).any() and (batch.table[used] >= border).any()
    batch.table_d.copy_(torch.from_numpy(batch.table))
    batch.caches = caches
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, 2)
    batch.check(o, lse, 2)
    for x in caches:
        x[first:first + pool] = 0


@pytest.mark.parametrize("form", FORMS)
def test_the_same_bits_again(gpu_runner, form):
    """Eager calls one behind the other in one workspace, which holds any bytes, then what the call before left there."""
    batch = batch_of(form, 64)
    o, lse = batch.outputs(True)
    ws = batch.attend(gpu_runner, o, lse, 2)
    batch.check(o, lse, 2)
    first = o.clone(), lse.clone()
    for fill in (None, 0xff, None, 0x3f):
        if fill is not None:
            ws.fill_(fill)
        o, lse = batch.outputs(True)
        assert batch.attend(gpu_runner, o, lse, 2, workspace=ws) is ws
        assert torch.equal(o, first[0]) and torch.equal(lse, first[1])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("which,scale", [(1, 255), (3, 254)])
def test_keys_and_queries_that_are_no_numbers(gpu_runner, form, which, scale):
    """Rows that see such a key, or are one, get NaN; all others what they get without it."""
    batch = batch_of(form, 64)
    g = batch.heads // batch.kv_heads
    nan = torch.zeros(batch.total, batch.heads, dtype=torch.bool, device=batch.dev)
    for b, (sq, sk) in enumerate(batch.lens):
        key, head = (sk - 1, 1) if b % 2 == 0 else (sk - sq // 2 - 1, 6)
        batch.caches[which][batch.table[b, key // 64], head, key % 64, b % 4] = scale
        at, end = int(batch.offsets[b]), int(batch.offsets[b + 1])
        nan[at + max(0, key - (sk - sq)):end, head * g:head * g + g] = True
        batch.q[at, 4 * g, 100] = float("nan")
        nan[at, 4 * g] = True
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, 2)
    batch.check(o, lse, 2, nan_rows=nan)


# Heads of one K/V head that fill more than a row tile, so that a token's rows lie in several.
WIDE = [(96, 1, [(1, 700), (1, 0), (1, 65)]), (300, 1, [(1, 700), (3, 2), (2, 1300)]), (512, 1, [(1, 3000), (5, 90)]),
        (516, 2, [(7, 2000), (0, 3), (1, 1)] * 3), (2000, 1, [(30, 500)])]


@pytest.mark.parametrize("causal", [0, 2])
@pytest.mark.parametrize("heads,kv_heads,lens", WIDE, ids=str)
def test_wide_groups(gpu_runner, heads, kv_heads, lens, causal):
    batch = Cache4(heads, kv_heads, 32, lens)
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, causal)
    batch.check(o, lse, causal)
    assert_guard_rows_untouched(batch)


@pytest.mark.parametrize("sequences", [1, 600_000])
def test_queries_past_4_gib(gpu_runner, sequences):
    """600000 tokens of 32 heads, of one sequence or of one each; looked at are some at both ends and in the middle."""
    tokens, keys = 600_000, 70
    batch = Cache4(32, 8, 64, [(1, keys)])
    gen = torch.Generator(device=batch.dev).manual_seed(2)
    q = torch.randn(tokens, 32, 128, generator=gen, device=batch.dev, dtype=torch.bfloat16)
    assert q.nbytes > 1 << 32
    o, lse = torch.full_like(q, float("nan")), torch.full((32, tokens), float("nan"), device=batch.dev)
    cu = torch.arange(0, tokens + 1, tokens // sequences, dtype=torch.int32, device=batch.dev)
    table = batch.table_d.expand(sequences, -1).contiguous()
    seqlens = batch.seqlens.expand(sequences).contiguous()
    gpu_runner.call_paged_mx4(q, *batch.caches, o, lse, cu, seqlens, table, tokens // sequences, keys, causal=0)
    middle = (1 << 32) // (32 * 256)
    for at in (0, middle - 150, tokens - 300):
        part = slice(at, at + 300)
        batch.lens, batch.offsets, batch.total = [(300, keys)], np.array([0, 300]), 300
        batch.check(o[part], lse[:, part], 0, q=q[part])
    assert not o.isnan().any() and not lse.isnan().any()


@pytest.mark.parametrize("form", FORMS)
def test_infinite_queries(gpu_runner, form):
    """Scores are then infinite or no numbers: O and LSE are NaN, or where all of a row's are -inf those of a row that sees
    no key.  Other rows do not notice."""
    batch = batch_of(form, 64)
    g, dim, head = batch.heads // batch.kv_heads, 37, 5
    kinds = torch.zeros(batch.total, dtype=torch.long, device=batch.dev)       # 1: no number, 2: as without keys
    for b, (sq, sk) in enumerate(batch.lens):
        k = batch.keys(b)[0][:, head // g, dim]
        gain = float("inf") if b % 2 else float("-inf")
        rows = slice(int(batch.offsets[b]), int(batch.offsets[b + 1]))
        batch.q[rows, head, dim] = gain
        sees_other = torch.cumsum((k * np.sign(gain) >= 0).long(), 0)[sk - sq:] > 0    # a key whose score is not -inf
        kinds[rows] = torch.where(sees_other, 1, 2)
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, 2)
    assert o[kinds == 1, head].isnan().all() and lse[head, kinds == 1].isnan().all()
    assert (o[kinds == 2, head] == 0).all() and torch.isneginf(lse[head, kinds == 2]).all()
    # The others, with those rows as any.
    want, want_lse = batch.outputs(True)
    batch.q[:, head, dim] = 1
    batch.attend(gpu_runner, want, want_lse, 2)
    o[:, head], lse[head] = want[:, head], want_lse[head]
    assert torch.equal(o, want) and torch.equal(lse, want_lse)
    batch.check(want, want_lse, 2)


@pytest.mark.parametrize("form", FORMS)
def test_the_largest_keys_touch_only_rows_that_see_them(gpu_runner, form):
    """Keys of 6 * 2^125 in all dims, whose scores and weighted sums pass FP32: whatever the rows get that see them, the
    others get the bits that they get without."""
    batch = batch_of(form, 64)
    want = [x.clone() for x in batch.outputs(True)]
    batch.attend(gpu_runner, *want, 2)
    batch.check(*want, 2)
    sees = torch.zeros(batch.total, batch.heads, dtype=torch.bool, device=batch.dev)
    g = batch.heads // batch.kv_heads
    for b, (sq, sk) in enumerate(batch.lens):
        key, head = sk - max(1, sq // 3), b % batch.kv_heads
        page, slot = batch.table[b, key // 64], key % 64
        for x, byte in zip(batch.caches, (0xf7, 252, 0x7f, 252)):
            x[page, head, slot] = byte
        at, end = int(batch.offsets[b]), int(batch.offsets[b + 1])
        sees[at + max(0, key - (sk - sq)):end, head * g:head * g + g] = True
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, 2)
    assert torch.equal(o[~sees], want[0][~sees]) and torch.equal(lse.T[~sees], want[1].T[~sees])
    assert (~sees).any() and not torch.equal(o[sees], want[0][sees])
