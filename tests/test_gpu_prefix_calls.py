"""GPU checks of attention behind shared prefixes called as a serving engine calls it: workspaces of exactly the size
asked for and of larger steps, slots and sizes padded for a captured graph, sequences in any order of prefixes."""
import numpy as np
import pytest
import torch

from tests.serving import Batch, offsets

pytestmark = pytest.mark.gpu

# (heads, kv_heads, page, prefixes, sequences of no prefix, causal) of the three cuts, and of batches whose plan is
# read from memory.
CUTS = {
    "few_rows_a_prefix": (32, 8, 64, [(1024, [(1, 1100), (1, 1025), (1, 800)]), (256, [(1, 300)])], [(1, 50)], 0),
    "few_rows_a_sequence": (32, 8, 64, [(1024, [(2, 1100 + 9 * i) for i in range(12)])], [(1, 70)], 2),
    "many_rows_a_sequence": (8, 2, 64, [(512, [(40, 600), (9, 900)])], [(33, 100)], 2),
    "over_512_sequences": (4, 1, 32, [(160, [(1, 170 + i % 90) for i in range(530)])], [], 0),
    "more_kv_heads_than_cus": (300, 300, 32, [(64, [(1, 100), (2, 70)])], [(1, 9)], 0),
}


def size_of(runner, x, causal, **over):
    a = dict(batch=len(x.lens), heads=x.heads, kv_heads=x.kv_heads, max_q=x.max_q, max_k=x.max_k,
             total_q=x.q.shape[0], page_size=x.page, max_pages=x.table.shape[1], num_pages=x.k.shape[0],
             num_prefixes=len(x.members), max_prefix_pages=x.prefix_table.shape[1], causal=causal)
    a.update(over)
    return runner.prefix_paged_workspace_size(**a)


@pytest.mark.parametrize("name", CUTS)
def test_workspace_of_exactly_its_size(gpu_runner, name):
    """Nothing is written before or behind the workspace, and a larger one gives bitwise the same."""
    heads, kvh, page, prefixes, alone, causal = CUTS[name]
    print("prefix workspace", name, flush=True)
    x = Batch(heads, kvh, page, prefixes, alone)
    need = size_of(gpu_runner, x, causal)
    assert need > 0
    buf = torch.full((need + 8192,), 0xA5, dtype=torch.uint8, device=x.dev)
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, causal, workspace=buf[4096:4096 + need])
    torch.cuda.synchronize()
    assert (buf[:4096] == 0xA5).all() and (buf[4096 + need:] == 0xA5).all()
    x.check(o, l, causal)
    o2, l2 = torch.empty_like(o), torch.empty_like(l)
    x.attend(gpu_runner, o2, l2, causal, workspace=buf)
    torch.cuda.synchronize()
    assert torch.equal(o2.view(torch.int16), o.view(torch.int16)) and torch.equal(l2, l)
    with pytest.raises(RuntimeError):
        x.attend(gpu_runner, o, l, causal, workspace=buf[4096:4096 + need - 1])


def test_workspace_of_the_largest_step_serves_smaller_ones(gpu_runner):
    """One workspace for steps of all three cuts."""
    steps = [(64, 8, [(512, [(60, 700), (60, 800), (50, 520)])], 2),
             (64, 8, [(512, [(1, 700 + i) for i in range(40)])], 0),
             (64, 8, [(512, [(1, 600)]), (128, [(1, 300), (1, 129)])], 0)]
    xs = [Batch(h, kvh, 64, p, seed=i) for i, (h, kvh, p, _) in enumerate(steps)]
    need = max(size_of(gpu_runner, x, c) for x, (*_, c) in zip(xs, steps))
    assert need <= size_of(gpu_runner, xs[0], 2, batch=40, num_prefixes=2, max_q=60, total_q=170, max_prefix_pages=8)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=xs[0].dev)
    outs = [x.outputs(True) for x in xs]
    for _ in range(2):
        for x, (o, l), (*_, c) in zip(xs, outs, steps):
            x.attend(gpu_runner, o, l, c, workspace=ws)
    torch.cuda.synchronize()
    for x, (o, l), (*_, c) in zip(xs, outs, steps):
        x.check(o, l, c)


@pytest.mark.parametrize("name", CUTS)
def test_sequences_before_the_first_prefix(gpu_runner, name):
    """cu_prefix_seqs starts behind 0: the sequences of no prefix come first."""
    heads, kvh, page, prefixes, alone, causal = CUTS[name]
    alone = alone + [(2, 90), (1, 0), (0, 70), (1, 33)]
    print("prefix behind others", name, flush=True)
    x = Batch(heads, kvh, page, prefixes, alone)
    n, m = len(x.lens), len(alone)
    turn = list(range(n - m, n)) + list(range(n - m))               # those of no prefix first
    x.lens, x.pages = [x.lens[i] for i in turn], [x.pages[i] for i in turn]
    x.table = np.ascontiguousarray(x.table[turn])
    x.offsets = offsets([q for q, _ in x.lens])
    x.cu.copy_(torch.from_numpy(x.offsets))
    x.seqlens.copy_(torch.tensor([k for _, k in x.lens], dtype=torch.int32))
    x.table_d.copy_(torch.from_numpy(x.table))
    x.cu_prefix += m
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, causal)
    torch.cuda.synchronize()
    x.check(o, l, causal)


@pytest.mark.parametrize("slots,keys", [(1, 0), (63, 0), (63, 640), (300, 640)])
@pytest.mark.parametrize("queries,causal", [(1, 0), (9, 2)])
def test_padded_prefix_slots(gpu_runner, slots, keys, queries, causal):
    """Prefix slots without sequences, with and without keys, before and behind one with many rows: their tables are
    not read."""
    print("prefix slots", slots, keys, queries, flush=True)
    x = Batch(32, 8, 64, [(640, [(queries, 660 + 5 * i) for i in range(40)])])
    before = slots // 3
    empty = lambda n, v: torch.full((n, *v.shape[1:]), 1 << 30, dtype=torch.int32, device=x.dev)
    x.prefix_table_d = torch.cat([empty(before, x.prefix_table_d), x.prefix_table_d,
                                  empty(slots - before, x.prefix_table_d)])
    lens = [keys] * before + [640] + [keys] * (slots - before)
    x.prefix_lens = torch.tensor(lens, dtype=torch.int32, device=x.dev)
    x.cu_prefix = torch.tensor([0] * (before + 1) + [40] * (slots - before + 1), dtype=torch.int32, device=x.dev)
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, causal)
    torch.cuda.synchronize()
    x.check(o, l, causal)


def test_prefixes_of_the_same_pages(gpu_runner):
    """Two prefixes may hold the same pages (a beam's group split in two)."""
    x = Batch(16, 4, 64, [(512, [(1, 600), (2, 513), (1, 700), (1, 520)])])
    x.prefix_table_d = x.prefix_table_d.repeat(2, 1)
    x.prefix_lens = x.prefix_lens.repeat(2)
    x.cu_prefix = torch.tensor([0, 2, 4], dtype=torch.int32, device=x.dev)
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, 2)
    torch.cuda.synchronize()
    x.check(o, l, 2)


@pytest.mark.parametrize("causal", [0, 2])
def test_a_graph_of_a_padded_batch(gpu_runner, causal):
    """Captured for more queries, tokens and keys than a step has; replayed with batches of other shapes, with eager
    calls between."""
    heads, kvh, page, slots = 16, 4, 64, 6
    x = Batch(heads, kvh, page, [(256, [(30, 1000), (20, 900), (25, 800)]), (128, [(10, 700), (1, 600)])], [(1, 500)])
    x.max_q, x.max_k = 64, 1024
    x.table = np.concatenate([x.table, np.full((slots, 17 - x.table.shape[1]), -1, np.int32)], 1)
    x.table_d = torch.from_numpy(x.table).to(x.dev)
    o, l = x.outputs(True)
    ws = x.attend(gpu_runner, o, l, causal)
    torch.cuda.synchronize()
    x.check(o, l, causal)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.attend(gpu_runner, o, l, causal, workspace=ws)
    for lens in ([(1, 900), (1, 800), (1, 300), (1, 600), (1, 129), (1, 1)],
                 [(0, 900), (60, 800), (0, 0), (1, 0), (5, 100), (3, 500)],
                 [(1, 1000), (1, 0), (1, 0), (1, 0), (1, 0), (1, 0)],
                 [(30, 1000), (20, 900), (25, 800), (10, 700), (1, 600), (1, 500)]):
        x.lens, x.offsets = lens, offsets([q for q, _ in lens])
        x.cu.copy_(torch.from_numpy(x.offsets))
        x.seqlens.copy_(torch.tensor([k for _, k in lens], dtype=torch.int32))
        x.q.copy_(torch.randn(x.q.shape, device=x.dev).to(torch.bfloat16))
        for _ in range(2):
            o.fill_(float("nan"))
            l.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            x.check(o, l, causal)
            n = int(x.offsets[-1])
            assert torch.isnan(o[n:]).all() and torch.isnan(l[:, n:]).all()
            eager, el = torch.full_like(o, float("nan")), torch.full_like(l, float("nan"))
            x.attend(gpu_runner, eager, el, causal)
            torch.cuda.synchronize()
            assert torch.equal(o[:n].view(torch.int16), eager[:n].view(torch.int16)) and torch.equal(l[:, :n], el[:, :n])


@pytest.mark.parametrize("name", CUTS)
def test_calls_repeat_bitwise(gpu_runner, name):
    heads, kvh, page, prefixes, alone, causal = CUTS[name]
    x = Batch(heads, kvh, page, prefixes, alone, seed=4)
    o, l = x.outputs(True)
    ws = x.attend(gpu_runner, o, l, causal)
    torch.cuda.synchronize()
    again, al = torch.empty_like(o), torch.empty_like(l)
    for _ in range(20):
        x.attend(gpu_runner, again, al, causal, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(again.view(torch.int16), o.view(torch.int16)) and torch.equal(al, l)


@pytest.mark.parametrize("prefix", [0, 1024])
@pytest.mark.parametrize("heads,kvh,queries,own", [(8, 1, 9, 4000), (8, 1, 33, 2000), (16, 2, 9, 6000), (32, 8, 40, 9000)])
def test_many_own_parts_of_a_row(gpu_runner, heads, kvh, queries, own, prefix):
    """More than 32 rows a sequence, and long keys of its own: as many parts as there are key tiles, or workgroups."""
    x = Batch(heads, kvh, 64, [(prefix, [(queries, prefix + own), (queries, prefix + own - 1000)])])
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, 2)
    torch.cuda.synchronize()
    x.check(o, l, 2)
