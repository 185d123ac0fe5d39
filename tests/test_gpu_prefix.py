"""GPU checks of attention behind shared prefixes (fav4_bshd_forward_prefix_paged): every sequence against its own
64-bit attention over all of its keys."""
import numpy as np
import pytest
import torch

from tests.serving import Batch, angles, assert_rotated

pytestmark = pytest.mark.gpu

# (heads, kv_heads, page, prefixes, sequences of no prefix, causal)
CASES = {
    "one_token": (8, 8, 32, [(32, [(1, 33)])], [], 0),
    "decode_gqa": (32, 8, 64, [(1024, [(1, 1025), (1, 1100), (1, 1500), (1, 1024 + 64)])], [], 0),
    "decode_mqa_small_pages": (8, 1, 32, [(4096, [(1, 4097 + 37 * i) for i in range(24)])], [], 0),
    "mha": (4, 4, 96, [(960, [(1, 961), (1, 1300), (1, 1000)])], [], 0),
    "odd_groups": (10, 2, 32, [(320, [(3, 400), (1, 321), (7, 777)])], [], 2),
    "prefixes_of_all_kinds": (32, 8, 64, [(640, [(1, 700), (1, 641)]), (0, [(1, 50)]), (100, [(1, 300), (1, 65)]),
                                          (2048, [(1, 2048), (1, 2049), (1, 3000), (1, 2500)]), (512, [])], [(1, 77)], 0),
    "empty_sequences": (16, 4, 64, [(256, [(1, 0), (0, 300), (1, 300), (1, 256), (0, 0)])], [(1, 0), (0, 9), (1, 3)], 0),
    "shorter_than_the_prefix": (8, 2, 64, [(512, [(1, 100), (1, 600), (1, 1), (2, 512), (1, 448)])], [], 0),
    "shorter_than_the_prefix_causal": (8, 2, 64, [(512, [(9, 100), (4, 600), (5, 3), (70, 512), (2, 450)])], [], 2),
    "speculative": (32, 8, 64, [(2048, [(4, 2100), (4, 2052), (4, 4000), (3, 2060)])], [], 2),
    "dense_queries": (8, 2, 128, [(256, [(5, 300), (40, 512)])], [(33, 100)], 0),
    "prefill": (16, 4, 64, [(1024, [(200, 1300), (64, 1088), (129, 1153), (1, 1025)])], [(300, 300)], 2),
    "prefill_mqa": (8, 1, 32, [(96, [(130, 226), (61, 157)])], [], 2),
    "more_queries_than_keys": (4, 2, 64, [(64, [(90, 70), (3, 66)])], [(5, 2)], 2),
    "no_prefix_at_all": (8, 2, 64, [(0, [(1, 500), (2, 64)])], [(1, 1000)], 0),
    "more_row_tiles_than_workgroups": (64, 64, 32, [(128, [(300, 428), (290, 420), (310, 450), (257, 400)])], [], 2),
    "more_row_tiles_than_workgroups_decode": (128, 128, 32, [(96, [(1, 97 + i % 60) for i in range(300)])], [], 0),
    "rows_of_prefixes_uneven": (8, 2, 64, [(1024, [(1, 1025 + 9 * i) for i in range(30)])] +
                                [(64 * i, [(1, 64 * i + 30)]) for i in range(6)], [], 0),
    "rows_of_prefixes_uneven_causal": (16, 2, 32, [(416, [(3, 400 + 7 * i) for i in range(5)])] +
                                       [(32 * i, [(1, 32 * i + 1)]) for i in range(9)], [(2, 70)], 2),
    "more_kv_heads_than_cus": (300, 300, 32, [(64, [(1, 100), (2, 70)])], [(1, 9)], 0),
    "more_kv_heads_than_cus_prefill": (300, 300, 32, [(64, [(40, 140), (33, 70)])], [], 2),
    "large_pages": (8, 2, 1024, [(2048, [(1, 3000), (1, 2049)])], [(1, 10)], 0),
    "widest_group": (256, 1, 64, [(320, [(1, 321), (2, 700)])], [(1, 65)], 2),
    "wide_group": (64, 2, 32, [(1600, [(2, 1700), (3, 1605)])], [], 2),
}


@pytest.mark.parametrize("lse", [False, True], ids=["o", "lse"])
@pytest.mark.parametrize("name", CASES)
def test_prefix(gpu_runner, name, lse):
    heads, kvh, page, prefixes, alone, causal = CASES[name]
    print("prefix", name, "lse", lse, flush=True)
    x = Batch(heads, kvh, page, prefixes, alone)
    o, l = x.outputs(lse)
    x.attend(gpu_runner, o, l, causal)
    torch.cuda.synchronize()
    x.check(o, l, causal)
    assert torch.isnan(x.o_all[o.shape[0]:]).all()


@pytest.mark.parametrize("seed", range(16))
def test_prefix_random(gpu_runner, seed):
    rng = np.random.default_rng(900 + seed)
    kvh = int(rng.choice([1, 2, 4, 8]))
    heads = kvh * int(rng.choice([1, 2, 4, 5, 8]))
    page = int(rng.choice([32, 64, 96, 128]))
    causal = int(rng.choice([0, 2]))
    most_q = int(rng.choice([1, 1, 4, 40, 150]))
    prefixes = []
    for _ in range(int(rng.integers(1, 6))):
        p = int(rng.choice([0, rng.integers(1, 300), rng.integers(300, 3001)]))
        prefixes.append((p, [(int(rng.integers(0, most_q + 1)), p + int(rng.integers(0, 700)))
                             for _ in range(int(rng.integers(0, 9)))]))
    alone = [(1, int(rng.integers(0, 400))) for _ in range(int(rng.integers(0, 3)))] + [(1, 40)]
    print("prefix random", seed, heads, kvh, page, causal, prefixes, alone, flush=True)
    x = Batch(heads, kvh, page, prefixes, alone, seed=seed)
    o, l = x.outputs(seed % 2 == 0)
    x.attend(gpu_runner, o, l, causal)
    torch.cuda.synchronize()
    x.check(o, l, causal)


def test_prefix_many_sequences_and_prefixes(gpu_runner):
    """More sequences and prefixes than a wave has lanes."""
    rng = np.random.default_rng(5)
    prefixes = [(int(rng.integers(0, 6)) * 32, [(int(rng.integers(0, 3)), int(rng.integers(160, 300)))
                                               for _ in range(int(rng.integers(0, 7)))]) for _ in range(150)]
    x = Batch(4, 2, 32, prefixes, [(1, 5)] * 3)
    assert len(x.lens) > 256
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, 0)
    torch.cuda.synchronize()
    x.check(o, l, 0)


# (heads, kv_heads, prefixes, sequences of each, most queries of a sequence, causal)
LARGE_BATCHES = {
    "rows_of_many_sequences": (8, 1, 3, 230, 1, 0),
    "few_rows_a_prefix": (4, 2, 290, 2, 1, 0),
    "many_prefixes": (64, 2, 300, 2, 1, 0),
    "many_prefixes_and_sequences": (16, 1, 300, 3, 2, 2),
    "many_rows_a_sequence": (32, 2, 5, 104, 9, 2),
    "many_rows_a_sequence_and_prefixes": (16, 1, 280, 2, 6, 2),
}


@pytest.mark.parametrize("name", LARGE_BATCHES)
def test_prefix_large_batches(gpu_runner, name):
    """More than 512 sequences or 256 prefixes: each workgroup reads their lengths from global memory."""
    heads, kvh, n, members, most_q, causal = LARGE_BATCHES[name]
    rng = np.random.default_rng(31)
    prefixes = []
    for i in range(n):
        p = 32 * int(rng.integers(0, 8))
        prefixes.append((p, [(int(rng.integers(min(most_q, j), most_q + 1)), p + int(rng.integers(0, 120)))
                             for j in range(members)]))
    print("prefix large", name, flush=True)
    x = Batch(heads, kvh, 32, prefixes, [(1, 40)] * 3)
    assert len(x.lens) > 512 or n > 256
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, causal)
    torch.cuda.synchronize()
    x.check(o, l, causal)
    assert torch.isnan(x.o_all[o.shape[0]:]).all()


def test_prefix_long(gpu_runner):
    """Keys over many ranges: a prefix of 50000 keys, and one sequence's own 20000 behind a short prefix."""
    for prefixes in ([(49984, [(1, 50000), (1, 51000), (2, 50001)])], [(64, [(1, 20000), (1, 70)])]):
        x = Batch(8, 2, 64, prefixes)
        o, l = x.outputs(True)
        x.attend(gpu_runner, o, l, 0)
        torch.cuda.synchronize()
        x.check(o, l, 0)


def test_prefix_large_logits(gpu_runner):
    """Logits far apart (q times 24): the weights of whole parts vanish in the merge."""
    x = Batch(8, 2, 64, [(512, [(1, 600), (1, 513), (3, 900)])])
    x.q.copy_((x.q.float() * 24).to(torch.bfloat16))
    o, l = x.outputs(False)
    x.attend(gpu_runner, o, l, 2)
    torch.cuda.synchronize()
    x.check(o, None, 2, weight_err=24 * 2e-4)


def test_prefix_leaves_other_rows(gpu_runner):
    """Rows before the first and behind the last sequence stay as they were."""
    x = Batch(8, 2, 64, [(128, [(3, 200), (2, 140)])])
    o, l = x.outputs(True)
    x.cu.copy_(torch.tensor([1, 3, 4], dtype=torch.int32))
    x.attend(gpu_runner, o, l, 0)
    torch.cuda.synchronize()
    x.lens, x.offsets = [(2, 200), (1, 140)], np.array([1, 3, 4])
    x.check(o, l, 0)
    assert torch.isnan(o[0]).all() and torch.isnan(o[4:]).all() and torch.isnan(l[:, 0]).all() and torch.isnan(l[:, 4:]).all()


def test_prefix_workspace_contents_and_repeats(gpu_runner):
    """Bitwise the same from call to call, whatever the workspace holds, and with a larger one."""
    x = Batch(16, 4, 64, [(640, [(1, 700), (1, 641), (2, 1000)])], [(1, 90)])
    o, l = x.outputs(True)
    ws = x.attend(gpu_runner, o, l, 0)
    torch.cuda.synchronize()
    first = o.clone(), l.clone()
    for fill in (0xFF, 0x7F, 0):
        ws.fill_(fill)
        o.fill_(0)
        l.fill_(0)
        x.attend(gpu_runner, o, l, 0, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(o.view(torch.int16), first[0].view(torch.int16)) and torch.equal(l, first[1])


def test_prefix_in_a_graph(gpu_runner):
    """Captured once, replayed with other lengths, queries and an emptied slot."""
    x = Batch(16, 4, 64, [(256, [(1, 500), (1, 400), (1, 300)]), (128, [(1, 600), (1, 222)])])
    o, l = x.outputs(True)
    ws = x.attend(gpu_runner, o, l, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.attend(gpu_runner, o, l, 0, workspace=ws)
    for keys in ([500, 400, 300, 600, 222], [257, 310, 256, 129, 128], [499, 0, 300, 128, 100], [300, 300, 300, 300, 222]):
        x.lens = [(1, k) for k in keys]
        x.seqlens.copy_(torch.tensor(keys, dtype=torch.int32))
        x.q.copy_(torch.randn(x.q.shape, device=x.dev).to(torch.bfloat16))
        o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        x.check(o, l, 0)
        eager, el = torch.empty_like(o), torch.empty_like(l)
        x.attend(gpu_runner, eager, el, 0)
        torch.cuda.synchronize()
        assert torch.equal(o.view(torch.int16), eager.view(torch.int16)) and torch.equal(l, el)


@pytest.mark.parametrize("heads,kvh,queries,causal", [(64, 2, 1, 0), (32, 2, 2, 2), (16, 4, 9, 2), (8, 1, 40, 2)])
def test_prefix_in_a_graph_of_more_rows(gpu_runner, heads, kvh, queries, causal):
    """More rows than one wave's for each prefix, and for each sequence: replayed with other lengths and prefixes."""
    x = Batch(heads, kvh, 64, [(256, [(queries, 500), (queries, 400), (queries, 300)]), (128, [(queries, 600), (queries, 222)])])
    o, l = x.outputs(True)
    ws = x.attend(gpu_runner, o, l, causal)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.attend(gpu_runner, o, l, causal, workspace=ws)
    for keys in ([500, 400, 300, 600, 222], [257, 310, 256, 129, 128], [499, 0, 300, 128, 100], [300, 300, 300, 300, 222]):
        x.lens = [(queries, k) for k in keys]
        x.seqlens.copy_(torch.tensor(keys, dtype=torch.int32))
        x.q.copy_(torch.randn(x.q.shape, device=x.dev).to(torch.bfloat16))
        o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        x.check(o, l, causal)


def test_prefix_far_pages(gpu_runner):
    """Caches of more than 2^31 elements: shared and own pages past 4 GiB."""
    x = Batch(8, 8, 128, [(256, [(1, 300), (2, 257)])], seed=3)
    pool, far = x.k.shape[0], 17000
    k = torch.zeros((far, 128, 8, 128), dtype=torch.bfloat16, device=x.dev)
    v = torch.zeros_like(k)
    k[far - pool:], v[far - pool:] = x.k, x.v
    x.k, x.v = k, v
    for t in (x.table, x.prefix_table):
        t[(t >= 0) & (t < pool)] += far - pool
        t[t == pool] = far
    x.pages = [p + far - pool for p in x.pages]
    x.table_d.copy_(torch.from_numpy(x.table))
    x.prefix_table_d.copy_(torch.from_numpy(x.prefix_table))
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, 2)
    torch.cuda.synchronize()
    x.check(o, l, 2)


def test_prefix_bad_pages_stay_with_their_sequence(gpu_runner):
    """Page numbers out of range are clamped: the sequence that has them gets some value, the others theirs."""
    x = Batch(8, 2, 64, [(128, [(1, 200), (1, 400), (1, 300)])])
    x.k.nan_to_num_(0.0)
    x.v.nan_to_num_(0.0)
    x.table_d[1, 2:] = torch.tensor([-7, 1 << 30, x.k.shape[0], -1, 5], dtype=torch.int32)[:x.table_d.shape[1] - 2]
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, 0)
    torch.cuda.synchronize()
    assert torch.isfinite(o).all()
    x.lens[1] = (0, 400)                    # not checked
    x.check(o, l, 0)


def test_prefix_on_two_streams(gpu_runner):
    """Two calls at once, each on a stream and with a workspace of its own."""
    xs = [Batch(16, 4, 64, [(1024, [(1, 1100 + 10 * i) for i in range(8)])], seed=s) for s in (1, 2)]
    outs = [x.outputs(False) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for x, (o, _), s in zip(xs, outs, streams):
            x.attend(gpu_runner, o, None, 0, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for x, (o, _) in zip(xs, outs):
        x.check(o, None, 0)


def test_prefix_against_the_paged_call(gpu_runner):
    """The same batch through call_splitkv_paged, which reads the shared pages from every sequence's own table."""
    x = Batch(32, 8, 64, [(2048, [(1, 2100), (1, 2500), (1, 2048), (1, 2049)])])
    for b, pages in enumerate(x.pages):
        x.table[b, :len(pages)] = pages
    x.table_d.copy_(torch.from_numpy(x.table))
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, 0)
    o2, l2 = torch.empty_like(o), torch.empty_like(l)
    gpu_runner.call_splitkv_paged(x.q, x.k, x.v, o2, l2, x.cu, x.seqlens, x.table_d, x.max_q, x.max_k, causal=0)
    torch.cuda.synchronize()
    x.check(o, l, 0)
    x.check(o2, l2, 0)


def test_step(gpu_runner):
    """Append, then attend, over three decode steps of one batch: keys that the append stored are attended to."""
    x = Batch(32, 8, 64, [(512, [(1, 512), (1, 600), (1, 575)]), (64, [(1, 100), (1, 127)])], spare=8)
    x.max_k += 4
    x.table = np.concatenate([x.table, np.full((5, 1), -1, np.int32)], 1)
    used = set(np.concatenate(x.pages).tolist())
    free = [p for p in range(x.k.shape[0]) if p not in used]
    for b, (_, sk) in enumerate(x.lens):               # a page for the keys to come
        n = len(x.pages[b])
        if n * 64 < sk + 3:
            page = free.pop()
            x.table[b, n] = page
            x.pages[b] = np.append(x.pages[b], page)
            x.k[page] = 0
            x.v[page] = 0
    x.table_d = torch.from_numpy(x.table).to(x.dev)
    cos, sin = angles(1024, 128, x.dev)
    gen = torch.Generator(device=x.dev).manual_seed(4)
    ws = None
    for _ in range(3):
        x.lens = [(1, sk + 1) for _, sk in x.lens]
        x.seqlens.copy_(torch.tensor([sk for _, sk in x.lens], dtype=torch.int32))
        qkv = torch.randn((5, 48, 128), generator=gen, device=x.dev).to(torch.bfloat16)
        q, k, v = qkv[:, :32], qkv[:, 32:40], qkv[:, 40:]
        turned = torch.empty_like(q, memory_format=torch.contiguous_format)
        o, l = x.outputs(True)
        gpu_runner.call_append_paged(q, k, v, turned, x.k, x.v, x.cu, x.seqlens, x.table_d, cos=cos, sin=sin)
        ws = x.attend(gpu_runner, o, l, 0, q=turned, workspace=ws)
        torch.cuda.synchronize()
        at = torch.tensor([sk - 1 for _, sk in x.lens], device=x.dev)
        assert_rotated(turned, q, cos[at], sin[at], False)
        for b, (_, sk) in enumerate(x.lens):
            page = x.pages[b][(sk - 1) // 64]
            assert torch.equal(x.v[page, (sk - 1) % 64], v[b])
        x.check(o, l, 0, q=turned)
