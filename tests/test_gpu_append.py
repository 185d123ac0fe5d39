"""GPU checks of appending to paged K/V caches (fav4_bshd_append_paged): every
stored row, every rotated query and every slot that must stay as it was."""
import numpy as np
import pytest
import torch

from tests.serving import D, angles, assert_rotated, offsets

pytestmark = pytest.mark.gpu

# (heads, kv_heads, page, [(new tokens, keys with them), ...], rotary_dim, interleaved, packed, positions, in place)
CASES = [
    (32, 8, 64, [(1, 1), (1, 64), (1, 65), (1, 2000)], 128, False, False, False, False),
    (32, 8, 64, [(1, 700), (1, 33), (1, 128)], 128, True, True, False, True),
    (8, 1, 32, [(5, 5), (17, 100), (1, 31)], 64, False, True, True, False),
    (6, 3, 16, [(40, 40), (0, 12), (7, 30)], 96, True, False, True, False),
    (5, 5, 7, [(13, 13), (2, 90)], 16, False, False, False, True),
    (4, 2, 1, [(3, 9), (6, 6)], 32, True, False, False, False),
    (12, 4, 256, [(300, 800), (511, 511), (1, 256)], 128, False, True, False, False),
    (16, 4, 48, [(9, 50), (1, 48)], 0, False, False, False, False),
    (1, 1, 5, [(1, 3)], 128, False, False, True, False),
]


class Append:
    def __init__(self, heads, kv_heads, page, lens, rotary_dim, interleaved, packed, positions, in_place, seed=3,
                 behind=0, dev="cuda:0", rows=4096):
        gen = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.cu, self.lens, self.page, self.dev = offsets([n for n, _ in lens]), lens, page, dev
        self.tokens = int(self.cu[-1]) + behind
        pages = [-(-sk // page) for _, sk in lens]
        self.pool = sum(pages) + 3
        order = rng.permutation(self.pool)
        self.table = np.full((len(lens), max(pages + [1])), -1, np.int32)
        for b, at in enumerate(offsets(pages)[:-1]):
            self.table[b, :pages[b]] = order[at:at + pages[b]]
        rand = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(dev)
        if packed:
            qkv = rand(self.tokens, heads + 2 * kv_heads + 1, D)       # one head of padding
            self.q, self.k, self.v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, -kv_heads - 1:-1]
        else:
            self.q, self.k, self.v = rand(self.tokens, heads, D), rand(self.tokens, kv_heads, D), rand(self.tokens, kv_heads, D)
        self.q_in = self.q.clone()
        self.q_out = self.q if in_place else torch.full((self.tokens, heads, D), float("nan"), dtype=torch.bfloat16, device=dev)
        self.kc, self.vc = rand(self.pool, page, kv_heads, D), rand(self.pool, page, kv_heads, D)
        self.before = self.kc.clone(), self.vc.clone()
        self.cos = self.sin = None
        if rotary_dim:
            self.cos, self.sin = angles(rows, rotary_dim, dev)
        self.interleaved = interleaved
        self.positions = None
        if positions:
            self.positions = torch.from_numpy(rng.integers(0, rows, self.tokens).astype(np.int32)).to(dev)
        i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)
        self.cu_d, self.seqlens, self.table_d = i32(self.cu), i32([sk for _, sk in lens]), i32(self.table)

    def call(self, runner, **more):
        runner.call_append_paged(self.q, self.k, self.v, self.q_out, self.kc, self.vc, self.cu_d, self.seqlens,
                                 self.table_d, cos=self.cos, sin=self.sin, interleaved=self.interleaved,
                                 positions=self.positions, **more)

    def where(self):
        """Per token of a sequence: its slot and the flat cache row, or -1."""
        slots, rows = [], []
        for b, (n, sk) in enumerate(self.lens):
            for i in range(n):
                s = sk - n + i
                slots.append(s)
                ok = 0 <= s < self.table.shape[1] * self.page and 0 <= self.table[b, s // self.page] < self.pool
                rows.append(self.table[b, s // self.page] * self.page + s % self.page if ok else -1)
        return np.array(slots), np.array(rows)

    def check(self):
        slots, rows = self.where()
        n = int(self.cu[-1])
        pos = slots if self.positions is None else self.positions[:n].cpu().numpy()
        if self.cos is None:
            cos = sin = torch.empty(n, 0, device=self.dev)
        else:
            p = torch.from_numpy(np.clip(pos, 0, self.cos.shape[0] - 1).astype(np.int64)).to(self.dev)
            cos, sin = self.cos[p], self.sin[p]
        if self.q_out is not None:
            assert_rotated(self.q_out[:n], self.q_in[:n], cos, sin, self.interleaved, "q")
            left = self.q_in if self.q_out is self.q else torch.full_like(self.q_in, float("nan"))
            assert torch.equal(self.q_out[n:].contiguous().view(torch.int16), left[n:].contiguous().view(torch.int16))
        kvh = self.k.shape[1]
        kept = torch.from_numpy(np.flatnonzero(rows >= 0)).to(self.dev)
        at = torch.from_numpy(rows[rows >= 0].astype(np.int64)).to(self.dev)
        k, v = self.kc.view(-1, kvh, D), self.vc.view(-1, kvh, D)
        assert_rotated(k[at], self.k[kept], cos[kept], sin[kept], self.interleaved, "k")
        assert torch.equal(v[at].view(torch.int16), self.v[kept].contiguous().view(torch.int16))
        rest = torch.ones(k.shape[0], dtype=torch.bool, device=self.dev)
        rest[at] = False
        for now, was in zip((k, v), self.before):
            assert torch.equal(now[rest].view(torch.int16), was.view(-1, kvh, D)[rest].view(torch.int16))


@pytest.mark.parametrize("case", CASES, ids=lambda c: "h%dkv%d_p%d_r%d%s%s%s%s" % (
    c[0], c[1], c[2], c[4], "i" * c[5], "_packed" * c[6], "_pos" * c[7], "_inplace" * c[8]))
def test_append(gpu_runner, case):
    print("append", case, flush=True)
    x = Append(*case, behind=2)
    x.call(gpu_runner)
    torch.cuda.synchronize()
    x.check()


def test_append_without_queries(gpu_runner):
    x = Append(8, 4, 64, [(3, 70), (1, 1)], 128, False, False, False, False)
    x.q = x.q_out = None
    x.call(gpu_runner)
    torch.cuda.synchronize()
    x.check()


def test_append_skips_slots_that_do_not_exist(gpu_runner):
    """More new tokens than keys, pages of -1 and past the pool, slots past the table: not stored; positions clamped."""
    x = Append(8, 2, 16, [(5, 3), (4, 40), (3, 20), (2, 33), (1, 0)], 64, False, False, False, False, rows=30)
    x.table[1, 2] = -1                     # slots 32..: of slots 36..39 none is stored
    x.table[2, 1] = x.pool                 # slots 17..19
    x.lens[3] = (2, 49)                    # slots 47 and 48 of a table of 48
    x.table[3, 2] = x.table[1, 1]          # a page of its own for slot 47 (sequence 1 stores nothing there)
    x.table_d.copy_(torch.from_numpy(x.table))
    x.seqlens.copy_(torch.tensor([sk for _, sk in x.lens], dtype=torch.int32))
    _, rows = x.where()
    assert (rows >= 0).tolist() == [False, False, True, True, True] + [False] * 4 + [False] * 3 + [True, False] + [False]
    x.call(gpu_runner)
    torch.cuda.synchronize()
    x.check()


@pytest.mark.parametrize("batch", [63, 64, 65, 129, 4097, 5000])
def test_append_many_sequences(gpu_runner, batch):
    """Batches around the steps of the search for a token's sequence, some without tokens."""
    rng = np.random.default_rng(batch)
    lens = [(int(n), int(n) + int(r)) for n, r in zip(rng.choice([0, 1, 1, 3], batch), rng.integers(0, 20, batch))]
    x = Append(2, 1, 8, lens, 32, False, False, False, False)
    x.call(gpu_runner)
    torch.cuda.synchronize()
    x.check()


def test_append_special_values(gpu_runner):
    """NaN and infinities in dims that are not turned and in V pass bit by bit."""
    x = Append(4, 2, 16, [(6, 20)], 64, False, False, False, False)
    for t in (x.k, x.q):
        t[0, :, 70], t[1, :, 127], t[2, :, 64] = float("nan"), float("inf"), float("-inf")
    x.v[3, :, 5], x.v[4, :, 99] = float("nan"), float("-inf")
    x.q_in = x.q.clone()
    x.call(gpu_runner)
    torch.cuda.synchronize()
    slots, rows = x.where()
    k, v = x.kc.view(-1, 2, D), x.vc.view(-1, 2, D)
    for i, r in enumerate(rows):
        assert torch.equal(k[r, :, 64:].view(torch.int16), x.k[i, :, 64:].view(torch.int16))
        assert torch.equal(v[r].view(torch.int16), x.v[i].view(torch.int16))
    assert torch.equal(x.q_out[:, :, 64:].view(torch.int16), x.q[:, :, 64:].view(torch.int16))


def test_append_far_slots(gpu_runner):
    """A cache of more than 2^31 elements (rows past 4 GiB): the last page of the pool."""
    kvh, page, pool = 8, 128, 17000
    dev = "cuda:0"
    kc = torch.zeros((pool, page, kvh, D), dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    gen = torch.Generator(device=dev).manual_seed(1)
    k, v = (torch.randn((3, kvh, D), generator=gen, device=dev).to(torch.bfloat16) for _ in range(2))
    table = torch.full((1, pool), -1, dtype=torch.int32, device=dev)
    table[0, pool - 2], table[0, pool - 1] = pool - 1, pool - 2
    cu = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    seqlens = torch.tensor([(pool - 1) * page + 2], dtype=torch.int32, device=dev)
    gpu_runner.call_append_paged(None, k, v, None, kc, vc, cu, seqlens, table)
    torch.cuda.synchronize()
    assert torch.equal(kc[pool - 1, page - 1], k[0]) and torch.equal(kc[pool - 2, :2], k[1:])
    assert torch.equal(vc[pool - 1, page - 1], v[0]) and torch.equal(vc[pool - 2, :2], v[1:])
    kc[pool - 1, page - 1] = 0
    kc[pool - 2, :2] = 0
    assert not kc.view(torch.int16).any()


def test_append_in_a_graph_and_on_a_stream(gpu_runner):
    """Captured once and replayed with new tokens and lengths, and a call on another stream."""
    x = Append(8, 2, 16, [(1, 20), (1, 37), (1, 5)], 128, False, False, False, False)
    x.call(gpu_runner)
    torch.cuda.synchronize()
    x.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.call(gpu_runner)
    for step in range(3):
        x.lens = [(1, sk + 1 if sk % 16 else sk) for _, sk in x.lens]
        x.seqlens.copy_(torch.tensor([sk for _, sk in x.lens], dtype=torch.int32))
        for t in (x.q, x.k, x.v):
            t.copy_(torch.randn(t.shape, device=x.dev).to(torch.bfloat16))
        x.q_in.copy_(x.q)
        x.before = x.kc.clone(), x.vc.clone()
        graph.replay()
        torch.cuda.synchronize()
        x.check()
    y = Append(8, 2, 16, [(9, 20), (2, 37)], 128, False, False, False, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y.call(gpu_runner, stream=side.cuda_stream)
    side.synchronize()
    y.check()
