"""Storing in 4-bit paged caches and reading them back: bit by bit what the definitions say."""
import numpy as np
import pytest
import torch

from tests.mx4 import quantise, rotated32, values
from tests.serving import D, angles, offsets

pytestmark = pytest.mark.gpu


class Tokens:
    """New tokens of sequences (new, all keys), caches of random bytes, pages anywhere; slots of tokens in `lost`
    (sequence, entry of its table) lie in no page."""

    def __init__(self, lens, heads=4, kv_heads=2, page=16, rotary_dim=128, interleaved=False, packed=False,
                 positions=False, lost=(), tail=0, seed=3, dev="cuda:0", gain=1.0):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.kv_heads, self.page, self.interleaved = lens, heads, kv_heads, page, interleaved
        new, keys = zip(*lens)
        self.offsets = offsets(new)
        self.n, total = int(self.offsets[-1]), int(self.offsets[-1]) + tail
        pages = [max(1, -(-k // page)) for k in keys]
        pool = sum(pages) + 2
        order = rng.permutation(pool)
        self.table = np.full((len(lens), max(pages)), -1, dtype=np.int32)
        at = 0
        for b, n in enumerate(pages):
            self.table[b, :n] = order[at:at + n]
            at += n
        for b, e in lost:
            self.table[b, e] = [-1, pool, 1 << 30][(b + e) % 3]
        self.pool, self.dev = pool, dev
        rand = lambda *s: (torch.randn(*s, generator=gen) * gain).to(torch.bfloat16)
        if packed:
            self.qkv = rand(total, heads + 2 * kv_heads, D).to(dev)
            self.q, self.k, self.v = self.qkv.split([heads, kv_heads, kv_heads], dim=1)
        else:
            self.q, self.k, self.v = (rand(total, h, D).to(dev) for h in (heads, kv_heads, kv_heads))
        i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)
        self.cu, self.seqlens, self.table_d = i32(self.offsets), i32(keys), i32(self.table)
        self.cos, self.sin = angles(max(keys) + 7, rotary_dim, dev) if rotary_dim else (None, None)
        self.positions = i32(rng.integers(0, max(keys) + 7, total)) if positions else None
        shape = (pool, kv_heads, page)
        self.caches = [torch.from_numpy(rng.integers(0, 256, (*shape, w), dtype=np.uint8)).to(dev) for w in (64, 4, 64, 4)]
        self.q_out = torch.full_like(self.q, float("nan"), memory_format=torch.contiguous_format)
        # Per token: its slot, and the page and the place in it (page -1: none).
        self.slot = np.concatenate([np.arange(k - n, k) for n, k in lens] or [[]]).astype(np.int64)
        seq = np.repeat(np.arange(len(lens)), new)
        entry = np.clip(self.slot // page, 0, self.table.shape[1] - 1)
        self.at = self.table[seq, entry].astype(np.int64)
        self.at[(self.at >= pool) | (self.slot < 0)] = -1
        self.place = self.slot % page

    def append(self, runner, q=True, q_out=None, **more):
        out = self.q_out if q_out is None else q_out
        runner.call_append_paged_mx4(self.q if q else None, self.k, self.v, out if q else None, *self.caches, self.cu,
                                     self.seqlens, self.table_d, cos=self.cos, sin=self.sin,
                                     interleaved=self.interleaved, positions=self.positions, **more)

    def turned(self, x):
        x = x[:self.n]
        if self.cos is None:
            return x.float().cpu().numpy()
        p = self.slot if self.positions is None else self.positions[:self.n].cpu().numpy()
        p = torch.from_numpy(np.clip(p, 0, self.cos.shape[0] - 1)).to(self.dev)
        return rotated32(x, self.cos[p], self.sin[p], self.interleaved)

    def want(self):
        """The caches after the append, as numpy."""
        out = [x.cpu().numpy().copy() for x in self.caches]
        for j, x in ((0, self.turned(self.k)), (2, self.v[:self.n].float().cpu().numpy())):
            codes, scales = quantise(x)
            ok = self.at >= 0
            out[j][self.at[ok], :, self.place[ok]] = codes[ok]
            out[j + 1][self.at[ok], :, self.place[ok]] = scales[ok]
        return out

    def check(self, want, q=True):
        for name, got, ref in zip(("k_cache", "k_scales", "v_cache", "v_scales"), self.caches, want):
            bad = got.cpu().numpy() != ref
            assert not bad.any(), (name, int(bad.sum()), np.argwhere(bad)[:4])
        if q:
            ref = torch.from_numpy(self.turned(self.q)).to(torch.bfloat16)
            assert torch.equal(self.q_out[:self.n].cpu().view(torch.int16), ref.view(torch.int16))


@pytest.mark.parametrize("rotary_dim", [0, 16, 32, 48, 64, 112, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("packed,positions", [(False, False), (True, True)])
def test_append(gpu_runner, rotary_dim, interleaved, packed, positions):
    t = Tokens([(1, 1), (5, 40), (0, 9), (33, 33), (16, 100)], rotary_dim=rotary_dim, interleaved=interleaved,
               packed=packed, positions=positions and rotary_dim > 0)
    want = t.want()
    t.append(gpu_runner)
    torch.cuda.synchronize()
    t.check(want)


@pytest.mark.parametrize("heads,kv_heads,page", [(32, 8, 64), (8, 1, 1), (3, 3, 17), (10, 5, 128)])
def test_append_layouts(gpu_runner, heads, kv_heads, page):
    t = Tokens([(1, 200), (300, 301), (1, 1), (2, 77)], heads, kv_heads, page)
    want = t.want()
    t.append(gpu_runner)
    torch.cuda.synchronize()
    t.check(want)


def test_append_of_keys_alone_and_in_place(gpu_runner):
    t = Tokens([(3, 10), (20, 50)])
    want = t.want()
    t.append(gpu_runner, q=False)
    torch.cuda.synchronize()
    t.check(want, q=False)
    assert t.q_out.isnan().all()
    ref = torch.from_numpy(t.turned(t.q)).to(torch.bfloat16)
    t.append(gpu_runner, q_out=t.q)
    assert torch.equal(t.q.cpu(), ref)


def test_append_leaves_out_what_has_no_place(gpu_runner):
    """Pages out of the pool, negative slots, rows behind the last sequence: nothing is stored, other rows are."""
    t = Tokens([(40, 40), (3, 64), (9, 5), (1, 0)], lost=[(0, 1), (1, 3)], tail=4)
    want = t.want()
    t.append(gpu_runner)
    torch.cuda.synchronize()
    assert (t.at < 0).sum() == 16 + 3 + 4 + 1
    t.check(want)
    assert t.q_out[t.n:].isnan().all()


def test_append_of_special_numbers(gpu_runner):
    """Ties, zeros of both signs, blocks of tiny and of the largest numbers, infinities and NaN."""
    rows = [np.tile([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0], 16),        # ties of the grid at a scale of 1
            np.tile([0.25, -0.75, 6.0, -7.03125, 2.5, -3.5, 5.0, 0.5], 16),   # the largest just above 7: the next scale
            np.zeros(D), -np.zeros(D), np.full(D, 2.0 ** -126), np.full(D, 3.0 * 2.0 ** -126),
            np.full(D, 3.3e38), np.r_[np.full(64, -3.3e38), np.full(64, 1e-37)],
            np.r_[np.inf, np.ones(127)], np.r_[np.ones(40), np.nan, np.ones(87)],
            np.r_[np.ones(96), -np.inf, np.nan, np.ones(30)], np.linspace(-8, 8, D), np.exp2(np.linspace(-100, 100, D))]
    t = Tokens([(len(rows), len(rows))], kv_heads=1, rotary_dim=0)
    x = torch.tensor(np.array(rows), dtype=torch.float32).to(torch.bfloat16)[:, None]
    t.k.copy_(x)
    t.v.copy_(-x)
    want = t.want()
    t.append(gpu_runner)
    torch.cuda.synchronize()
    t.check(want)
    got = values(t.caches[0], t.caches[1])[t.at, 0, t.place].cpu()
    assert got[8, :32].isnan().all() and not got[8, 32:].isnan().any()
    assert got[9, 32:64].isnan().all() and got[10, 96:].isnan().all() and not got[10, :96].isnan().any()
    assert (got[2] == 0).all() and torch.isfinite(got[6]).all()


@pytest.mark.parametrize("gain", [1e-30, 1.0, 1e30])
def test_values_are_near(gpu_runner, gain):
    """A number is off by at most half a step of the grid, a quarter of the step's upper end; 6 to 7 become 6."""
    t = Tokens([(200, 200)], rotary_dim=0, gain=gain)
    t.append(gpu_runner)
    k, v = (torch.empty_like(x) for x in (t.k, t.v))
    gpu_runner.call_gather_paged_mx4(*t.caches, k, v, t.cu, t.table_d)
    for x, y in ((t.k, k), (t.v, v)):
        x, y = x.double(), y.double()
        most = x.unflatten(-1, (4, 32)).abs().amax(-1).repeat_interleave(32, -1)
        # Steps of 0.5, 1 and 2 at a scale of more than most / 7 / 2 and at most 2 most / 7.
        assert ((x - y).abs() <= torch.maximum(x.abs() / 3, most / 14)).all()


@pytest.mark.parametrize("kv_heads,page", [(8, 64), (1, 16), (3, 5)])
@pytest.mark.parametrize("packed", [False, True])
def test_gather(gpu_runner, kv_heads, page, packed):
    """Any bytes, starts inside a sequence, rows of no page, rows behind the last sequence."""
    lens = [(0, 0), (30, 100), (7, 7), (0, 50), (1, 90), (64, 64), (100, 130)]
    t = Tokens(lens, kv_heads=kv_heads, page=page, lost=[(6, 100 // page)])
    starts = np.array([0, 70, 0, 3, -1, 0, 28], dtype=np.int32)
    rows = t.n + 3
    if packed:
        both = torch.full((rows, 2 * kv_heads, D), 3.0, dtype=torch.bfloat16, device=t.dev)
        k, v = both[:, :kv_heads], both[:, kv_heads:]
    else:
        k, v = (torch.full((rows, kv_heads, D), 3.0, dtype=torch.bfloat16, device=t.dev) for _ in range(2))
    for given in (starts, None):
        k.fill_(3.0), v.fill_(3.0)
        gpu_runner.call_gather_paged_mx4(*t.caches, k, v, t.cu, t.table_d,
                                         starts=None if given is None else torch.from_numpy(given).to(t.dev))
        torch.cuda.synchronize()
        first = starts if given is not None else starts * 0
        key = np.concatenate([np.arange(s, s + n) for s, (n, _) in zip(first, lens)]).astype(np.int64)
        seq = np.repeat(np.arange(len(lens)), [n for n, _ in lens])
        at = t.table[seq, np.clip(key // page, 0, t.table.shape[1] - 1)].astype(np.int64)
        ok = (key >= 0) & (key < t.table.shape[1] * page) & (at >= 0) & (at < t.pool)
        assert (~ok).any() or given is None
        for j, x in ((0, k), (2, v)):
            ref = values(t.caches[j], t.caches[j + 1])[np.where(ok, at, 0), :, np.where(ok, key % page, 0)]
            ref[torch.from_numpy(~ok)] = 0
            assert (x[t.n:] == 3).all()
            got = x[:t.n].double()
            # Numbers below 2^-126 may count as 0.
            same = (got == ref) | (got.isnan() & ref.isnan()) | ((ref.abs() < 2.0 ** -126) & (got == 0))
            assert same.all(), (j, int((~same).sum()))


def test_append_then_gather_of_many_sequences(gpu_runner):
    """More sequences than a wave has lanes, most of them without new tokens."""
    rng = np.random.default_rng(8)
    lens = [(int(n), int(n) + int(k)) for n, k in zip(rng.integers(0, 2, 300) * rng.integers(0, 4, 300), rng.integers(0, 40, 300))]
    t = Tokens(lens)
    want = t.want()
    t.append(gpu_runner)
    torch.cuda.synchronize()
    t.check(want)
    k, v = (torch.empty(t.n, t.kv_heads, D, dtype=torch.bfloat16, device=t.dev) for _ in range(2))
    starts = torch.tensor([k - n for n, k in lens], dtype=torch.int32, device=t.dev)
    gpu_runner.call_gather_paged_mx4(*t.caches, k, v, t.cu, t.table_d, starts=starts)
    for j, x in ((0, k), (2, v)):
        assert torch.equal(x.double(), values(t.caches[j], t.caches[j + 1])[t.at, :, t.place])
