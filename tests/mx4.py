"""Inputs and references of the tests of 4-bit paged caches.

What is stored has one right answer, bit by bit: the products and sums of the rotation are rounded one by one in FP32,
a block's scale and the nearest numbers of the grid follow from that.  Reading back is exact.  The tolerances of the
attention are those of tests/serving.py (its K and V are exact in BF16): BF16 weights and the output's rounding."""
import numpy as np
import torch

from tests.serving import D, HALF_STEP, LSE_TOL, SCALE, offsets

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def values(codes, scales):
    """float64 numbers of codes [..., 64] and scales [..., 4] (uint8 numpy or torch, returned alike)."""
    if isinstance(codes, torch.Tensor):
        grid = torch.tensor(np.concatenate([GRID, -GRID]), device=codes.device)
        code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
        power = torch.tensor(np.r_[np.ldexp(1.0, np.arange(253) - 127), [np.nan] * 3], device=codes.device)
        return grid[code] * power[scales.long()].repeat_interleave(32, -1)
    return values(torch.from_numpy(codes), torch.from_numpy(scales)).numpy()


def quantise(x):
    """(codes, scales) of float32 x [..., 128], element by element from the definition."""
    x = np.asarray(x, dtype=np.float32)
    b = x.reshape(*x.shape[:-1], 4, 32)
    most = np.abs(b).max(-1)
    fin = np.isfinite(b).all(-1)
    with np.errstate(divide="ignore", invalid="ignore"):
        mant, exp = np.frexp(np.where(fin, most, 1).astype(np.float64))       # most = mant 2^exp, mant in [0.5, 1)
    e = np.clip(np.where(most == 0, -125, exp - 3 + (mant > 0.875)), -125, 125)   # 7 2^e = 0.875 2^(e + 3)
    y = np.abs(np.where(fin[..., None], b, 0).astype(np.float64)) / np.exp2(e)[..., None]
    edges = (GRID[1:] + GRID[:-1]) / 2
    code = np.searchsorted(edges, y, side="left")                             # at an edge the lower one ...
    code += (y == edges[np.minimum(code, 6)]) & (code % 2 == 1) & (code < 7)    # ... or the even one
    code = code.astype(np.uint8) | (np.signbit(b).astype(np.uint8) << 3)
    code = np.where(fin[..., None], code, 0).reshape(x.shape).astype(np.uint8)
    return code[..., ::2] | (code[..., 1::2] << 4), np.where(fin, e + 127, 255).astype(np.uint8)


def rotated32(x, cos, sin, interleaved):
    """x [tokens, heads, 128] (BF16 torch) turned by the tokens' angles, every product and sum rounded to FP32."""
    x = x.float().cpu().numpy()
    r = 2 * cos.shape[1]
    out = x.copy()
    i = np.arange(r // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    c, s = (t.cpu().numpy()[:, None] for t in (cos, sin))
    with np.errstate(over="ignore", invalid="ignore"):
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
    return out


class Cache4:
    """4-bit caches of a batch whose pages lie anywhere in the pool.  Unused pages and slots hold any bytes, scales of
    255 among them, and table entries that must not be read numbers out of range."""

    def __init__(self, heads, kv_heads, page, lens, seed=1, dev="cuda:0", spare=3, extra_pages=0):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.page, self.dev, self.lens = heads, kv_heads, page, dev, lens
        sq, sk = zip(*lens)
        cu = offsets(sq)
        self.offsets, self.total = cu, int(cu[-1])
        self.max_q, self.max_k = max(max(sq), 1), max(max(sk), 1)
        pages = [-(-k // page) for k in sk]
        pool = sum(pages) + spare
        order = rng.permutation(pool)
        width = -(-self.max_k // page) + extra_pages
        self.table = rng.choice([-3, pool, 1 << 30], size=(len(lens), width)).astype(np.int32)
        shape = (pool, kv_heads, page)
        caches = [torch.from_numpy(rng.integers(0, 256, (*shape, n), dtype=np.uint8)) for n in (64, 4, 64, 4)]
        for x in caches[1::2]:
            x[torch.from_numpy(rng.random(x.shape) < 0.3)] = 255
        at, self.pages = 0, []
        for b, n in enumerate(pages):
            mine = order[at:at + n]
            at += n
            self.table[b, :n] = mine
            self.pages.append(mine.astype(np.int64))
            for i, pg in enumerate(mine):
                rows = min(page, sk[b] - i * page)
                for j in (0, 2):
                    codes, scales = quantise(torch.randn(kv_heads, rows, D, generator=gen).numpy())
                    caches[j][pg, :, :rows], caches[j + 1][pg, :, :rows] = torch.from_numpy(codes), torch.from_numpy(scales)
        self.caches = [x.to(dev) for x in caches]
        i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)
        self.q = torch.randn(max(self.total, 1), heads, D, generator=gen).to(torch.bfloat16).to(dev)
        self.cu, self.seqlens, self.table_d = i32(cu), i32(sk), i32(self.table)

    def outputs(self, lse, guard=3):
        """O and LSE filled with NaN, O with guard rows behind the tokens."""
        n = self.q.shape[0]
        self.o_all = torch.full((n + guard, self.heads, D), float("nan"), dtype=torch.bfloat16, device=self.dev)
        self.lse = torch.full((self.heads, n), float("nan"), device=self.dev) if lse else None
        return self.o_all[:n], self.lse

    def attend(self, runner, o, lse, causal, q=None, **more):
        more.setdefault("max_q", self.max_q)
        more.setdefault("max_k", self.max_k)
        return runner.call_paged_mx4(self.q if q is None else q, *self.caches, o, lse, self.cu, self.seqlens,
                                     self.table_d, causal=causal, **more)

    def keys(self, b):
        """K and V [sk, kv_heads, 128] of sequence b in 64 bits."""
        pages = torch.from_numpy(self.pages[b]).to(self.dev)
        sk = self.lens[b][1]
        return tuple(values(self.caches[j][pages], self.caches[j + 1][pages]).transpose(1, 2)
                     .reshape(-1, self.kv_heads, D)[:sk] for j in (0, 2))

    def check(self, o, lse, causal, q=None, weight_err=2e-4, nan_rows=None):
        """Every sequence against its own 64-bit attention.  nan_rows: bool [total, heads], rows whose query or a key
        that they see is no number: all of O and the LSE is NaN there, and all else is as ever."""
        q = self.q if q is None else q
        g = self.heads // self.kv_heads
        for b, (sq, sk) in enumerate(self.lens):
            if sq == 0:
                continue
            rows = slice(int(self.offsets[b]), int(self.offsets[b + 1]))
            k, v = self.keys(b)
            seen = (sk - sq + torch.arange(sq, device=self.dev) if causal == 2
                    else torch.full((sq,), sk - 1, device=self.dev))
            hidden = (torch.arange(sk, device=self.dev)[None] > seen[:, None]).repeat_interleave(g, 0)
            by_head = lambda x: x.double().reshape(sq, self.kv_heads, g, -1).transpose(0, 1).reshape(
                self.kv_heads, sq * g, -1)
            k, v = k.transpose(0, 1).nan_to_num(0.0).contiguous(), v.transpose(0, 1).nan_to_num(0.0).contiguous()
            got, x = by_head(o[rows]), by_head(q[rows]).nan_to_num(0.0)
            nan = (torch.zeros(got.shape[:2], dtype=torch.bool, device=self.dev) if nan_rows is None
                   else by_head(nan_rows[rows][..., None])[..., 0] > 0)
            assert got[nan].isnan().all(), b
            assert torch.isfinite(got[~nan]).all(), b
            s = torch.bmm(x, k.transpose(1, 2).contiguous()).mul_(SCALE).masked_fill_(hidden, -np.inf)
            want_lse = (torch.logsumexp(s, 2) if sk else
                        torch.full((self.kv_heads, sq * g), -np.inf, dtype=torch.float64, device=self.dev))
            w = torch.exp(s - torch.where(torch.isneginf(want_lse), 0.0, want_lse)[..., None])
            ref = torch.bmm(w, v)
            # sum_j w_j |v_j - o| <= sqrt(sum_j w_j (v_j - o)^2), the weights' sum being 1 (0 in empty rows).
            spread = (torch.bmm(w, v.square()) - ref.square()).clamp(min=0).sqrt()
            tol = (1.01 * HALF_STEP + weight_err) * spread + 1.01 * HALF_STEP * ref.abs() + 1e-5
            worst = ((got - ref).abs() / tol)[~nan]
            assert worst.numel() == 0 or worst.max().item() <= 1, (b, sq, sk, worst.max().item())
            if lse is not None:
                l = lse[:, rows].double().reshape(self.kv_heads, g, sq).transpose(1, 2).reshape(self.kv_heads, sq * g)
                assert l[nan].isnan().all(), b
                assert torch.equal(torch.isneginf(l[~nan]), torch.isneginf(want_lse[~nan])), b
                fin = torch.isfinite(want_lse) & ~nan
                assert ((l - want_lse)[fin].abs() <= LSE_TOL).all(), (b, (l - want_lse)[fin].abs().max())


def assert_guard_rows_untouched(batch):
    assert batch.o_all[batch.q.shape[0]:].isnan().all()
