"""Inputs and 64-bit references of the serving tests.

Tolerances, from the number of roundings on the way:
* append: one BF16 rounding of an FP32 value, half a step = 2^-8 of it, and
  three FP32 roundings of the two products, 3 * 2^-24 (|x| + |y|);
* attention: every weight is rounded to BF16 (2^-8 of it) before the product
  with V, numerator and denominator alike, so o moves by at most
  2^-8 / (1 - 2^-8) * sum_j w_j |v_j - o|; the output's own rounding is 2^-8 |o|.
  FP32 scores of 128 products of N(0, 1) values carry at most 128 * 2^-24 *
  sum |q k| scale, about 6e-5 of a weight for the inputs here (2e-4 for both
  the scores and exp2's argument, with a margin); larger scores carry more in proportion.
* LSE: the same 2e-4, absolute.
"""
import numpy as np
import torch

D = 128
SCALE = 1.0 / D ** 0.5
HALF_STEP = 2.0 ** -8                 # BF16
LSE_TOL = 2e-4


def offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


class Batch:
    """Caches whose pages lie anywhere in the pool.  prefixes: [(shared keys, [(queries, all keys), ...]), ...];
    `alone`: sequences of no prefix, behind them.  Unused pages and slots hold NaN, and table entries that must not be
    read numbers out of range."""

    def __init__(self, heads, kv_heads, page, prefixes, alone=(), seed=1, dev="cuda:0", spare=5):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.page, self.dev = heads, kv_heads, page, dev
        self.lens = [s for _, m in prefixes for s in m] + list(alone)
        self.members = [len(m) for _, m in prefixes]
        self.shared = [p // page * page for p, m in prefixes for _ in m] + [0] * len(alone)
        owner = [i for i, (_, m) in enumerate(prefixes) for _ in m] + [None] * len(alone)
        sq, sk = zip(*self.lens)
        cu = offsets(sq)
        self.max_q, self.max_k, self.total = max(max(sq), 1), max(max(sk), max((p for p, _ in prefixes), default=1), 1), int(cu[-1])
        shared_pages = [p // page for p, _ in prefixes]
        own_pages = [max(0, -(-k // page) - s // page) for k, s in zip(sk, self.shared)]
        pool = sum(shared_pages) + sum(own_pages) + spare
        order = rng.permutation(pool)
        bad = [-3, pool, 1 << 30]
        self.table = rng.choice(bad, size=(len(self.lens), -(-self.max_k // page))).astype(np.int32)
        self.prefix_table = rng.choice(bad, size=(len(prefixes), max(shared_pages + [1]))).astype(np.int32)
        at, first = 0, []
        k = torch.full((pool, page, kv_heads, D), float("nan"))
        v = torch.full_like(k, float("nan"))
        rand = lambda *s: torch.randn(*s, generator=gen)
        for p, n in enumerate(shared_pages):
            first.append(order[at:at + n])
            self.prefix_table[p, :n] = first[p]
            idx = torch.from_numpy(first[p].astype(np.int64))
            k[idx], v[idx] = rand(n, page, kv_heads, D), rand(n, page, kv_heads, D)
            at += n
        self.pages = []                                   # every sequence's pages, the shared ones first
        for b, n in enumerate(own_pages):
            mine = order[at:at + n]
            at += n
            s = self.shared[b] // page
            self.table[b, s:s + n] = mine
            for i, pg in enumerate(mine):
                rows = min(page, sk[b] - (s + i) * page)
                k[pg, :rows], v[pg, :rows] = rand(rows, kv_heads, D), rand(rows, kv_heads, D)
            self.pages.append(np.concatenate([first[owner[b]] if owner[b] is not None else [], mine]).astype(np.int64))
        i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)
        self.q = rand(max(self.total, 1), heads, D).to(torch.bfloat16).to(dev)
        self.k, self.v = k.to(torch.bfloat16).to(dev), v.to(torch.bfloat16).to(dev)
        self.cu, self.seqlens, self.table_d = i32(cu), i32(sk), i32(self.table)
        self.prefix_table_d, self.prefix_lens = i32(self.prefix_table), i32([p for p, _ in prefixes])
        self.cu_prefix = i32(offsets(self.members))
        self.offsets = cu

    def outputs(self, lse, guard=3):
        """O and LSE filled with NaN, O with guard rows behind the tokens."""
        n = self.q.shape[0]
        self.o_all = torch.full((n + guard, self.heads, D), float("nan"), dtype=torch.bfloat16, device=self.dev)
        self.lse = torch.full((self.heads, n), float("nan"), device=self.dev) if lse else None
        return self.o_all[:n], self.lse

    def attend(self, runner, o, lse, causal, q=None, **more):
        return runner.call_prefix_paged(self.q if q is None else q, self.k, self.v, o, lse, self.cu, self.seqlens,
                                        self.table_d, self.prefix_table_d, self.prefix_lens, self.cu_prefix,
                                        self.max_q, self.max_k, causal=causal, **more)

    def check(self, o, lse, causal, q=None, weight_err=2e-4):
        """Every sequence against its own 64-bit attention."""
        q = self.q if q is None else q
        g = self.heads // self.kv_heads
        for b, (sq, sk) in enumerate(self.lens):
            rows = slice(int(self.offsets[b]), int(self.offsets[b + 1]))
            if sq == 0:
                continue
            pages = torch.from_numpy(self.pages[b]).to(self.dev)
            k, v = (c[pages].reshape(-1, self.kv_heads, D)[:sk].double() for c in (self.k, self.v))
            seen = (sk - sq + torch.arange(sq, device=self.dev) if causal == 2
                    else torch.full((sq,), sk - 1, device=self.dev))
            hidden = (torch.arange(sk, device=self.dev)[None] > seen[:, None]).repeat_interleave(g, 0)
            by_head = lambda x: x.double().reshape(sq, self.kv_heads, g, D).transpose(0, 1).reshape(
                self.kv_heads, sq * g, D)
            k, v = k.transpose(0, 1).contiguous(), v.transpose(0, 1).contiguous()
            got, x = by_head(o[rows]), by_head(q[rows])
            assert torch.isfinite(got).all(), b
            s = torch.bmm(x, k.transpose(1, 2).contiguous()).mul_(SCALE).masked_fill_(hidden, -np.inf)
            want_lse = (torch.logsumexp(s, 2) if sk else
                        torch.full((self.kv_heads, sq * g), -np.inf, dtype=torch.float64, device=self.dev))
            w = torch.exp(s - torch.where(torch.isneginf(want_lse), 0.0, want_lse)[..., None])
            ref = torch.bmm(w, v)
            # sum_j w_j |v_j - o| <= sqrt(sum_j w_j (v_j - o)^2), the weights' sum being 1 (0 in empty rows).
            spread = (torch.bmm(w, v.square()) - ref.square()).clamp(min=0).sqrt()
            tol = (1.01 * HALF_STEP + weight_err) * spread + 1.01 * HALF_STEP * ref.abs() + 1e-5
            worst = ((got - ref).abs() / tol).max().item()
            assert worst <= 1, (b, sq, sk, worst)
            if lse is not None:
                l = lse[:, rows].double().reshape(self.kv_heads, g, sq).transpose(1, 2).reshape(self.kv_heads, sq * g)
                assert torch.equal(torch.isneginf(l), torch.isneginf(want_lse)), b
                fin = torch.isfinite(want_lse)
                assert ((l - want_lse)[fin].abs() <= LSE_TOL).all(), (b, (l - want_lse)[fin].abs().max())


def angles(rows, rotary_dim, dev):
    rates = 10000.0 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    x = torch.arange(rows, dtype=torch.float64)[:, None] * rates
    return x.cos().float().to(dev), x.sin().float().to(dev)


def rotated(x, cos, sin, interleaved):
    """(x turned by the tokens' angles, |x| + |y| of each dim's pair) in 64 bits; cos, sin: [tokens, rotary_dim / 2]."""
    x = x.double()
    out, size = x.clone(), x.abs()
    r = 2 * cos.shape[1]
    if r == 0:
        return out, size * 0
    i = torch.arange(r // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    c, s = cos.double()[:, None], sin.double()[:, None]
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    both = x[..., a].abs() + x[..., b].abs()
    size = torch.zeros_like(x)
    size[..., a], size[..., b] = both, both
    return out, size


def assert_rotated(got, x, cos, sin, interleaved, what=""):
    """got against x turned, each rounded once; dims that are not turned are copied bit by bit."""
    ref, size = rotated(x, cos, sin, interleaved)
    r = 2 * cos.shape[1]
    assert torch.equal(got[..., r:].view(torch.int16), x[..., r:].view(torch.int16)), what
    err = (got.double() - ref).abs()
    tol = HALF_STEP * ref.abs() * (1 + 2.0 ** -8) + 3 * 2.0 ** -24 * size
    bad = err > tol
    assert not bad.any(), (what, int(bad.sum()), (err / tol.clamp(min=1e-30)).max().item())
