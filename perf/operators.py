"""The serving operators of this library's paged K/V caches that are timed, with
their plain forms: what a decode or prefill step does to the caches and reads
from them.

* ``append``  the new tokens' K and V go into the paged caches, K (and Q)
  rotated by position on the way (``Runner.call_append_paged``);
* ``prefix``  attention of a batch whose sequences share leading pages (one
  system prompt, several samples of a prompt, beams), those keys attended once
  for all that share them (``Runner.call_prefix_paged``);
* ``step``    the two as a decode step runs them.

Where ``own`` is false the operators are computed in elementary torch
operations in 32 bits; where it is true, by the library.  Everything is BF16
at head dimension 128, as in the rest of the library; there is no backward
pass on a serving path.  ``draw`` gives more cases of the listed ranges.
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128
SCALE = 1.0 / math.sqrt(D)
DEVICE = "cuda"
BOTTOM_RIGHT = 2          # Runner's mask code: query i of sq sees keys j <= sk - sq + i
THETA = 10000.0


def listed():
    return [
        # One decode step of four chats: four tokens, where only latency counts.
        dict(name="append_small", op="append", seqs=4, heads=32, kv_heads=8, min_q=1, max_q=1, min_sk=100, max_sk=2000,
             page_size=64, rotary_dim=128, interleaved=False, packed=False, positions=False, lens_seed=1),
        # One decode step of a full serving batch.
        dict(name="append_batch", op="append", seqs=128, heads=32, kv_heads=8, min_q=1, max_q=1, min_sk=64, max_sk=1000,
             page_size=64, rotary_dim=128, interleaved=False, packed=False, positions=False, lens_seed=2),
        # Chunked prefill from the output of one QKV projection: ragged chunks
        # behind what is cached, half of each head rotated in neighbouring
        # pairs, positions of the caller's own.
        dict(name="append_chunks", op="append", seqs=4, heads=32, kv_heads=8, min_q=333, max_q=1024, min_sk=1024,
             max_sk=8192, page_size=64, rotary_dim=64, interleaved=True, packed=True, positions=True, lens_seed=3),
        # Whole prompts of mixed lengths, the largest call: bound by memory.
        dict(name="append_prompts", op="append", seqs=16, heads=32, kv_heads=8, min_q=500, max_q=4096, min_sk=0,
             max_sk=0, page_size=64, rotary_dim=128, interleaved=False, packed=False, positions=False, lens_seed=4),
        # Four chats behind a short system prompt: launches and latency.
        dict(name="prefix_small", op="prefix", prefixes=1, seqs=4, idle=0, heads=32, kv_heads=8, min_prefix=1024,
             max_prefix=1024, min_own=1, max_own=100, min_q=1, max_q=1, page_size=64, mask=0, lse=False, lens_seed=5),
        # A full decode batch behind one long system prompt.
        dict(name="prefix_batch", op="prefix", prefixes=1, seqs=64, idle=0, heads=32, kv_heads=8, min_prefix=8192,
             max_prefix=8192, min_own=16, max_own=1000, min_q=1, max_q=1, page_size=64, mask=0, lse=False,
             lens_seed=6),
        # Many questions on one long document, each with a history of its own.
        dict(name="prefix_long", op="prefix", prefixes=1, seqs=128, idle=0, heads=32, kv_heads=8, min_prefix=32768,
             max_prefix=32768, min_own=64, max_own=4096, min_q=1, max_q=1, page_size=64, mask=0, lse=False,
             lens_seed=7),
        # Four samples of each of sixteen prompts of mixed lengths, in a batch
        # padded to a fixed size by idle slots without keys; the LSE kept.
        dict(name="prefix_samples", op="prefix", prefixes=16, seqs=64, idle=3, heads=32, kv_heads=8, min_prefix=300,
             max_prefix=8192, min_own=16, max_own=500, min_q=1, max_q=1, page_size=64, mask=0, lse=True, lens_seed=8),
        # Speculative decoding: four draft tokens of each sequence at once.
        dict(name="prefix_speculative", op="prefix", prefixes=1, seqs=32, idle=0, heads=32, kv_heads=8, min_prefix=4096,
             max_prefix=4096, min_own=64, max_own=2000, min_q=4, max_q=4, page_size=64, mask=BOTTOM_RIGHT, lse=False,
             lens_seed=9),
        # One K/V head for all query heads, small pages.
        dict(name="prefix_mqa", op="prefix", prefixes=1, seqs=24, idle=0, heads=8, kv_heads=1, min_prefix=16384,
             max_prefix=16384, min_own=1, max_own=300, min_q=1, max_q=1, page_size=32, mask=0, lse=False,
             lens_seed=10),
        # Prefill chunks of many users behind one system prompt, the largest
        # call: bound by the matrix products.
        dict(name="prefix_prefill", op="prefix", prefixes=1, seqs=16, idle=0, heads=32, kv_heads=8, min_prefix=4096,
             max_prefix=4096, min_own=64, max_own=1000, min_q=64, max_q=256, page_size=64, mask=BOTTOM_RIGHT, lse=True,
             lens_seed=11),
        # A decode step as a serving engine runs it: append, then attend.
        dict(name="decode_step", op="step", prefixes=1, seqs=48, idle=0, heads=32, kv_heads=8, min_prefix=2048,
             max_prefix=2048, min_own=16, max_own=500, min_q=1, max_q=1, page_size=64, mask=0, lse=False,
             rotary_dim=128, interleaved=False, packed=False, positions=False, lens_seed=12),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the listed ranges (rng: random.Random)."""
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= 2.0e11 and w["bytes"] <= 6.0e8:
            return case


def _draw(rng):
    heads = rng.choice([8, 16, 32])
    kv_heads = heads // rng.choice([1, 4, 4, 8])
    page = rng.choice([32, 64, 64, 128])
    rotary = dict(rotary_dim=rng.choice([32, 64, 128, 128]), interleaved=rng.random() < 0.3,
                  packed=rng.random() < 0.5, positions=rng.random() < 0.3)
    seed = rng.randrange(1 << 30)
    if rng.random() < 0.4:
        if rng.random() < 0.5:
            q, sk, seqs = rng.choice([1, 1, 1, 4]), _log_int(rng, 100, 2000), _log_int(rng, 1, 128)
            return dict(op="append", seqs=seqs, heads=heads, kv_heads=kv_heads, min_q=q, max_q=q,
                        min_sk=max(q, sk // 8), max_sk=sk, page_size=page, lens_seed=seed, **rotary)
        q, sk = _log_int(rng, 64, 4096), rng.choice([0, 0, _log_int(rng, 1024, 8192)])
        return dict(op="append", seqs=_log_int(rng, 1, 16), heads=heads, kv_heads=kv_heads, min_q=max(1, q // 4),
                    max_q=q, min_sk=sk // 4, max_sk=sk, page_size=page, lens_seed=seed, **rotary)
    prefixes = rng.choice([1, 1, _log_int(rng, 2, 16)])
    seqs = max(prefixes, _log_int(rng, 2, 128))
    high = _log_int(rng, 512, 32768)
    own_keys = _log_int(rng, 16, 4096)
    q = rng.choice([1, 1, 1, 1, rng.randint(2, 8), _log_int(rng, 33, 256)])
    case = dict(op="prefix", prefixes=prefixes, seqs=seqs, idle=rng.choice([0, 0, 2]), heads=heads, kv_heads=kv_heads,
                min_prefix=max(page, high // rng.choice([1, 8])), max_prefix=high, min_own=max(1, own_keys // 16),
                max_own=own_keys, min_q=q if q <= 8 else q // 4, max_q=q, page_size=page,
                mask=0 if q == 1 else BOTTOM_RIGHT, lse=rng.random() < 0.4, lens_seed=seed)
    if q == 1 and rng.random() < 0.25:
        case.update(op="step", lse=False, idle=0, **rotary)
    return case


# ---- shapes ----------------------------------------------------------------
def _spread(rng, n, low, high):
    """n lengths spread over [low, high] (over their logarithm), the longest among them."""
    lens = [_log_int(rng, low, high) for _ in range(n)]
    lens[rng.randrange(n)] = high
    return lens


def _shape(case):
    """Per sequence the new tokens, the keys and the shared leading keys; per
    prefix its keys and the number of sequences that share it."""
    rng = random.Random(case["lens_seed"])
    n = case["seqs"]
    queries = _spread(rng, n, case["min_q"], case["max_q"])
    if case["op"] == "append":
        keys = [max(q, sk) for q, sk in zip(queries, _spread(rng, n, max(1, case["min_sk"]), max(1, case["max_sk"])))]
        return queries, keys, [0] * n, [], []
    page, count = case["page_size"], case["prefixes"]
    lens = [max(1, p // page) * page for p in _spread(rng, count, case["min_prefix"], case["max_prefix"])]
    members = [n // count + (i < n % count) for i in range(count)]
    own_keys = [max(q, sk) for q, sk in zip(queries, _spread(rng, n, case["min_own"], case["max_own"]))]
    shared = [lens[p] for p in range(count) for _ in range(members[p])]
    keys = [p + sk for p, sk in zip(shared, own_keys)]
    # Idle slots: one query row, no keys, no prefix.
    idle = case["idle"]
    return queries + [1] * idle, keys + [0] * idle, shared + [0] * idle, lens, members


def _visible(sq, sk, mask):
    """(query, key) pairs that attend to each other."""
    if sk == 0:
        return 0
    return sq * sk if mask != BOTTOM_RIGHT else sum(sk - sq + i + 1 for i in range(sq))


def work(case):
    queries, keys, shared, lens, _ = _shape(case)
    h, kvh, row = case["heads"], case["kv_heads"], D * 2
    tokens, size, flops = sum(queries), 0, 0
    if case["op"] != "prefix":
        # Q, K and V read and written once, a row of the angles' cosines and sines for each token.
        rot = case["rotary_dim"]
        size += tokens * (2 * (h + 2 * kvh) * row + rot * 4)
        flops += tokens * (h + kvh) * rot * 3
    if case["op"] != "append":
        # Each shared key once, each key of a sequence's own once.
        own_keys = sum(sk - p for sk, p in zip(keys, shared))
        size += tokens * h * (2 * row + (4 if case["lse"] else 0)) + (sum(lens) + own_keys) * kvh * 2 * row
        flops += 4 * h * D * sum(_visible(sq, sk, case["mask"]) for sq, sk in zip(queries, keys))
    return {"bytes": size, "flops": flops}


# ---- inputs ----------------------------------------------------------------
def _randn(shape, gen):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(torch.bfloat16)


def _offsets(lens):
    total, out = 0, [0]
    for n in lens:
        total += n
        out.append(total)
    return out


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    """New tokens, caches that hold what came before them, and where it lies:
    every sequence's pages are anywhere in the pool, shared ones in the tables
    of all sequences that share them."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    queries, keys, shared, lens, members = _shape(case)
    h, kvh, page = case["heads"], case["kv_heads"], case["page_size"]
    cu_q = _offsets(queries)
    tokens, n = cu_q[-1], len(queries)
    prefix_pages = [p // page for p in lens]
    own_pages = [-(-sk // page) - p // page for sk, p in zip(keys, shared)]
    pool = sum(prefix_pages) + sum(own_pages)
    order = torch.randperm(pool, generator=gen, device=DEVICE, dtype=torch.int32).cpu()
    table = torch.zeros((n, max(1, max(-(-sk // page) for sk in keys))), dtype=torch.int32)
    prefix_table = torch.zeros((max(1, len(lens)), max(prefix_pages, default=1)), dtype=torch.int32)
    for p, at in enumerate(_offsets(prefix_pages)[:-1]):
        prefix_table[p, :prefix_pages[p]] = order[at:at + prefix_pages[p]]
    owner = [p for p, m in enumerate(members) for _ in range(m)] + [0] * case.get("idle", 0)
    for b, at in enumerate(_offsets(own_pages)[:-1]):
        at += sum(prefix_pages)
        first = shared[b] // page
        if first:
            table[b, :first] = prefix_table[owner[b], :first]
        table[b, first:first + own_pages[b]] = order[at:at + own_pages[b]]
    s = dict(case=case, cu_q=_int32(cu_q), seqlens=_int32(keys), table=table.to(DEVICE),
             prefix_table=prefix_table.to(DEVICE), prefix_lens=_int32(lens), cu_prefix=_int32(_offsets(members)),
             max_q=max(queries), max_k=max(keys), max_own=max(sk - p for sk, p in zip(keys, shared)),
             max_shared=max(lens, default=0), total_k=sum(keys),
             max_sharing=max((sum(queries[i:j]) for i, j in zip(_offsets(members), _offsets(members)[1:])), default=0),
             k_cache=_randn((pool, page, kvh, D), gen), v_cache=_randn((pool, page, kvh, D), gen))
    if case["op"] != "prefix":
        if case["packed"]:
            qkv = _randn((tokens, h + 2 * kvh, D), gen)
            s.update(q=qkv[:, :h], k=qkv[:, h:h + kvh], v=qkv[:, h + kvh:])
        else:
            s.update(q=_randn((tokens, h, D), gen), k=_randn((tokens, kvh, D), gen), v=_randn((tokens, kvh, D), gen))
        rot = case["rotary_dim"]
        rates = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEVICE) / rot)
        angles = torch.arange(max(keys) + 64, dtype=torch.float64, device=DEVICE)[:, None] * rates
        s.update(cos=angles.cos().float(), sin=angles.sin().float(), positions=None)
        if case["positions"]:
            s["positions"] = torch.randint(0, max(keys) + 64, (tokens,), generator=gen, device=DEVICE,
                                           dtype=torch.int32)
        s["q_out"] = torch.empty((tokens, h, D), dtype=torch.bfloat16, device=DEVICE)
    else:
        s["q"] = _randn((tokens, h, D), gen)
    if case["op"] != "append":
        s["o"] = torch.empty((tokens, h, D), dtype=torch.bfloat16, device=DEVICE)
        s["lse"] = torch.empty((h, tokens), dtype=torch.float32, device=DEVICE) if case["lse"] else None
    return s


# ---- plain forms -------------------------------------------------------------
def _sequence_of_tokens(s):
    """Sequence of each token, and its place among the sequence's keys."""
    t = torch.arange(s["q"].shape[0], device=DEVICE)
    b = torch.searchsorted(s["cu_q"][1:].contiguous(), t, right=True)
    return b, s["seqlens"].long()[b] - s["cu_q"].long()[b + 1] + t


def _rotate(x, cos, sin, interleaved):
    """The first 2 * cos.shape[1] dims of x [tokens, heads, D] turned by the tokens' angles, rounded once."""
    x, half = x.float(), cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1).to(torch.bfloat16)


def _plain_append(s):
    case, page = s["case"], s["case"]["page_size"]
    b, slot = _sequence_of_tokens(s)
    where = s["positions"].long() if s["positions"] is not None else slot
    cos, sin = s["cos"][where], s["sin"][where]
    rows = s["table"][b, slot // page].long() * page + slot % page
    kvh = case["kv_heads"]
    s["k_cache"].view(-1, kvh, D)[rows] = _rotate(s["k"], cos, sin, case["interleaved"])
    s["v_cache"].view(-1, kvh, D)[rows] = s["v"]
    return _rotate(s["q"], cos, sin, case["interleaved"])


def _attend_part(q, k, v, hidden):
    """q [n, kvh, r, D] (scaled), k and v [n, kvh, keys, D], hidden [n, r, keys]:
    each row's maximum, sum of exponentials and weighted sum of V."""
    scores = (q @ k.transpose(-1, -2).contiguous()).masked_fill_(hidden[:, None], -math.inf)
    m = scores.amax(-1)
    weights = torch.exp(scores - torch.where(m == -math.inf, 0.0, m)[..., None])
    return m, weights.sum(-1), weights @ v


def _plain_prefix(s, q):
    case, page = s["case"], s["case"]["page_size"]
    h, kvh = case["heads"], case["kv_heads"]
    g, tokens = h // kvh, q.shape[0]
    q = (q.float() * SCALE).view(tokens, kvh, g, D)
    b, place = _sequence_of_tokens(s)
    cu_q, seqlens = s["cu_q"].long(), s["seqlens"].long()
    # The last key that each token sees, and the shared keys of its sequence.
    last = place if case["mask"] == BOTTOM_RIGHT else seqlens[b] - 1
    prefix_of = torch.searchsorted(s["cu_prefix"][1:].contiguous(), torch.arange(seqlens.shape[0], device=DEVICE),
                                   right=True)
    lens = torch.cat((s["prefix_lens"].long(), torch.zeros(1, dtype=torch.long, device=DEVICE)))
    shared = lens[prefix_of]

    def part(first, most, pages, start, end):
        """Rows [first, first + most) of each group against the keys [start, end) of its pages."""
        at = (first[:, None] + torch.arange(most, device=DEVICE)).clamp(max=tokens - 1)
        n, span = at.shape[0], s["max_shared"] if start is None else s["max_own"]
        key = torch.arange(span, device=DEVICE).expand(n, span) + (0 if start is None else start[:, None])
        slot = (key // page).clamp(max=pages.shape[1] - 1)
        rows = torch.gather(pages.long(), 1, slot) * page + key % page
        k, v = (s[c].view(-1, kvh, D)[rows].float().transpose(1, 2).contiguous() for c in ("k_cache", "v_cache"))
        hidden = (key[:, None] > last[at][..., None]) | (key[:, None] >= end[:, None, None])
        hidden = hidden[:, :, None].expand(n, most, g, span).reshape(n, most * g, span)
        rows = q[at].transpose(1, 2).reshape(n, kvh, most * g, D)
        m, l, acc = _attend_part(rows, k, v, hidden)
        return (x.view(n, kvh, most, g, -1).transpose(1, 2) for x in (m, l, acc))

    first = cu_q[s["cu_prefix"].long()[:-1]]
    mp, lp, ap = part(first, s["max_sharing"], s["prefix_table"], None, lens[:-1])
    group = prefix_of[b].clamp(max=first.shape[0] - 1)
    row = (torch.arange(tokens, device=DEVICE) - first[group]).clamp(max=s["max_sharing"] - 1)
    none = (prefix_of[b] >= first.shape[0])[:, None, None, None]
    mp = torch.where(none, -math.inf, mp[group, row])
    lp, ap = torch.where(none, 0.0, lp[group, row]), torch.where(none, 0.0, ap[group, row])
    mo, lo, ao = part(cu_q[:-1], s["max_q"], s["table"], shared, seqlens)
    row = torch.arange(tokens, device=DEVICE) - cu_q[b]
    mo, lo, ao = mo[b, row], lo[b, row], ao[b, row]
    m = torch.maximum(mp, mo)
    base = torch.where(m == -math.inf, 0.0, m)
    wp, wo = torch.exp(mp - base), torch.exp(mo - base)
    total = lp * wp + lo * wo
    o = (ap * wp + ao * wo) / torch.where(total == 0, 1.0, total)
    o = o.reshape(tokens, h, D).to(torch.bfloat16)
    return o, (m + torch.log(total)).view(tokens, h).T.contiguous() if case["lse"] else None


# ---- one pass ------------------------------------------------------------------
_kept = {}


def _runner():
    if "runner" not in _kept:
        import __graft_entry__
        _kept["runner"] = __graft_entry__.import_package().Runner()
    return _kept["runner"]


def _own_append(s):
    _runner().call_append_paged(s["q"], s["k"], s["v"], s["q_out"], s["k_cache"], s["v_cache"], s["cu_q"], s["seqlens"],
                                s["table"], cos=s["cos"], sin=s["sin"], interleaved=s["case"]["interleaved"],
                                positions=s["positions"])
    return s["q_out"]


def _own_prefix(s, q):
    # A serving loop keeps its workspace between steps: call_prefix_paged returns the one that it used.
    s["workspace"] = _runner().call_prefix_paged(q, s["k_cache"], s["v_cache"], s["o"], s["lse"], s["cu_q"],
                                                 s["seqlens"], s["table"], s["prefix_table"], s["prefix_lens"],
                                                 s["cu_prefix"], s["max_q"], s["max_k"],
                                                 workspace=s.get("workspace"), total_k=s["total_k"],
                                                 causal=s["case"]["mask"])
    return s["o"], s["lse"]


def run(state):
    s, op = state, state["case"]["op"]
    append, prefix = (_own_append, _own_prefix) if own else (_plain_append, _plain_prefix)
    if op == "append":
        return append(s), s["k_cache"], s["v_cache"]
    if op == "prefix":
        o, lse = prefix(s, s["q"])
        return (o, lse) if lse is not None else o
    o, _ = prefix(s, append(s))
    return o, s["k_cache"], s["v_cache"]


# ---- the same in 64 bits -------------------------------------------------------
def _exact_append(s, x):
    """x [tokens, heads, D] rotated in 64 bits, as complex numbers times the unit of the token's angle."""
    case, rot = s["case"], s["case"]["rotary_dim"]
    lens = (s["cu_q"][1:] - s["cu_q"][:-1]).tolist()
    slots = torch.cat([torch.arange(sk - n, sk) for n, sk in zip(lens, s["seqlens"].tolist())]).to(DEVICE)
    where = slots if s["positions"] is None else s["positions"].long()
    unit = torch.complex(s["cos"][where].double(), s["sin"][where].double())[:, None]
    out = x.double().clone()
    turned = out[..., :rot]
    if case["interleaved"]:
        turned.copy_(torch.view_as_real(torch.view_as_complex(turned.unflatten(-1, (-1, 2)).contiguous()) * unit)
                     .flatten(-2))
    else:
        z = torch.complex(turned[..., :rot // 2].contiguous(), turned[..., rot // 2:].contiguous()) * unit
        turned.copy_(torch.cat((z.real, z.imag), dim=-1))
    return out


def _exact_caches(s):
    """Both caches after the append, in 64 bits."""
    page, kvh = s["case"]["page_size"], s["case"]["kv_heads"]
    k, v = s["k_cache"].double(), s["v_cache"].double()
    turned = _exact_append(s, s["k"])
    table, cu = s["table"].cpu(), s["cu_q"].tolist()
    for b, sk in enumerate(s["seqlens"].tolist()):
        n = cu[b + 1] - cu[b]
        slots = torch.arange(sk - n, sk)
        rows = (table[b, slots // page].long() * page + slots % page).to(DEVICE)
        k.view(-1, kvh, D)[rows] = turned[cu[b]:cu[b + 1]]
        v.view(-1, kvh, D)[rows] = s["v"][cu[b]:cu[b + 1]].double()
    return k, v


def _exact_prefix(s, q, k_cache, v_cache):
    """Every sequence on its own, over all of its keys."""
    case, page = s["case"], s["case"]["page_size"]
    h, kvh = case["heads"], case["kv_heads"]
    g, cu = h // kvh, s["cu_q"].tolist()
    o = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
    lse = torch.full((h, q.shape[0]), -math.inf, dtype=torch.float64, device=DEVICE)
    for b, sk in enumerate(s["seqlens"].tolist()):
        if sk == 0:
            continue
        pages = s["table"][b, :-(-sk // page)].long()
        k, v = (c[pages].reshape(-1, kvh, D)[:sk].double() for c in (k_cache, v_cache))
        rows = slice(cu[b], cu[b + 1])
        n = cu[b + 1] - cu[b]
        for j in range(kvh):
            x = q[rows, j * g:(j + 1) * g].double().reshape(n * g, D)
            scores = (x @ k[:, j].T) * SCALE
            if case["mask"] == BOTTOM_RIGHT:
                query = torch.arange(n * g, device=DEVICE) // g
                scores.masked_fill_(torch.arange(sk, device=DEVICE)[None] > (sk - n + query)[:, None], -math.inf)
            o[rows, j * g:(j + 1) * g] = (torch.softmax(scores, dim=1) @ v[:, j]).view(n, g, D)
            lse[j * g:(j + 1) * g, rows] = torch.logsumexp(scores, dim=1).view(n, g).T
    return o, lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return (_exact_append(s, s["q"]), *_exact_caches(s))
    if case["op"] == "prefix":
        o, lse = _exact_prefix(s, s["q"], s["k_cache"], s["v_cache"])
        return (o, lse) if case["lse"] else o
    # The step's operators pass BF16 on to each other.
    k, v = _exact_caches(s)
    q = _exact_append(s, s["q"]).to(torch.bfloat16)
    o, _ = _exact_prefix(s, q, k.to(torch.bfloat16), v.to(torch.bfloat16))
    return o, k, v
