"""The operators of 4-bit paged K/V caches that are timed, with their plain
forms: what a serving step stores in such caches, reads back and attends to.

A cache row (128 dims of one key and head) is held as MXFP4: 128 E2M1 numbers,
two to a byte, and for each block of 32 dims an E8M0 byte s that scales them by
2^(s - 127).  68 bytes instead of the 256 of BF16.

* ``append``  the new tokens' K and V, K (and Q) rotated by position, are
  quantised and stored (``Runner.call_append_paged_mx4``), and read back as the
  values that they now stand for (``Runner.call_gather_paged_mx4``), as an
  engine does that prefills over the values its later steps will see;
* ``read``    whole histories are read back to BF16 rows of a packed batch;
* ``attend``  attention over the caches (``Runner.call_paged_mx4``);
* ``step``    all three as an engine runs them that mirrors each step's new keys
  elsewhere.

Where ``own`` is false the operators are computed in elementary torch
operations in 32 bits; where it is true, by the library.  Q, O and the rows that
are stored and read back are BF16 at head dimension 128, as in the rest of the
library; there is no backward pass on a serving path.  ``draw`` gives more cases
of the listed ranges.
"""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128
BLOCK = 32                # dims that share a scale
SCALE = 1.0 / math.sqrt(D)
DEVICE = "cuda"
BOTTOM_RIGHT = 2          # Runner's mask code: query i of sq sees keys j <= sk - sq + i
THETA = 10000.0


def listed():
    return [
        # One decode step of four chats: four tokens, where only latency counts.
        dict(name="append_small", op="append", seqs=4, heads=32, kv_heads=8, min_q=1, max_q=1, min_sk=100, max_sk=2000,
             page_size=64, rotary_dim=128, interleaved=False, packed=False, positions=False, lens_seed=21),
        # Chunked prefill from the output of one QKV projection: ragged chunks
        # behind what is cached, half of each head rotated in neighbouring
        # pairs, positions of the caller's own.
        dict(name="append_chunks", op="append", seqs=4, heads=32, kv_heads=8, min_q=333, max_q=1024, min_sk=1024,
             max_sk=8192, page_size=64, rotary_dim=64, interleaved=True, packed=True, positions=True, lens_seed=22),
        # Whole prompts of mixed lengths: bound by memory.
        dict(name="append_prompts", op="append", seqs=16, heads=32, kv_heads=8, min_q=500, max_q=4096, min_sk=0,
             max_sk=0, page_size=64, rotary_dim=128, interleaved=False, packed=True, positions=False, lens_seed=23),
        # Histories of mixed lengths read back, for the packed forward or to be sent elsewhere.
        dict(name="read_histories", op="read", seqs=12, heads=32, kv_heads=8, min_q=1, max_q=1, min_sk=300,
             max_sk=16384, page_size=64, lens_seed=24),
        # A decode step of four chats: launches and latency.
        dict(name="attend_small", op="attend", seqs=4, heads=32, kv_heads=8, min_q=1, max_q=1, min_sk=100, max_sk=2000,
             page_size=64, mask=0, lse=False, lens_seed=25),
        # A full decode batch of mixed lengths.
        dict(name="attend_batch", op="attend", seqs=64, heads=32, kv_heads=8, min_q=1, max_q=1, min_sk=500, max_sk=8192,
             page_size=64, mask=0, lse=False, lens_seed=26),
        # Long contexts, what a 4-bit cache is for: bound by memory.
        dict(name="attend_long", op="attend", seqs=32, heads=32, kv_heads=8, min_q=1, max_q=1, min_sk=4096,
             max_sk=32768, page_size=64, mask=0, lse=False, lens_seed=27),
        # Speculative decoding: four draft tokens of each sequence at once, the LSE kept.
        dict(name="attend_speculative", op="attend", seqs=32, heads=32, kv_heads=8, min_q=4, max_q=4, min_sk=200,
             max_sk=4096, page_size=64, mask=BOTTOM_RIGHT, lse=True, lens_seed=28),
        # One K/V head for all query heads, small pages.
        dict(name="attend_mqa", op="attend", seqs=24, heads=8, kv_heads=1, min_q=1, max_q=1, min_sk=1000, max_sk=16384,
             page_size=32, mask=0, lse=False, lens_seed=29),
        # Chunked prefill behind what is cached.
        dict(name="attend_chunks", op="attend", seqs=8, heads=32, kv_heads=8, min_q=64, max_q=512, min_sk=1024,
             max_sk=8192, page_size=64, mask=BOTTOM_RIGHT, lse=True, lens_seed=30),
        # Whole prompts, bound by the matrix products: the largest call.
        dict(name="attend_prompts", op="attend", seqs=8, heads=32, kv_heads=8, min_q=500, max_q=2500, min_sk=0,
             max_sk=0, page_size=64, mask=BOTTOM_RIGHT, lse=False, lens_seed=31),
        # A decode step as a serving engine runs it: append, attend, and the new rows read back.
        dict(name="decode_step", op="step", seqs=48, heads=32, kv_heads=8, min_q=1, max_q=1, min_sk=100, max_sk=4096,
             page_size=64, mask=0, lse=False, rotary_dim=128, interleaved=False, packed=True, positions=False,
             lens_seed=32),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the listed ranges (rng: random.Random)."""
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= 2.0e11 and w["bytes"] <= 6.0e8 and _plain_values(case) <= 1.6e9:
            return case


def _draw(rng):
    heads = rng.choice([8, 16, 32])
    kv_heads = heads // rng.choice([1, 4, 4, 8])
    page = rng.choice([16, 32, 64, 64, 128])
    rotary = dict(rotary_dim=rng.choice([32, 64, 128, 128]), interleaved=rng.random() < 0.3,
                  packed=rng.random() < 0.5, positions=rng.random() < 0.3)
    case = dict(heads=heads, kv_heads=kv_heads, page_size=page, lens_seed=rng.randrange(1 << 30))
    op = rng.choice(["append", "append", "read", "attend", "attend", "attend", "attend", "attend", "step"])
    if op == "append" and rng.random() < 0.5:
        q, sk = _log_int(rng, 64, 4096), rng.choice([0, 0, _log_int(rng, 1024, 8192)])
        return dict(op=op, seqs=_log_int(rng, 1, 16), min_q=max(1, q // 4), max_q=q, min_sk=sk // 4, max_sk=sk, **case,
                    **rotary)
    if op == "read":
        sk = _log_int(rng, 100, 32768)
        return dict(op=op, seqs=_log_int(rng, 1, 64), min_q=1, max_q=1, min_sk=max(1, sk // 16), max_sk=sk, **case)
    if op != "attend":
        q, sk = rng.choice([1, 1, 1, 4]), _log_int(rng, 100, 4096)
        case.update(op=op, seqs=_log_int(rng, 1, 128), min_q=q, max_q=q, min_sk=max(q, sk // 8), max_sk=sk, **rotary)
        return case if op == "append" else dict(case, mask=0 if q == 1 else BOTTOM_RIGHT, lse=rng.random() < 0.3)
    q = rng.choice([1, 1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 512), 0])
    if q == 0:                                   # whole prompts
        q, sk = _log_int(rng, 100, 2500), 0
    else:
        sk = _log_int(rng, max(100, q), 32768)
    return dict(op=op, seqs=_log_int(rng, 1, 64 if q <= 8 else 8), min_q=q if q <= 8 else q // 4, max_q=q,
                min_sk=sk // rng.choice([1, 8, 16]), max_sk=sk, mask=0 if q == 1 else BOTTOM_RIGHT,
                lse=rng.random() < 0.4, **case)


def _plain_values(case):
    """Scores and gathered values that the plain form holds at once."""
    queries, keys = _shape(case)
    padded = max(keys) * len(keys) if case["op"] in ("attend", "step") else 0
    return padded * (case["kv_heads"] * D + case["heads"] * max(queries))


# ---- shapes ----------------------------------------------------------------
def _spread(rng, n, low, high):
    """n lengths spread over [low, high] (over their logarithm), the longest among them."""
    lens = [_log_int(rng, low, high) for _ in range(n)]
    lens[rng.randrange(n)] = high
    return lens


def _shape(case):
    """Per sequence the new tokens and the keys, the new ones included."""
    rng = random.Random(case["lens_seed"])
    n = case["seqs"]
    queries = _spread(rng, n, case["min_q"], case["max_q"])
    cached = _spread(rng, n, max(1, case["min_sk"]), max(1, case["max_sk"]))
    return queries, [max(q, sk) for q, sk in zip(queries, cached)]


def _visible(sq, sk, mask):
    """(query, key) pairs that attend to each other."""
    return sq * sk if mask != BOTTOM_RIGHT else sum(sk - sq + i + 1 for i in range(sq))


def work(case):
    queries, keys = _shape(case)
    h, kvh, op = case["heads"], case["kv_heads"], case["op"]
    row, row4 = D * 2, D // 2 + D // BLOCK
    tokens, size, flops = sum(queries), 0, 0
    if op in ("append", "step"):
        # Q, K and V read, Q written, K and V stored, then read back and written; a row of the angles' cosines and
        # sines for each token.
        rot = case["rotary_dim"]
        size += tokens * (2 * h * row + 2 * kvh * (2 * row + row4) + rot * 4)
        flops += tokens * ((h + kvh) * rot * 3 + 2 * kvh * D * 4)
    if op == "read":
        size += sum(keys) * 2 * kvh * (row4 + row)
        flops += sum(keys) * 2 * kvh * D
    if op in ("attend", "step"):
        size += tokens * h * (2 * row + (4 if case["lse"] else 0)) + sum(keys) * kvh * 2 * row4
        flops += 4 * h * D * sum(_visible(sq, sk, case["mask"]) for sq, sk in zip(queries, keys))
    return {"bytes": size, "flops": flops}


# ---- inputs ----------------------------------------------------------------
def _randn(shape, gen, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)


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
    every sequence's pages are anywhere in the pool.  Some channels of K are
    much larger than others, as they are in trained models."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    queries, keys = _shape(case)
    h, kvh, page, op = case["heads"], case["kv_heads"], case["page_size"], case["op"]
    cu_q = _offsets(queries)
    tokens, n = cu_q[-1], len(queries)
    pages = [-(-sk // page) for sk in keys]
    pool = sum(pages)
    order = torch.randperm(pool, generator=gen, device=DEVICE, dtype=torch.int32).cpu()
    table = torch.zeros((n, max(pages)), dtype=torch.int32)
    for b, at in enumerate(_offsets(pages)[:-1]):
        table[b, :pages[b]] = order[at:at + pages[b]]
    gains = torch.exp(0.5 * torch.randn((kvh, 1, D), generator=gen, device=DEVICE))
    s = dict(case=case, cu_q=_int32(cu_q), seqlens=_int32(keys), table=table.to(DEVICE), max_q=max(queries),
             max_k=max(keys), total_k=sum(keys), starts=_int32([sk - q for q, sk in zip(queries, keys)]))
    shape = (pool, kvh, page, D)
    s["k_cache"], s["k_scales"] = _quantised(_randn(shape, gen, torch.float32) * gains)
    s["v_cache"], s["v_scales"] = _quantised(_randn(shape, gen, torch.float32))
    if op in ("append", "step"):
        gains = gains.view(1, kvh, D).to(torch.bfloat16)
        if case["packed"]:
            qkv = _randn((tokens, h + 2 * kvh, D), gen)
            qkv[:, h:h + kvh] *= gains
            s.update(q=qkv[:, :h], k=qkv[:, h:h + kvh], v=qkv[:, h + kvh:])
        else:
            s.update(q=_randn((tokens, h, D), gen), k=_randn((tokens, kvh, D), gen) * gains,
                     v=_randn((tokens, kvh, D), gen))
        rot = case["rotary_dim"]
        rates = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEVICE) / rot)
        angles = torch.arange(max(keys) + 64, dtype=torch.float64, device=DEVICE)[:, None] * rates
        s.update(cos=angles.cos().float(), sin=angles.sin().float(), positions=None)
        if case["positions"]:
            s["positions"] = torch.randint(0, max(keys) + 64, (tokens,), generator=gen, device=DEVICE,
                                           dtype=torch.int32)
        s["q_out"] = torch.empty((tokens, h, D), dtype=torch.bfloat16, device=DEVICE)
    elif op == "attend":
        s["q"] = _randn((tokens, h, D), gen)
    if op != "attend":
        rows = sum(keys) if op == "read" else tokens
        s["k_rows"], s["v_rows"] = (torch.empty((rows, kvh, D), dtype=torch.bfloat16, device=DEVICE) for _ in range(2))
        s["cu_rows"] = _int32(_offsets(keys)) if op == "read" else s["cu_q"]
    if op in ("attend", "step"):
        s["o"] = torch.empty((tokens, h, D), dtype=torch.bfloat16, device=DEVICE)
        s["lse"] = torch.empty((h, tokens), dtype=torch.float32, device=DEVICE) if case["lse"] else None
    return s


# ---- plain forms -------------------------------------------------------------
def _quantised(x):
    """x [..., D] in 32 bits as (codes [..., D / 2], scales [..., D / 32]), bytes.  A block's scale is the smallest
    power of two with max |x| <= 7 * 2^e (2^-125 to 2^125): what lies between 6 and 7 is nearer to 6 than to the next
    scale's grid.  Each number goes to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times the scale, ties to the even
    code; even dims lie in the low halves of the bytes, the sign is a code's top bit."""
    x = x.unflatten(-1, (-1, BLOCK))
    most = x.abs().amax(-1).view(torch.int32)
    scales = (((most + 0x1fffff) >> 23) - 2).clamp(2, 252)
    y = x * ((254 - scales) << 23).view(torch.float32)[..., None]
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a * 0.5 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(x).to(torch.uint8) << 3)).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), scales.to(torch.uint8)


def _values(codes, scales):
    """The numbers that codes and scales stand for, in 32 bits (exact)."""
    code = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).int()
    a, sign = code & 7, 1.0 - 2.0 * (code >> 3)
    a = torch.where(a < 4, a * 0.5, torch.where(a < 6, a - 2.0, a * 2.0 - 8.0)) * sign
    return (a.unflatten(-1, (-1, BLOCK)) * (scales.int() << 23).view(torch.float32)[..., None]).flatten(-2)


def _sequence_of_tokens(s):
    """Sequence of each token, and its place among the sequence's keys."""
    t = torch.arange(s["q"].shape[0], device=DEVICE)
    b = torch.searchsorted(s["cu_q"][1:].contiguous(), t, right=True)
    return b, s["seqlens"].long()[b] - s["cu_q"].long()[b + 1] + t


def _rotate(x, cos, sin, interleaved):
    """The first 2 * cos.shape[1] dims of x [tokens, heads, D] turned by the tokens' angles, in 32 bits."""
    x, half = x.float(), cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _plain_append(s):
    case, page = s["case"], s["case"]["page_size"]
    b, slot = _sequence_of_tokens(s)
    where = s["positions"].long() if s["positions"] is not None else slot
    cos, sin = s["cos"][where], s["sin"][where]
    at, slot = s["table"][b, slot // page].long(), slot % page
    for name, x in (("k", _rotate(s["k"], cos, sin, case["interleaved"])), ("v", s["v"].float())):
        codes, scales = _quantised(x)
        s[name + "_cache"][at, :, slot] = codes
        s[name + "_scales"][at, :, slot] = scales
    return _rotate(s["q"], cos, sin, case["interleaved"]).to(torch.bfloat16)


def _plain_read(s):
    """Keys [starts[b], ...) of each sequence, as many as it has rows."""
    page, cu = s["case"]["page_size"], s["cu_rows"].long()
    t = torch.arange(s["k_rows"].shape[0], device=DEVICE)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    key = t - cu[b] + (0 if s["case"]["op"] == "read" else s["starts"].long()[b])
    at, slot = s["table"][b, key // page].long(), key % page
    return tuple(_values(s[name + "_cache"][at, :, slot], s[name + "_scales"][at, :, slot]).to(torch.bfloat16)
                 for name in "kv")


def _plain_attend(s, q):
    case, page = s["case"], s["case"]["page_size"]
    h, kvh, most = case["heads"], case["kv_heads"], s["max_q"]
    g, tokens, n, span = h // kvh, q.shape[0], s["seqlens"].shape[0], s["max_k"]
    cu_q, seqlens = s["cu_q"].long(), s["seqlens"].long()
    key = torch.arange(span, device=DEVICE)
    at = s["table"][:, key // page].long()
    k, v = (_values(s[name + "_cache"][at, :, key % page], s[name + "_scales"][at, :, key % page])
            .transpose(1, 2).contiguous() for name in "kv")
    row = (cu_q[:-1, None] + torch.arange(most, device=DEVICE)).clamp(max=tokens - 1)
    x = (q.float() * SCALE).view(tokens, kvh, g, D)[row].transpose(1, 2).reshape(n, kvh, most * g, D)
    last = (seqlens[:, None] - 1).expand(n, most)
    if case["mask"] == BOTTOM_RIGHT:
        last = seqlens[:, None] - (cu_q[1:] - cu_q[:-1])[:, None] + torch.arange(most, device=DEVICE)
    hidden = (key > last[..., None]) | (key >= seqlens[:, None, None])
    hidden = hidden[:, :, None].expand(n, most, g, span).reshape(n, 1, most * g, span)
    scores = (x @ k.transpose(-1, -2).contiguous()).masked_fill_(hidden, -math.inf)
    m = scores.amax(-1)
    scores.sub_(torch.where(m == -math.inf, 0.0, m)[..., None]).exp_()
    total = scores.sum(-1)
    o = (scores @ v) / torch.where(total == 0, 1.0, total)[..., None]
    b, _ = _sequence_of_tokens(s)
    row = torch.arange(tokens, device=DEVICE) - cu_q[b]
    by_token = lambda y: y.view(n, kvh, most, g, -1).transpose(1, 2)[b, row].reshape(tokens, h, -1)
    lse = by_token(m + torch.log(total))[..., 0].T.contiguous() if case["lse"] else None
    return by_token(o).to(torch.bfloat16), lse


# ---- one pass ------------------------------------------------------------------
_kept = {}


def _runner():
    if "runner" not in _kept:
        import __graft_entry__
        _kept["runner"] = __graft_entry__.import_package().Runner()
    return _kept["runner"]


def _own_append(s):
    _runner().call_append_paged_mx4(s["q"], s["k"], s["v"], s["q_out"], s["k_cache"], s["k_scales"], s["v_cache"],
                                    s["v_scales"], s["cu_q"], s["seqlens"], s["table"], cos=s["cos"], sin=s["sin"],
                                    interleaved=s["case"]["interleaved"], positions=s["positions"])
    return s["q_out"]


def _own_read(s):
    _runner().call_gather_paged_mx4(s["k_cache"], s["k_scales"], s["v_cache"], s["v_scales"], s["k_rows"], s["v_rows"],
                                    s["cu_rows"], s["table"],
                                    starts=None if s["case"]["op"] == "read" else s["starts"])
    return s["k_rows"], s["v_rows"]


def _own_attend(s, q):
    # A serving loop keeps its workspace between steps: call_paged_mx4 returns the one that it used.
    s["workspace"] = _runner().call_paged_mx4(q, s["k_cache"], s["k_scales"], s["v_cache"], s["v_scales"], s["o"],
                                              s["lse"], s["cu_q"], s["seqlens"], s["table"], s["max_q"], s["max_k"],
                                              workspace=s.get("workspace"), total_k=s["total_k"],
                                              causal=s["case"]["mask"])
    return s["o"], s["lse"]


def run(state):
    s, op = state, state["case"]["op"]
    append, read, attend = (_own_append, _own_read, _own_attend) if own else (_plain_append, _plain_read, _plain_attend)
    if op == "append":
        return (append(s), *read(s))
    if op == "read":
        return read(s)
    if op == "attend":
        o, lse = attend(s, s["q"])
        return (o, lse) if lse is not None else o
    o, lse = attend(s, append(s))
    return (o, lse, *read(s)) if lse is not None else (o, *read(s))


# ---- the same in 64 bits -------------------------------------------------------
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_values(codes, scales):
    """What bytes stand for, by a table of the 256 pairs."""
    signed = torch.tensor(GRID + tuple(-x for x in GRID), dtype=torch.float64, device=DEVICE)
    pairs = torch.stack((signed.repeat(16), signed.repeat_interleave(16)), dim=-1)
    power = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=DEVICE), scales.double() - 127)
    return pairs[codes.long()].flatten(-2) * power.repeat_interleave(BLOCK, dim=-1)


def _exact_rotated(s, x):
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


def _exact_stored(x):
    """x [..., D] in 64 bits as the cache holds it: the nearest multiple of its block's scale on the grid."""
    y = x.unflatten(-1, (-1, BLOCK))
    power = torch.exp2(torch.ceil(torch.log2(y.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -120) / 7)))
    a = (y / power).abs()
    grid = torch.tensor(GRID, dtype=torch.float64, device=DEVICE)
    below = (torch.searchsorted(grid, a.contiguous(), right=True) - 1).clamp(0, 6)
    low, high = grid[below], grid[below + 1]
    up = (a - low > high - a) | ((a - low == high - a) & (below % 2 == 1))
    return (torch.where(up, high, low) * power * torch.sign(y)).flatten(-2)


def _exact_attend(s, q, k_all, v_all):
    """Every sequence on its own; k_all, v_all: each one's keys [sk, kv_heads, D] in 64 bits."""
    case = s["case"]
    h, kvh = case["heads"], case["kv_heads"]
    g, cu = h // kvh, s["cu_q"].tolist()
    o = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
    lse = torch.full((h, q.shape[0]), -math.inf, dtype=torch.float64, device=DEVICE)
    for b, sk in enumerate(s["seqlens"].tolist()):
        k, v, n = k_all(b), v_all(b), cu[b + 1] - cu[b]
        rows = slice(cu[b], cu[b + 1])
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
    page, table, lens = case["page_size"], s["table"], s["seqlens"].tolist()

    def keys_of(name, new=None):
        def of(b):
            pages = table[b, :-(-lens[b] // page)].long()
            rows = _exact_values(s[name + "_cache"][pages], s[name + "_scales"][pages])
            rows = rows.transpose(1, 2).reshape(-1, case["kv_heads"], D)[:lens[b]]
            if new is not None:
                first, end = s["cu_q"][b:b + 2].tolist()
                rows[lens[b] - (end - first):] = new[first:end]
            return rows
        return of

    if case["op"] == "read":
        return tuple(torch.cat([keys_of(name)(b) for b in range(len(lens))]) for name in "kv")
    if case["op"] == "attend":
        o, lse = _exact_attend(s, s["q"], keys_of("k"), keys_of("v"))
        return (o, lse) if case["lse"] else o
    q, k, v = _exact_rotated(s, s["q"]), _exact_stored(_exact_rotated(s, s["k"])), _exact_stored(s["v"].double())
    if case["op"] == "append":
        return q, k, v
    # The step's operators pass BF16 on to each other.
    o, lse = _exact_attend(s, q.to(torch.bfloat16), keys_of("k", k), keys_of("v", v))
    return (o, lse, k, v) if case["lse"] else (o, k, v)
