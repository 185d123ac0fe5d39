"""GPU checks of the serving operators at more rows than one pass of their grids takes (2^22 workgroups)."""
import pytest
import torch

from tests.serving import D, HALF_STEP, LSE_TOL, SCALE

pytestmark = pytest.mark.gpu
GRID = 1 << 22
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_append_of_more_tokens_than_one_pass(gpu_runner):
    """One K/V head, four tokens a workgroup: bit by bit, pages in reverse order."""
    page, first, tokens = 256, 5000, 4 * GRID + 1000
    print("append", tokens, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randint(-1 << 15, 1 << 15, (tokens, 1, D), generator=gen, device=DEV, dtype=torch.int16)
            for _ in range(2))
    lens = (first, tokens - first)
    pages = [-(-n // page) for n in lens]
    pool = sum(pages)
    table = torch.full((2, pages[1]), -1, dtype=torch.int32, device=DEV)
    order = torch.arange(pool - 1, -1, -1, dtype=torch.int32, device=DEV)
    table[0, :pages[0]], table[1] = order[:pages[0]], order[pages[0]:]
    kc, vc = (torch.zeros((pool, page, 1, D), dtype=torch.int16, device=DEV) for _ in range(2))
    bf16 = lambda x: x.view(torch.bfloat16)
    gpu_runner.call_append_paged(None, bf16(k), bf16(v), None, bf16(kc), bf16(vc), i32(0, first, tokens), i32(*lens), table)
    torch.cuda.synchronize()
    for new, cache in ((k, kc), (v, vc)):
        rows = cache.flip(0).view(-1, 1, D)
        start = pages[0] * page
        assert torch.equal(rows[:first], new[:first]) and torch.equal(rows[start:start + lens[1]], new[first:])
        assert not rows[first:start].any() and not rows[start + lens[1]:].any()
        del rows


def test_prefix_of_more_rows_than_the_merge_takes_in_one_pass(gpu_runner):
    """16 rows a workgroup of the merge: two sequences of queries over a prefix and a few keys of their own."""
    page, rows = 64, 16 * GRID + 5000
    print("prefix", rows, flush=True)
    gen = torch.Generator(device=DEV).manual_seed(2)
    q = torch.empty((rows, 1, D), dtype=torch.bfloat16, device=DEV)
    q.normal_(generator=gen)
    kc, vc = (torch.randn((4, page, 1, D), generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2))
    cut = 40_000_000
    o = torch.full_like(q, float("nan"))
    lse = torch.full((1, rows), float("nan"), device=DEV)
    ws = gpu_runner.call_prefix_paged(q, kc, vc, o, lse, i32(0, cut, rows), i32(100, 128), i32(-1, 3, -1, 0).view(2, 2),
                                      i32(2).view(1, 1), i32(64), i32(0, 2), cut, 128)
    torch.cuda.synchronize()
    del ws
    assert not torch.isnan(lse).any()
    border = 16 * GRID
    at = torch.cat([torch.arange(a, b, device=DEV) for a, b in (
        (0, 600), (cut - 600, cut + 600), (border - 600, border + 600), (rows - 600, rows))] +
        [torch.randint(0, rows, (20000,), generator=gen, device=DEV)])
    for own, sk, mine in ((3, 100, at[at < cut]), (0, 128, at[at >= cut])):
        k, v = (torch.cat([c[2, :, 0], c[own, :, 0]])[:sk].double() for c in (kc, vc))
        s = q[mine, 0].double() @ k.T.contiguous() * SCALE
        want = torch.logsumexp(s, 1)
        w = torch.exp(s - want[:, None])
        ref = w @ v
        spread = (w @ v.square() - ref.square()).clamp(min=0).sqrt()
        tol = (1.01 * HALF_STEP + 2e-4) * spread + 1.01 * HALF_STEP * ref.abs() + 1e-5
        assert ((o[mine, 0].double() - ref).abs() <= tol).all()
        assert ((lse[0, mine].double() - want).abs() <= LSE_TOL).all()
