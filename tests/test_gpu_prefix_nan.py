"""GPU checks of attention behind shared prefixes with queries that are not numbers: their rows are not numbers
either, and no other row changes."""
import pytest
import torch

from tests.serving import Batch

pytestmark = pytest.mark.gpu

# (heads, kv_heads, page, prefixes, sequences of no prefix, causal); the merge takes 1, 4 or 16 teams a row.
CASES = {
    "one_part": (8, 8, 32, [(0, [(1, 20)])], [(1, 9)], 0),
    "few_rows_a_prefix": (32, 8, 64, [(1024, [(1, 1100), (1, 1025), (1, 800)])], [], 0),
    "few_rows_a_sequence": (32, 8, 64, [(1024, [(2, 1100 + 9 * i) for i in range(12)])], [(1, 70)], 2),
    "many_rows_a_sequence": (8, 2, 64, [(512, [(40, 600), (9, 900)])], [(33, 100)], 2),
    "many_parts_a_row": (8, 1, 32, [(16384, [(1, 16385 + 37 * i) for i in range(24)])], [], 0),
    "many_rows": (32, 8, 64, [(1024, [(1, 1030 + i % 50) for i in range(150)])], [], 0),
}


@pytest.mark.parametrize("value", ["nan", "inf"])
@pytest.mark.parametrize("name", CASES)
def test_a_query_that_is_no_number(gpu_runner, name, value):
    heads, kvh, page, prefixes, alone, causal = CASES[name]
    print("prefix nan", name, value, flush=True)
    x = Batch(heads, kvh, page, prefixes, alone)
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, causal)
    torch.cuda.synchronize()
    x.check(o, l, causal)
    rows = [(0, 0), (x.total // 2, heads - 1), (x.total - 1, heads // 2)]
    for t, h in rows:
        x.q[t, h, 5 * h % 128] = float(value)        # an infinity: scores of both signs, and their softmax is no number
    bad, bl = torch.empty_like(o), torch.empty_like(l)
    x.attend(gpu_runner, bad, bl, causal)
    torch.cuda.synchronize()
    hit = torch.zeros(o.shape[:2], dtype=torch.bool, device=x.dev)
    for t, h in rows:
        hit[t, h] = True
    assert torch.isnan(bad[hit]).all() and torch.isnan(bl.T[hit]).all()
    assert torch.equal(bad[~hit].view(torch.int16), o[~hit].view(torch.int16))
    assert torch.equal(bl.T[~hit], l.T[~hit])


def test_a_query_that_is_no_number_and_sees_no_key(gpu_runner):
    """Rows without a visible key have O = 0 and LSE = -inf, whatever their query."""
    x = Batch(8, 2, 64, [(128, [(5, 3), (1, 0)])], [(3, 1)])
    x.q.fill_(float("nan"))
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, 2)
    torch.cuda.synchronize()
    for t, empty in enumerate([True, True, False, False, False, True, True, True, False]):
        if empty:
            assert (o[t] == 0).all() and torch.isneginf(l[:, t]).all(), t
        else:
            assert torch.isnan(o[t]).all() and torch.isnan(l[:, t]).all(), t
