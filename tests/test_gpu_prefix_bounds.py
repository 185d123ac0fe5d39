"""GPU checks of attention behind shared prefixes where the call's sizes lie close: max_seqlen_k is what it is said
to be, a bound on the sequences' key counts, and may lie inside a prefix."""
import numpy as np
import pytest
import torch

from tests.serving import Batch

pytestmark = pytest.mark.gpu


class ShortBatch(Batch):
    """max_seqlen_k is the longest sequence's key count, and the block table has no columns past it."""

    def __init__(self, *args, **more):
        super().__init__(*args, **more)
        self.max_k = max(max(sk for _, sk in self.lens), 1)
        self.table = np.ascontiguousarray(self.table[:, :-(-self.max_k // self.page)])
        self.table_d = torch.from_numpy(self.table).to(self.dev)


# (heads, kv_heads, page, prefixes, sequences of no prefix, causal); the three cuts: up to 32 rows a prefix, up to 32
# a sequence, more.
SHORT = {
    "few_rows_a_prefix": (32, 8, 64, [(1024, [(1, 1000), (1, 963)])], [], 0),
    "few_rows_a_prefix_causal": (32, 8, 64, [(1024, [(2, 1000), (3, 961)])], [], 2),
    "few_rows_a_sequence": (32, 8, 64, [(1024, [(1, 1000 - 3 * i) for i in range(12)])], [], 0),
    "few_rows_a_sequence_causal": (8, 1, 32, [(320, [(3, 310 - i) for i in range(4)])], [(1, 7)], 2),
    "many_rows_a_sequence": (8, 2, 64, [(1024, [(40, 1000), (9, 990)])], [], 0),
    "many_rows_a_sequence_causal": (8, 2, 64, [(1024, [(40, 1000), (9, 990)])], [], 2),
    "within_the_first_page": (8, 2, 64, [(128, [(1, 40), (1, 64), (1, 1)])], [], 0),
    "shorter_than_a_page": (8, 2, 64, [(128, [(1, 40), (1, 63)])], [], 0),
    "shorter_than_a_page_causal": (16, 4, 96, [(192, [(5, 40), (30, 50)])], [], 2),
    "shorter_than_a_page_many_rows": (8, 1, 256, [(512, [(60, 100), (3, 255)])], [], 0),
    "single_keys": (8, 8, 32, [(64, [(1, 1), (1, 1)])], [], 0),
    "prefixes_longer_and_shorter": (16, 4, 64, [(64, [(1, 90)]), (640, [(1, 100), (1, 30)]), (128, [(1, 0)])],
                                    [(1, 99)], 0),
    "a_long_prefix": (8, 2, 64, [(8192, [(1, 4100), (1, 17)])], [], 0),
    "over_512_sequences": (4, 1, 32, [(160, [(1, 1 + i % 150) for i in range(530)])], [], 0),
    "over_256_prefixes": (4, 2, 32, [(96, [(1, 70 + i % 9)]) for i in range(260)], [], 2),
}


@pytest.mark.parametrize("seed", [1, 2])
@pytest.mark.parametrize("name", SHORT)
def test_sequences_shorter_than_their_prefixes(gpu_runner, name, seed):
    """max_seqlen_k ends inside a prefix, and inside a page: the keys of that page are the prefix's all the same."""
    heads, kvh, page, prefixes, alone, causal = SHORT[name]
    print("prefix short", name, seed, flush=True)
    x = ShortBatch(heads, kvh, page, prefixes, alone, seed=seed)
    assert x.max_k < max(p for p, _ in prefixes)
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, causal)
    torch.cuda.synchronize()
    x.check(o, l, causal)
    assert torch.isnan(x.o_all[o.shape[0]:]).all()


@pytest.mark.parametrize("causal", [0, 2])
def test_more_keys_than_the_paged_call_takes(gpu_runner, causal):
    """Over 2^19 keys, most of them shared."""
    x = Batch(4, 1, 128, [(600064, [(1, 600200), (2, 660000)])])
    o, l = x.outputs(True)
    x.attend(gpu_runner, o, l, causal)
    torch.cuda.synchronize()
    x.check(o, l, causal)
