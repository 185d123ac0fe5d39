"""Host-only: which kernel each batch of the GPU tests of the 4-bit caches' attention gets, so that a change of the rules
does not move a test off the kernel that it is there for."""
import pytest

from tests import launches
from tests.test_gpu_mx4_calls import KINDS
from tests.test_gpu_mx4_forms import FORMS, PAGES, WIDE


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return launches.build(tmp_path_factory.mktemp("mx4"))


def form(launched):
    return (*launches.kind(launched), launched[0][2])


@pytest.mark.parametrize("causal", [0, 2])
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("name", FORMS)
def test_forms(lib, name, page, causal):
    want, heads, kv_heads, lens = FORMS[name]
    assert form(launches.attention(lib, heads, kv_heads, page, lens, causal)) == want


def test_every_form_has_a_batch():
    assert len({f for f, *_ in FORMS.values()}) == len(FORMS) == 9


# tests/test_gpu_mx4_calls.py: what its batches get at 8 heads, 2 K/V heads, pages of 16 to 64 and the lengths' sum unknown.
CALLS = {"whole": ("decode", "whole", 16, 512), "line": ("decode", "line", 16, 256), "long_whole": ("decode", "whole", 16, 768),
         "drafts": ("decode", "whole", 32, 512), "drafts_line": ("decode", "line", 32, 256),
         "prompts": ("decode", "whole", 32, 512), "chunks": ("decode", "line", 32, 256),
         "long_chunks": ("prefill", "line", 256, 512), "many_prompts": ("prefill", "whole", 128, 256),
         "many_chunks": ("prefill", "line", 128, 256)}


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("name", KINDS)
def test_kinds(lib, name, page):
    for lse in (False, True):
        assert form(launches.attention(lib, 8, 2, page, KINDS[name], 2, lse=lse)) == CALLS[name]


def test_a_sum_that_is_not_known(lib):
    """total_k 0 is taken as batch * max_seqlen_k; the rule of the BF16 call, one less, is not this one's."""
    for lens, causal in (([(1, 32768)] + [(1, 300)] * 31, 0), ([(4, 3000), (4, 100)] * 9, 2), ([(300, 4000), (20, 30)] * 5, 2)):
        most = len(lens) * max(k for _, k in lens)
        not_known = launches.attention(lib, 32, 8, 64, lens, causal)
        assert not_known == launches.attention(lib, 32, 8, 64, lens, causal, total_k=most)
    skewed = [(1, 32768)] + [(1, 300)] * 31
    assert launches.kind(launches.attention(lib, 32, 8, 64, skewed, 0))[1] == "whole"
    assert launches.kind(launches.attention(lib, 32, 8, 64, skewed, 0, total_k=32768 + 31 * 300))[1] == "line"


def test_wide_groups(lib):
    """More rows a token than a row tile has, in three of the kernels."""
    got = [launches.kind(launches.attention(lib, h, kvh, 32, lens, 2)) for h, kvh, lens in WIDE]
    assert {k for k, *_ in got} == {"decode", "prefill"} and {c for _, c, _ in got} == {"whole", "line"}, got
    assert all(h // kvh > rows for (h, kvh, _), (*_, rows) in zip(WIDE, got)), got


def test_queries_past_4_gib(lib):
    one = launches.attention(lib, 32, 8, 64, [(600_000, 70)], 0)
    each = launches.attention(lib, 32, 8, 64, [(1, 70)] * 600_000, 0)
    assert launches.kind(one)[0] == "prefill" and launches.kind(each)[0] == "decode"


def test_launches_fit_a_grid(lib):
    """Less than 2^32 threads each, at the largest plans that are accepted."""
    for heads, kv_heads, lens, max_q in ((8, 8, [(1 << 19, 64)], None), (64, 64, [(100, 64)] * 60_000, None),
                                         (1 << 15, 1 << 15, [(1, 1 << 15)], None)):
        for name, grid, threads in launches.attention(lib, heads, kv_heads, 64, lens, 2, max_q=max_q):
            assert 0 < grid * threads < 1 << 32, (name, grid, threads)
