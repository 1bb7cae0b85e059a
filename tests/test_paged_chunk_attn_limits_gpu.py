"""Attention of new tokens over the paged cache at the edge of what a call may hold."""
import pytest
import torch

from gpu_util import native, status_word
from test_paged_chunk_attn_gpu import Case

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n", [3, 60, 700])
def test_starts_that_go_back_give_nothing(n, eight):
    """Every second sequence would own the same rows. n: the three forms of the kernel (700 over 8 bits: the cache is converted first)."""
    c = Case([(n, 700), (0, 300), (0, 700)], 12, 2, 128, 16, eight, pad=2, seed=n)
    good = c.starts.clone()
    for bad in ([0, n, 0, n], [n, 0, n, n], [2, n, n, 1]):
        c.starts.copy_(torch.tensor(bad))
        c.call()
        assert int(c.status) == 6
        assert bool((c.out == 7).all())
        c.status.zero_()
    c.starts.copy_(good)
    c.call()
    c.check()


@pytest.mark.parametrize("eight", [False, True])
def test_starts_that_go_back_thousands_of_times(eight):
    """4096 sequences that would own the same 10922 rows: 4e9 tiles of keys, where the call's rows have 2e6."""
    c = Case([(10922, 700)], 12, 2, 128, 16, eight, seed=1)
    c.table = c.table.expand(8192, -1)
    c.lens = c.lens.repeat(8192)
    c.starts = (torch.arange(8193, device=DEV) % 2 * 10922).int()
    c.call()
    assert int(c.status) == 6
    assert bool((c.out == 7).all())
