"""Attention of new tokens over the paged cache at the edge of what a call may hold."""
import math

import pytest
import torch

from async_grpo_nccl_b200.ops import reference as R
from gpu_util import native
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


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("kind", [math.nan, math.inf])
@pytest.mark.parametrize("n,total", [(1, 3000), (3, 700), (1, 17), (40, 5000), (300, 600)])
def test_values_that_are_no_numbers_count_under_any_probability(n, total, kind, eight):
    """The first 64 tokens' logits lie so far below the others' (24 * 217 / 128^0.5 * log2 e: about 600 binades) that their probabilities are zero in 32 bits, in a
    part of their own or not: 0 * NaN and 0 * inf are no numbers, whoever adds the parts."""
    c = Case([(n, total)], 12, 2, 128, 16, eight, seed=n)
    c.rows.copy_(c.rows.abs() + 0.5)  # |q| of 1.7 on average, 217 a head
    for b in range(min(4, total // 16)):
        page = int(c.table[0, b])
        if eight:
            c.kv[0].view(torch.uint8)[page] = 0xf4  # -192
            c.scales[0][page] = 127 - 3                # times 2^-3
        else:
            c.kv[0][page] = -24
    page = int(c.table[0, 0])
    if eight:
        c.scales[1][page, 1, 5] = 255
    else:
        c.kv[1][page, 1, 5, 7] = kind
    c.call()
    heads = c.out.view(n, 2, 6, 128)
    assert bool(heads[:, 0].isfinite().all())
    assert not bool(heads[:, 1, :, 7].isfinite().any())
    if eight:
        assert bool(heads[:, 1].isnan().all())


@pytest.mark.parametrize("seqs,power", [([(1, 700)], 113), ([(1, 17)], 113), ([(2, 700)] * 40, 113), ([(40, 900)], 105), ([(1100, 1200)], 105),
                                        ([(1, 700)], -110), ([(1, 17)], -110), ([(2, 700)] * 40, -110), ([(40, 900)], -110), ([(1100, 1200)], -110)])
def test_eight_bit_values_near_the_ends_of_the_range(seqs, power):
    """Values of 2^power. Sums are 32 bits, relative to a maximum that may be behind by 2 (few rows) or 8 binades: 700 * 2^2 * 2^(113 + 2.6) and 1200 * 2^8 * 2^(105 + 2.6)
    are below 2^128. At the lower end a part of a row is off by 2^-126 for each key's product and each part, against 2^-8 * 2^-110 allowed."""
    c = Case(seqs, 12, 2, 128, 16, True, seed=7)
    held = c.scales[1] != 255
    assert float(c.values[1].abs().max()) <= 2 ** 2.6
    codes, s = R.kv8_quantise((c.values[1] * 2.0 ** power).bfloat16())
    c.values[1] = R.kv8_values(codes, s)
    c.kv[1], c.scales[1] = codes, s.masked_fill(~held, 255)
    c.call()
    c.check()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n", [1, 60, 1100])
def test_scales_that_32_bits_do_not_hold_are_refused(n, eight):
    """A scale of zero in 32 bits would make hidden scores 0 * -inf. Next to that end it still is the mean of the values that a row sees."""
    c = Case([(n, 1100)], 12, 2, 128, 16, eight, seed=3)

    def call(scale):
        native().paged_chunk_attn(c.rows, c.kv[0], c.kv[1], c.table, c.lens, c.starts, c.out, 12, 2, 128, scale, c.status, c.scales[0], c.scales[1])

    for scale in (0.0, -0.1, math.nan, math.inf, 1e-60, 1e-39, 1e39, 3e38):
        with pytest.raises(RuntimeError, match="softmax_scale"):
            call(scale)
    assert bool((c.out == 7).all())
    call(1e-37)
    want, size = R.paged_chunk_attention(c.rows, c.values[0], c.values[1], c.table, c.lens, c.starts, 12, 2, 128, 1e-37)
    assert bool(((c.out.double() - want).abs() <= want.abs() * 2.0 ** -8 + size * (2.0 ** -8 + 2.0 ** -10)).all())
    assert int(c.status) == 0


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("seqs,Hq", [
    ([(20 if b % 2 else 0, 100 + b % 9) for b in range(700)], 12),            # more sequences than the kernel has threads
    ([(800 if b % 331 == 7 else 0, 800 + b % 9) for b in range(2000)], 12),   # hundreds of idle ones between those that have rows
    ([(40 if b % 140 < 3 else 0, 60) for b in range(300)] * 2, 64),           # shares of short sequences go across idle ones
    ([(900, 950)] * 3 + [(0, 40)] * 130 + [(900, 900)] * 3, 64),              # over 8 bits the cache is converted first
    ([(1, 30 + b % 50) for b in range(3000)] + [(2500, 2500)], 64),           # single tokens beside a long prompt
])
def test_many_rows_among_many_sequences(seqs, Hq, eight):
    """More sequences than a CTA has at hand (128) and than it has threads, in the kernel of many rows: Tq * (query heads a kv head) > 16 * sequences."""
    assert sum(n for n, _ in seqs) * Hq // 2 > 16 * len(seqs)
    c = Case(seqs, Hq, 2, 128, 16, eight, pad=1, seed=35)
    c.call()
    c.check()
