"""Attention of new tokens over the paged cache against 64 bits.

Tolerance: bf16 results are off by 2^-8 of their value, the probabilities, rounded to bf16 for the second product, by 2^-8 each, which adds at
most 2^-8 sum p|v|. What is left is fp32: a logit of 128 products is off by less than 2^-16 here (|q.k| s log2 e summed by magnitude is below 2^6),
the exponential and the running sums by 2^-20 and a few thousand times 2^-24; 2^-10 sum p|v| covers them."""
import math

import pytest
import torch

from async_grpo_nccl_b200.ops import reference as R
from gpu_util import native, status_word

pytestmark = pytest.mark.gpu
DEV = "cuda"

# (new rows, tokens in the cache): single tokens around the tiles' edges, idle and empty ones, rows that see nothing, chunks
MIXED = [(1, 1), (1, 0), (0, 5), (0, 0), (3, 2), (1, 127), (1, 128), (1, 129), (17, 17), (2, 700), (130, 1000), (257, 300), (5, 0), (1, 2049)]


class Case:
    def __init__(self, seqs, Hq, Hkv, D, bs, eight, pad=0, pitch=0, seed=0, q_scale=1.5):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.Hq, self.Hkv, self.D, self.bs = Hq, Hkv, D, bs
        per = [-(-L // bs) for _, L in seqs]
        blocks = sum(per) + 2
        order = torch.randperm(blocks, device=DEV, generator=g).int().tolist()
        width = max(1, max(per))
        self.table = torch.full((len(seqs), width + 3), 2 ** 30, dtype=torch.int32, device=DEV)[:, :width]  # entries behind a sequence mean nothing
        at, kv = 0, [torch.randn(blocks, Hkv, bs, D, device=DEV, generator=g).bfloat16() + i for i in range(2)]
        held = torch.zeros(blocks, bs, dtype=torch.bool, device=DEV)
        for b, n in enumerate(per):
            pages = order[at:at + n]
            at += n
            if n:
                self.table[b, :n] = torch.tensor(pages, dtype=torch.int32, device=DEV)
                held.view(-1)[(torch.tensor(pages, device=DEV)[:, None] * bs + torch.arange(bs, device=DEV)).reshape(-1)[:seqs[b][1]]] = True
        self.scales = [None, None]
        if eight:
            both = [R.kv8_quantise(c.float()) for c in kv]
            self.values = [R.kv8_values(*b) for b in both]
            kv, self.scales = [b[0] for b in both], [b[1] for b in both]
            for c, s in zip(kv, self.scales):
                c.view(torch.uint8).masked_fill_(~held[:, None, :, None], 0x7f)  # NaN where no sequence has a token
                s.masked_fill_(~held[:, None], 255)
        else:
            self.values = [c.clone() for c in kv]
            for c in kv:
                c.masked_fill_(~held[:, None, :, None], math.nan)
        self.kv = kv
        n = [a for a, _ in seqs]
        self.Tq = sum(n) + pad
        self.rows = (torch.randn(self.Tq, (Hq + 2 * Hkv) * D + pitch, device=DEV, generator=g) * q_scale).bfloat16()[:, :(Hq + 2 * Hkv) * D]
        self.starts = torch.tensor([0] + n, device=DEV).cumsum(0).int()
        self.lens = torch.tensor([b for _, b in seqs], device=DEV).int()
        self.out = torch.full((self.Tq, Hq * D + pitch), 7.0, device=DEV, dtype=torch.bfloat16)[:, :Hq * D]
        self.status = status_word()

    def call(self, **kw):
        a = dict(status=self.status, k_scale=self.scales[0], v_scale=self.scales[1])
        a.update(kw)
        native().paged_chunk_attn(self.rows, self.kv[0], self.kv[1], self.table, self.lens, self.starts, self.out, self.Hq, self.Hkv, self.D,
                                  1 / math.sqrt(self.D), **a)

    def check(self):
        want, size = R.paged_chunk_attention(self.rows, self.values[0], self.values[1], self.table, self.lens, self.starts, self.Hq, self.Hkv, self.D,
                                             1 / math.sqrt(self.D))
        n = int(self.starts[-1])
        off = (self.out[:n].double() - want[:n]).abs() - (want[:n].abs() * 2.0 ** -8 + size[:n] * (2.0 ** -8 + 2.0 ** -10))
        assert bool(self.out[:n].isfinite().all())
        assert n == 0 or float(off.max()) <= 0, (float(off.max()), torch.nonzero(off > 0)[:8].tolist())
        assert bool((self.out[n:] == 7).all())
        assert int(self.status) == 0


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,bs", [(12, 2, 128, 16), (28, 4, 128, 16), (5, 1, 64, 16), (8, 8, 128, 32), (64, 2, 128, 16), (14, 2, 64, 64), (3, 3, 64, 128),
                                         (16, 2, 128, 128)])
def test_mixed_lengths(Hq, Hkv, D, bs, eight):
    c = Case(MIXED, Hq, Hkv, D, bs, eight, pad=3, pitch=64, seed=Hq)
    c.call()
    c.check()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("seqs", [[(1, 1)], [(1, 700)], [(1, 40000)], [(4, 4)], [(1, 50)] * 300, [(1, L) for L in range(0, 400, 3)], [(7, 3000)] * 9, [(1000, 1000)],
                                  [(333, 5000), (1, 9)], [(64, 64 + i) for i in range(40)], [(0, 3)] * 5 + [(1, 3)], [(2100, 2100), (0, 0), (1500, 1777)],
                                  [(1, 5000)] * 150])
def test_uses(seqs, eight):
    """Decode steps, drafts, prompts and portions at one layout each."""
    c = Case(seqs, 12, 2, 128, 16, eight, seed=len(seqs))
    c.call()
    c.check()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n", [1, 40])
def test_large_logits(n, eight):
    """Softmax over one or two keys of thousands: logits of several hundred, maxima that keep growing along the sequence."""
    c = Case([(n, 3000)], 6, 1, 128, 16, eight, seed=n, q_scale=1.5)
    big = 1 + 8 * torch.arange(c.kv[0].shape[0] * 16, device=DEV).float().view(-1, 1, 16, 1) / (c.kv[0].shape[0] * 16)
    vals = (c.values[0].float() * big).bfloat16()
    if eight:
        codes, s = R.kv8_quantise(vals.float())
        c.kv[0], c.scales[0], c.values[0] = codes, s, R.kv8_values(codes, s)
    else:
        c.kv[0] = c.values[0] = vals
    c.call()
    c.check()


@pytest.mark.parametrize("seqs", [[(1, 900)] * 3, [(60, 900), (200, 500)]])
@pytest.mark.parametrize("which,spread", [(0, 8), (0, 60), (1, 8), (1, 20), (1, 60), (2, 30)])
def test_keys_and_values_of_very_different_sizes(seqs, which, spread):
    """8 bits: every vector with a power of its own, up to 2^spread apart (0: keys, 1: values, 2: both); a third of the values' vectors is zero."""
    c = Case(seqs, 12, 2, 128, 16, True, seed=spread)
    g = torch.Generator(device=DEV).manual_seed(which)
    for i in range(2):
        if which not in (i, 2):
            continue
        held = c.scales[i] != 255
        e = torch.randint(-spread, 1, held.shape, device=DEV, generator=g)
        x = torch.randn(c.kv[i].shape, device=DEV, generator=g).double() * torch.exp2(e.double())[..., None]
        if i == 1:
            x[torch.rand(held.shape, device=DEV, generator=g) < 0.33] = 0
        codes, s = R.kv8_quantise(x.bfloat16().float())
        c.values[i] = R.kv8_values(codes, s)
        codes.view(torch.uint8).masked_fill_(~held[..., None], 0x7f)
        c.kv[i], c.scales[i] = codes, s.masked_fill(~held, 255)
    c.call()
    c.check()


@pytest.mark.parametrize("seqs", [[(1, 900)] * 3, [(60, 900), (200, 500)]])
def test_values_that_grow_along_the_sequence(seqs):
    """8 bits: later pages hold values up to 2^40 larger, whose probabilities are small."""
    c = Case(seqs, 12, 2, 128, 16, True, seed=9)
    held = c.scales[1] != 255
    where = torch.zeros(held.shape[0], device=DEV)
    for b, (_, total) in enumerate(seqs):
        n = -(-total // 16)
        where[c.table[b, :n].long()] = torch.arange(n, device=DEV) * 40.0 / n
    x = torch.randn(c.kv[1].shape, device=DEV) * torch.exp2(where.floor())[:, None, None, None]
    codes, s = R.kv8_quantise(x)
    c.values[1] = R.kv8_values(codes, s)
    c.kv[1], c.scales[1] = codes, s.masked_fill(~held, 255)
    c.call()
    c.check()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("seqs", [[(1, 300), (1, 300)], [(70, 300), (70, 300)], [(200, 300), (200, 300)]])
def test_a_nan_stays_with_the_rows_that_see_it(seqs, eight):
    """A key or a value that is NaN makes its own sequence's rows NaN, those that see it and no other sequence's."""
    for i in range(2):
        c = Case(seqs, 12, 2, 128, 16, eight, seed=11)
        page, off = int(c.table[0, 3]), 5   # token 53 of sequence 0, kv head 1
        if eight:
            c.scales[i][page, 1, off] = 255
        else:
            c.kv[i][page, 1, off, 7] = math.nan
        c.call()
        n = seqs[0][0]
        heads = c.out.view(-1, 2, 6 * 128)
        assert bool(heads[n:].isfinite().all()) and bool(heads[:n, 0].isfinite().all())
        bad = heads[:n, 1].view(n, 6, 128)
        assert bool(bad.isnan().all()) if i == 0 or eight else bool(bad[..., 7].isnan().all()) and bool(bad[..., :7].isfinite().all())


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 2, 128), (8, 1, 64), (3, 3, 128), (20, 2, 64)])
@pytest.mark.parametrize("seqs", [[(3, 40), (2, 700), (5, 5)], [(1, 300), (2, 3), (1, 17)], [(60, 300), (200, 500), (9, 3)], [(300, 2300), (300, 300)]])
def test_values_that_are_no_numbers_do_not_reach_rows_that_do_not_see_them(seqs, Hq, Hkv, D, eight):
    """NaN and infinite values at tokens that some rows see and others do not: those rows are as if the values were zero, the others not finite
    in the places that the values have."""
    c = Case(seqs, Hq, Hkv, D, 16, eight, seed=13)
    clean = c.values[1].clone()
    bad = torch.zeros(clean.shape, dtype=torch.bool, device=DEV)
    for b, (n, total) in enumerate(seqs):
        for back, kind in ((1, math.inf), (1 + n // 2, math.nan), (max(n - 1, 1), -math.inf)):
            token = total - back
            if not 0 <= token or back >= n:
                continue
            page, off, h = int(c.table[b, token // 16]), token % 16, b % Hkv
            if eight:
                c.scales[1][page, h, off] = 255
                c.kv[1].view(torch.uint8)[page, h, off] = 0
                bad[page, h, off] = True
                clean[page, h, off] = 0
            else:
                for d in (back % D, D - 1):
                    c.kv[1][page, h, off, d] = kind
                    bad[page, h, off, d] = True
                    clean[page, h, off, d] = 0
    assert bool(bad.any())
    c.call()
    want, size = R.paged_chunk_attention(c.rows, c.values[0], clean, c.table, c.lens, c.starts, Hq, Hkv, D, 1 / math.sqrt(D))
    # the largest probability-weighted sum of marks: what sees one has a number above zero there
    marks, _ = R.paged_chunk_attention(c.rows, torch.zeros_like(c.values[0]), bad.double(), c.table, c.lens, c.starts, Hq, Hkv, D, 1.0)
    seen = marks > 0
    assert bool(seen.any()) and bool((~seen).any())
    assert bool((c.out.isfinite() == ~seen).all())
    off = (c.out.double() - want).abs() - (want.abs() * 2.0 ** -8 + size * (2.0 ** -8 + 2.0 ** -10))
    assert float(off[~seen].max()) <= 0
    assert int(c.status) == 0


@pytest.mark.parametrize("eight", [False, True])
def test_queries_of_any_size(eight):
    """Rows of Q from subnormal to 2^60, one of zeros: with keys as small as the queries are large, logits stay moderate."""
    for n in (1, 50):
        c = Case([(n, 300)] * 2, 12, 2, 128, 16, eight, seed=12)
        e = torch.tensor([-100.0, -30.0, 0.0, 1.0], device=DEV)[torch.arange(c.rows.shape[0], device=DEV) % 4]
        c.rows = (c.rows.double() * torch.exp2(e.double())[:, None]).bfloat16()
        c.rows[0] = 0
        c.call()
        c.check()
        c.rows = (c.rows.float() * 2.0 ** 59).bfloat16()
        small = c.values[0].double() * 2.0 ** -59
        if eight:
            codes, s = R.kv8_quantise(small.float())
            c.kv[0], c.scales[0], c.values[0] = codes, s, R.kv8_values(codes, s)
        else:
            c.kv[0] = c.values[0] = small.bfloat16()
        c.out.fill_(7)
        c.call()
        c.check()


def test_a_sequence_does_not_depend_on_where_its_pages_are():
    a = Case([(5, 700), (300, 900)], 12, 2, 128, 16, False, seed=1)
    a.call()
    blocks = a.kv[0].shape[0]
    perm = torch.randperm(blocks, device=DEV)
    first = a.out.clone()
    a.kv = [torch.empty_like(c).index_copy_(0, perm, c) for c in a.kv]
    inside = a.table < blocks
    a.table[inside] = perm[a.table[inside].long()].int()
    a.out.fill_(7)
    a.call()
    assert torch.equal(a.out, first)


@pytest.mark.parametrize("eight", [False, True])
def test_the_same_call_gives_the_same_bits(eight):
    c = Case([(1, 3000)] * 20 + [(200, 2000)], 12, 2, 128, 16, eight)
    c.call()
    first = c.out.clone()
    for _ in range(5):
        c.out.fill_(7)
        c.call()
        assert torch.equal(c.out, first)


@pytest.mark.parametrize("eight", [False, True])
def test_captured_calls_follow_the_lengths(eight):
    """Two graphs captured one after the other, replayed in turn on two streams with other lengths than at capture, beside an eager call."""
    cases = [Case([(1, 900), (1, 300), (1, 40)], 12, 2, 128, 16, eight, seed=3), Case([(60, 1500), (3, 700)], 12, 2, 128, 16, eight, seed=4)]
    graphs = []
    for c in cases:
        c.call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.call()
        graphs.append(g)
    cases[0].lens.copy_(torch.tensor([17, 300, 0]))
    cases[1].lens.copy_(torch.tensor([1300, 3]))
    eager = Case([(1, 2000)] * 7, 12, 2, 128, 16, eight, seed=5)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(4):
        for s, f in zip(streams, (graphs[0].replay, graphs[1].replay, eager.call)):
            with torch.cuda.stream(s):
                f()
    torch.cuda.synchronize()
    for c in cases + [eager]:
        c.check()


def test_captured_calls_with_a_converted_copy():
    """Two graphs of many rows over 8 bits replayed on two streams at once, and an eager call on a third, lengths changed in between."""
    cases = [Case([(n, 1500), (900, 1000)], 12, 2, 128, 16, True, seed=n) for n in (600, 800, 1000)]
    graphs = []
    for c in cases[:2]:
        c.call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.call()
        graphs.append(g)
    cases[0].lens.copy_(torch.tensor([700, 901]))
    cases[1].lens.copy_(torch.tensor([30, 0]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        for s, f in zip(streams, (graphs[0].replay, graphs[1].replay, cases[2].call)):
            with torch.cuda.stream(s):
                f()
    torch.cuda.synchronize()
    for c in cases:
        c.check()


@pytest.mark.parametrize("Hq,Hkv,D,bs", [(12, 2, 128, 16), (6, 3, 64, 64), (8, 8, 128, 128)])
def test_the_converted_copy_of_an_eight_bit_cache(Hq, Hkv, D, bs):
    """Many rows a sequence: the cache is converted once, ahead. With a table so wide that the copy would be too large the attention converts the keys itself; both
    give the same bits."""
    seqs = [(1100, 1200), (0, 500), (1, 300), (2200, 2200), (40, 0), (0, 0)]
    c = Case(seqs, Hq, Hkv, D, bs, True, pad=3, pitch=64, seed=21)
    c.call()
    c.check()
    first = c.out.clone()
    wide = torch.full((len(seqs), (128 << 20) // (len(seqs) * 4 * Hkv * bs * D) + 1), 2 ** 30, dtype=torch.int32, device=DEV)
    wide[:, :c.table.shape[1]] = c.table
    c.table = wide
    c.out.fill_(7)
    c.call()
    c.check()
    assert torch.equal(c.out, first)


def test_a_page_that_does_not_exist_under_many_rows():
    c = Case([(700, 700), (900, 1000)], 12, 2, 128, 16, True)
    c.call()
    first = c.out.clone()
    page = int(c.table[0, 7])
    for bad in (-1, 10 ** 6):
        c.table[0, 7] = bad
        c.out.fill_(7)
        c.call()
        assert int(c.status) == 6
        c.status.zero_()
        assert torch.equal(c.out[700:], first[700:]) and torch.equal(c.out[:7 * 16], first[:7 * 16])
    c.table[0, 7] = page
    c.lens[0] = 2 ** 30  # more than its table holds
    c.call()
    assert int(c.status) == 6
    c.status.zero_()
    c.lens[0] = 700
    c.out.fill_(7)
    c.call()
    assert int(c.status) == 0 and torch.equal(c.out, first)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("seqs", [[(1, 300)] * 3, [(40, 300), (300, 300)]])
def test_output_rows_on_sixteen_bytes(seqs, eight):
    c = Case(seqs, 12, 2, 128, 16, eight, pitch=8, seed=30)
    c.call()
    c.check()


@pytest.mark.parametrize("eight", [False, True])
def test_more_sequences_than_a_cta_has_at_hand(eight):
    """Hundreds of idle sequences between those that have rows, in both kernels."""
    for n in (1, 90):
        seqs = [(n if b % 331 == 7 else 0, 100 + b % 9) for b in range(2000)]
        c = Case(seqs, 12, 2, 128, 16, eight, seed=31)
        c.call()
        c.check()


def test_rows_and_output_in_one_buffer():
    for n in (1, 60):
        c = Case([(n, 300)] * 3, 12, 2, 128, 16, False, seed=33)
        both = torch.zeros(c.Tq, 2048 + 1536, dtype=torch.bfloat16, device=DEV)
        for q, o in ((slice(0, 2048), slice(2048, 3584)), (slice(1536, 3584), slice(0, 1536))):
            both[:, q] = c.rows
            c.rows, c.out = both[:, q], both[:, o]
            c.call()
            c.check()


def test_tables_without_columns_and_rows_that_are_one_row():
    c = Case([(4, 0), (2, 0)], 12, 2, 128, 16, False)
    c.table = c.table[:, :0]
    c.call()
    assert bool((c.out == 0).all()) and int(c.status) == 0
    c.lens[0] = 1  # more than its table holds
    c.call()
    assert int(c.status) == 6
    one = Case([(300, 300)], 12, 2, 128, 16, True, seed=32)
    one.rows = one.rows[:1].expand(300, -1)
    one.call()
    one.check()


def test_pages_and_lengths_that_do_not_exist_are_reported():
    for page in (-1, 10 ** 6):
        c = Case([(1, 100), (1, 100)], 12, 2, 128, 16, False)
        c.table[0, 2] = page
        c.call()
        assert int(c.status) == 6
        c.status.zero_()
        want = c.out[1].clone()
        c.table[0, 2] = c.table[1, 0]
        c.call()
        assert int(c.status) == 0 and torch.equal(c.out[1], want)
    c = Case([(1, 100), (1, 50)], 12, 2, 128, 16, True)
    c.lens[0] = 2 ** 30  # more than its table holds
    c.call()
    assert int(c.status) == 6
    c = Case([(1, 100), (2, 50)], 12, 2, 128, 16, True)
    for bad in ([0, 9, 3], [0, 2, 1], [-5, 1, 3]):  # starts that leave the rows or go back
        c.status.zero_()
        c.out.fill_(7)
        c.starts.copy_(torch.tensor(bad))
        c.call()
        assert int(c.status) == 6


def test_a_cache_behind_two_gigabytes():
    Hkv, D, bs = 8, 128, 16
    blocks = (1 << 31) // (Hkv * D * bs) + 40
    c = Case([(1, 300), (9, 200)], 16, Hkv, D, bs, True)
    n = c.kv[0].shape[0]
    k, v = (torch.empty(blocks, Hkv, bs, D, dtype=torch.uint8, device=DEV) for _ in range(2))
    s = [torch.zeros(blocks, Hkv, bs, dtype=torch.uint8, device=DEV) for _ in range(2)]
    for big, small, sb, ss in zip((k, v), c.kv, s, c.scales):
        big[-n:] = small.view(torch.uint8)
        sb[-n:] = ss
    c.call()
    first = c.out.clone()
    c.kv, c.scales = [k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)], s
    c.table += blocks - n
    c.out.fill_(7)
    c.call()
    assert torch.equal(c.out, first) and int(c.status) == 0


@pytest.mark.parametrize("eight", [False, True])
def test_pages_behind_two_billion_elements(eight):
    """A single token, some, and many (which an 8-bit cache is converted for)."""
    Hkv, D, bs = 8, 128, 16
    blocks = (1 << 31) // (Hkv * D * bs) + 400
    for seqs in ([(1, 300), (1, 200)], [(9, 200), (40, 300)], [(1100, 1200)]):
        c = Case(seqs, 16, Hkv, D, bs, eight, seed=34)
        n = c.kv[0].shape[0]
        big = [torch.empty(blocks, *k.shape[1:], dtype=torch.uint8 if eight else k.dtype, device=DEV) for k in c.kv]
        scales = [torch.zeros(blocks, Hkv, bs, dtype=torch.uint8, device=DEV) if eight else None for _ in c.kv]
        for b, k, s, t in zip(big, c.kv, scales, c.scales):
            b[-n:] = k.view(torch.uint8) if eight else k
            if eight:
                s[-n:] = t
        c.call()
        first = c.out.clone()
        c.kv = [b.view(torch.float8_e4m3fn) if eight else b for b in big]
        c.scales = scales
        c.table += blocks - n
        c.out.fill_(7)
        c.call()
        assert torch.equal(c.out, first) and int(c.status) == 0


def test_the_cache_that_was_written_is_what_is_attended():
    """Operators in a row, as an engine runs them: rows written in 8 bits, attended in place, and the same over what is read back."""
    C = native()
    Hq, Hkv, D, bs, T = 12, 2, 128, 16, 333
    c = Case([(T, T)], Hq, Hkv, D, bs, True)
    slots = (c.table[0, :, None] * bs + torch.arange(bs, device=DEV)).reshape(-1)[:T].int().contiguous()
    C.kv_cache_write(c.rows, slots, c.kv[0], c.kv[1], Hq, Hkv, D, c.status, 0, c.scales[0], c.scales[1])
    both = c.rows.float().view(T, Hq + 2 * Hkv, D)[:, Hq:]
    for i in range(2):
        c.values[i] = c.values[i].clone()
        c.values[i].transpose(1, 2).reshape(-1, Hkv, D)
        flat = c.values[i].transpose(1, 2).reshape(-1, Hkv, D).clone()
        flat[slots.long()] = R.kv8_values(*R.kv8_quantise(both[:, i * Hkv:(i + 1) * Hkv]))
        c.values[i] = flat.view(-1, bs, Hkv, D).transpose(1, 2)
    c.call()
    c.check()
    back = c.rows.clone()
    C.kv_cache_read(c.kv[0], c.kv[1], slots, back, Hq, Hkv, D, c.status, c.scales[0], c.scales[1])
    k, v = (torch.zeros(c.kv[0].shape, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    C.kv_cache_write(back, slots, k, v, Hq, Hkv, D, c.status)
    eight = c.out.clone()
    c.kv, c.scales = [k, v], [None, None]
    c.call()
    c.check()
    assert torch.equal(c.out, eight)  # the same values, the same products


def test_refusals():
    c = Case([(2, 40)], 12, 2, 128, 16, True)

    def refused(match, **kw):
        a = dict(qkv=c.rows, k=c.kv[0], v=c.kv[1], table=c.table, lens=c.lens, starts=c.starts, out=c.out, Hq=12, Hkv=2, D=128, ks=c.scales[0], vs=c.scales[1])
        a.update(kw)
        with pytest.raises(RuntimeError, match=match):
            native().paged_chunk_attn(a["qkv"], a["k"], a["v"], a["table"], a["lens"], a["starts"], a["out"], a["Hq"], a["Hkv"], a["D"], 0.1, c.status, a["ks"], a["vs"])

    refused("head_dim", D=96)
    refused("1 to 32", Hq=13)
    refused("1 to 32", Hq=128)
    refused("cache of", Hq=4, Hkv=4, out=c.out[:, :512])
    refused("cache of|heads of this rank", Hkv=1)
    refused("needs k_scale", ks=None)
    refused("scales uint8", vs=c.scales[1][:1])
    refused("out \\[rows", out=c.out[:1])
    refused("out bf16", out=c.out.float())
    refused("must not be qkv", out=c.rows[:, :1536])
    refused("rows overlap", out=c.out[:1].expand(2, -1))
    both = torch.zeros(2, 4096, dtype=torch.bfloat16, device=DEV)
    refused("must not be qkv", qkv=both[:, :2048], out=both[:, 1528:3064])
    refused("must not be qkv", qkv=both[:, 2048:], out=both[:, 1000:2536])
    refused("must not be qkv", qkv=both[:, 8:2056], out=both[:, :1536])
    refused("q_starts int32", starts=c.starts.long())
    refused("seq_lens int32", lens=c.lens[:0])
    refused("block_tables", table=c.table.long())
    refused("block_tables", table=c.table[:0])
    refused("on the device", lens=c.lens.cpu())
    small = torch.zeros(4, 2, 8, 128, dtype=torch.float8_e4m3fn, device=DEV)
    sc = torch.zeros(4, 2, 8, dtype=torch.uint8, device=DEV)
    refused("block size", k=small, v=small, ks=sc, vs=sc)
    many = Case([(1, 1)] * 2048, 12, 2, 128, 16, True)  # of up to 2^29 tokens each
    refused("too many rows", qkv=many.rows, lens=many.lens, starts=many.starts, out=many.out, k=many.kv[0], v=many.kv[1], ks=many.scales[0], vs=many.scales[1],
            table=many.table[:1, :1].expand(2048, 1).new_zeros(1, 1 << 25).expand(2048, -1))
    # nothing to do
    native().paged_chunk_attn(c.rows[:0], c.kv[0], c.kv[1], c.table[:0], c.lens[:0], c.starts[:1], c.out[:0], 12, 2, 128, 0.1, c.status, c.scales[0], c.scales[1])
    assert bool((c.out == 7).all()) and int(c.status) == 0
