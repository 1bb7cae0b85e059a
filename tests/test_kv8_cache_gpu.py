"""The 8-bit KV cache on the GPU: written from rows, written by a decode step, read back. Every value is compared bit for bit: a power of
two scales without a rounding, and a code is exact in bf16."""
import math

import pytest
import torch

from async_grpo_nccl_b200.ops import reference as R
from gpu_util import native, status_word

pytestmark = pytest.mark.gpu
DEV = "cuda"


def empty_cache(blocks, heads, bs, D):
    """Every code and byte set to something that no test writes there."""
    k, v = (torch.full((blocks, heads, bs, D), 0x15, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.full((blocks, heads, bs), 99, dtype=torch.uint8, device=DEV) for _ in range(2))
    return k, v, ks, vs


def rows_of(T, heads, D, pitch=0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, heads * D + pitch, device=DEV, generator=g)
    x *= torch.exp2(torch.randint(-20, 20, (T, 1), device=DEV, generator=g).float())
    return x.bfloat16()[:, :heads * D]


def same(a, b):
    return torch.equal(a.nan_to_num(nan=12345.0), b.nan_to_num(nan=12345.0)) and torch.equal(a.isnan(), b.isnan())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,Hq,Hkv,bs,pitch", [(1, 1, 1, 16, 0), (37, 12, 2, 16, 0), (130, 3, 3, 7, 64), (1025, 8, 8, 32, 8)])
def test_written_entries_are_the_nearest_codes(D, T, Hq, Hkv, bs, pitch):
    C = native()
    blocks = T // bs + 3
    x = rows_of(T, Hq + 2 * Hkv, D, pitch)
    kv = x.view(T, -1) if pitch == 0 else x
    if T > 20:  # zeros, subnormals, the top, infinities and NaN
        h = Hq * D
        kv[3, h:] = 0
        kv[4, h:] = 1e-39
        kv[5, h] = torch.finfo(torch.bfloat16).max
        kv[6, h] = math.inf
        kv[7, h + D - 1] = -math.nan
        kv[8, h:] = -kv[9, h:]
        kv[10, h] = 448
        kv[11, h] = -450
    slots = torch.randperm(blocks * bs, device=DEV)[:T].int()
    slots[::5] = -1
    k, v, ks, vs = empty_cache(blocks, Hkv, bs, D)
    before = [t.clone() for t in (k.view(torch.uint8), v.view(torch.uint8), ks, vs)]
    st = status_word()
    C.kv_cache_write(x, slots, k, v, Hq, Hkv, D, st, 0, ks, vs)
    want = x.float().view(T, Hq + 2 * Hkv, D)[:, Hq:] if pitch == 0 else x.float().reshape(T, Hq + 2 * Hkv, D)[:, Hq:]
    codes, scale = R.kv8_quantise(want)
    on = slots >= 0
    blk, off = slots[on].long() // bs, slots[on].long() % bs
    for i, (c, s, was_c, was_s) in enumerate(((k, ks, before[0], before[2]), (v, vs, before[1], before[3]))):
        mine = slice(i * Hkv, (i + 1) * Hkv)
        was_s[blk, :, off] = scale[on][:, mine]
        assert torch.equal(s, was_s)  # nothing else was touched
        bad = (scale[on][:, mine] == R.KV8_NAN_BYTE)[..., None]
        got = c.view(torch.uint8)[blk, :, off]
        assert torch.equal(torch.where(bad, 0, got), torch.where(bad, 0, codes[on][:, mine].view(torch.uint8)))
        was_c[blk, :, off] = got
        assert torch.equal(c.view(torch.uint8), was_c)
    # back into rows: only the k and v columns of rows with a slot
    back = torch.full((T, (Hq + 2 * Hkv) * D + 16), 7.0, device=DEV, dtype=torch.bfloat16)[:, :(Hq + 2 * Hkv) * D]
    C.kv_cache_read(k, v, slots, back, Hq, Hkv, D, st, ks, vs)
    values = R.kv8_values(codes, scale).flatten(1)
    assert same(back[on][:, Hq * D:].double(), values[on])
    assert bool((back[~on] == 7).all()) and bool((back[:, :Hq * D] == 7).all())
    assert int(st) == 0


@pytest.mark.parametrize("D", [64, 128])
def test_every_code_under_every_scale_reads_as_what_it_stands_for(D):
    C = native()
    codes = torch.arange(256, dtype=torch.uint8, device=DEV)
    codes = codes[(codes & 0x7f) != 0x7f]
    codes = torch.cat([codes, codes[:2]]).view(-1, D)            # 256 codes = whole vectors
    bytes_ = torch.arange(R.KV8_MIN_BYTE, 247, dtype=torch.uint8, device=DEV)
    n = len(codes) * len(bytes_)
    k = codes.repeat(len(bytes_), 1).view(n, 1, 1, D).view(torch.float8_e4m3fn)
    s = bytes_.repeat_interleave(len(codes)).view(n, 1, 1)
    out = torch.zeros(n, 2 * D, device=DEV, dtype=torch.bfloat16)
    C.kv_cache_read(k, k, torch.arange(n, device=DEV).int(), out, 0, 1, D, None, s, s)
    want = R.kv8_values(k.view(n, D), s.view(n))
    assert torch.equal(out[:, :D].double(), want) and torch.equal(out[:, D:].double(), want)


def test_a_rank_writes_its_share_of_the_heads():
    C = native()
    T, Hq, Hkv, D, bs = 20, 4, 4, 128, 16
    x = rows_of(T, Hq + 2 * Hkv, D)
    slots = torch.arange(T, device=DEV).int()
    whole, part = empty_cache(2, Hkv, bs, D), empty_cache(2, 2, bs, D)
    for c, at in ((whole, 0), (part, 1)):
        C.kv_cache_write(x, slots, c[0], c[1], Hq, Hkv, D, None, at, c[2], c[3])
    for a, b in zip(whole, part):
        assert torch.equal(a.view(torch.uint8)[:, 1:3], b.view(torch.uint8))


def test_a_bf16_cache_reads_back_too():
    C = native()
    T, Hq, Hkv, D, bs = 45, 3, 2, 64, 16
    x = rows_of(T, Hq + 2 * Hkv, D)
    k, v = (torch.zeros(5, Hkv, bs, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    slots = torch.randperm(5 * bs, device=DEV)[:T].int()
    C.kv_cache_write(x, slots, k, v, Hq, Hkv, D)
    back = torch.zeros_like(x)
    C.kv_cache_read(k, v, slots, back, Hq, Hkv, D)
    assert torch.equal(back[:, Hq * D:], x[:, Hq * D:]) and bool((back[:, :Hq * D] == 0).all())


@pytest.mark.parametrize("Hq,Hkv,D,B", [(12, 2, 128, 1), (28, 4, 128, 70), (5, 5, 64, 33)])
def test_a_decode_step_rotates_and_writes(Hq, Hkv, D, B):
    """The rotated rows have the bits of the kernel for a bf16 cache, and the entries are those of the rotated rows."""
    C = native()
    bs, g = 16, torch.Generator().manual_seed(B)
    lens = torch.randint(0, 300, (B,), generator=g)
    lens[B // 2] = 0  # idle
    nb = 20
    table = torch.randperm(B * nb, generator=g).view(B, nb).int().to(DEV)
    lens = lens.int().to(DEV)
    angle = torch.arange(250)[:, None] * 1e4 ** (-torch.arange(0, D, 2) / D)   # fewer positions than the longest sequence: clamped
    cos_t, sin_t = angle.cos().float().to(DEV), angle.sin().float().to(DEV)
    rows = rows_of(B, Hq + 2 * Hkv, D, seed=B)
    a, b = rows.clone(), rows.clone()
    kb, vb = (torch.zeros(B * nb, Hkv, bs, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    k, v, ks, vs = empty_cache(B * nb, Hkv, bs, D)
    st = status_word()
    C.rope_kv_write_decode(a, cos_t, sin_t, table, lens, kb, vb, Hq, Hkv, D, st)
    C.rope_kv_write_decode(b, cos_t, sin_t, table, lens, k, v, Hq, Hkv, D, st, ks, vs)
    assert torch.equal(a, b) and int(st) == 0
    last = (lens.long() - 1).clamp(min=0)
    slots = (table.gather(1, (last // bs)[:, None])[:, 0] * bs + last % bs).int()
    slots[lens == 0] = -1
    k2, v2, ks2, vs2 = empty_cache(B * nb, Hkv, bs, D)
    C.kv_cache_write(b, slots, k2, v2, Hq, Hkv, D, st, 0, ks2, vs2)
    for p, q in ((k, k2), (v, v2), (ks, ks2), (vs, vs2)):
        assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("eight", [False, True])
def test_rows_on_sixteen_bytes_read_and_write_the_same(D, eight):
    """Every other row lies off the 32-byte sectors, a bf16 cache as a whole does."""
    C = native()
    T, Hq, Hkv, bs = 70, 3, 2, 16
    cols = (Hq + 2 * Hkv) * D
    x = rows_of(T, Hq + 2 * Hkv, D)
    slots = torch.randperm(6 * bs, device=DEV)[:T].int()
    seen = []
    for pitch, off in ((0, 0), (8, 0), (8, 8)):
        rows = torch.zeros(T, cols + pitch + off, device=DEV, dtype=torch.bfloat16)[:, off:off + cols]
        rows.copy_(x)
        scales = (None, None)
        if eight:
            k, v, *scales = empty_cache(6, Hkv, bs, D)
        else:
            k, v = (torch.zeros(6 * Hkv * bs * D + 8, device=DEV, dtype=torch.bfloat16)[off:off + 6 * Hkv * bs * D].view(6, Hkv, bs, D) for _ in range(2))
        C.kv_cache_write(rows, slots, k, v, Hq, Hkv, D, None, 0, *scales)
        back = torch.full((T, cols + pitch + off), 7.0, device=DEV, dtype=torch.bfloat16)[:, off:off + cols]
        C.kv_cache_read(k, v, slots, back, Hq, Hkv, D, None, *scales)
        assert bool((back[:, :Hq * D] == 7).all())
        seen.append(back[:, Hq * D:].clone())
    assert torch.equal(seen[1], seen[0]) and torch.equal(seen[2], seen[0])
    if not eight:
        assert torch.equal(seen[0], x[:, Hq * D:])


def test_slots_behind_the_cache_are_reported_and_left_out():
    C = native()
    x = rows_of(3, 3, 64)
    k, v, ks, vs = empty_cache(2, 1, 16, 64)
    st = status_word()
    C.kv_cache_write(x, torch.tensor([3, 32, 2 ** 31 - 1], device=DEV, dtype=torch.int32), k, v, 1, 1, 64, st, 0, ks, vs)
    assert int(st) == 6 and int((ks != 99).sum()) == 1
    st.zero_()
    back = torch.zeros_like(x)
    C.kv_cache_read(k, v, torch.tensor([3, 32, 2 ** 31 - 1], device=DEV, dtype=torch.int32), back, 1, 1, 64, st, ks, vs)
    assert int(st) == 6 and bool((back[1:] == 0).all()) and bool((back[0, 64:] != 0).any())
    st.zero_()
    ones = torch.ones(4, 32, device=DEV)
    C.rope_kv_write_decode(x[:1], ones, ones, torch.tensor([[7]], device=DEV, dtype=torch.int32), torch.tensor([5], device=DEV, dtype=torch.int32), k, v, 1, 1,
                           64, st, ks, vs)
    assert int(st) == 6
    st.zero_()  # a position behind the table's last block
    C.rope_kv_write_decode(x[:1], ones, ones, torch.tensor([[1]], device=DEV, dtype=torch.int32), torch.tensor([17], device=DEV, dtype=torch.int32), k, v, 1, 1,
                           64, st, ks, vs)
    assert int(st) == 6 and int((ks != 99).sum()) == 1


def test_offsets_behind_two_gigabytes():
    C = native()
    Hkv, D, bs = 8, 128, 16
    blocks = (1 << 31) // (Hkv * D * bs) + 9
    k, v = (torch.zeros(blocks, Hkv, bs, D, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.zeros(blocks, Hkv, bs, dtype=torch.uint8, device=DEV) for _ in range(2))
    x = rows_of(32, 2 * Hkv, D)
    slots = ((blocks - 2) * bs + torch.arange(32, device=DEV)).int()
    C.kv_cache_write(x, slots, k, v, 0, Hkv, D, None, 0, ks, vs)
    back = torch.zeros_like(x)
    C.kv_cache_read(k, v, slots, back, 0, Hkv, D, None, ks, vs)
    assert torch.equal(back.double(), R.kv8_values(*R.kv8_quantise(x.float().view(32, 2 * Hkv, D))).flatten(1))


def test_refusals():
    C = native()
    k, v, ks, vs = empty_cache(2, 2, 16, 64)
    x = rows_of(4, 6, 64)
    s = torch.zeros(4, dtype=torch.int32, device=DEV)

    def refused(match, *args):
        with pytest.raises(RuntimeError, match=match):
            C.kv_cache_write(*args)

    refused("needs k_scale", x, s, k, v, 2, 2, 64)
    refused("scales uint8", x, s, k, v, 2, 2, 64, None, 0, ks, vs[:1])
    refused("scales uint8", x, s, k, v, 2, 2, 64, None, 0, ks, vs.int())
    refused("heads of this rank", x, s, k, v, 2, 2, 64, None, 1, ks, vs)
    refused("heads of this rank", x, s, k[..., :32], v[..., :32], 2, 2, 32, None, 0, ks, vs)
    refused("slot for each row", x, s[:3], k, v, 2, 2, 64, None, 0, ks, vs)
    refused("slots int32", x, s.long(), k, v, 2, 2, 64, None, 0, ks, vs)
    refused("16-byte aligned", x[:, 1:], s, k, v, 1, 2, 64, None, 0, ks, vs)
    refused("one type", x, s, k, v.to(torch.bfloat16), 2, 2, 64, None, 0, ks, vs)
    refused("float8_e4m3fn", x, s, k.view(torch.float8_e5m2), v.view(torch.float8_e5m2), 2, 2, 64, None, 0, ks, vs)
    b = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    refused("has no scales", x, s, b, b, 2, 2, 64, None, 0, ks, vs)
    with pytest.raises(RuntimeError, match="rows overlap"):
        C.kv_cache_read(k, v, s, x[:1].expand(4, -1), 2, 2, 64, None, ks, vs)
    with pytest.raises(RuntimeError, match="cache of"):
        C.kv_cache_read(k, v, s, x, 2, 1, 64, None, ks, vs)
    # nothing to do
    C.kv_cache_write(x[:0], s[:0], k, v, 2, 2, 64, None, 0, ks, vs)
    C.kv_cache_read(k, v, s[:0], x[:0], 2, 2, 64, None, ks, vs)
