"""The rollout cache in 8 bits and the attention of new tokens over the paged cache, as cases that can be timed and compared.

Three kinds of work, each as the rollout engine does it:

* ``cache``: the keys and values of a prompt's tokens go into their cache slots in 8 bits, and the values of a context come back
  (a prompt that shares a known beginning);
* ``step``: a decode step's rows are rotated, their keys and values go into the cache in 8 bits, and what was written is read back;
* ``attn``: attention of the newest tokens of every sequence (one token, a few drafted ones, a portion of a prompt) over the paged
  cache, which holds bf16 or 8 bits.

A cache in 8 bits holds, for a token's ``D`` values of one kv head, e4m3 codes and one power of two 2^e: the smallest with
max|x| <= 448 * 2^e, e >= -116, stored as the byte e + 127. What a code stands for is exact in bf16.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"


def listed():
    return [
        # the last sample of a group decodes alone: the smallest call, all latency
        dict(name="attn_one", kind="attn", cache="bf16", B=1, n_lo=1, n_hi=1, past_lo=699, past_hi=699, Hq=12, Hkv=2, D=128, bs=16, pad=0, lens=1),
        # a decode step in the middle of a generation phase, ragged contexts, idle rows behind the running ones
        dict(name="attn_step_8bit", kind="attn", cache="e4m3", B=61, n_lo=1, n_hi=1, past_lo=200, past_hi=4000, Hq=12, Hkv=2, D=128, bs=16, pad=3, lens=2),
        # a full decode batch on long contexts, more kv heads: the bandwidth of the cache
        dict(name="attn_step_long_8bit", kind="attn", cache="e4m3", B=128, n_lo=1, n_hi=1, past_lo=1000, past_hi=8000, Hq=40, Hkv=8, D=128, bs=16, pad=0, lens=3),
        # the same with a bf16 cache and two to six drafted tokens a sequence
        dict(name="attn_drafts", kind="attn", cache="bf16", B=32, n_lo=2, n_hi=6, past_lo=500, past_hi=4000, Hq=28, Hkv=4, D=128, bs=16, pad=0, lens=4),
        # prompts of many lengths at once, some wholly known, behind shared beginnings of other lengths
        dict(name="attn_prompts", kind="attn", cache="bf16", B=24, n_lo=0, n_hi=900, past_lo=0, past_hi=700, Hq=12, Hkv=2, D=128, bs=16, pad=5, lens=5),
        # one portion of a long prompt
        dict(name="attn_portion", kind="attn", cache="bf16", B=1, n_lo=4096, n_hi=4096, past_lo=12288, past_hi=12288, Hq=28, Hkv=4, D=128, bs=16, pad=0, lens=6),
        # a shorter portion far into a long document, 8-bit cache
        dict(name="attn_portion_8bit", kind="attn", cache="e4m3", B=2, n_lo=700, n_hi=1000, past_lo=15000, past_hi=28000, Hq=12, Hkv=2, D=128, bs=16, pad=0, lens=7),
        # heads of 64, larger pages
        dict(name="attn_heads64_8bit", kind="attn", cache="e4m3", B=9, n_lo=33, n_hi=500, past_lo=0, past_hi=3000, Hq=14, Hkv=2, D=64, bs=32, pad=0, lens=8),
        # a short prompt's tokens written and read back
        dict(name="cache_short", kind="cache", T=37, R=53, skip=4, Hq=12, Hkv=2, D=128, bs=16, lens=9),
        # a prefill batch of the engine's 16384 tokens
        dict(name="cache_prefill", kind="cache", T=16384, R=16000, skip=0, Hq=40, Hkv=8, D=128, bs=16, lens=10),
        # odd counts, heads of 64, larger pages
        dict(name="cache_odd", kind="cache", T=1537, R=2049, skip=130, Hq=4, Hkv=2, D=64, bs=32, lens=11),
        # the rows of a decode step on their way into the cache
        dict(name="step_rows", kind="step", B=256, past_lo=0, past_hi=9000, Hq=28, Hkv=4, D=128, bs=16, lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


LARGEST = 4 * 128 * 28 * 4096 * (12288 + 2048)  # products of the largest listed case


def draw(rng):
    Hkv, D, bs = rng.choice([1, 2, 2, 4, 8]), rng.choice([64, 128, 128]), rng.choice([16, 16, 32])
    Hq = Hkv * rng.randint(1, 8)
    lens = rng.randrange(1 << 30)
    kind = rng.choice(["attn", "attn", "attn", "attn", "cache", "step"])
    if kind == "cache":
        T = _log(rng, 1, 16384)
        return dict(kind=kind, T=T, R=_log(rng, 1, 16384), skip=rng.randint(0, T // 8), Hq=Hq, Hkv=Hkv, D=D, bs=bs, lens=lens)
    if kind == "step":
        return dict(kind=kind, B=_log(rng, 1, 512), past_lo=0, past_hi=_log(rng, 16, 16000), Hq=Hq, Hkv=Hkv, D=D, bs=bs, lens=lens)
    use = rng.choice(["step", "drafts", "prompts", "portion"])
    if use == "step":
        B, n, past = _log(rng, 1, 256), (1, 1), (_log(rng, 1, 500), _log(rng, 500, 8000))
    elif use == "drafts":
        B, n, past = _log(rng, 1, 64), (rng.randint(1, 3), rng.randint(4, 12)), (_log(rng, 1, 500), _log(rng, 500, 8000))
    elif use == "prompts":
        B, n, past = _log(rng, 2, 24), (0, _log(rng, 10, 1000)), (0, _log(rng, 10, 1000))
    else:
        a, b = _log(rng, 16, 4096), _log(rng, 16, 16000)
        B, n, past = rng.randint(1, 2), (a // 2, a), (b // 2, b)
    case = dict(kind=kind, cache=rng.choice(["bf16", "e4m3"]), B=B, n_lo=n[0], n_hi=n[1], past_lo=past[0], past_hi=past[1], Hq=Hq, Hkv=Hkv, D=D, bs=bs, pad=rng.choice([0, 0, 3]), lens=lens)
    while work(case)["flops"] > LARGEST or case["B"] * past[1] * Hkv * D > 1 << 30:
        case["B"] = max(1, case["B"] // 2)
        if case["B"] == 1:
            case["n_hi"] //= 2
            case["n_lo"] = min(case["n_lo"], case["n_hi"])
    return case


def _lengths(case):
    """(new tokens, tokens in the cache) of every sequence."""
    rng = random.Random(case["lens"])
    if case["kind"] == "step":
        n = [1] * case["B"]
    else:
        n = [rng.randint(case["n_lo"], case["n_hi"]) for _ in range(case["B"])]
    return n, [a + rng.randint(case["past_lo"], case["past_hi"]) for a in n]


def work(case):
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "cache":
        rows = (case["T"] - case["skip"]) + case["R"]
        return {"bytes": rows * 2 * Hkv * (3 * D + 1) + 4 * (case["T"] + case["R"]), "flops": 2 * rows * 2 * Hkv * D}
    if case["kind"] == "step":
        B = case["B"]
        return {"bytes": B * D * (4 * (Hq + Hkv) + 2 * Hkv + 4) + B * 2 * Hkv * (D + 1) + B * 2 * Hkv * (3 * D + 1),
                "flops": 3 * B * (Hq + Hkv) * D + 2 * B * 2 * Hkv * D}
    n, total = _lengths(case)
    token = 2 * Hkv * (2 * D if case["cache"] == "bf16" else D + 1)
    pairs = sum(a * b - a * (a - 1) // 2 for a, b in zip(n, total))
    return {"bytes": sum(b * token for a, b in zip(n, total) if a) + sum(n) * Hq * D * 4 + sum(-(-b // case["bs"]) * 4 for b in total),
            "flops": 4 * D * Hq * pairs}


# ---------------------------------------------------------------------------------------------------- 8 bits
def _power(e):
    """2^e from the bits of the number."""
    return ((e + 127) << 23).view(torch.float32)


def _quantise(x):
    """(codes, scale bytes) of the vectors along the last dimension of ``x``."""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))
    e = (e - 9 + (m > 0.875).int()).clamp(min=-116)  # 448 = 0.875 * 2^9
    return (x * _power(-e)[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _values(cache, scales, *at):
    """What the vectors at these indices of a cache stand for."""
    if scales is None:
        return cache[at].float()
    codes = cache.view(torch.uint8)[at].view(torch.float8_e4m3fn)
    return codes.float() * _power(scales[at].int() - 127)[..., None]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    plan = torch.Generator(device=DEV).manual_seed(seed + 1)
    Hq, Hkv, D, bs = case["Hq"], case["Hkv"], case["D"], case["bs"]
    i32 = dict(dtype=torch.int32, device=DEV)
    s = dict(case=case, status=torch.zeros(1, **i32))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    if case["kind"] == "cache":
        slots_of = case["T"] + case["R"]
        blocks = -(-slots_of // bs) + 2
    else:
        n, total = _lengths(case)
        per_seq = [-(-t // bs) for t in total]
        blocks = sum(per_seq) + 2
    # what the cache holds: keys with a few strong channels, values with a mean, as layers have them
    strong = 1 + 3 * (torch.rand(Hkv, 1, D, generator=gen, device=DEV) < 0.05)
    caches = [(normal(blocks, Hkv, bs, D) * strong).bfloat16(), (normal(blocks, Hkv, bs, D) + normal(Hkv, 1, D)).bfloat16()]
    s["scales"] = [None, None]
    if case.get("cache", "e4m3") == "e4m3":
        both = [_quantise(c) for c in caches]
        caches, s["scales"] = [b[0] for b in both], [b[1] for b in both]
    s["caches"] = caches
    order = torch.randperm(blocks, generator=plan, device=DEV).int()
    if case["kind"] == "cache":
        T, R = case["T"], case["R"]
        s["qkv"] = normal(T, (Hq + 2 * Hkv) * D).bfloat16()
        s["back"] = torch.zeros(R, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device=DEV)
        at = (order[:, None] * bs + torch.arange(bs, **i32)).reshape(-1)  # slots in the order in which tokens come
        slots = at[:T].clone()
        slots[torch.randperm(T, generator=plan, device=DEV)[:case["skip"]]] = -1  # padding and tokens that are known already
        s["slots"], s["rows"] = slots, torch.nonzero(slots >= 0)[:, 0]
        s["read"] = at[T // 2:T // 2 + R].contiguous()  # the later half of what was written and older tokens
        return s
    if case["kind"] == "step":
        B = case["B"]
        s["rows"] = normal(B, (Hq + 2 * Hkv) * D).bfloat16()
        s["qkv"] = torch.empty_like(s["rows"])
        far = max(total)
        angle = torch.arange(far, device=DEV, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["back"] = torch.zeros_like(s["rows"])
    else:
        Tq = sum(n) + case["pad"]
        s["qkv"] = normal(Tq, (Hq + 2 * Hkv) * D).bfloat16()
        s["out"] = torch.zeros(Tq, Hq * D, dtype=torch.bfloat16, device=DEV)
        s["starts"] = torch.tensor([0] + n, **i32).cumsum(0).int()
        s["n_most"] = max(n)
    s["kv_most"] = max(total)
    s["lens"] = torch.tensor(total, **i32)
    table = torch.zeros(len(total), max(1, max(per_seq)), dtype=torch.int32)
    at = 0
    host = order.cpu()
    for b, k in enumerate(per_seq):
        table[b, :k] = host[at:at + k]
        at += k
    s["table"] = table.to(DEV)
    if case["kind"] == "step":
        last = s["lens"].long() - 1
        s["read"] = (s["table"].gather(1, (last // bs)[:, None])[:, 0] * bs + last % bs).int()
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _write(s, kv, slots):
    """kv [rows, 2 Hkv, D] into the slots."""
    bs, Hkv = s["case"]["bs"], s["case"]["Hkv"]
    codes, scale = _quantise(kv)
    blk, off = slots.long() // bs, slots.long() % bs
    for i, (cache, scales) in enumerate(zip(s["caches"], s["scales"])):
        mine = slice(i * Hkv, (i + 1) * Hkv)
        cache.view(torch.uint8)[blk, :, off] = codes[:, mine].view(torch.uint8)
        scales[blk, :, off] = scale[:, mine]


def _read(s, slots, rows):
    """The slots' values into the key and value columns of the rows."""
    Hq, Hkv, D, bs = (s["case"][k] for k in ("Hq", "Hkv", "D", "bs"))
    blk, off = slots.long() // bs, slots.long() % bs
    out = rows.view(len(slots), Hq + 2 * Hkv, D)
    for i, (cache, scales) in enumerate(zip(s["caches"], s["scales"])):
        out[:, Hq + i * Hkv:Hq + (i + 1) * Hkv] = _values(cache, scales, blk, slice(None), off).bfloat16()


def _plain_step(s):
    Hq, Hkv, D = (s["case"][k] for k in ("Hq", "Hkv", "D"))
    x = s["rows"].view(-1, Hq + 2 * Hkv, D).float()
    pos = s["lens"].long() - 1
    c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]
    a, b = x[:, :Hq + Hkv, :D // 2], x[:, :Hq + Hkv, D // 2:]
    turned = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    s["qkv"].copy_(torch.cat([turned, x[:, Hq + Hkv:]], 1).view_as(s["qkv"]))
    _write(s, s["qkv"].view(-1, Hq + 2 * Hkv, D)[:, Hq:], s["read"])


def _plain_attn(s):
    case = s["case"]
    Hq, Hkv, D, B = case["Hq"], case["Hkv"], case["D"], case["B"]
    n, kv = s["n_most"], s["kv_most"]
    if n == 0 or kv == 0:
        return
    dev = s["qkv"].device
    starts, lens = s["starts"].long(), s["lens"].long()
    count = starts[1:] - starts[:-1]
    i = torch.arange(n, device=dev)
    rows = (starts[:-1, None] + i).clamp(max=len(s["qkv"]) - 1)
    q = s["qkv"][rows, :Hq * D].float().view(B, n, Hkv, Hq // Hkv, D)
    k, v = (_values(c, sc, s["table"].long()).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)[:, :, :kv] for c, sc in zip(s["caches"], s["scales"]))
    last = lens - count  # a row sees the keys up to its own
    see = torch.arange(kv, device=dev) <= (last[:, None] + i)[:, :, None]
    q = (q / math.sqrt(D)).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    z = (q @ k.transpose(2, 3)).view(B, Hkv, Hq // Hkv, n, kv)
    z.masked_fill_(~see[:, None, None], float("-inf"))
    top = z.amax(-1, keepdim=True).clamp_(min=-1e30)
    z.sub_(top).exp_()
    total = z.sum(-1, keepdim=True)
    o = (z.view(B, Hkv, -1, kv) @ v).view(B, Hkv, Hq // Hkv, n, D) / total.clamp_(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, Hq * D).bfloat16()
    there = i < count[:, None]
    s["out"][rows[there]] = o[there]


def run(s):
    case = s["case"]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    (k, v), (ks, vs) = s["caches"], s["scales"]
    if own:
        from async_grpo_nccl_b200.ops import native

        C = native()
    if case["kind"] == "cache":
        if own:
            C.kv_cache_write(s["qkv"], s["slots"], k, v, Hq, Hkv, D, s["status"], 0, ks, vs)
            C.kv_cache_read(k, v, s["read"], s["back"], Hq, Hkv, D, s["status"], ks, vs)
        else:
            _write(s, s["qkv"].view(-1, Hq + 2 * Hkv, D)[s["rows"], Hq:], s["slots"][s["rows"]])
            _read(s, s["read"], s["back"])
        return s["back"][:, Hq * D:]
    if case["kind"] == "step":
        if own:
            s["qkv"].copy_(s["rows"])  # the product before this writes the rows anew in every step
            C.rope_kv_write_decode(s["qkv"], s["cos"], s["sin"], s["table"], s["lens"], k, v, Hq, Hkv, D, s["status"], ks, vs)
            C.kv_cache_read(k, v, s["read"], s["back"], Hq, Hkv, D, s["status"], ks, vs)
        else:
            _plain_step(s)
            _read(s, s["read"], s["back"])
        return s["qkv"], s["back"][:, Hq * D:]
    if own:
        C.paged_chunk_attn(s["qkv"], k, v, s["table"], s["lens"], s["starts"], s["out"], Hq, Hkv, D, 1 / math.sqrt(D), s["status"], ks, vs)
    else:
        _plain_attn(s)
    return s["out"]


# ---------------------------------------------------------------------------------------------------- 64 bits
def _exact_round(x):
    """What a vector of the last dimension reads as from the cache, without float8 types: the grid of 3 mantissa bits by hand."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -116)))
    e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
    e = torch.where((top <= 448 * torch.exp2(e - 1)) & (e > -116), e - 1, e)
    y = x / torch.exp2(e)
    grid = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)  # below 2^-6 the grid stays
    return torch.round(y / grid) * grid * torch.exp2(e)  # half to even


def exact(case, seed):
    s = prepare(case, seed)
    Hq, Hkv, D, bs = case["Hq"], case["Hkv"], case["D"], case["bs"]
    held = [c.double() if sc is None else c.float().double() * torch.exp2(sc.double() - 127)[..., None] for c, sc in zip(s["caches"], s["scales"])]
    if case["kind"] == "cache":
        rows, out = s["qkv"].view(-1, Hq + 2 * Hkv, D), []
        for i, c in enumerate(held):
            flat = c.permute(0, 2, 1, 3).reshape(-1, Hkv, D)
            flat[s["slots"][s["rows"]].long()] = _exact_round(rows[s["rows"], Hq + i * Hkv:Hq + (i + 1) * Hkv])
            out.append(flat[s["read"].long()])
        return torch.cat(out, 1).reshape(case["R"], -1)
    if case["kind"] == "step":
        x = s["rows"].double().view(-1, Hq + 2 * Hkv, D)
        z = torch.complex(x[:, :Hq + Hkv, :D // 2], x[:, :Hq + Hkv, D // 2:])
        pos = s["lens"].long() - 1
        z = z * torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])[:, None]
        # next to a border of the 8-bit grid the last bit of a rotated key decides: no value there
        return torch.cat([torch.cat([z.real, z.imag], -1), x[:, Hq + Hkv:]], 1).view(len(x), -1), None
    out = torch.zeros(len(s["qkv"]), Hq, D, dtype=torch.float64, device=DEV)
    starts, table = s["starts"].tolist(), s["table"].long()
    for b, total in enumerate(s["lens"].tolist()):
        a, z = starts[b], starts[b + 1]
        if z == a or total == 0:
            continue
        pages = table[b, :-(-total // bs)]
        past = torch.arange(z - a, device=DEV)[:, None] + (total - (z - a))
        hidden = torch.arange(total, device=DEV)[None] > past
        for h in range(Hkv):
            k, v = (c[pages, h].reshape(-1, D)[:total] for c in held)
            for g in range(h * Hq // Hkv, (h + 1) * Hq // Hkv):
                w = s["qkv"][a:z, g * D:(g + 1) * D].double() @ k.T * D ** -0.5
                out[a:z, g] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v
    return out.view(len(out), -1)
