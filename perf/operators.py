"""Cases of the paged KV cache's operators: append with rotation, decode attention, gather.

A cache is a pool of pages; a page holds ``page`` tokens of every KV head. A sequence's tokens
lie in the pages that its row of the page table names, in order. Two forms of a page:

- ``bf16``: the rotated keys and the values as they are;
- ``int4``: four bits an element. Keys: groups of 32 along the head dim, value = (code - 8) * s
  with a bf16 scale s = bf16(amax / 7). Values: the same groups, value = (code - 8) * r * 2^e
  with one exponent e a token and head, e = floor(log2(amax of the row / 7)), and fp16 scales
  r = fp16(amax of the group / 7 * 2^-e). code = round-half-even(x / scale) + 8, in 1 .. 15.

The bytes of a page and head are 16-token granules, laid out for the attention kernel's
registers: ``_pack`` writes that layout, ``_unpack`` reads it back, and ``exact`` reads it by
its own byte addresses.

Positions: row i of sequence b stands at ``starts[b] + i`` for i < ``counts[b]``; rows behind
that are padding, and a sequence with a negative start is inactive. Attention is causal: a row
sees the cached tokens up to and with its own position.
"""

import math
import random

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
GRANULE = 16


# ------------------------------------------------------------------------------- the cases


def listed():
    return [
        # One user's chat, an early token of the answer: latency of a single short sequence.
        dict(name="attend int4 short", op="attend", form="int4", batch=1, heads=28, kv_heads=4, dim=128, page=64,
             rows=1, longest=512, shortest=512),
        # The full-model prompt of the benchmark, decoded one token at a time.
        dict(name="attend int4 prompt 32640", op="attend", form="int4", batch=1, heads=28, kv_heads=4, dim=128,
             page=64, rows=1, longest=32641, shortest=32641),
        # The longest layer configuration.
        dict(name="attend int4 128K", op="attend", form="int4", batch=1, heads=28, kv_heads=4, dim=128, page=128,
             rows=1, longest=131072, shortest=131072),
        # A server's batch: sequences of all lengths, one token each.
        dict(name="attend int4 batch 32 ragged", op="attend", form="int4", batch=32, heads=28, kv_heads=4, dim=128,
             page=64, rows=1, longest=32768, shortest=4096),
        # The 40-head layer of two long sequences with a cache that is kept in bf16.
        dict(name="attend bf16 2 x 64K", op="attend", form="bf16", batch=2, heads=40, kv_heads=8, dim=128, page=32,
             rows=1, longest=65536, shortest=65536),
        # Head dim 256, five drafted tokens a sequence checked in one call, small pages, odd lengths.
        dict(name="attend int4 d256 verify 5", op="attend", form="int4", batch=4, heads=16, kv_heads=4, dim=256,
             page=16, rows=5, longest=9173, shortest=1031),
        # A decode step's new tokens of a batch: a few rows, latency.
        dict(name="append int4 step of 64", op="append", form="int4", batch=64, heads=28, kv_heads=4, dim=128,
             page=64, rows=1, longest=4096, shortest=1, rotary=128),
        # A whole prompt into the cache.
        dict(name="append int4 prompt 32640", op="append", form="int4", batch=1, heads=28, kv_heads=4, dim=128,
             page=64, rows=32640, longest=32640, shortest=32640, rotary=128),
        # A padded batch of prompts, head dim 256 with a rotation of its first quarter.
        dict(name="append bf16 d256 padded", op="append", form="bf16", batch=3, heads=16, kv_heads=4, dim=256,
             page=16, rows=4097, longest=5000, shortest=3001, rotary=64),
        # A cached prefix read back for the prefill of a follow-up prompt.
        dict(name="gather int4 prefix 32768", op="gather", form="int4", batch=1, heads=28, kv_heads=4, dim=128,
             page=64, rows=32768, longest=32768, shortest=32768),
        # Prefixes of a ragged batch out of bf16 pages.
        dict(name="gather bf16 batch 8 ragged", op="gather", form="bf16", batch=8, heads=40, kv_heads=8, dim=128,
             page=32, rows=4095, longest=4095, shortest=97),
    ]


def draw(rng: random.Random):
    """One more case: any operator and form, head layouts of the configurations and of their tensor-parallel
    shards, lengths over their logarithm; no more cached rows than the largest listed case pads to."""
    op = rng.choice(["attend", "attend", "append", "gather"])
    heads, kv_heads, dim = rng.choice([(28, 4, 128), (40, 8, 128), (16, 4, 256), (7, 1, 128), (4, 1, 128),
                                       (12, 2, 128), (16, 1, 128)])
    log = lambda lo, hi: min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))  # noqa: E731
    batch, form = log(1, 64), rng.choice(["int4", "int4", "bf16"])
    case = dict(op=op, form=form, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128]),
                batch=batch)
    # token rows of one KV head at head dim 128, so that the bytes stay below the largest listed case's
    most = {"attend": 3500000 // (4 if form == "bf16" else 1), "gather": 500000, "append": 20000 * kv_heads}[op]
    most //= kv_heads * (dim // 128)
    if op == "attend":
        case["rows"] = rng.choice([1, 1, 1, 2, 3, 4, 8])
        case["longest"] = log(16, max(16, min(131072, most // batch // case["rows"])))
        case["shortest"] = rng.randint(case["rows"], max(case["rows"], case["longest"]))
        case["longest"] = max(case["longest"], case["shortest"])
    else:
        case["longest"] = log(1, min(32768, most // batch))
        case["shortest"] = rng.randint(1, case["longest"])
        case["rows"] = case["longest"] if rng.random() < 0.5 else rng.randint(1, case["longest"])
        if op == "append":
            case["rotary"] = rng.choice([dim, dim, dim // 2, dim // 4])
    return case


def _lengths(case):
    """Tokens in the cache after the call, a sequence each: from the case alone, so that the work is its own."""
    r = random.Random(case["batch"] * 1000003 + case["longest"] * 31 + case["shortest"])
    got = [r.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
    got[0] = case["longest"]
    return got


def _counts(case):
    return [min(n, case["rows"]) for n in _lengths(case)]


def _row_bytes(case):
    """Bytes of one token of one KV head in the pool: K and V."""
    return 4 * case["dim"] if case["form"] == "bf16" else 9 * case["dim"] // 8 + 2


def work(case):
    b, h, g, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    lengths, counts = _lengths(case), _counts(case)
    new = sum(counts)
    if case["op"] == "attend":
        table = 4 * sum(-(-n // case["page"]) for n in lengths)
        seen = sum(c * n - c * (c - 1) // 2 for n, c in zip(lengths, counts))
        return {"bytes": sum(lengths) * g * _row_bytes(case) + 2 * 2 * new * h * d + table, "flops": 4 * d * h * seen}
    if case["op"] == "append":
        # q, k and v in; q rotated, the cached rows, and their values (read from the cache) out
        read = new * (h + 2 * g) * d * 2 + new * case["rotary"] * 4
        return {"bytes": read + new * h * d * 2 + 2 * new * g * _row_bytes(case) + new * 2 * g * d * 2,
                "flops": 3 * new * (h + g) * case["rotary"] + 4 * new * g * d}
    return {"bytes": new * g * _row_bytes(case) + new * 2 * g * d * 2, "flops": 2 * new * g * d}


# ------------------------------------------------------------------------------ the inputs


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _rope(positions, rotary, theta=1e6):
    """[positions, rotary] fp32: cosines, then sines, of position * theta^(-2i / rotary); angles in 64 bits."""
    inv = theta ** (-torch.arange(0, rotary, 2, device=DEV, dtype=torch.float64) / rotary)
    ang = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * inv
    return torch.cat((ang.cos(), ang.sin()), 1).float()


def prepare(case, seed):
    g = _generator(seed)
    b, h, kv, d, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    lengths, counts = _lengths(case), _counts(case)
    pages = -(-case["longest"] // page)
    order = torch.randperm(b * pages + 3, generator=g, device=DEV)[: b * pages]  # pages as an allocator leaves them
    table = order.view(b, pages).to(torch.int32).contiguous()
    starts = torch.tensor([n - c for n, c in zip(lengths, counts)], dtype=torch.int32, device=DEV)
    count = torch.tensor(counts, dtype=torch.int32, device=DEV)
    if case["form"] == "int4":  # what no sequence has written yet is whatever the memory held
        pool = torch.full((b * pages + 3, kv, page, _row_bytes(case)), 255, dtype=torch.uint8, device=DEV)
    else:
        pool = torch.full((b * pages + 3, kv, page, 2 * d), float("nan"), dtype=torch.bfloat16, device=DEV)
    state = dict(case=case, pool=pool, table=table, starts=starts, counts=count, scale=d ** -0.5)
    if case["op"] != "append":
        # keys whose channels differ in size and have an offset, as trained projections give them
        size = 0.5 + torch.rand(d, generator=g, device=DEV)
        shift = 0.5 * _randn(g, kv, 1, d)
        for i in range(b):
            n = -(-lengths[i] // page) * page
            k = (_randn(g, kv, n, d) * size + shift).to(torch.bfloat16)
            v = _randn(g, kv, n, d).to(torch.bfloat16)
            rows = _pack(case, k, v).view(kv, n // page, -1).transpose(0, 1)
            live = (torch.arange(n, device=DEV) < lengths[i]).view(-1, 1, page)
            del k, v
            pool[table[i, : n // page].long()] = _masked_granules(case, rows, live)
    if case["op"] == "attend":
        state["q"] = _randn(g, b, case["rows"], h, d).to(torch.bfloat16)
    if case["op"] == "append":
        qkv = _randn(g, b, case["rows"], (h + 2 * kv) * d).to(torch.bfloat16)  # a fused projection's output
        state["q"] = qkv[..., : h * d].view(b, -1, h, d)
        state["k"] = qkv[..., h * d:(h + kv) * d].view(b, -1, kv, d)
        state["v"] = qkv[..., (h + kv) * d:].view(b, -1, kv, d)
        state["rope"] = _rope(case["longest"], case["rotary"])
    return state


def _masked_granules(case, rows, live):
    """The packed pages [pages, kv, bytes or elements] in the pool's shape, whole granules behind a sequence's end
    left as unwritten memory."""
    pages, kv, page = rows.shape[0], rows.shape[1], case["page"]
    rows = rows.reshape(pages, kv, page // GRANULE, -1)
    keep = live.view(pages, 1, page // GRANULE, GRANULE).any(-1, keepdim=True)
    blank = torch.full_like(rows[:1, :1, :1], 255 if rows.dtype == torch.uint8 else float("nan"))
    return torch.where(keep, rows, blank).view(pages, kv, page, -1)


# ---------------------------------------------------------------------------- the 4-bit form


def _quantise_k(x):
    """x fp32 [..., d] -> codes 1 .. 15 (uint8), scales bf16 [..., d / 32]."""
    x = x.unflatten(-1, (-1, 32))
    seven = torch.full((), 7.0, device=x.device)
    s = (x.abs().amax(-1) / seven).to(torch.bfloat16)
    return _codes(x, s.float()[..., None]).flatten(-2), s


def _quantise_v(x):
    """x fp32 [..., d] -> codes, scales fp16 [..., d / 32], exponents int32 [...]."""
    x = x.unflatten(-1, (-1, 32))
    seven = torch.full((), 7.0, device=x.device)
    amax = x.abs().amax(-1) / seven
    top = amax.amax(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 1, -60).clamp(-60, 126).to(torch.int32)
    r = (amax * _two(-e[..., None])).to(torch.float16)
    return _codes(x, (r.float() * _two(e[..., None]))[..., None]).flatten(-2), r, e


def _two(e):
    """2^e in fp32 for int32 e in -126 .. 127, by its bits."""
    return ((e + 127) << 23).view(torch.float32)


def _codes(x, s):
    return (torch.where(s > 0, torch.round(x / s), torch.zeros_like(x)).clamp(-7, 7) + 8).to(torch.uint8)


def _chunk_order(device):
    """[8, 8]: the 16-byte chunk of value codes that lies at place c of token pair q is c ^ 2 (q mod 4)."""
    q = torch.arange(8, device=device)
    return q[None] ^ (2 * (q % 4))[:, None]


def _pack(case, k, v):
    """k, v bf16 or fp32 [kv, n, d], n a multiple of 16 -> granules [kv, n / 16, bytes or elements]."""
    kv, n, d = k.shape
    if case["form"] == "bf16":  # rows of 16-byte chunks, chunk c of row r at place c ^ (r mod 8); K beside V
        c, r = torch.arange(d // 8, device=k.device), torch.arange(GRANULE, device=k.device)
        place = (c[None] ^ (r % 8)[:, None])
        both = torch.stack((k, v), 2).to(torch.bfloat16).view(kv, n // GRANULE, GRANULE, 2, d // 8, 8)
        return both[:, :, r[:, None], :, place].permute(2, 3, 0, 4, 1, 5).reshape(kv, n // GRANULE, -1)
    kc, ks = _quantise_k(k.float())
    vc, vr, ve = _quantise_v(v.float())
    half = d // 128
    kb = (kc[..., 0::2] + 16 * kc[..., 1::2]).view(kv, -1, GRANULE, half, 4, 4, 4)  # half, group, word, byte
    kb = kb.transpose(4, 5).reshape(kv, -1, GRANULE * d // 2)
    vb = (vc[..., 0::2] + 16 * vc[..., 1::2]).view(kv, -1, 8, 2, half, 4, 8, 2)     # pair, of pair, half, group, chunk, byte
    vb = vb.permute(0, 1, 4, 2, 6, 3, 5, 7)                                           # half, pair, chunk, of pair, group, byte
    vb = vb[:, :, :, torch.arange(8, device=k.device)[:, None], _chunk_order(k.device)].reshape(kv, -1, GRANULE * d // 2)
    ks = ks.view(torch.uint8).reshape(kv, -1, GRANULE * d // 16)
    vs = vr.view(kv, -1, 8, 2, d // 32).transpose(3, 4).contiguous().view(torch.uint8).reshape(kv, -1, GRANULE * d // 16)
    ve = ve.to(torch.bfloat16).contiguous().view(torch.uint8).reshape(kv, -1, GRANULE * 2)
    return torch.cat((kb, vb, ks, vs, ve), -1)


def _unpack(case, pages):
    """Pool rows [..., page, bytes or elements] -> k, v fp32 [..., page, d]."""
    d, lead = case["dim"], pages.shape[:-2]
    if case["form"] == "bf16":
        c, r = torch.arange(d // 8, device=pages.device), torch.arange(GRANULE, device=pages.device)
        place = (c[None] ^ (r % 8)[:, None])
        g = pages.reshape(-1, GRANULE, 2, d // 8, 8)
        g = g[:, r[:, None], :, place].permute(2, 0, 3, 1, 4).reshape(*lead, -1, 2, d).float()
        return g[..., 0, :], g[..., 1, :]
    half = d // 128
    g = pages.reshape(-1, GRANULE * (9 * d // 8 + 2))
    kb, vb, ks, vs, ve = g.split([GRANULE * d // 2, GRANULE * d // 2, GRANULE * d // 16, GRANULE * d // 16, 32], -1)
    kb = kb.reshape(-1, GRANULE, half, 4, 4, 4).transpose(3, 4)
    vb = vb.reshape(-1, half, 8, 8, 2, 4, 2)[:, :, torch.arange(8, device=g.device)[:, None], _chunk_order(g.device)]
    vb = vb.permute(0, 2, 4, 1, 5, 3, 6)
    nibbles = lambda x: torch.stack((x & 15, x >> 4), -1).reshape(-1, GRANULE, d // 32, 32).float() - 8  # noqa: E731
    ks = ks.contiguous().view(torch.bfloat16).view(-1, GRANULE, d // 32, 1).float()
    vr = vs.contiguous().view(torch.float16).view(-1, 8, d // 32, 2).transpose(2, 3).reshape(-1, GRANULE, d // 32, 1)
    ve = ve.contiguous().view(torch.bfloat16).view(-1, GRANULE, 1, 1).float()
    k = nibbles(kb) * ks
    v = nibbles(vb) * (vr.float() * _two(ve.to(torch.int32)))
    return k.reshape(*lead, -1, d), v.reshape(*lead, -1, d)


# --------------------------------------------------------------------------- the operators


def run(state):
    case = state["case"]
    if own:
        from exp3_b200 import paged
        where = (state["pool"], state["table"], state["starts"])
        if case["op"] == "attend":
            return paged.paged_decode_attention(state["q"], *where, state["scale"], counts=state["counts"])
        if case["op"] == "gather":
            return paged.paged_gather(*where, state["counts"], case["rows"])
        q = paged.paged_append(state["k"], state["v"], *where, counts=state["counts"], q=state["q"],
                               rope=state["rope"])
        return q, *paged.paged_gather(*where, state["counts"], case["rows"])
    if case["op"] == "attend":
        return _attend(state)
    if case["op"] == "gather":
        return _gather(state)
    return _append(state)


def _at(state):
    """Positions [B, rows] of the call's rows, and which of them are no padding."""
    i = torch.arange(state["case"]["rows"], device=DEV)
    return state["starts"][:, None] + i, i < state["counts"][:, None]


def _cached(state):
    """The sequences' pages as k, v fp32 [B, kv, tokens, d]."""
    rows = state["pool"][state["table"].long()].transpose(1, 2)  # [B, kv, pages, page, row]
    k, v = _unpack(state["case"], rows)
    return k.flatten(2, 3), v.flatten(2, 3)


def _attend(state):
    case, q = state["case"], state["q"].float()
    b, rows, h, d = q.shape
    k, v = _cached(state)
    pos, valid = _at(state)
    seen = (torch.arange(k.shape[2], device=DEV) <= pos[..., None]) & valid[..., None]  # [B, rows, tokens]
    any_row = seen.any(1)[:, None, :, None]
    k, v = torch.where(any_row, k, 0.0), torch.where(any_row, v, 0.0)  # what no row sees may be NaN
    q = q.view(b, rows, case["kv_heads"], -1, d).permute(0, 2, 1, 3, 4).reshape(b, case["kv_heads"], -1, d)
    s = (q @ k.transpose(2, 3)).view(b, case["kv_heads"], rows, -1, k.shape[2]) * state["scale"]
    s = s.masked_fill(~seen[:, None, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
    l = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).view(b, case["kv_heads"], rows, -1, d)
    o = torch.where(l > 0, o / l, 0.0)
    return o.permute(0, 2, 1, 3, 4).reshape(b, rows, h, d).to(torch.bfloat16)


def _gather(state):
    pos, valid = _at(state)
    k, v = _cached(state)
    at = torch.where(valid, pos, 0).long()[:, None, :, None].expand(-1, k.shape[1], -1, k.shape[3])
    pick = lambda x: torch.where(valid[:, :, None, None], x.gather(2, at).transpose(1, 2), 0.0).to(torch.bfloat16)  # noqa: E731
    return pick(k), pick(v)


def _rotate(x, rope, rotary):
    """x fp32 [B, rows, heads, d], rope [B, rows, rotary]."""
    half = rotary // 2
    c, s = rope[:, :, None, :half], rope[:, :, None, half:]
    a, b = x[..., :half], x[..., half:rotary]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., rotary:]), -1)


def _append(state):
    case = state["case"]
    pos, valid = _at(state)
    rope = state["rope"][torch.where(valid, pos, 0).long()]
    q = _rotate(state["q"].float(), rope, case["rotary"])
    k = _rotate(state["k"].float(), rope, case["rotary"])
    v = state["v"].float()
    if case["form"] == "int4":
        c, s = _quantise_k(k)
        k = ((c.float() - 8).unflatten(-1, (-1, 32)) * s.float()[..., None]).flatten(-2)
        c, r, e = _quantise_v(v)
        v = ((c.float() - 8).unflatten(-1, (-1, 32)) * (r.float() * _two(e[..., None]))[..., None]).flatten(-2)
    out = lambda x: torch.where(valid[:, :, None, None], x, 0.0).to(torch.bfloat16)  # noqa: E731
    return out(q), out(k), out(v)


# ----------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, state)
    if case["op"] == "gather":
        return _exact_gather(case, state)
    return _exact_attend(case, state)


def _exact_rows(case, state, i, head, first, n):
    """K and V of tokens first .. first + n - 1 of sequence i, one KV head, in 64 bits, by byte addresses."""
    d, page, dev = case["dim"], case["page"], state["pool"].device
    at = torch.arange(first, first + n, device=dev)
    number = state["table"][i].long()[at // page]
    within, t = (at % page) // GRANULE, at % GRANULE
    x = torch.arange(d, device=dev)[None]
    t, within = t[:, None], within[:, None]
    flat = state["pool"][:, head].reshape(state["pool"].shape[0], -1)
    look = lambda a: flat[number[:, None].expand_as(a), a]  # noqa: E731
    if case["form"] == "bf16":
        base = within * GRANULE * 2 * d + t * 2 * d
        a = ((x // 8) ^ (t % 8)) * 8 + x % 8  # K and V of one row lie side by side
        return look(base + a).double(), look(base + d + a).double()
    base = within * GRANULE * (9 * d // 8 + 2)
    hi, group, rest = x // 128, (x % 128) // 32, x % 32
    nibble = lambda a, odd: ((look(a).long() >> (4 * odd)) & 15).double() - 8  # noqa: E731
    k_at = base + t * (d // 2) + hi * 64 + (rest // 8) * 16 + group * 4 + (rest % 8) // 2
    pair = t // 2
    v_at = (base + GRANULE * (d // 2) + hi * 1024 + pair * 128 + ((rest // 4) ^ (2 * (pair % 4))) * 16 + (t % 2) * 8
            + group * 2 + (rest % 4) // 2)
    j = x // 32
    two = lambda a: look(a).long() + 256 * look(a + 1).long()  # noqa: E731
    bf16 = lambda u: (u << 16).to(torch.int32).view(torch.float32).double()  # noqa: E731
    ks = bf16(two(base + GRANULE * d + (t * (d // 32) + j) * 2))
    vs = two(base + GRANULE * d + GRANULE * (d // 16) + ((pair * (d // 32) + j) * 2 + t % 2) * 2)
    vs = vs.to(torch.int16).view(torch.float16).double()
    ve = bf16(two(base + GRANULE * d + 2 * GRANULE * (d // 16) + 2 * t))
    return nibble(k_at, x % 2) * ks, nibble(v_at, x % 2) * vs * 2.0 ** ve


def _exact_attend(case, state):
    starts, counts = state["starts"].tolist(), state["counts"].tolist()
    q = state["q"].double()
    out = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    for i in range(case["batch"]):
        n = starts[i] + counts[i]
        for g in range(case["kv_heads"]):
            mine = slice(g * group, (g + 1) * group)
            most = torch.full((counts[i], group, 1), -math.inf, dtype=torch.float64, device=DEV)
            total, acc = torch.zeros_like(most), torch.zeros(counts[i], group, case["dim"], dtype=torch.float64, device=DEV)
            for first in range(0, n, 65536):
                k, v = _exact_rows(case, state, i, g, first, min(65536, n - first))
                s = torch.einsum("rhd,td->rht", q[i, : counts[i], mine], k) * state["scale"]
                t = torch.arange(first, first + k.shape[0], device=DEV)
                limit = starts[i] + torch.arange(counts[i], device=DEV)
                s = s.masked_fill(t > limit[:, None, None], -math.inf)
                new = torch.maximum(most, s.amax(-1, keepdim=True))
                keep = torch.exp(most - new)
                p = torch.exp(s - new)
                total = total * keep + p.sum(-1, keepdim=True)
                acc = acc * keep + torch.einsum("rht,td->rhd", p, v)
                most = new
            out[i, : counts[i], mine] = acc / total
    return out


def _exact_gather(case, state):
    if case["batch"] * case["kv_heads"] > 512:
        return None
    starts, counts = state["starts"].tolist(), state["counts"].tolist()
    shape = (case["batch"], case["rows"], case["kv_heads"], case["dim"])
    k, v = (torch.zeros(shape, dtype=torch.float64, device=DEV) for _ in range(2))
    for i in range(case["batch"]):
        for g in range(case["kv_heads"]):
            k[i, : counts[i], g], v[i, : counts[i], g] = _exact_rows(case, state, i, g, starts[i], counts[i])
    return k, v


def _exact_append(case, state):
    b, rows, half = case["batch"], case["rows"], case["rotary"] // 2
    counts = state["counts"][:, None]
    live = (torch.arange(rows, device=DEV)[None] < counts)[..., None, None]
    pos = (state["starts"][:, None] + torch.arange(rows, device=DEV)).clamp(max=case["longest"] - 1).long()
    table = state["rope"].double()[pos][:, :, None]

    def turned(x):
        z = torch.complex(x[..., :half].double(), x[..., half:2 * half].double())
        z = z * torch.complex(table[..., :half], table[..., half:])
        return torch.cat((z.real, z.imag, x[..., 2 * half:].double()), -1)

    q, k, v = turned(state["q"]), turned(state["k"]), state["v"].double()
    if case["form"] == "int4":
        x = k.reshape(b, rows, case["kv_heads"], -1, 32)
        s = (x.abs().amax(-1, keepdim=True) / 7).float().to(torch.bfloat16).double()
        k = (torch.round(x / s).nan_to_num() * s).view_as(k)
        x = v.reshape(b, rows, case["kv_heads"], -1, 32)
        size = x.abs().amax(-1, keepdim=True) / 7
        e = torch.floor(torch.log2(size.amax(-2, keepdim=True))).clamp(-60, 126)
        s = (size * 2.0 ** -e).float().to(torch.float16).double() * 2.0 ** e
        v = (torch.round(x / s).nan_to_num() * s).view_as(v)
    return tuple(torch.where(live, x, 0.0) for x in (q, k, v))
