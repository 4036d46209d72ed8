"""Rotary positions and a paged cache held in 8 bits: the cases that are measured, their inputs, one pass as a caller's program makes
it, the same in plain torch operations, and what a pass cannot do without.

A case is a dict of plain values.  `op` says what it is:

  rotary   functional.rotary without gradients: queries and keys turned by their positions
  turn     functional.rotary, forward and torch.autograd backward
  store    capi.kv_store into 8 bits and capi.kv_load of all that the sequences hold then, as a piece of a prompt needs it
  load     capi.kv_load alone: what sequences hold, from 8 bits to packed bf16 rows
  decode   functional.sdpa_paged on 8 bits: one or a few new tokens per sequence, a prefix shared by the batch or none

Lengths are texts of numbers with commas between them.  Eight bits are "int8" (codes from -127 to 127) or "e4m3" (largest value 448);
a code stands for code * scale, with a scale for every `block` tokens of a head.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}
LEAST = 2.0 ** -100                 # of the scales


# ---------------------------------------------------------------------------------------------------------------- cases
def _text(lens):
    return ",".join(str(n) for n in lens)


def _lens(text):
    return [int(n) for n in text.split(",")]


def _rotary(name, form, H, Hkv, D, turned, lens, start, op="rotary", dtype="bf16", interleaved=False, base=10000.0, scaling="none", factor=1.0,
            original=4096):
    """form: "packed", rows of sequences by their bounds and first positions; "rows", a position for every row; "batch",
    [B, H, S, D] with a position for every token."""
    return dict(name=name, op=op, form=form, H=H, Hkv=Hkv, D=D, turned=turned, lens=_text(lens), start=_text(start), dtype=dtype, interleaved=interleaved,
                base=base, scaling=scaling, factor=factor, original=original)


def _pages(name, op, code, Hkv, D, page, block, lens, start=None):
    """lens: rows that are stored (store) or held (load); start: tokens that each sequence holds before."""
    return dict(name=name, op=op, code=code, Hkv=Hkv, D=D, page=page, block=block, lens=_text(lens), start=_text(start or [0] * len(lens)))


def _decode(name, code, H, Hkv, D, page, block, new, prefix, lens):
    return dict(name=name, op="decode", code=code, H=H, Hkv=Hkv, D=D, page=page, block=block, new=new, prefix=prefix, lens=_text(lens))


def listed():
    return [
        # a token of each of 64 sequences, far positions of a stretched range: a launch's time decides
        _rotary("rotary_step", "rows", 32, 8, 128, 128, [1] * 64, [(7919 * i) % 120000 for i in range(64)], base=500000.0, scaling="yarn", factor=32.0),
        # joint attention at a head dim of 96, of which 64 are turned, in 32 bits, neighbours in pairs
        _rotary("rotary_part_fp32", "batch", 12, 12, 96, 64, [1024] * 2, [0, 333], dtype="fp32", interleaved=True),
        # prompts of a serving batch and the next pieces of others
        _rotary("rotary_prompts", "packed", 32, 8, 128, 128, [4096, 513, 2049, 77, 1024, 3333, 1, 1500], [0, 8192, 0, 5, 64, 0, 40000, 0]),
        # training on packed documents
        _rotary("turn_packed", "packed", 32, 8, 128, 128, [4096, 1101, 2049, 333, 4608, 1024], [0] * 6, op="turn"),
        # new tokens of many short sequences, one to four each, in the middle of their blocks
        _pages("store_tokens", "store", "e4m3", 8, 128, 16, 16, [1 + i % 4 for i in range(64)], [(37 * i) % 61 for i in range(64)]),
        # pieces of prompts behind what is there already
        _pages("store_prompt", "store", "int8", 8, 128, 64, 32, [4096, 513, 2049, 77, 1024], [0, 5, 64, 1000, 17]),
        # short sequences with a scale for every token
        _pages("load_short", "load", "int8", 4, 64, 16, 1, [300, 1, 77, 16, 129, 512]),
        # long contexts for the packed attention of their next pieces
        _pages("load_long", "load", "e4m3", 8, 128, 64, 16, [8192, 2560, 5001, 16384, 333]),
        # a step of few sequences: latency decides
        _decode("decode_few", "int8", 32, 8, 128, 16, 16, 1, 0, [300, 1024, 77, 611]),
        # a serving batch: the largest case
        _decode("decode_batch", "e4m3", 32, 8, 128, 64, 16, 1, 0, [2000 + (1237 * i) % 4001 for i in range(64)]),
        # many answers to one long prompt: the prefix is common to all of them
        _decode("decode_shared_prefix", "int8", 32, 8, 128, 64, 64, 1, 8192, [(97 * i) % 509 + 1 for i in range(64)]),
        # long contexts, four drafted tokens each, a scale for every token, a head dim of 64
        _decode("decode_long", "int8", 16, 4, 64, 128, 1, 4, 0, [32000, 24577, 40000, 16385, 28001, 36000, 20000, 31999]),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, most=32):
    while True:
        hkv, g = rng.choice([1, 2, 3, 4, 8, 12]), rng.choice([1, 2, 3, 4, 6, 8])
        if hkv * g <= most:
            return hkv * g, hkv


def draw(rng: random.Random):
    op = rng.choice(["rotary", "rotary", "turn", "store", "store", "load", "decode", "decode", "decode"])
    if op in ("rotary", "turn"):
        H, Hkv = _heads(rng)
        D = rng.choice([64, 128]) if rng.random() < 0.5 else 2 * rng.randint(8, 96)
        turned = D if rng.random() < 0.6 else 2 * rng.randint(2, D // 2)
        n, longest = _log(rng, 1, 64), _log(rng, 1, 4608)
        while n * longest * (H + Hkv) * D > 13000 * 40 * 128:
            n, longest = max(1, n - 1), max(1, int(longest * 0.9))
        form = rng.choice(["packed", "rows", "batch"])
        lens = [longest] * n if form == "batch" else [max(1, int(longest * rng.random())) for _ in range(n)]
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if dtype == "fp32" and n > 1 and form != "batch":
            lens = lens[:(n + 1) // 2]
        elif dtype == "fp32":
            lens = [-(-m // 2) for m in lens]
        scaling = rng.choice(["none", "linear", "ntk", "yarn", "bands"])
        return dict(op=op, form=form, H=H, Hkv=Hkv, D=D, turned=turned, lens=_text(lens), start=_text([_log(rng, 1, 1000000) - 1 for _ in lens]), dtype=dtype,
                    interleaved=rng.random() < 0.5, base=rng.choice([10000.0, 500000.0]), scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0]), original=rng.choice([2048, 4096, 8192]))
    code, page = rng.choice(["int8", "e4m3"]), rng.choice([16, 32, 64, 128])
    block = 2 ** rng.randint(0, page.bit_length() - 1)
    D = rng.choice([64, 128]) if rng.random() < 0.6 else 16 * rng.randint(2, 8)
    if op == "decode":
        H, Hkv = _heads(rng)
        new = rng.choice([1, 1, 1, 2, 4, 7])
        B, longest = _log(rng, 1, 96), _log(rng, 16, 32000)
        while B * longest * Hkv * D > 64 * 4000 * 8 * 128:
            B, longest = max(1, B - 1), int(longest * 0.9)
        lens = [max(new, int(longest * rng.uniform(0.2, 1.0))) for _ in range(B)]
        prefix = page * (_log(rng, page, 16384) // page) if rng.random() < 0.5 else 0
        return dict(op=op, code=code, H=H, Hkv=Hkv, D=D, page=page, block=block, new=new, prefix=prefix, lens=_text(lens))
    n, most, Hkv = _log(rng, 1, 64), _log(rng, 1, 4096), rng.choice([1, 2, 4, 8])
    while n * most > 40000:
        n, most = max(1, n - 1), int(most * 0.9)
    lens = [max(1, int(most * rng.random())) for _ in range(n)]
    start = [_log(rng, 1, 400) - 1 for _ in lens] if op == "store" else [0] * n
    return dict(op=op, code=code, Hkv=Hkv, D=D, page=page, block=block, lens=_text(lens), start=_text(start))


# --------------------------------------------------------------------------------------------------------------- inputs
def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _bounds(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return _ints(at)


def _table(rng, lens, page, spare=3):
    """Pages of every sequence in no order, as after some time of taking and freeing: (table, pages of the cache)."""
    need = [max(1, -(-n // page)) for n in lens]
    places = list(range(sum(need) + spare))
    rng.shuffle(places)
    rows, at = [], 0
    for n in need:
        rows.append(places[at:at + n] + [0] * (max(need) - n))
        at += n
    return _ints(rows), len(places)


def _tokens(g, *shape):
    """Keys or values as they come: some channels larger than the others, tokens of different magnitude.  shape: [..., heads, D]"""
    wide = 1.0 + 7.0 * (torch.rand(shape[-2:], device="cuda", generator=g) < 0.03)
    size = torch.exp(0.4 * _randn(g, *shape[:-1], 1))
    return _randn(g, *shape) * wide * size


def _cache(g, case, pages):
    """(codes [pages, Hkv, page, D], scales [pages, Hkv, page / block]) of a cache in use"""
    Hkv, page, D, block, code = (case[n] for n in ("Hkv", "page", "D", "block", "code"))
    x = _tokens(g, pages, page, Hkv, D).transpose(1, 2).reshape(pages, Hkv, page // block, block, D)
    scale = _round_up(x.abs().amax((-1, -2)) / LARGEST[code])
    x = (x / scale[..., None, None]).reshape(pages, Hkv, page, D)
    return (torch.round(x) if code == "int8" else x).to(CODES[code]), scale


def _frequencies(case):
    """(radians per position of every pair, what the result is multiplied with)"""
    R, base, factor, original, kind = (case[n] for n in ("turned", "base", "factor", "original", "scaling"))
    if kind == "ntk" and R > 2:
        base = base * factor ** (R / (R - 2))
    f = [base ** (-2.0 * i / R) for i in range(R // 2)]
    if kind == "linear":
        return [x / factor for x in f], 1.0
    if kind == "yarn":              # pairs that turn often keep their pace, those that turn less than once are slowed down
        lo, hi = (R * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(base)) for turns in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), R - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for i in range(R // 2)]
        return [x / factor * r + x * (1.0 - r) for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1.0
    if kind == "bands":             # the same by wave lengths: a quarter of the range and shorter, all of it and longer
        smooth = [min(max((original * x / (2.0 * math.pi) - 1.0) / 3.0, 0.0), 1.0) for x in f]
        return [x / factor * (1.0 - s) + x * s for x, s in zip(f, smooth)], 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    op, D, lens = case["op"], case["D"], _lens(case["lens"])
    st = {"case": case}
    if op in ("rotary", "turn"):
        start, dt = _lens(case["start"]), DTYPES[case["dtype"]]
        if case["form"] == "batch":
            lead, shape = len(lens), lambda H: (len(lens), H, lens[0], D)
            st["positions"] = _ints([list(range(a, a + n)) for a, n in zip(start, lens)])
        else:
            lead, shape = sum(lens), lambda H: (lead, H, D)
            if case["form"] == "packed":
                st.update(cu=_bounds(lens), start=_ints(start))
            else:
                st["positions"] = _ints([p for a, n in zip(start, lens) for p in range(a, a + n)])
        for name, H in (("q", case["H"]), ("k", case["Hkv"])):
            st[name] = _randn(g, *shape(H)).to(dt)
            if op == "turn":
                st["d" + name] = _randn(g, *shape(H)).to(dt)
                st[name].requires_grad_(True)
        if own:
            from flame_amd.rotary import Rotary
            st["rope"] = Rotary(D, base=case["base"], rotary_dim=case["turned"], interleaved=case["interleaved"],
                                scaling=None if case["scaling"] == "none" else case["scaling"], factor=case["factor"], original_length=case["original"])
        else:
            f, st["size"] = _frequencies(case)
            st["f"] = torch.tensor(f, dtype=torch.float64, device="cuda")
        return st
    if op == "decode":
        page, prefix = case["page"], case["prefix"]
        both, n_pages = _table(rng, [prefix] + lens, page)
        st.update(kv_len=_ints(lens), q=_randn(g, len(lens), case["H"], case["new"], D).to(torch.bfloat16),
                  page_table=both[1:, :max(-(-n // page) for n in lens)].contiguous())
        if prefix:
            st.update(prefix_table=both[0, :prefix // page].contiguous(), prefix_len=_ints([prefix]))
    else:
        start = _lens(case["start"])
        held = [a + b for a, b in zip(start, lens)]
        st["page_table"], n_pages = _table(rng, held, case["page"])
        st.update(cu_all=_bounds(held), none=_ints([0] * len(lens)), rows=sum(held))
        if op == "store":
            st.update(cu=_bounds(lens), start=_ints(start), k=_tokens(g, sum(lens), case["Hkv"], D).to(torch.bfloat16),
                      v=_tokens(g, sum(lens), case["Hkv"], D).to(torch.bfloat16))
    st["k_cache"], st["k_scale"] = _cache(g, case, n_pages)
    st["v_cache"], st["v_scale"] = _cache(g, case, n_pages)
    return st


# --------------------------------------------------------------------------------------------------------- the framework
def _own(st):
    from flame_amd import capi, functional
    op = st["case"]["op"]
    if op in ("rotary", "turn"):
        q, k = functional.rotary(st["rope"], st["q"], st["k"], positions=st.get("positions"), cu_seqlens=st.get("cu"), start=st.get("start"))
        if op == "rotary":
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))]
    if op == "decode":
        return functional.sdpa_paged(st["q"], st["k_cache"], st["v_cache"], st["page_table"], st["kv_len"], st.get("prefix_table"), st.get("prefix_len"),
                                     k_scale=st["k_scale"], v_scale=st["v_scale"])
    if op == "store":
        capi.kv_store(st["k"], st["v"], st["k_cache"], st["v_cache"], st["page_table"], st["cu"], st["start"], st["k_scale"], st["v_scale"])
    k, v = capi.kv_load(st["k_cache"], st["v_cache"], st["page_table"], st["cu_all"], st["none"], st["rows"], st["k_scale"], st["v_scale"])
    return [k, v] if op == "load" else [k, v, st["k_scale"], st["v_scale"]]


# ------------------------------------------------------------------------------------------------------------ plain forms
def _row_positions(st):
    """Position of every row (packed, rows) or token [B, S]; angles of far positions need 64 bits."""
    if "positions" in st:
        return st["positions"].double()
    t = torch.arange(len(st["q"]), device="cuda")
    b = torch.searchsorted(st["cu"][1:].contiguous(), t.to(torch.int32), right=True)
    return (st["start"][b] + t - st["cu"][b]).double()


def _turn(x, cos, sin, R, interleaved):
    y = x.float()
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
    pair = [a * cos - b * sin, b * cos + a * sin]
    both = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat([both, y[..., R:]], -1).to(x.dtype)


def _plain_rotary(st):
    case = st["case"]
    angle = _row_positions(st)[..., None] * st["f"]
    axis = -3 if case["form"] == "batch" else -2
    cos, sin = (x.mul(st["size"]).float().unsqueeze(axis) for x in (angle.cos(), angle.sin()))
    out = [_turn(st[n].detach(), cos, sin, case["turned"], case["interleaved"]) for n in ("q", "k")]
    if case["op"] == "turn":        # the way back is the turn by the opposite angle
        out += [_turn(st[n], cos, -sin, case["turned"], case["interleaved"]) for n in ("dq", "dk")]
    return out


def _round_up(s):
    """The next number with a leading bit and three more: quotients of bf16 numbers by it are far from the borders of the codes or on them."""
    return ((s.view(torch.int32) + 0xFFFFF) & ~0xFFFFF).view(torch.float32).clamp_min(LEAST)


def _doubled(x, n):
    """x * 2^n, exactly (torch.ldexp goes through a power that is not)"""
    return x * ((n.clamp(-126, 127) + 127) << 23).to(torch.int32).view(torch.float32)


def _to_code(y, code):
    return (torch.round(y) if code == "int8" else y).to(CODES[code])


def _bytes(x):
    return x.view(torch.uint8)


def _places(table, page, cu, start, rows):
    """Page and token of every packed row."""
    t = torch.arange(rows, device="cuda")
    b = torch.searchsorted(cu[1:].contiguous(), t.to(torch.int32), right=True)
    pos = start[b] + t - cu[b]
    return table[b, pos // page].long(), pos % page


def _plain_load(st):
    block = st["case"]["block"]
    at, off = _places(st["page_table"], st["case"]["page"], st["cu_all"], st["none"], st["rows"])
    out = []
    for n in ("k", "v"):
        c = _bytes(st[n + "_cache"])[at, :, off].view(st[n + "_cache"].dtype).float()
        out.append((c * st[n + "_scale"][at, :, off // block][..., None]).to(torch.bfloat16))
    return out


def _plain_store(st):
    case = st["case"]
    page, block, code, Hkv = (case[n] for n in ("page", "block", "code", "Hkv"))
    Q = LARGEST[code]
    at, off = _places(st["page_table"], page, st["cu"], st["start"], len(st["k"]))
    number = at * (page // block) + off // block              # of the block in the cache
    touched, row = torch.unique(number, return_inverse=True)
    first = torch.full((len(touched),), block, device="cuda").scatter_reduce_(0, row, off % block, "amin")       # new tokens from here on
    before = torch.arange(block, device="cuda") < first[:, None]
    for n in ("k", "v"):
        x = st[n].float()
        codes, scales = st[n + "_cache"], st[n + "_scale"]
        most = torch.zeros((len(touched), Hkv), device="cuda").index_reduce_(0, row, x.abs().amax(-1), "amax")
        s = scales[touched // (page // block), :, touched % (page // block)]
        m, e = torch.frexp(most / (Q * s))
        grow = torch.where(m > 0.5, e, e - 1).clamp_min(0)                       # doublings until the new rows fit
        kept = (first > 0)[:, None]
        s = torch.where(kept, _doubled(s, grow), _round_up((most.double() / Q).float()))        # (by a number torch divides in 32 bits with two roundings)
        by = _bytes(codes).view(len(codes), Hkv, page // block, block, -1)
        old = by[touched // (page // block), :, touched % (page // block)]       # [touched, Hkv, block, D]
        again = _to_code(_doubled(old.view(codes.dtype).float(), -grow[..., None, None]), code)
        by[touched // (page // block), :, touched % (page // block)] = torch.where((before[:, None] & kept[..., None])[..., None], _bytes(again), old)
        _bytes(codes)[at, :, off] = _bytes(_to_code(x / s[row][..., None], code))
        scales[touched // (page // block), :, touched % (page // block)] = s
    return _plain_load(st) + [st["k_scale"], st["v_scale"]]


def _plain_decode(st):
    q, lens, block = st["q"], st["kv_len"], st["case"]["block"]
    B, H, N, D = q.shape
    Hkv = st["k_cache"].shape[1]
    G, scale = H // Hkv, 1.0 / math.sqrt(D)
    qh = q.float().view(B, Hkv, G * N, D)

    def keys(n, table):             # [..., pages] -> [..., Hkv, keys, D]
        codes = st[n + "_cache"]
        c = _bytes(codes)[table].view(codes.dtype).float()
        c = c.unflatten(-2, (-1, block)).mul_(st[n + "_scale"][table][..., None, None]).flatten(-3, -2)
        return c.transpose(-4, -3).flatten(-3, -2)

    table = st["page_table"].long()
    s = torch.matmul(qh, keys("k", table).transpose(-1, -2)).mul_(scale).view(B, Hkv, G, N, -1)
    j, i = torch.arange(s.shape[-1], device=q.device), torch.arange(N, device=q.device)
    keep = j < (lens[:, None] - N + 1 + i).clamp(min=0)[:, :, None]
    s = s.masked_fill_(~keep[:, None, None], -math.inf).view(B, Hkv, G * N, -1)
    top = s.amax(-1, keepdim=True)
    if "prefix_table" in st:        # the scores of all sequences at once
        pre = st["prefix_table"].long()
        pk, pv = keys("k", pre[None])[0], keys("v", pre[None])[0]
        sp = torch.matmul(qh.transpose(0, 1).reshape(Hkv, -1, D), pk.transpose(-1, -2)).mul_(scale)
        sp = sp.masked_fill_(torch.arange(sp.shape[-1], device=q.device) >= st["prefix_len"], -math.inf)
        top = torch.maximum(top, sp.amax(-1, keepdim=True).view(Hkv, B, G * N, 1).transpose(0, 1))
        sp = sp.view(Hkv, B, G * N, -1).sub_(top.transpose(0, 1)).exp_()
    top = top.clamp_min(-1e30)
    s = s.sub_(top).exp_()
    o, total = torch.matmul(s, keys("v", table)), s.sum(-1, keepdim=True)
    if "prefix_table" in st:
        o = o + torch.matmul(sp.reshape(Hkv, B * G * N, -1), pv).view(Hkv, B, G * N, D).transpose(0, 1)
        total = total + sp.sum(-1, keepdim=True).transpose(0, 1)
    return (o / total.clamp_min(1e-30)).to(torch.bfloat16).view(B, H, N, D)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    with torch.no_grad():
        return {"rotary": _plain_rotary, "turn": _plain_rotary, "store": _plain_store, "load": _plain_load, "decode": _plain_decode}[op](state)


# ------------------------------------------------------------------------------------------------- what a pass has to do
def _pairs(q, k):
    """Attended (query, key) pairs of one head of a sequence, causal from the end."""
    first = k - q + 1               # keys of the first query
    lo = max(0, 1 - first)          # queries without a key
    return (first + lo + k) * (q - lo) // 2


def work(case):
    op, Hkv, D, lens = case["op"], case["Hkv"], case["D"], _lens(case["lens"])
    if op in ("rotary", "turn"):
        numbers = sum(lens) * (case["H"] + Hkv)
        passes = 2 if op == "turn" else 1
        return {"bytes": passes * (2 * numbers * D * DTYPES[case["dtype"]].itemsize + 4 * sum(lens)), "flops": passes * numbers * case["turned"] * 3}
    each = 2 * Hkv * D                                          # numbers of a token, keys and values
    scales = lambda tokens: 8 * Hkv * -(-tokens // case["block"])
    if op == "decode":
        H, N = case["H"], case["new"]
        own_pairs = sum(_pairs(min(N, n), n) for n in lens)
        return {"bytes": each * (case["prefix"] + sum(lens)) + scales(case["prefix"]) + sum(scales(n) for n in lens) + 4 * D * H * N * len(lens),
                "flops": 4 * D * H * (own_pairs + N * len(lens) * case["prefix"])}
    held = [a + b for a, b in zip(_lens(case["start"]), lens)]
    read = each * 2 * sum(held) + sum(scales(n) for n in held)
    if op == "load":
        return {"bytes": read + each * sum(held), "flops": each * sum(held)}
    return {"bytes": read + each * (sum(held) - sum(lens)) + each * 3 * sum(lens), "flops": each * (sum(held) + 3 * sum(lens))}


# ------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_rotary(case, st):
    """Pairs as complex numbers, turned by exp(i position f)."""
    R, D = case["turned"], case["D"]
    f, size = _frequencies(case)
    f = torch.tensor(f, dtype=torch.float64, device="cuda")
    if case["form"] == "batch":
        pos = st["positions"].double()[:, None]                 # [B, 1, S]
    else:
        pos = torch.cat([torch.arange(a, a + n, dtype=torch.float64, device="cuda") for a, n in zip(_lens(case["start"]), _lens(case["lens"]))])[:, None]
    wave = torch.polar(torch.full_like(pos[..., None] * f, size), pos[..., None] * f)
    out = []
    for names, w in ((("q", "k"), wave), (("dq", "dk") if case["op"] == "turn" else (), wave.conj())):
        for n in names:
            x = st[n].detach().double()
            pairs = x[..., :R].unflatten(-1, (R // 2, 2)) if case["interleaved"] else x[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2)
            y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w)
            y = y if case["interleaved"] else y.transpose(-1, -2)
            out.append(torch.cat([y.flatten(-2), x[..., R:D]], -1))
    return out


def _two_to(n):
    return ((n.long() + 1023) << 52).view(torch.float64)


def _nearest64(y, code):
    """The nearest code, the even one of two."""
    if code == "int8":
        return torch.round(y)
    step = _two_to(torch.frexp(y)[1].clamp_min(-5) - 4)       # of e4m3: 2^-9 below 2^-6
    return torch.round(y / step) * step


def _exact_pages(case, st):
    """Sequence by sequence: its tokens' codes in their order, then the new rows block by block."""
    page, block, code = case["page"], case["block"], case["code"]
    Q, out, scales = LARGEST[code], [], []
    lens, start, table = _lens(case["lens"]), _lens(case["start"]), st["page_table"].tolist()
    for name in ("k", "v"):
        codes, all_scales = st[name + "_cache"], st[name + "_scale"].double()
        parts, row = [], 0
        for b, n in enumerate(lens):
            held = start[b] + n
            pages = table[b][:max(1, -(-held // page))]
            c = _bytes(codes)[pages].view(codes.dtype).double().transpose(1, 2).flatten(0, 1).clone()            # [tokens, Hkv, D]
            s = all_scales[pages].transpose(1, 2).flatten(0, 1).clone()                                         # [blocks, Hkv]
            if case["op"] == "store":
                x = st[name][row:row + n].double()
                row += n
                for i in range(start[b] // block, (held - 1) // block + 1):
                    lo, hi = max(start[b], i * block), min(held, (i + 1) * block)
                    new = x[lo - start[b]:hi - start[b]]
                    most = new.abs().amax((0, 2))
                    if lo == i * block:
                        m, e = torch.frexp(most / Q)
                        s[i] = (torch.ceil(m * 16) / 16 * _two_to(e)).clamp_min(LEAST)
                    else:
                        m, e = torch.frexp(most / (Q * s[i]))
                        grow = torch.where(m > 0.5, e, e - 1).clamp_min(0)
                        s[i] *= _two_to(grow)
                        c[i * block:lo] = _nearest64(c[i * block:lo] * _two_to(-grow)[:, None], code)
                    c[lo:hi] = _nearest64(new / s[i][:, None], code)
                all_scales[pages] = s.unflatten(0, (len(pages), -1)).transpose(1, 2)
            parts.append(c[:held] * s[torch.arange(held, device="cuda") // block][..., None])
        out.append(torch.cat(parts))
        scales.append(all_scales)
    return out if case["op"] == "load" else out + scales


def _exact_decode(case, st):
    q = st["q"].double()
    N, G, page, D, block = case["new"], case["H"] // case["Hkv"], case["page"], case["D"], case["block"]
    o = torch.zeros_like(q)
    pre = st["prefix_table"].long() if case["prefix"] else torch.zeros(0, dtype=torch.long, device=q.device)
    for b, n in enumerate(_lens(case["lens"])):
        table = torch.cat([pre, st["page_table"][b, :-(-n // page)].long()])
        kv = []
        for name in ("k", "v"):
            codes = st[name + "_cache"]
            s = st[name + "_scale"][table].double().repeat_interleave(block, 2)
            kv.append((_bytes(codes)[table].view(codes.dtype).double() * s[..., None]).transpose(0, 1).flatten(1, 2)[:, :case["prefix"] + n])
        k, v = kv
        keep = torch.ones((N, k.shape[1]), dtype=torch.bool, device=q.device).tril(k.shape[1] - N)
        keep[:, :case["prefix"]] = True
        for h in range(case["H"]):
            s = q[b, h] @ k[h // G].T * D ** -0.5
            s[~keep] = -math.inf
            e = torch.exp(s - torch.where(keep.any(1), s.max(1).values, 0.0)[:, None])
            o[b, h] = e @ v[h // G] / torch.where(keep.any(1), e.sum(1), 1.0)[:, None]
    return o


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("rotary", "turn"):
        return _exact_rotary(case, st)
    return _exact_decode(case, st) if case["op"] == "decode" else _exact_pages(case, st)
