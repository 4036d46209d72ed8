"""Attention over packed sequences and over a paged cache: the cases that are measured, their inputs, one pass as a caller's
program makes it, the same in plain torch operations, and what a pass cannot do without.

A case is a dict of plain values.  `op` says what it is:

  prompt   functional.sdpa_packed without gradients: causal attention of packed sequences of different lengths, grouped heads
  train    functional.sdpa_packed, forward and torch.autograd backward
  decode   functional.sdpa_paged: one or a few new tokens per sequence against a paged cache, a prefix shared by the batch or none
  store    capi.kv_store: rows of new keys and values to their places in the pages
  pages    capi.kv_copy_pages: copies of whole pages over all layers (forked sequences, compaction)

Lengths are texts of numbers with commas between them.
"""
from __future__ import annotations

import math
import random

import torch

own = False


# ---------------------------------------------------------------------------------------------------------------- cases
def _text(lens):
    return ",".join(str(n) for n in lens)


def _lens(text):
    return [int(n) for n in text.split(",")]


def _prompt(name, H, Hkv, D, q, k=None, op="prompt"):
    return dict(name=name, op=op, H=H, Hkv=Hkv, D=D, lens_q=_text(q), lens_k=_text(q if k is None else k))


def _decode(name, H, Hkv, D, page, new, prefix, lens):
    return dict(name=name, op="decode", H=H, Hkv=Hkv, D=D, page=page, new=new, prefix=prefix, lens=_text(lens))


def _pages(name, Hkv, D, page, layers, pages, moved):
    return dict(name=name, op="pages", Hkv=Hkv, D=D, page=page, layers=layers, pages=pages, moved=moved)


def listed():
    return [
        # one short prompt: a launch's time decides
        _prompt("prompt_short", 24, 8, 128, [77]),
        # prompts of a serving batch, lengths far apart, four query heads to a key head
        _prompt("prompt_batch", 32, 8, 128, [4096, 513, 2049, 77, 1024, 3333, 1, 1500]),
        # the next pieces of long prompts, whose earlier keys are there already; keys without gradients, one head dim of 64
        _prompt("prompt_pieces", 16, 4, 64, [512, 512, 300, 512], [8192, 2560, 5001, 512]),
        # training on short packed samples, as many key heads as query heads
        _prompt("train_short", 16, 16, 64, [256, 31, 200, 77, 128, 5, 333, 64], op="train"),
        # training on packed documents, grouped heads: the largest case
        _prompt("train_packed", 32, 8, 128, [4096, 1101, 2049, 333, 4608, 1024], op="train"),
        # training at a head dim between the usual ones
        _prompt("train_head_dim_96", 12, 4, 96, [1024, 700, 1500, 257], op="train"),
        # a step of few sequences: latency decides
        _decode("decode_few", 32, 8, 128, 16, 1, 0, [300, 1024, 77, 611]),
        # many answers to one long prompt: the prefix is common to all of them
        _decode("decode_shared_prefix", 32, 8, 128, 64, 1, 8192, [(97 * i) % 509 + 1 for i in range(64)]),
        # long contexts, four drafted tokens each, no common prefix
        _decode("decode_long", 32, 4, 128, 128, 4, 0, [32000, 24577, 40000, 16385, 28001, 36000, 20000, 31999]),
        # the keys and values of a batch of prompts to their pages
        dict(name="store_prompt", op="store", Hkv=8, D=128, page=16, lens=_text([4096, 513, 2049, 77, 1024]), start=_text([0, 5, 64, 1000, 17])),
        # forked sequences: their last, partly filled pages, in all layers
        _pages("pages_fork", 8, 128, 16, 24, 512, 32),
        # compaction after many sequences ended
        _pages("pages_compact", 8, 128, 16, 24, 1536, 600),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, most=32):
    while True:
        hkv, g = rng.choice([1, 2, 3, 4, 8, 12]), rng.choice([1, 2, 3, 4, 6, 8])
        if hkv * g <= most:
            return hkv * g, hkv


def _head_dim(rng):
    return rng.choice([64, 128]) if rng.random() < 0.6 else 8 * rng.randint(4, 16)


def draw(rng: random.Random):
    op = rng.choice(["prompt", "prompt", "train", "train", "decode", "decode", "decode", "store", "pages"])
    D = _head_dim(rng)
    if op in ("prompt", "train"):
        H, Hkv = _heads(rng)
        n, longest = _log(rng, 1, 24), _log(rng, 16, 4608)
        # plain forms work on padded batches: as much room as the largest listed case takes
        while n * longest * longest * H > 6 * 4608 * 4608 * 32 // 2:
            n, longest = max(1, n - 1), int(longest * 0.9)
        q = [max(1, int(longest * rng.random() ** 2)) for _ in range(n)]
        q[rng.randrange(n)] = longest
        k = list(q)
        if op == "prompt" and rng.random() < 0.3:       # later pieces of prompts
            k, q = q, [max(1, int(m * rng.uniform(0.05, 1.0))) for m in q]
        return dict(op=op, H=H, Hkv=Hkv, D=D, lens_q=_text(q), lens_k=_text(k))
    if op == "decode":
        H, Hkv = _heads(rng)
        page, new = rng.choice([16, 32, 64, 128]), rng.choice([1, 1, 1, 2, 4, 7])
        B, longest = _log(rng, 1, 96), _log(rng, 16, 32000)
        while B * longest * Hkv * D > 8 * 40000 * 4 * 128:
            B, longest = max(1, B - 1), int(longest * 0.9)
        lens = [max(new, int(longest * rng.uniform(0.2, 1.0))) for _ in range(B)]
        prefix = page * (_log(rng, page, 16384) // page) if rng.random() < 0.5 else 0
        return dict(op=op, H=H, Hkv=Hkv, D=D, page=page, new=new, prefix=prefix, lens=_text(lens))
    Hkv, page = rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 64, 128])
    if op == "store":
        n = _log(rng, 1, 64)
        most = _log(rng, 1, 2048)
        lens = [max(1, int(most * rng.random())) for _ in range(n)]
        return dict(op=op, Hkv=Hkv, D=D, page=page, lens=_text(lens), start=_text([_log(rng, 1, 2000) - 1 for _ in range(n)]))
    pages = _log(rng, 64, 1024) * 16 // page + 16
    return dict(op=op, Hkv=Hkv, D=D, page=page, layers=rng.randint(1, 24), pages=pages, moved=rng.randint(1, max(1, pages * 2 // 5)))


# --------------------------------------------------------------------------------------------------------------- inputs
def _bf16(g, *shape):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(torch.bfloat16)


def _bounds(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _table(rng, lens, page, spare=3):
    """Pages of every sequence in no order, as after some time of taking and freeing: (table, pages of the cache)."""
    need = [-(-n // page) for n in lens]
    places = list(range(sum(need) + spare))
    rng.shuffle(places)
    rows, at = [], 0
    for n in need:
        rows.append(places[at:at + n] + [0] * (max(need) - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), len(places)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    op, Hkv, D = case["op"], case["Hkv"], case["D"]
    st = {"case": case}
    if op in ("prompt", "train"):
        lq, lk = _lens(case["lens_q"]), _lens(case["lens_k"])
        st.update(cu_q=_bounds(lq), cu_k=_bounds(lk), most_q=max(lq), most_k=max(lk), q=_bf16(g, sum(lq), case["H"], D), k=_bf16(g, sum(lk), Hkv, D),
                  v=_bf16(g, sum(lk), Hkv, D))
        if op == "train":
            st["do"] = _bf16(g, sum(lq), case["H"], D)
            for name in ("q", "k", "v"):
                st[name].requires_grad_(True)
    elif op == "decode":
        lens, page, prefix = _lens(case["lens"]), case["page"], case["prefix"]
        both, n_pages = _table(rng, [prefix] + lens, page)
        st.update(kv_len=torch.tensor(lens, dtype=torch.int32, device="cuda"), q=_bf16(g, len(lens), case["H"], case["new"], D),
                  k_cache=_bf16(g, n_pages, Hkv, page, D), v_cache=_bf16(g, n_pages, Hkv, page, D),
                  page_table=both[1:, :max(-(-n // page) for n in lens)].contiguous())
        if prefix:
            st.update(prefix_table=both[0, :prefix // page].contiguous(), prefix_len=torch.tensor([prefix], dtype=torch.int32, device="cuda"))
    elif op == "store":
        lens, start = _lens(case["lens"]), _lens(case["start"])
        table, n_pages = _table(rng, [a + b for a, b in zip(lens, start)], case["page"])
        st.update(cu=_bounds(lens), start=torch.tensor(start, dtype=torch.int32, device="cuda"), page_table=table, k=_bf16(g, sum(lens), Hkv, D),
                  v=_bf16(g, sum(lens), Hkv, D), k_cache=_bf16(g, n_pages, Hkv, case["page"], D), v_cache=_bf16(g, n_pages, Hkv, case["page"], D))
    else:
        places = rng.sample(range(case["pages"]), 2 * case["moved"])
        st.update(src=places[:case["moved"]], dst=places[case["moved"]:], k_cache=_bf16(g, case["layers"], case["pages"], Hkv, case["page"], D),
                  v_cache=_bf16(g, case["layers"], case["pages"], Hkv, case["page"], D))
    return st


# --------------------------------------------------------------------------------------------------------- the framework
def _own(st):
    from flame_amd import capi, functional
    op = st["case"]["op"]
    if op == "prompt":
        return functional.sdpa_packed(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], is_causal=True)
    if op == "train":
        o = functional.sdpa_packed(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], is_causal=True)
        return [o.detach(), *torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"])]
    if op == "decode":
        return functional.sdpa_paged(st["q"], st["k_cache"], st["v_cache"], st["page_table"], st["kv_len"], st.get("prefix_table"), st.get("prefix_len"))
    if op == "store":
        capi.kv_store(st["k"], st["v"], st["k_cache"], st["v_cache"], st["page_table"], st["cu"], st["start"])
    else:
        capi.kv_copy_pages(st["k_cache"], st["v_cache"], st["src"], st["dst"])
    return [st["k_cache"], st["v_cache"]]


# ------------------------------------------------------------------------------------------------------------ plain forms
def _places(cu, most, total):
    """Rows of a padded batch in the packed tensor: where each is read, where it is written (the row behind the end for those
    that a sequence does not have), and which exist."""
    pos = torch.arange(most, device=cu.device)
    there = pos < (cu[1:] - cu[:-1])[:, None]
    at = cu[:-1, None] + pos
    return torch.where(there, at, 0), torch.where(there, at, total), there


def _plain_packed(st):
    H, Hkv, D = (st["case"][n] for n in ("H", "Hkv", "D"))
    G, scale = H // Hkv, 1.0 / math.sqrt(D)
    q, k, v = (st[n].detach() for n in ("q", "k", "v"))
    n, Sq, Sk = len(st["cu_q"]) - 1, st["most_q"], st["most_k"]
    rq, wq, _ = _places(st["cu_q"], Sq, len(q))
    rk, wk, has_k = _places(st["cu_k"], Sk, len(k))
    past = (st["cu_k"][1:] - st["cu_k"][:-1]) - (st["cu_q"][1:] - st["cu_q"][:-1])
    i, j = torch.arange(Sq, device=q.device), torch.arange(Sk, device=q.device)
    no = ~(has_k[:, None, :] & (j <= i[:, None] + past[:, None, None]))[:, None, None]

    def by_heads(x, rows, S):       # [n, Hkv, G or 1 heads one behind the other, D] in 32 bits
        return x[rows].float().view(n, S, Hkv, -1, D).permute(0, 2, 3, 1, 4).reshape(n, Hkv, -1, D)

    def packed(x, places, S, total):
        out = torch.zeros((total + 1, x.numel() // (n * S * D), D), dtype=torch.bfloat16, device=x.device)
        out[places] = x.reshape(n, Hkv, -1, S, D).permute(0, 3, 1, 2, 4).reshape(n, S, -1, D).to(torch.bfloat16)
        return out[:total]

    qh, kh, vh = by_heads(q, rq, Sq), by_heads(k, rk, Sk), by_heads(v, rk, Sk)
    p = torch.matmul(qh, kh.transpose(-1, -2)).mul_(scale).view(n, Hkv, G, Sq, Sk).masked_fill_(no, -math.inf)
    top = p.amax(-1, keepdim=True).clamp_min_(-1e30)
    p = p.sub_(top).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min_(1e-30)).view(n, Hkv, G * Sq, Sk)
    o = torch.matmul(p, vh)
    out = packed(o, wq, Sq, len(q))
    if st["case"]["op"] == "prompt":
        return out
    doh = by_heads(st["do"], rq, Sq) * (torch.arange(Sq, device=q.device) < (st["cu_q"][1:] - st["cu_q"][:-1])[:, None])[:, None, None, :, None].expand(
        n, 1, G, Sq, 1).reshape(n, 1, G * Sq, 1)
    dv = torch.matmul(p.transpose(-1, -2), doh)
    ds = torch.matmul(doh, vh.transpose(-1, -2)).sub_((doh * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, kh), torch.matmul(ds.transpose(-1, -2), qh)
    return [out, packed(dq, wq, Sq, len(q)), packed(dk, wk, Sk, len(k)), packed(dv, wk, Sk, len(k))]


def _plain_decode(st):
    q, kc, vc, lens = (st[n] for n in ("q", "k_cache", "v_cache", "kv_len"))
    B, H, N, D = q.shape
    Hkv, page = kc.shape[1], kc.shape[2]
    G, scale = H // Hkv, 1.0 / math.sqrt(D)
    qh = q.float().view(B, Hkv, G * N, D)

    def keys(cache, table):         # [..., pages] -> [..., Hkv, keys, D]
        return cache[table].float().transpose(-4, -3).flatten(-3, -2)

    table = st["page_table"].long()
    s = torch.matmul(qh, keys(kc, table).transpose(-1, -2)).mul_(scale).view(B, Hkv, G, N, -1)
    j, i = torch.arange(s.shape[-1], device=q.device), torch.arange(N, device=q.device)
    keep = j < (lens[:, None] - N + 1 + i).clamp(min=0)[:, :, None]
    s = s.masked_fill_(~keep[:, None, None], -math.inf).view(B, Hkv, G * N, -1)
    top = s.amax(-1, keepdim=True)
    if "prefix_table" in st:        # the scores of all sequences at once
        pre = st["prefix_table"].long()
        pk, pv = keys(kc, pre[None])[0], keys(vc, pre[None])[0]
        sp = torch.matmul(qh.transpose(0, 1).reshape(Hkv, -1, D), pk.transpose(-1, -2)).mul_(scale)
        sp = sp.masked_fill_(torch.arange(sp.shape[-1], device=q.device) >= st["prefix_len"], -math.inf)
        top = torch.maximum(top, sp.amax(-1, keepdim=True).view(Hkv, B, G * N, 1).transpose(0, 1))
        sp = sp.view(Hkv, B, G * N, -1).sub_(top.transpose(0, 1)).exp_()
    top = top.clamp_min(-1e30)
    s = s.sub_(top).exp_()
    o, total = torch.matmul(s, keys(vc, table)), s.sum(-1, keepdim=True)
    if "prefix_table" in st:
        o = o + torch.matmul(sp.reshape(Hkv, B * G * N, -1), pv).view(Hkv, B, G * N, D).transpose(0, 1)
        total = total + sp.sum(-1, keepdim=True).transpose(0, 1)
    return (o / total.clamp_min(1e-30)).to(torch.bfloat16).view(B, H, N, D)


def _plain_store(st):
    page, t = st["case"]["page"], torch.arange(len(st["k"]), device="cuda")
    b = torch.searchsorted(st["cu"][1:].contiguous(), t.to(torch.int32), right=True)
    pos = st["start"][b] + t - st["cu"][b]
    at, off = st["page_table"][b, pos // page].long(), pos % page
    st["k_cache"][at, :, off] = st["k"]
    st["v_cache"][at, :, off] = st["v"]
    return [st["k_cache"], st["v_cache"]]


def _plain_pages(st):
    src, dst = (torch.tensor(st[n], device="cuda") for n in ("src", "dst"))
    for c in (st["k_cache"], st["v_cache"]):
        c[:, dst] = c[:, src]
    return [st["k_cache"], st["v_cache"]]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    with torch.no_grad():
        return {"prompt": _plain_packed, "train": _plain_packed, "decode": _plain_decode, "store": _plain_store, "pages": _plain_pages}[op](state)


# ------------------------------------------------------------------------------------------------- what a pass has to do
def _pairs(q, k):
    """Attended (query, key) pairs of one head of a sequence, causal from the end."""
    first = k - q + 1               # keys of the first query
    lo = max(0, 1 - first)          # queries without a key
    return (first + lo + k) * (q - lo) // 2


def work(case):
    op, Hkv, D = case["op"], case["Hkv"], case["D"]
    if op in ("prompt", "train"):
        lq, lk, H = _lens(case["lens_q"]), _lens(case["lens_k"]), case["H"]
        pairs = sum(_pairs(a, b) for a, b in zip(lq, lk)) * H
        rows = 2 * D * (sum(lq) * H + sum(lk) * Hkv)        # bytes of q and k, or of o and v, or of dq and dk
        if op == "prompt":
            return {"bytes": 2 * rows, "flops": 4 * D * pairs}
        return {"bytes": 4 * rows, "flops": 14 * D * pairs}        # q k v dO, O dQ dK dV; two products forward, five backward
    if op == "decode":
        lens, H, N = _lens(case["lens"]), case["H"], case["new"]
        own_pairs = sum(_pairs(min(N, n), n) for n in lens)
        return {"bytes": 4 * D * Hkv * (case["prefix"] + sum(lens)) + 4 * D * H * N * len(lens),
                "flops": 4 * D * H * (own_pairs + N * len(lens) * case["prefix"])}
    if op == "store":
        return {"bytes": 8 * D * Hkv * sum(_lens(case["lens"])), "flops": 0}
    return {"bytes": 8 * D * Hkv * case["page"] * case["layers"] * case["moved"], "flops": 0}


# ------------------------------------------------------------------------------------------------------------- 64 bits
def _attend64(q, k, v, keep, scale):
    """One head's queries [a, D] on keys [b, D]: (O, P), a row without keys is zero."""
    s = (q @ k.T) * scale
    s[~keep] = -math.inf
    e = torch.exp(s - torch.where(keep.any(1), s.max(1).values, 0.0)[:, None])
    p = e / torch.where(keep.any(1), e.sum(1), 1.0)[:, None]
    return p @ v, p


def _exact_packed(case, st):
    H, D = case["H"], case["D"]
    G, scale = H // case["Hkv"], D ** -0.5
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    do = st["do"].double() if case["op"] == "train" else None
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    a = b = 0
    for m, n in zip(_lens(case["lens_q"]), _lens(case["lens_k"])):
        keep = torch.ones((m, n), dtype=torch.bool, device=q.device).tril(n - m)
        Q, K = slice(a, a + m), slice(b, b + n)
        for h in range(H):
            c = h // G
            o[Q, h], p = _attend64(q[Q, h], k[K, c], v[K, c], keep, scale)
            if do is not None:
                dp = do[Q, h] @ v[K, c].T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
                dq[Q, h] = ds @ k[K, c]
                dk[K, c] += ds.T @ q[Q, h]
                dv[K, c] += p.T @ do[Q, h]
        a, b = a + m, b + n
    return o if do is None else [o, dq, dk, dv]


def _exact_decode(case, st):
    q, kc, vc = (st[n].double() for n in ("q", "k_cache", "v_cache"))
    N, G, page, D = case["new"], case["H"] // case["Hkv"], case["page"], case["D"]
    o = torch.zeros_like(q)
    pre = st["prefix_table"].long() if case["prefix"] else torch.zeros(0, dtype=torch.long, device=q.device)
    for b, n in enumerate(_lens(case["lens"])):
        table = torch.cat([pre, st["page_table"][b, :-(-n // page)].long()])
        for c in range(case["Hkv"]):
            k, v = (x[table, c].reshape(-1, D)[:case["prefix"] + n] for x in (kc, vc))
            keep = torch.ones((N, len(k)), dtype=torch.bool, device=q.device).tril(len(k) - N)
            keep[:, :case["prefix"]] = True
            for h in range(c * G, c * G + G):
                o[b, h] = _attend64(q[b, h], k, v, keep, D ** -0.5)[0]
    return o


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("prompt", "train"):
        return _exact_packed(case, st)
    if op == "decode":
        return _exact_decode(case, st)
    if op == "store":               # row by row
        lens, start, table = _lens(case["lens"]), _lens(case["start"]), st["page_table"].tolist()
        pages, offs = [], []
        for b, n in enumerate(lens):
            for pos in range(start[b], start[b] + n):
                pages.append(table[b][pos // case["page"]])
                offs.append(pos % case["page"])
        out = []
        for c, x in ((st["k_cache"], st["k"]), (st["v_cache"], st["v"])):
            rows = c.transpose(1, 2).contiguous().view(-1, case["Hkv"], case["D"])
            rows[[p * case["page"] + f for p, f in zip(pages, offs)]] = x
            out.append(rows.view(c.shape[0], case["page"], case["Hkv"], case["D"]).transpose(1, 2).contiguous())
        return out
    for a, b in zip(st["src"], st["dst"]):
        for c in (st["k_cache"], st["v_cache"]):
            c[:, b].copy_(c[:, a])
    return [st["k_cache"], st["v_cache"]]
