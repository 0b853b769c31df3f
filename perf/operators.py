"""Operators of the token-paged 8-bit cache: what is measured, and their plain forms.

Four operators that work on one cache, as a serving loop uses them: rotary positions on Q and K, quantised append into
pages of a few tokens, attention over those pages, and the page bookkeeping (reserve, fork, copy, free, compact).
`run` computes them with elementary torch operations, or, where `own` is true, through the package's entry points.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

D = 128          # channels of a head, the one size that the cache has
E_MIN, E_MAX = -60, 60


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one sequence, one new token: the latency of a single decode step
        {"name": "attn one token", "op": "attn", "seqs": 1, "len_lo": 777, "len_hi": 777, "q_lo": 1, "q_hi": 1, "hq": 48, "hkv": 8, "page": 64, "window": 0},
        # a serving batch of ragged lengths, one token each
        {"name": "attn batch decode", "op": "attn", "seqs": 64, "len_lo": 300, "len_hi": 8191, "q_lo": 1, "q_hi": 1, "hq": 48, "hkv": 8, "page": 64, "window": 0},
        # few long contexts: the cache is all the traffic
        {"name": "attn long decode", "op": "attn", "seqs": 8, "len_lo": 100001, "len_hi": 131072, "q_lo": 1, "q_hi": 1, "hq": 24, "hkv": 8, "page": 128, "window": 0},
        # several proposed tokens verified at once on one rank of eight (one kv head), small pages, a sliding window
        {"name": "attn verify window", "op": "attn", "seqs": 16, "len_lo": 900, "len_hi": 20011, "q_lo": 2, "q_hi": 5, "hq": 6, "hkv": 1, "page": 16, "window": 4099},
        # prompts read in after a cached prefix
        {"name": "attn prompt", "op": "attn", "seqs": 3, "len_lo": 2600, "len_hi": 9001, "q_lo": 700, "q_hi": 2500, "hq": 48, "hkv": 8, "page": 32, "window": 0},
        # one token for every sequence of a batch
        {"name": "append one token", "op": "append", "seqs": 64, "len_lo": 1, "len_hi": 4000, "new_lo": 1, "new_hi": 1, "hkv": 8, "page": 64},
        # prompts of up to a chunk of 21600 tokens
        {"name": "append prompt", "op": "append", "seqs": 5, "len_lo": 0, "len_hi": 333, "new_lo": 2001, "new_hi": 21600, "hkv": 8, "page": 128},
        # branches of a prompt that share its pages, each about to take one more token
        {"name": "fork branches", "op": "fork", "seqs": 8, "branches": 4, "len_lo": 500, "len_hi": 4001, "layers": 4, "hkv": 8, "page": 32},
        # sequences copied page by page, to be changed apart
        {"name": "copy sequences", "op": "copy", "seqs": 4, "branches": 1, "len_lo": 3000, "len_hi": 9000, "layers": 6, "hkv": 8, "page": 64},
        # a pool with holes made dense, so that its upper part can be given away
        {"name": "compact pool", "op": "compact", "seqs": 40, "branches": 0, "len_lo": 200, "len_hi": 6001, "layers": 4, "hkv": 8, "page": 64},
        # the query heads of one decode step, part of the head, far positions
        {"name": "rotary decode", "op": "rotary", "tokens": 64, "heads": 48, "dim": 128, "rot": 96, "layout": "half", "dtype": "bfloat16", "pos_hi": 1000000, "factor": 16.0, "inverse": False},
        # a chunk's worth of tokens, the transposed rotation that a gradient takes
        {"name": "rotary long transposed", "op": "rotary", "tokens": 21600, "heads": 24, "dim": 128, "rot": 128, "layout": "interleaved", "dtype": "float32", "pos_hi": 40000, "factor": 1.0, "inverse": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "append", "fork", "copy", "compact", "rotary"])
    page = rng.choice([16, 32, 64, 128])
    hq, hkv = rng.choice([(48, 8), (24, 8), (6, 1), (8, 8), (6, 2), (16, 1)])
    if op == "attn":
        kind = rng.choice(["decode", "decode", "few", "prompt"])
        window = rng.choice([0, 0, _log(rng, 17, 6000)])
        if kind == "prompt":
            q = _log(rng, 17, 2500)
            hi = q + _log(rng, 1, 6000)
            return {"op": op, "seqs": rng.randint(1, 3), "len_lo": rng.randint(q, hi), "len_hi": hi, "q_lo": rng.randint(1, q), "q_hi": q, "hq": hq, "hkv": hkv, "page": page, "window": window}
        q = 1 if kind == "decode" else rng.randint(2, 16)
        hi = _log(rng, max(q, 3), 120000)
        seqs = min(_log(rng, 1, 200), max(1, 900000 // hi))
        return {"op": op, "seqs": seqs, "len_lo": rng.randint(q, hi), "len_hi": hi, "q_lo": rng.randint(1, q), "q_hi": q, "hq": hq, "hkv": hkv, "page": page, "window": window}
    if op == "append":
        new = rng.choice([1, rng.randint(2, 9), _log(rng, 10, 12000)])
        seqs = min(_log(rng, 1, 200), max(1, 60000 // new))
        return {"op": op, "seqs": seqs, "len_lo": 0, "len_hi": _log(rng, 1, 5000), "new_lo": rng.randint(1, new), "new_hi": new, "hkv": hkv, "page": page}
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([dim, 2 * rng.randint(1, dim // 2)])
        heads = rng.choice([1, 2, 5, 8, 24, 48])
        tokens = min(_log(rng, 1, 21600), 60000000 // (heads * dim))
        return {"op": op, "tokens": tokens, "heads": heads, "dim": dim, "rot": rot, "layout": rng.choice(["half", "interleaved"]), "dtype": rng.choice(["bfloat16", "float16", "float32"]),
                "pos_hi": _log(rng, 2, 1000000), "factor": rng.choice([1.0, 4.0, 16.0]), "inverse": rng.random() < 0.5}
    hi = _log(rng, 20, 6000)
    return {"op": op, "seqs": rng.randint(1, 24), "branches": 0 if op == "compact" else rng.randint(1, 3 if op == "fork" else 1), "len_lo": rng.randint(0, hi), "len_hi": hi, "layers": rng.randint(1, 3), "hkv": hkv, "page": page}


def _spread(lo, hi, n, salt):
    """n whole numbers from lo to hi, in an order of their own: the same for every seed."""
    v = [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(salt).shuffle(v)
    return v


def _lens(case):
    return _spread(case["len_lo"], case["len_hi"], case["seqs"], 7)


def _n_q(case):
    return _spread(case["q_lo"], case["q_hi"], case["seqs"], 11)


def _n_new(case):
    return _spread(case["new_lo"], case["new_hi"], case["seqs"], 13)


def _pages(n, page):
    return -(-n // page)


# ------------------------------------------------------------------------------------------------ inputs
def _codes(shape, g):
    """e4m3 codes of normal values, as a quantised block of tokens holds them."""
    out = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    for part in out.view(-1, shape[-1]).split(1 << 21):
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 96).clamp_(-448, 448))
    return out


def _scales(shape, g):
    return _two_to(torch.randint(-8, -5, shape, generator=g, device="cuda"))


def _two_to(e):
    """2^e for whole e, from its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _cache(lens, pages_of, extra, rows, layers, hkv, page, seed, g):
    """A cache as a program has it after some work: `lens[i]` tokens in row i, its pages scattered over the pool."""
    counts = [_pages(n, page) for n in pages_of]
    n_pages = sum(counts) + extra
    per_row = max(counts + [1])
    order = np.random.RandomState(seed % (1 << 31)).permutation(n_pages).astype(np.int32)
    table, refs, at = np.full((rows, per_row), -1, np.int32), np.zeros(n_pages, np.int32), 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        refs[order[at:at + c]] = 1
        at += c
    seq_lens = np.zeros(rows, np.int32)
    seq_lens[:len(lens)] = lens
    shape = (layers, n_pages, hkv, page, D)
    s = {"k8": _codes(shape, g), "v8": _codes(shape, g), "k_scale": _scales(shape[:3], g), "v_scale": _scales(shape[:3], g),
         "page_table": torch.from_numpy(table).cuda(), "seq_lens": torch.from_numpy(seq_lens).cuda(), "page_refs": torch.from_numpy(refs).cuda()}
    if own:
        # the program's handle: the package's cache, with the same pages in it
        c = _package().TokenPagedKVCache(n_layers=layers, n_pages=n_pages, page_tokens=page, n_kv_heads=hkv, max_seqs=rows, max_pages_per_seq=per_row)
        for k in list(s):
            getattr(c, k).view(torch.uint8).copy_(s[k].view(torch.uint8))
            s[k] = getattr(c, k)
        s["cache"] = c
    return s


def _package():
    root = os.path.join(os.getcwd(), "magi-1_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import magi_b200
    return magi_b200


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cu(counts):
    return _i32(np.concatenate([[0], np.cumsum(counts)]).tolist())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "rotary":
        dtype, half = getattr(torch, case["dtype"]), case["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) * 2 / case["rot"]) / case["factor"]
        return {"case": case, "mb": _package() if own else None, "x": torch.randn(case["tokens"], case["heads"], case["dim"], generator=g, device="cuda").to(dtype),
                "positions": torch.randint(0, case["pos_hi"], (case["tokens"],), generator=g, device="cuda", dtype=torch.int32),
                "inv_freq": freq.cuda(), "mscale": 0.1 * math.log(case["factor"]) + 1.0}
    lens, hkv, page = _lens(case), case["hkv"], case["page"]
    n = len(lens)
    if op == "attn":
        n_q = _n_q(case)
        s = _cache(lens, lens, 3, n, 1, hkv, page, seed, g)
        s |= {"q": torch.randn(sum(n_q), case["hq"], D, generator=g, device="cuda").to(torch.bfloat16), "seqs": _i32(list(range(n))), "cu_q": _cu(n_q), "max_q": max(n_q), "max_len": max(lens)}
    elif op == "append":
        # the tokens are reserved already: the lengths count them, `starts` says where each sequence's go
        new = _n_new(case)
        after = [a + b for a, b in zip(lens, new)]
        s = _cache(after, after, 2, n, 1, hkv, page, seed, g)
        # values that grow from token to token, so that some pages take a larger scale
        k, v = [(torch.randn(sum(new), hkv, D, generator=g, device="cuda") * torch.exp(torch.randn(sum(new), 1, 1, generator=g, device="cuda"))).to(torch.bfloat16) for _ in range(2)]
        s |= {"k": k, "v": v, "seqs": _i32(list(range(n))), "starts": _i32(lens), "cu_new": _cu(new), "max_new": max(new)}
    elif op == "compact":
        # every second sequence has ended: its pages are the holes
        s = _cache(lens, lens, 5, n, case["layers"], hkv, page, seed, g)
        dead = torch.arange(0, n, 2, device="cuda")
        gone = s["page_table"][dead]
        s["page_refs"][gone[gone >= 0].long()] = 0
        s["page_table"][dead] = -1
        s["seq_lens"][dead] = 0
        s["saved"] = [s[k].clone() for k in ("page_table", "seq_lens", "page_refs")]
    else:
        m = n * case["branches"]
        extra = sum(_pages(v + 1, page) for v in lens) * case["branches"] if op == "copy" else 2 * m
        s = _cache(lens, [v + 1 for v in lens], extra, n + m, case["layers"], hkv, page, seed, g)
        # a row's spare page (a token more than the length) is not its own yet
        used = (s["seq_lens"] + page - 1) // page
        spare = torch.arange(s["page_table"].shape[1], device="cuda")[None] >= used[:, None]
        over = s["page_table"][spare]
        s["page_refs"][over[over >= 0].long()] = 0
        s["page_table"][spare] = -1
        s |= {"src": _i32([i for i in range(n) for _ in range(case["branches"])]), "dst": _i32(list(range(n, n + m))), "ones": _i32([1] * m)}
    return s | {"case": case, "mb": _package() if own else None}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    case, op, mb = s["case"], s["case"]["op"], s["mb"]
    if op == "attn":
        out, lse = mb.paged_attn(s["q"], s["cache"], 0, s["seqs"], s["cu_q"], max_q=s["max_q"], window=case["window"])
        return {"out": out, "lse": lse}
    if op == "rotary":
        return {"out": mb.rotary(s["x"], s["positions"], s["inv_freq"], layout=case["layout"], mscale=s["mscale"], inverse=case["inverse"])}
    c = s["cache"]
    if op == "append":
        c.append(0, s["seqs"], s["starts"], s["k"], s["v"], s["cu_new"], max_new=s["max_new"])
        return _pools(s)
    if op == "compact":
        for name, v in zip(("page_table", "seq_lens", "page_refs"), s["saved"]):
            s[name].copy_(v)
        c.compact()
        return _pools(s) | _tables(s)
    c.free(s["dst"])
    if op == "copy":
        c.copy(s["src"], s["dst"])
        return _pools(s) | _tables(s)
    c.fork(s["src"], s["dst"])
    starts = c.reserve(s["dst"], s["ones"])
    return _pools(s) | _tables(s) | {"starts": starts}


def _pools(s):
    return {k: s[k] for k in ("k8", "v8", "k_scale", "v_scale")}


def _tables(s):
    return {k: s[k] for k in ("page_table", "seq_lens", "page_refs")}


def _run_plain(s):
    op = s["case"]["op"]
    if op == "attn":
        return _plain_attn(s)
    if op == "rotary":
        return _plain_rotary(s)
    if op == "append":
        return _plain_append(s)
    if op == "compact":
        for name, v in zip(("page_table", "seq_lens", "page_refs"), s["saved"]):
            s[name].copy_(v)
        _plain_compact(s)
        return _pools(s) | _tables(s)
    _plain_free(s, s["dst"].long())
    _plain_branch(s, s["src"].long(), s["dst"].long(), shared=op == "fork")
    if op == "copy":
        return _pools(s) | _tables(s)
    starts = _plain_reserve(s, s["dst"].long(), s["ones"])
    return _pools(s) | _tables(s) | {"starts": starts}


def _plain_attn(s):
    case, q, page = s["case"], s["q"], s["case"]["page"]
    hq, hkv, window = case["hq"], case["hkv"], case["window"]
    n, rows, group = s["seqs"].numel(), s["max_q"], hq // hkv
    seqs = s["seqs"].long()
    table = s["page_table"][seqs, :_pages(s["max_len"], page)].clamp(min=0).long()
    lens = s["seq_lens"][seqs].long()
    span = table.shape[1] * page
    at = torch.arange(span, device="cuda")
    held = (at[None] < lens[:, None])[:, None, :, None]

    def values(codes, scale):
        v = codes[0].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * scale[0][table][..., None, None]
        return torch.where(held, v.transpose(1, 2).reshape(n, hkv, span, D), 0.0)

    cu = s["cu_q"].long()
    n_q = cu[1:] - cu[:-1]
    i = torch.arange(rows, device="cuda")
    there = i[None] < n_q[:, None]
    index = (cu[:-1, None] + i[None]).clamp(max=q.shape[0] - 1)
    qs = q[index].float().view(n, rows, hkv, group, D).permute(0, 2, 3, 1, 4).reshape(n, hkv, group * rows, D)
    last = lens[:, None] - n_q[:, None] + i[None]
    seen = (at[None, None] <= last[..., None]) & (at[None, None] < lens[:, None, None])
    if window:
        seen &= at[None, None] > last[..., None] - window
    score = torch.matmul(qs, values(s["k8"], s["k_scale"]).transpose(-1, -2)).view(n, hkv, group, rows, span)
    score = torch.where(seen[:, None, None], score * D ** -0.5, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, hkv, group * rows, span), values(s["v8"], s["v_scale"])).view(n, hkv, group, rows, D)
    out = torch.where(total > 0, out / total, 0.0)
    lse = top + torch.log(total)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, rows, hq, D)[there]
    lse = lse[..., 0].permute(0, 3, 1, 2).reshape(n, rows, hq)[there]
    return {"out": out.to(torch.bfloat16), "lse": lse}


def _plain_rotary(s):
    case, x = s["case"], s["x"].float()
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = (torch.cos(angle) * s["mscale"]).float()[:, None], (torch.sin(angle) * s["mscale"]).float()[:, None]
    if case["inverse"]:
        sin = -sin
    rot, half = case["rot"], case["rot"] // 2
    if case["layout"] == "half":
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return {"out": torch.cat([turned, x[..., rot:]], -1).to(s["x"].dtype)}


def _plain_append(s):
    page = s["case"]["page"]
    seqs, starts, cu = s["seqs"].long(), s["starts"].long(), s["cu_new"].long()
    n_new = cu[1:] - cu[:-1]
    total = s["k"].shape[0]
    entry = torch.repeat_interleave(torch.arange(seqs.numel(), device="cuda"), n_new, output_size=total)
    pos = starts[entry] + torch.arange(total, device="cuda") - cu[entry]
    pid, off = s["page_table"][seqs[entry], pos // page].long(), pos % page
    touched, slot = torch.unique(pid, return_inverse=True)
    fresh = torch.zeros(touched.numel(), page, dtype=torch.bool, device="cuda")
    fresh[slot, off] = True
    base = torch.zeros(touched.numel(), dtype=torch.long, device="cuda")
    base[slot] = pos - off
    length = torch.zeros_like(base)
    length[slot] = s["seq_lens"].long()[seqs[entry]]
    kept = (torch.arange(page, device="cuda")[None] < (length - base)[:, None]) & ~fresh
    _plain_write(s["k8"], s["k_scale"], s["k"], touched, slot, off, pid, kept)
    _plain_write(s["v8"], s["v_scale"], s["v"], touched, slot, off, pid, kept)
    return _pools(s)


def _plain_write(codes, scale, x, touched, slot, off, pid, kept):
    x = x.float()
    size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    top = torch.zeros(touched.numel(), x.shape[1], device="cuda").scatter_reduce_(0, slot[:, None].expand_as(size), size, "amax")
    m, e = torch.frexp(top)
    e = torch.where(top > 0, torch.where(m <= 0.875, e - 9, e - 8), E_MIN).clamp(E_MIN, E_MAX)
    before = scale[0][touched]
    after = _two_to(e)
    after = torch.where(kept.any(1)[:, None], torch.maximum(before, after), after)
    raw = codes[0].view(torch.uint8)
    old = raw[touched]
    again = (old.view(torch.float8_e4m3fn).float() * (before / after)[..., None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    raw[touched] = torch.where(kept[:, None, :, None], again, old)
    raw[pid, :, off] = (x / after[slot][..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    scale[0][touched] = after


def _plain_free(s, rows):
    old = s["page_table"][rows]
    old = old[old >= 0].long()
    s["page_refs"].index_add_(0, old, torch.full_like(old, -1, dtype=torch.int32))
    s["page_table"][rows] = -1
    s["seq_lens"][rows] = 0


def _plain_move(s, old, new):
    for k in ("k8", "v8"):
        raw = s[k].view(torch.uint8)
        raw[:, new] = raw[:, old]
    for k in ("k_scale", "v_scale"):
        s[k][:, new] = s[k][:, old]


def _plain_branch(s, src, dst, shared):
    page = s["case"]["page"]
    lens = s["seq_lens"].long()[src]
    own_from = lens // page if shared else torch.zeros_like(lens)
    at = torch.arange(s["page_table"].shape[1], device="cuda")[None]
    used = at < ((lens + page - 1) // page)[:, None]
    mine = used & (at >= own_from[:, None])
    rows = s["page_table"][src]
    old = rows[mine].long()
    held = rows[used & ~mine].long()
    new = torch.nonzero(s["page_refs"] == 0)[:old.numel(), 0]
    s["page_refs"].index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    s["page_refs"][new] = 1
    rows[mine] = new.int()
    rows[~used] = -1
    s["page_table"][dst] = rows
    s["seq_lens"][dst] = lens.int()
    _plain_move(s, old, new)


def _plain_reserve(s, rows, n_new):
    page = s["case"]["page"]
    lens = s["seq_lens"][rows]
    at = torch.arange(s["page_table"].shape[1], device="cuda")[None]
    want = (at >= ((lens + page - 1) // page)[:, None]) & (at < ((lens + n_new + page - 1) // page)[:, None])
    new = torch.nonzero(s["page_refs"] == 0)[:int(want.sum()), 0]
    table = s["page_table"][rows]
    table[want] = new.int()
    s["page_table"][rows] = table
    s["page_refs"][new] = 1
    s["seq_lens"][rows] = lens + n_new
    return lens


def _plain_compact(s):
    live = s["page_refs"] > 0
    n_live = int(live.sum())
    hole = torch.nonzero(~live[:n_live])[:, 0]
    mover = torch.nonzero(live[n_live:])[:, 0] + n_live
    _plain_move(s, mover, hole)
    to = torch.arange(live.numel(), device="cuda", dtype=torch.int32)
    to[mover] = hole.int()
    s["page_table"].copy_(torch.where(s["page_table"] >= 0, to[s["page_table"].clamp(min=0).long()], -1))
    s["page_refs"][hole] = s["page_refs"][mover]
    s["page_refs"][mover] = 0


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    op = case["op"]
    if op not in ("attn", "append", "rotary"):
        return None  # whole numbers and bytes that are moved: nothing is computed
    s = prepare(case, seed)
    if op == "rotary":
        x = s["x"].double()
        half = case["rot"] // 2
        turn = torch.polar(torch.full((1,), s["mscale"], dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * s["inv_freq"])[:, None]
        if case["inverse"]:
            turn = turn.conj()
        first, second = (slice(0, half), slice(half, 2 * half)) if case["layout"] == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return {"out": x}
    return _exact_attn(case, s) if op == "attn" else _exact_append(case, s)


def _exact_attn(case, s):
    page, hq, hkv, group = case["page"], case["hq"], case["hkv"], case["hq"] // case["hkv"]
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    lens, cu = s["seq_lens"].tolist(), s["cu_q"].tolist()
    for b, length in enumerate(lens):
        ids = s["page_table"][b, :_pages(length, page)].long()
        for h in range(hkv):
            k, v = [(s[c][0, :, h][ids].double() * s[z][0, :, h][ids].double()[:, None, None]).reshape(-1, D)[:length] for c, z in (("k8", "k_scale"), ("v8", "v_scale"))]
            last = length - (cu[b + 1] - cu[b]) + torch.arange(cu[b + 1] - cu[b], device="cuda")[:, None]
            at = torch.arange(length, device="cuda")[None]
            hidden = (at > last) | ((at <= last - case["window"]) if case["window"] else False)
            for j in range(h * group, (h + 1) * group):
                score = (s["q"][cu[b]:cu[b + 1], j].double() @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
                lse[cu[b]:cu[b + 1], j] = torch.logsumexp(score, 1)
                out[cu[b]:cu[b + 1], j] = torch.softmax(score, 1) @ v
    return {"out": out, "lse": lse}


def _nearest_e4m3(y):
    """The e4m3 value nearest to y, ties to even, magnitudes beyond 448 at 448."""
    size = y.abs()
    half, _ = torch.frexp(size.clamp(min=2.0 ** -6))
    step = size.clamp(min=2.0 ** -6) / half * 2.0 ** -4  # 2^(floor(log2(size)) - 3)
    return torch.sign(y) * torch.minimum(torch.round(size / step) * step, torch.full_like(y, 448.0))


def _exact_append(case, s):
    page, got = case["page"], {}
    lens, starts, cu, table = s["seq_lens"].tolist(), s["starts"].tolist(), s["cu_new"].tolist(), s["page_table"].tolist()
    if sum(_pages(n, page) for n in _n_new(case)) > 6000:
        return None
    for codes, scale, name in (("k8", "k_scale", "k"), ("v8", "v_scale", "v")):
        value, factor = s[codes].double(), s[scale].double()
        for b, (start, end) in enumerate(zip(starts, lens)):
            for slot in range(start // page, _pages(end, page)):
                pid, lo, hi = table[b][slot], max(start, slot * page), min(end, (slot + 1) * page)
                x = s[name][cu[b] + lo - start:cu[b] + hi - start].double()
                top = x.abs().amax((0, 2)) / 448.0
                half, _ = torch.frexp(top)
                power = torch.where(top > 0, top / half, 0.0)  # the power of two above it, or half that where it is one itself
                grown = torch.where(half == 0.5, power / 2, power).clamp(2.0 ** E_MIN, 2.0 ** E_MAX)
                if lo > slot * page:
                    before = factor[0, pid].clone()
                    grown = torch.maximum(grown, before)
                    kept = value[0, pid, :, :lo - slot * page]
                    kept.copy_(_nearest_e4m3(kept * (before / grown)[:, None, None]))
                factor[0, pid] = grown
                value[0, pid, :, lo - slot * page:hi - slot * page] = _nearest_e4m3(x.transpose(0, 1) / grown[:, None, None])
        got |= {codes: value, scale: factor}
    return got


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    op = case["op"]
    if op == "rotary":
        n = case["tokens"] * case["heads"] * case["dim"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * n * size + 4 * case["tokens"], "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    lens, hkv, page = _lens(case), case["hkv"], case["page"]
    token = 2 * hkv * D  # the codes of one token, K and V
    if op == "attn":
        n_q, window = _n_q(case), case["window"] or 1 << 40
        read = sum(min(n, window + q - 1) for n, q in zip(lens, n_q))
        seen = sum(min(window, n - q + i + 1) for n, q in zip(lens, n_q) for i in range(q))
        rows = sum(n_q) * case["hq"]
        return {"bytes": read * token + sum(_pages(min(n, window + q - 1), page) for n, q in zip(lens, n_q)) * (8 * hkv + 4) + rows * (4 * D + 4), "flops": 4 * D * case["hq"] * seen}
    if op == "append":
        new = _n_new(case)
        blocks = sum(_pages(a + b, page) - a // page for a, b in zip(lens, new))
        return {"bytes": sum(new) * token * 3 + blocks * 8 * hkv, "flops": 4 * sum(new) * token}
    if op == "compact":
        # about what stays alive beyond the border: every second sequence has left, its holes lie anywhere
        live = [n for i, n in enumerate(lens) if i % 2]
        total = sum(_pages(n, page) for n in lens) + 5
        alive = sum(_pages(n, page) for n in live)
        moved = alive * (total - alive) // total
    elif op == "copy":
        moved = sum(_pages(n, page) for n in lens) * case["branches"]
    else:
        moved = sum(n % page > 0 for n in lens) * case["branches"]
    rows = case["seqs"] * (1 + case["branches"])
    return {"bytes": 2 * moved * case["layers"] * (token * page + 8 * hkv) + 8 * rows * max(_pages(n, page) for n in lens + [1]), "flops": 0}
