"""Cases of the paged 8-bit KV cache: planning its pages, filling it, reading it back and attending over it.

The cache holds keys and values as codes of 8 bits (int8, or float8 e4m3)
in pages ``[pages, page, kv_heads, D]`` with one float32 scale for each
``block`` consecutive tokens of a page and each kv head.  Four operators:

* ``plan``       block tables, slot maps and the free-page ring of a serving
                 step from the requests' lengths;
* ``append``     quantises new K/V rows into their slots; a block that already
                 holds tokens keeps one scale, so a larger row raises the
                 scale and the block's earlier codes are rounded again;
* ``read``       the values that given slots hold, as bfloat16;
* ``attention``  causal attention of packed query rows over the cache: one
                 query per sequence (decode), a few (multi-token verify), or
                 a prefill chunk.

Lengths come from the case alone (``lens`` seeds them), so that ``work`` can
count them; everything else comes from the seed.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

TINY = 2.0 ** -100  # least magnitude a block's scale is made for
KINDS = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def listed():
    return [
        # one decode step of the 16-sequence serving batch: every request grows by one token
        {"name": "plan decode 16", "op": "plan", "batch": 16, "page": 64, "max_pages": 512, "lo": 1024, "hi": 32768,
         "prompt": 0, "lens": 1},
        # a continuous-batching step: mostly decodes, some prompts admitted, some requests released
        {"name": "plan mixed 512", "op": "plan", "batch": 512, "page": 64, "max_pages": 256, "lo": 1, "hi": 12000,
         "prompt": 1000, "lens": 2},
        # one decoded token for each of 64 sequences, the batch of the decode layer
        {"name": "append decode 64", "op": "append", "kind": "int8", "batch": 64, "page": 64, "block": 64, "kv": 2,
         "dim": 256, "lo": 1, "hi": 4096, "new_lo": 1, "new_hi": 1, "fused": False, "lens": 3},
        # the 5,000-token prefill chunk of one sequence, continuing a part-filled block
        {"name": "append chunk 5000", "op": "append", "kind": "int8", "batch": 1, "page": 64, "block": 64, "kv": 2,
         "dim": 256, "lo": 1237, "hi": 1237, "new_lo": 5000, "new_hi": 5000, "fused": False, "lens": 4},
        # ragged prompts, K and V as slices of a fused projection's rows, small pages
        {"name": "append ragged e4m3", "op": "append", "kind": "e4m3", "batch": 37, "page": 16, "block": 16, "kv": 8,
         "dim": 128, "lo": 0, "hi": 900, "new_lo": 1, "new_hi": 701, "fused": True, "lens": 5},
        # a 32k sequence's cache taken out whole (migration, a bfloat16 consumer)
        {"name": "read 32768", "op": "read", "kind": "int8", "rows": 32768, "page": 64, "block": 64, "kv": 2, "dim": 256},
        # a short odd piece of a cache with large pages
        {"name": "read 333 e4m3", "op": "read", "kind": "e4m3", "rows": 333, "page": 256, "block": 32, "kv": 4, "dim": 256},
        # the paged decode benchmark's shape: 16 sequences of 1k to 32k tokens
        {"name": "decode 16 x 1k-32k", "op": "attention", "kind": "int8", "batch": 16, "page": 64, "block": 64, "kv": 2,
         "group": 8, "dim": 256, "lo": 1024, "hi": 32768, "q_lo": 1, "q_hi": 1, "lens": 6},
        # one user, 1,000 tokens, the heads and page size of the attention selftest: latency
        {"name": "decode 1 x 1000", "op": "attention", "kind": "int8", "batch": 1, "page": 256, "block": 64, "kv": 4,
         "group": 6, "dim": 256, "lo": 1000, "hi": 1000, "q_lo": 1, "q_hi": 1, "lens": 7},
        # many short sequences, empty and one-token ones among them, small pages
        {"name": "decode 64 odd e4m3", "op": "attention", "kind": "e4m3", "batch": 64, "page": 16, "block": 16, "kv": 8,
         "group": 4, "dim": 128, "lo": 0, "hi": 5003, "q_lo": 1, "q_hi": 1, "lens": 8},
        # verify of up to 8 drafted tokens per sequence
        {"name": "verify 16 x 8", "op": "attention", "kind": "int8", "batch": 16, "page": 64, "block": 64, "kv": 2,
         "group": 8, "dim": 256, "lo": 1024, "hi": 16384, "q_lo": 1, "q_hi": 8, "lens": 9},
        # the 5,000-token prefill chunk
        {"name": "prefill 5000", "op": "attention", "kind": "int8", "batch": 1, "page": 64, "block": 64, "kv": 2,
         "group": 8, "dim": 256, "lo": 5000, "hi": 5000, "q_lo": 5000, "q_hi": 5000, "lens": 10},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "read", "attention", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128, 256])
    c = {"op": op, "page": page}
    if op == "plan":
        hi = _log(rng, 64, 32768)
        return dict(c, batch=_log(rng, 1, 600), max_pages=-(-(hi + 2000) // page), lo=rng.choice([0, 1]), hi=hi,
                    prompt=rng.choice([0, 1, _log(rng, 1, 1200)]), lens=rng.randrange(1 << 20))
    c.update(kind=rng.choice(sorted(KINDS)), block=rng.choice([b for b in (16, 32, 64, 128) if page % b == 0]),
             kv=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128, 256]))
    width = c["kv"] * c["dim"]
    if op == "read":
        return dict(c, rows=_log(rng, 1, min(60000, 32768 * 512 // width)))
    if op == "append":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, 5000 * 512 // (width * batch)))
        return dict(c, batch=batch, lo=0, hi=_log(rng, 1, 1000), new_lo=rng.choice([0, 1]), new_hi=hi,
                    fused=rng.random() < 0.5, lens=rng.randrange(1 << 20))
    batch = _log(rng, 1, 64)
    c.update(batch=batch, group=rng.choice([1, 2, 3, 4, 6, 8, 8, 12, 16]), lens=rng.randrange(1 << 20))
    form = rng.choice(["decode", "decode", "verify", "chunk"])
    heads = c["kv"] * c["group"]
    most = 250_000 * 512 // (width * batch)  # tokens a sequence may hold
    if form == "decode":
        hi, q_hi = _log(rng, 2, max(3, min(32768, most))), 1
    elif form == "verify":
        q_hi = rng.randint(2, 8)
        hi = _log(rng, q_hi + 1, max(q_hi + 2, min(16384, most)))
    else:  # at most half the largest case's padded scores, which the plain form holds whole
        q_hi = min(_log(rng, 16, 2000), most, int(math.sqrt(2e8 / (heads * batch))))
        hi = max(q_hi, min(most, int(2e8 / (heads * batch * q_hi)), 16384))
    return dict(c, lo=rng.choice([0, 1, hi // 2]) if form == "decode" else q_hi, hi=hi, q_lo=1, q_hi=q_hi)


def _lengths(case):
    """(tokens held after the call, new or query tokens) of every sequence, from the case alone."""
    r = random.Random(case["lens"])
    n = case["batch"]
    held = [r.randint(case["lo"], case["hi"]) for _ in range(n)]
    if case["op"] == "append":
        new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(n)]
        new[0] = max(new[0], 1)
        return [h + m for h, m in zip(held, new)], new
    new = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(n)]
    if n >= 4 and case["lo"] == 0:  # an empty sequence and a one-token one
        held[1], held[2] = 0, min(1, case["hi"])
    return held, new


def _plan_lengths(case):
    r = random.Random(case["lens"])
    n, cap = case["batch"], case["page"] * case["max_pages"]
    held = [r.randint(case["lo"], case["hi"]) for _ in range(n)]
    new, gone = [1] * n, [0] * n
    if case["prompt"]:
        for b in range(n):
            u = r.random()
            if u < 0.06:  # a finished request; its row starts another one at once, or stays empty
                gone[b], new[b] = 1, r.choice([0, r.randint(1, case["prompt"])])
            elif u < 0.10:
                new[b] = r.randint(1, case["prompt"])
            elif u < 0.14:
                new[b] = 0
    held = [min(h, cap - m) for h, m in zip(held, new)]
    return held, new, gone


def _cuda(a, dtype):
    return torch.tensor(a, dtype=dtype, device="cuda")


def _quantise(x, block, kind):
    """Codes and scales of x [tokens, heads, D], tokens a multiple of block."""
    dtype, top = KINDS[kind]
    t, h, d = x.shape
    b = x.view(t // block, block, h, d)
    s = b.abs().amax((1, 3)).clamp_min(TINY) / top
    y = (b * (1.0 / s)[:, None, :, None]).clamp(-top, top)
    return (y.round() if kind == "int8" else y).to(dtype).view(t, h, d), s


def _pool(case, pages, g):
    """A cache whose every slot holds something: keys with uneven channels, values evenly spread."""
    page, block, kv, d = case["page"], case["block"], case["kv"], case["dim"]
    got = []
    for gain in (torch.exp(0.5 * torch.randn(kv, d, device="cuda", generator=g)), torch.ones(kv, d, device="cuda")):
        codes = torch.empty(pages * page, kv, d, dtype=KINDS[case["kind"]][0], device="cuda")
        scales = torch.empty(pages * page // block, kv, device="cuda")
        step = max(page, (1 << 26) // (kv * d) // page * page)
        for at in range(0, pages * page, step):
            n = min(step, pages * page - at)
            x = (torch.randn(n, kv, d, device="cuda", generator=g) * gain).bfloat16().float()
            codes[at:at + n], scales[at // block:(at + n) // block] = _quantise(x, block, case["kind"])
        got += [codes.view(pages, page, kv, d), scales.view(pages, page // block, kv)]
    return {"k_cache": got[0], "k_scale": got[1], "v_cache": got[2], "v_scale": got[3]}


def _tables(case, held, g, spare=3):
    """A block table of randomly placed pages for sequences of these lengths."""
    page = case["page"]
    need = [-(-h // page) for h in held]
    pages = sum(need) + spare
    perm = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    at = np.concatenate([[0], np.cumsum(need)])
    table = torch.full((len(held), max(max(need), 1) + 1), -1, dtype=torch.int32, device="cuda")
    rows = torch.from_numpy(np.repeat(np.arange(len(held)), need)).cuda()
    cols = torch.from_numpy(np.arange(at[-1]) - np.repeat(at[:-1], need)).cuda()
    table[rows, cols] = perm[: int(at[-1])]
    return table, pages, rows, cols


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    if op == "plan":
        held, new, gone = _plan_lengths(case)
        page = case["page"]
        spare = sum(-(-m // page) + 1 for m in new)
        short, pages, _, _ = _tables(case, held, g, spare)
        table = torch.full((len(held), case["max_pages"]), -1, dtype=torch.int32, device="cuda")
        w = min(short.shape[1], case["max_pages"])
        table[:, :w] = short[:, :w]
        free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        taken = torch.zeros(pages, dtype=torch.bool, device="cuda")
        taken[short[short >= 0].long()] = True
        left = torch.nonzero(~taken).view(-1).to(torch.int32)
        left = left[torch.randperm(spare, device="cuda", generator=g)]
        head = seed * 7919 % pages  # the ring's first free page lies anywhere
        free[(head + torch.arange(spare, device="cuda")) % pages] = left
        return {"op": op, "page": page, "max_tokens": max(1, -(-sum(new) // 256) * 256 if case["prompt"] else len(new)),
                "seq_lens": _cuda(held, torch.int32), "new_lens": _cuda(new, torch.int32),
                "release": _cuda(gone, torch.int32), "block_table": table, "free_pages": free,
                "free_state": _cuda([head, spare], torch.int32)}
    page, block, kv, d = case["page"], case["block"], case["kv"], case["dim"]
    s = {"op": op, "kind": case["kind"], "page": page, "block": block}
    if op == "read":
        rows = case["rows"]
        s.update(_pool(case, -(-rows // page) + 2, g))
        order = torch.randperm(s["k_cache"].shape[0], device="cuda", generator=g)
        t = torch.arange(rows, device="cuda")
        s["slots"] = order[t // page] * page + t % page
        if rows > 8:
            s["slots"][rows // 2] = -1  # a token that was never given a slot
        return s
    held, new = _lengths(case)
    table, pages, rows, cols = _tables(case, held, g)
    s.update(_pool(case, pages, g))
    cu = np.concatenate([[0], np.cumsum(new)])
    total = int(cu[-1])
    if op == "append":
        seq = np.repeat(np.arange(len(new)), new)
        pos = np.arange(total) - cu[seq] + np.array(held)[seq] - np.array(new)[seq]
        seq_d, pos_d = torch.from_numpy(seq).cuda(), torch.from_numpy(pos).cuda()
        s["slot_map"] = table[seq_d, pos_d // page].long() * page + pos_d % page
        # every written slot of the blocks that the call touches
        first = [(h - m) // block * block for h, m in zip(held, new)]
        count = [h - f if m else 0 for h, m, f in zip(held, new, first)]
        seq = np.repeat(np.arange(len(new)), count)
        at = np.concatenate([[0], np.cumsum(count)])
        pos = np.arange(int(at[-1])) - at[seq] + np.array(first)[seq]
        seq_d, pos_d = torch.from_numpy(seq).cuda(), torch.from_numpy(pos).cuda()
        s["slots"] = table[seq_d, pos_d // page].long() * page + pos_d % page
        s["blocks"] = torch.unique(s["slot_map"] // block)
        # most new rows lie within the range of those held; one in a few raises its block's scale
        x = torch.randn(2, total, kv, d, device="cuda", generator=g)
        x *= torch.exp(0.3 * torch.randn(2, total, kv, 1, device="cuda", generator=g))
        if case["fused"]:
            row = torch.empty(total, 3 * kv * d, dtype=torch.bfloat16, device="cuda")
            row[:, kv * d:] = x.transpose(0, 1).reshape(total, 2 * kv * d).bfloat16()
            s["k"], s["v"] = row[:, kv * d:].view(total, 2, kv, d).unbind(1)
        else:
            s["k"], s["v"] = x[0].bfloat16(), x[1].bfloat16()
        return s
    s["block_table"], s["context_lens"] = table, _cuda(held, torch.int32)
    s["cu_q"] = None if case["q_hi"] == 1 else _cuda(cu.tolist(), torch.int32)
    s["n_max"], s["l_max"] = max(new), max(max(held), 1)
    s["q"] = torch.randn(total, kv * case["group"], d, device="cuda", generator=g).bfloat16()
    s["scale"] = d ** -0.5
    return s


# ---- the plain forms ----


def _plain_plan(s):
    page, cap = s["page"], s["max_tokens"]
    table, dev = s["block_table"], s["block_table"].device
    batch, width = table.shape
    num = s["free_pages"].shape[0]
    gone = s["release"] != 0
    had = s["seq_lens"].long()
    new = s["new_lens"].long()
    before = torch.where(gone, 0, had)
    pages0 = (before + page - 1) // page
    fits = before + new <= width * page
    need = torch.where(fits, (before + new + page - 1) // page - pages0, 0)
    want = torch.where(fits, new, 0)
    head, count = s["free_state"][0].long(), s["free_state"][1].long()
    c = need.cumsum(0)
    ok = fits & ((need == 0) | (c <= count)) & ((want == 0) | (want.cumsum(0) <= cap))
    n, need_ok = torch.where(ok, new, 0), torch.where(ok, need, 0)
    start = c - need
    lens = before + n
    # tables: a released row is cleared, then the new pages follow those held
    col = torch.arange(width, device=dev)[None]
    k = col - pages0[:, None]
    take = (k >= 0) & (k < need_ok[:, None])
    given = s["free_pages"][(head + start[:, None] + k.clamp_min(0)) % num]
    out = torch.where(take, given, torch.where(gone[:, None], -1, table))
    # released pages go to the ring's end, in the order of the sequences
    back = torch.where(gone, (had + page - 1) // page, 0).clamp_max(width)
    rb = back.cumsum(0)
    total_back = rb[-1]
    ring = s["free_pages"]
    i = torch.arange(num, device=dev)
    b = torch.searchsorted(rb, i, right=True).clamp_max(batch - 1)
    j = (i - (rb - back)[b]).clamp(0, width - 1)
    at = (head + count + i) % num
    ring[at] = torch.where(i < total_back, table[b, j], ring[at])
    used = need_ok.sum()
    state = torch.stack([(head + used) % num, count - used + total_back]).to(torch.int32)
    # packed tokens
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), n.cumsum(0)])
    t = torch.arange(cap, device=dev)
    seq = torch.searchsorted(cu, t, right=True) - 1
    live = t < cu[-1]
    q = seq.clamp(0, batch - 1)
    pos = before[q] + t - cu[q]
    slot = out[q, (pos // page).clamp(0, width - 1)].long() * page + pos % page
    return {"block_table": out, "seq_lens": lens.to(torch.int32), "free_pages": ring, "free_state": state,
            "slot_map": torch.where(live, slot, -1), "token_seq": torch.where(live, q, -1).to(torch.int32),
            "positions": torch.where(live, pos, -1).to(torch.int32), "cu_new": cu.to(torch.int32),
            "admitted": ok.to(torch.int32)}


def _plain_store(x, slots, blocks, codes, scales, block, kind):
    dtype, top = KINDS[kind]
    kv, d = codes.shape[2:]
    flat, sc = codes.view(-1, block, kv, d), scales.view(-1, kv)
    x = x.float()
    of = slots // block
    peak = torch.zeros(sc.shape, device=x.device).index_reduce_(0, of, x.abs().amax(-1), "amax")[blocks]
    start = torch.full((sc.shape[0],), block, device=x.device).index_reduce_(0, of, slots % block, "amin")[blocks]
    old = torch.where(start[:, None] > 0, sc[blocks], 0.0)
    new = torch.maximum(old, peak.clamp_min(TINY) / top)
    held = flat[blocks]
    again = (held.float() * (old / new)[:, None, :, None]).clamp(-top, top)
    again = (again.round() if kind == "int8" else again).to(dtype)
    earlier = torch.arange(block, device=x.device)[None] < start[:, None]
    bits = torch.where(earlier[:, :, None, None], again.view(torch.uint8), held.view(torch.uint8))
    flat.view(torch.uint8)[blocks] = bits
    sc[blocks] = new
    y = (x * (1.0 / sc)[of][:, :, None]).clamp(-top, top)
    y = (y.round() if kind == "int8" else y).to(dtype)
    codes.view(torch.uint8).view(-1, kv, d)[slots] = y.view(torch.uint8)


def _plain_values(slots, codes, scales, block):
    kv, d = codes.shape[2:]
    at = slots.clamp_min(0)
    x = codes.view(torch.uint8).view(-1, kv, d)[at].view(codes.dtype).float() * scales.view(-1, kv)[at // block][..., None]
    return torch.where(slots.view(*slots.shape, 1, 1) >= 0, x, 0.0)


def _plain_attention(s):
    q, table, ctx, page = s["q"], s["block_table"], s["context_lens"].long(), s["page"]
    rows, heads, d = q.shape
    kv = s["k_cache"].shape[2]
    batch, group, dev = table.shape[0], heads // kv, q.device
    cu = torch.arange(batch + 1, device=dev) if s["cu_q"] is None else s["cu_q"].long()
    n_max, l_max = s["n_max"], s["l_max"]
    i, j = torch.arange(n_max, device=dev), torch.arange(l_max, device=dev)
    here = table[:, (j // page).clamp_max(table.shape[1] - 1)].long()
    slots = torch.where(here >= 0, here * page + j % page, -1)
    k = _plain_values(slots, s["k_cache"], s["k_scale"], s["block"]).permute(0, 2, 3, 1)
    qq = q[(cu[:-1, None] + i).clamp_max(rows - 1)].float().view(batch, n_max, kv, group, d)
    qq = qq.permute(0, 2, 1, 3, 4).reshape(batch, kv, n_max * group, d)
    w = (qq @ k) * s["scale"]
    last = (ctx - cu.diff())[:, None] + i  # the position of query i
    seen = (j <= last[..., None]) & (slots >= 0)[:, None]
    seen = seen[:, None, :, None].expand(batch, 1, n_max, group, l_max).reshape(batch, 1, n_max * group, l_max)
    w = w.masked_fill_(~seen, -math.inf)
    m = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    v = _plain_values(slots, s["v_cache"], s["v_scale"], s["block"]).permute(0, 2, 1, 3)
    total = w.sum(-1, keepdim=True)
    o = (w @ v) / torch.where(total > 0, total, 1.0)
    o = o.view(batch, kv, n_max, group, d).permute(0, 2, 1, 3, 4).reshape(batch, n_max, heads, d)
    t = torch.arange(rows, device=dev)
    b = torch.searchsorted(cu, t, right=True) - 1
    return o[b, t - cu[b]].bfloat16()


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "macqwen-releases_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from flashnext_b200 import paged_q8

    return paged_q8


def run(s):
    op = s["op"]
    if not own:
        if op == "plan":
            return _plain_plan(s)
        if op == "attention":
            return _plain_attention(s)
        if op == "append":
            for x in "kv":
                _plain_store(s[x], s["slot_map"], s["blocks"], s[x + "_cache"], s[x + "_scale"], s["block"], s["kind"])
        k, v = (_plain_values(s["slots"], s[x + "_cache"], s[x + "_scale"], s["block"]).bfloat16() for x in "kv")
        return {"k": k, "v": v} if op == "read" else {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    q8 = _framework()
    if op == "plan":
        p = q8.page_plan(s["seq_lens"], s["new_lens"], s["block_table"], s["free_pages"], s["free_state"], s["page"],
                         s["max_tokens"], release=s["release"], out=s.get("plan"))
        s["plan"] = p  # a serving loop writes every step's plan into the same buffers
        return {"block_table": p.block_table, "seq_lens": p.seq_lens, "free_pages": p.free_pages,
                "free_state": p.free_state, "slot_map": p.slot_map, "token_seq": p.token_seq,
                "positions": p.positions, "cu_new": p.cu_new, "admitted": p.admitted}
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if op == "attention":
        return q8.paged_attention_q8(s["q"], *cache, s["block_table"], s["context_lens"], s["scale"], cu_q=s["cu_q"])
    if op == "append":
        q8.kv_append_q8(s["k"], s["v"], s["slot_map"], *cache)
    k, v = q8.kv_read_q8(s["slots"], *cache)
    return {"k": k, "v": v} if op == "read" else {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def work(case):
    op = case["op"]
    if op == "plan":
        held, new, gone = _plan_lengths(case)
        n, page = len(held), case["page"]
        cells = 2 * n * case["max_pages"]  # the table, in and out
        moved = sum(2 * (-(-h // page)) for h, x in zip(held, gone) if x)
        cap = max(1, -(-sum(new) // 256) * 256 if case["prompt"] else n)
        return {"bytes": 4 * (cells + moved + 6 * n) + 16 * cap, "flops": 0}
    row = case["kv"] * case["dim"]
    if op == "read":
        return {"bytes": case["rows"] * (2 * row * 3 + 8), "flops": 2 * case["rows"] * row}
    held, new = _lengths(case)
    block = case["block"]
    scales = lambda t: 2 * 4 * case["kv"] * -(-t // block)  # noqa: E731
    if op == "append":  # rows in, codes out, their scales; then the touched blocks as values
        old = sum((h - m) % block for h, m in zip(held, new) if m)
        t = sum(new)
        touched = old + t
        return {"bytes": t * (2 * row * 3 + 8) + 2 * scales(touched) + touched * (2 * row * 3 + 8), "flops": 8 * t * row}
    heads = case["kv"] * case["group"]
    pairs = sum(m * max(h - m, 0) + min(h, m) * (min(h, m) + 1) // 2 for h, m in zip(held, new))
    held_sum = sum(held)
    return {"bytes": held_sum * 2 * row + scales(held_sum) + 4 * sum(new) * heads * case["dim"],
            "flops": 4 * pairs * heads * case["dim"]}


# ---- 64 bits ----


def _f64(codes, scales, slot, block):
    """The values of one slot list, exactly."""
    kv, d = codes.shape[2:]
    c = codes.view(torch.uint8).reshape(-1, kv, d)[slot].view(codes.dtype)
    return c.to(torch.float32).double() * scales.reshape(-1, kv)[torch.div(slot, block, rounding_mode="floor")].double()[:, :, None]


def _round64(y, kind):
    """The nearest code's value, ties to even, of each element of a float64 array."""
    if kind == "int8":
        return np.clip(np.rint(y), -127, 127)
    a = np.minimum(np.abs(y), 448.0)
    e = np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -12))), -6)
    step = 2.0 ** (e - 3)
    return np.sign(y) * np.minimum(np.rint(a / step) * step, 448.0)


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None
    s = prepare(case, seed)
    block = case["block"]
    if op == "read":
        got = {}
        for x in "kv":
            y = torch.zeros(case["rows"], case["kv"], case["dim"], dtype=torch.float64, device="cuda")
            there = torch.nonzero(s["slots"] >= 0).view(-1)
            y[there] = _f64(s[x + "_cache"], s[x + "_scale"], s["slots"][there], block)
            got[x] = y
        return got
    if op == "append":
        top = KINDS[case["kind"]][1]
        slots, read = s["slot_map"].cpu().numpy(), s["slots"].cpu().numpy()
        got = {}
        for x in "kv":
            scale = s[x + "_scale"].double().cpu().numpy().reshape(-1, case["kv"])
            rows = s[x].double().cpu().numpy()
            members = {}
            for t, slot in enumerate(slots.tolist()):
                members.setdefault(slot // block, []).append(t)
            values = {}
            for b, ts in members.items():
                first = int(slots[ts[0]] % block)
                r = rows[ts]
                sc = np.maximum(np.abs(r).max((0, 2)), TINY) / top
                if first:
                    sc = np.maximum(sc, scale[b])
                    idx = torch.arange(b * block, b * block + first, device="cuda")
                    before = _f64(s[x + "_cache"], torch.ones_like(s[x + "_scale"]), idx, block).cpu().numpy()
                    for k in range(first):
                        values[b * block + k] = _round64(before[k] * (scale[b] / sc)[:, None], case["kind"]) * sc[:, None]
                for t in ts:
                    values[int(slots[t])] = _round64(rows[t] / sc[:, None], case["kind"]) * sc[:, None]
                scale[b] = sc
            got[x] = np.stack([values[i] for i in read.tolist()])
            got[x + "_scale"] = scale.reshape(s[x + "_scale"].shape)
        return got
    held, new = _lengths(case)
    heads, kv, d, page = case["kv"] * case["group"], case["kv"], case["dim"], case["page"]
    out = torch.zeros(sum(new), heads, d, dtype=torch.float64, device="cuda")
    at = 0
    for b, (h, m) in enumerate(zip(held, new)):
        if h:
            slot = (s["block_table"][b, : -(-h // page)].long()[:, None] * page + torch.arange(page, device="cuda")).view(-1)[:h]
            k, v = (_f64(s[x + "_cache"], s[x + "_scale"], slot, block) for x in "kv")
            for lo in range(0, m, 512):
                n = min(512, m - lo)
                q = s["q"][at + lo:at + lo + n].double().view(n, kv, case["group"], d)
                z = torch.einsum("ikgd,jkd->kgij", q, k) / math.sqrt(d)
                future = torch.arange(h, device="cuda") > (torch.arange(lo, lo + n, device="cuda") + h - m)[:, None]
                p = torch.softmax(z.masked_fill(future, -1e300), -1).masked_fill(future, 0.0)
                out[at + lo:at + lo + n] = torch.einsum("kgij,jkd->ikgd", p, v).reshape(n, heads, d)
        at += m
    return out
