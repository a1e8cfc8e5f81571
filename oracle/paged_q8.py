"""Paged 8-bit KV cache oracle -- TEST INFRASTRUCTURE ONLY.

Plain restatements, in loops, of the operators of ``flashnext_b200.paged_q8``:
the page plan in Python integers, the quantising append in float32 (the codes
are defined by float32 operations, so they can be held bit for bit), the
attention in float64.
"""
from __future__ import annotations

import math

import numpy as np

TINY = np.float32(2.0 ** -100)
TOP = {"int8": np.float32(127.0), "e4m3": np.float32(448.0)}


def page_plan(seq_lens, new_lens, release, table, ring, head, count, page, cap):
    """-> dict of every output; the ring is returned as a new list."""
    batch, width = len(seq_lens), len(table[0])
    ring, num = list(ring), len(ring)
    rows = [list(r) for r in table]
    pages = lambda t: -(-t // page)  # noqa: E731
    want_pages = want_tokens = given = put = total = 0
    lens, admitted, cu, slots, seqs, positions = [], [], [0], [], [], []
    back, first_count = [], count
    for b in range(batch):
        had = max(seq_lens[b], 0)
        gone = bool(release[b]) if release is not None else False
        held, n = (0 if gone else had), max(new_lens[b], 0)
        if gone:
            back += rows[b][: min(pages(had), width)]
            rows[b] = [-1] * width
        need = pages(held + n) - pages(held)
        fits = held + n <= width * page
        if fits:
            want_pages += need
            want_tokens += n
        ok = fits and (need == 0 or want_pages <= first_count) and (n == 0 or want_tokens <= cap)
        admitted.append(int(ok))
        if not ok:
            n = need = 0
        for i in range(need):
            rows[b][pages(held) + i] = ring[(head + given + i) % num]
        given += need
        for i in range(n):
            p = held + i
            pg = rows[b][p // page]
            slots.append(-1 if pg < 0 else pg * page + p % page)
            seqs.append(b)
            positions.append(p)
        total += n
        cu.append(total)
        lens.append(held + n)
    for pg in back:
        ring[(head + first_count + put) % num] = pg
        put += 1
    pad = [-1] * (cap - total)
    return {"block_table": rows, "seq_lens": lens, "free_pages": ring, "slot_map": slots + pad,
            "free_state": [(head + given) % num, min(first_count - given + put, num)], "token_seq": seqs + pad,
            "positions": positions + pad, "cu_new": cu, "admitted": admitted}


def e4m3_round(y):
    """float32 values within +-448 rounded to e4m3 values, ties to even."""
    y = np.asarray(y, np.float64)
    a = np.abs(y)
    e = np.maximum(np.frexp(np.maximum(a, 1e-300))[1] - 1, -6)
    step = np.ldexp(1.0, e - 3)
    return np.copysign(np.minimum(np.rint(a / step) * step, 448.0), y).astype(np.float32)


def encode(x, inv, kind):
    """float32 rows times inv -> code values (float32)."""
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        y = (x * np.float32(inv)).astype(np.float32)
    y = np.where(np.isnan(x), np.float32(0), np.clip(np.nan_to_num(y, nan=0.0, posinf=3e38, neginf=-3e38), -TOP[kind], TOP[kind]))
    return np.rint(y).astype(np.float32) if kind == "int8" else e4m3_round(y)


def append(x, slots, codes, scales, block, kind):
    """x [T, H, D] float32 (bf16 values); codes [slots, H, D] code values and
    scales [slots / block, H] float32 are updated in place."""
    runs = {}
    for t, s in enumerate(slots):
        if 0 <= s < codes.shape[0]:
            runs.setdefault(int(s) // block, []).append(t)
    one = np.float32(1.0)
    for b, ts in runs.items():
        first = int(slots[ts[0]]) % block
        for h in range(x.shape[1]):
            mag = np.abs(x[ts, h])
            mag = mag[np.isfinite(mag)]
            peak = max(np.float32(mag.max()) if mag.size else np.float32(0), TINY)
            old = scales[b, h] if first else np.float32(0)
            s = max(old, np.float32(peak / TOP[kind]))
            if first and s != old:
                at = slice(b * block, b * block + first)
                codes[at, h] = encode(codes[at, h], np.float32(old / s), kind)
            inv = np.float32(one / s)
            for t in ts:
                codes[slots[t], h] = encode(x[t, h], inv, kind)
            scales[b, h] = s


def attention(q, k, v, seen, scale):
    """q [R, Hq, D]; k, v [T, Hkv, D] values; seen [R, T] -> (out, mean |v|) in
    float64: the softmax-weighted means of v and of |v|; 0 where nothing is seen."""
    rows, hq, d = q.shape
    hkv = k.shape[1]
    out, mag = np.zeros((rows, hq, d)), np.zeros((rows, hq, d))
    for h in range(hq):
        kk, vv = k[:, h // (hq // hkv)].astype(np.float64), v[:, h // (hq // hkv)].astype(np.float64)
        s = np.where(seen, (q[:, h].astype(np.float64) @ kk.T) * scale, -math.inf)
        m = s.max(1, initial=-math.inf, keepdims=True)
        w = np.exp(s - np.where(np.isfinite(m), m, 0.0))
        tot = w.sum(1, keepdims=True)
        w = w / np.where(tot > 0, tot, 1.0)
        out[:, h], mag[:, h] = w @ vv, w @ np.abs(vv)
    return out, mag
