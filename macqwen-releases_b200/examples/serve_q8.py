"""One attention layer served over the paged 8-bit KV cache.

    python macqwen-releases_b200/examples/serve_q8.py [--steps 64] [--codes int8|e4m3]

Requests of random lengths arrive, are prefilled, decode token by token, end
and make room for others, all through the device: each step plans pages and
slots (``PagedKVCacheQ8.plan``), stores the step's K/V rows and attends with
its packed queries.  The host keeps only what it knows anyway, how many tokens
each request still wants.  At the end one sequence's attention is compared
with attention over the bfloat16 rows that were stored.
"""
from __future__ import annotations

import argparse
import random
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from flashnext_b200.paged_q8 import PagedKVCacheQ8  # noqa: E402


def main(argv=None) -> float:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--codes", choices=("int8", "e4m3"), default="int8")
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    batch, kv, group, dim, page, width = 16, 2, 8, 256, 64, 64
    codes = torch.int8 if a.codes == "int8" else torch.float8_e4m3fn
    cache = PagedKVCacheQ8(batch * width, page, kv, dim, width, batch, max_tokens=8192, codes=codes)
    rng = random.Random(a.seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(a.seed)
    left = [0] * batch                # tokens that each row's request still decodes
    kept = [[] for _ in range(batch)]  # row 0's stored rows, for the check
    out, tokens = None, 0
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(a.steps):
        new, gone = [], []
        for b in range(batch):
            ended = left[b] == 0
            gone.append(int(ended))
            new.append(rng.randint(1, 400) if ended else 1)
            left[b] = rng.randint(8, 64) if ended else left[b] - 1
            if ended:
                kept[b] = []
        n = sum(new)
        cache.plan(torch.tensor(new, dtype=torch.int32, device="cuda"),
                   torch.tensor(gone, dtype=torch.int32, device="cuda"))
        # where a model would project its hidden states
        qkv = torch.randn(n, (group + 2) * kv, dim, device="cuda", generator=gen).bfloat16()
        q, k, v = qkv.split((group * kv, kv, kv), 1)
        cache.append(k, v)
        out = cache.attention(q, dim ** -0.5)
        kept[0].append((k[: new[0]], v[: new[0]], q[: new[0]]))
        last0, tokens = new[0], tokens + n
    end.record()
    torch.cuda.synchronize()
    assert cache.last.admitted.all()
    k, v = (torch.cat([s[i] for s in kept[0]]).double() for i in range(2))
    q = kept[0][-1][2].double().view(last0, kv, group, dim)
    s = torch.einsum("ikgd,jkd->kgij", q, k) * dim ** -0.5
    at = torch.arange(k.shape[0], device="cuda")
    s = s.masked_fill(at > (at[-1] - last0 + 1 + torch.arange(last0, device="cuda"))[:, None], float("-inf"))
    want = torch.einsum("kgij,jkd->ikgd", s.softmax(-1), v).reshape(last0, -1, dim)
    rel = float((out[:last0].double() - want).norm() / want.norm())
    print(f"{a.steps} steps, {tokens} tokens, {begin.elapsed_time(end) / a.steps:.3f} ms a step; "
          f"sequence 0 ({k.shape[0]} tokens) is {rel:.3g} from attention over its bfloat16 rows")
    return rel


if __name__ == "__main__":
    main()
