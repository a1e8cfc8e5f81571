"""A small decoder served token by token, from embedding row to next token.

    python macqwen-releases_b200/examples/decode_step.py [--tokens 32] [--eager]

Two layers of attention over the paged 8-bit KV cache and of sparse-MoE blocks,
with random weights: embedding rows, norms that add the residual and write 8-bit
rows, 8-bit query/key/value and output projections, the MoE block, the head and
the draw of the next token.  Prompts of random lengths are prefilled packed; the
decode steps are replayed from a CUDA graph (two steps in one graph: a cache's
tables alternate between two sets of buffers) and fed by nothing but the step's
uniform numbers.  Rotary positions are left out.
"""
from __future__ import annotations

import argparse
import random
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from flashnext_b200 import synthetic  # noqa: E402
from flashnext_b200.dense import add_rms_norm, linear, quantize_rows  # noqa: E402
from flashnext_b200.moe_block import SparseMoEBlock  # noqa: E402
from flashnext_b200.ngram import StreamingQuantizedEmbedding  # noqa: E402
from flashnext_b200.paged_q8 import PagedKVCacheQ8  # noqa: E402
from flashnext_b200.sampling import sample  # noqa: E402

HIDDEN, INTER, EXPERTS, TOP_K, VOCAB = 1024, 256, 32, 4, 4003
HEADS, KV, DIM, PAGE, PAGES = 8, 2, 128, 64, 8


class Layer:
    def __init__(self, batch, seed, gen):
        def weight(n, k):
            return quantize_rows(torch.randn(n, k, device="cuda", generator=gen) * k ** -0.5)

        self.attention_norm = 1 + 0.1 * torch.randn(HIDDEN, device="cuda", generator=gen)
        self.block_norm = 1 + 0.1 * torch.randn(HIDDEN, device="cuda", generator=gen)
        self.qkv, self.out = weight((HEADS + 2 * KV) * DIM, HIDDEN), weight(HIDDEN, HEADS * DIM)
        moe = synthetic.moe_layer(1, hidden=HIDDEN, inter=INTER, num_experts=EXPERTS, top_k=TOP_K, seed=seed)
        self.moe = SparseMoEBlock(moe.router_weight, moe.experts, top_k=TOP_K, shared=moe.shared,
                                  shared_expert_gate=moe.shared_expert_gate)
        self.cache = PagedKVCacheQ8(batch * PAGES, PAGE, KV, DIM, PAGES, batch, max_tokens=batch * PAGE)

    def __call__(self, x, residual, new_lens, release, one_row):
        """x [rows, HIDDEN] is what the last layer adds to ``residual`` (float32) -> the same of this layer."""
        n = add_rms_norm(x, self.attention_norm, residual, codes=torch.int8)
        qkv = linear(n.codes, self.qkv[0], x_scale=n.scales, weight_scale=self.qkv[1]).view(-1, HEADS + 2 * KV, DIM)
        q, k, v = qkv.split((HEADS, KV, KV), 1)
        self.cache.plan(new_lens, release)
        self.cache.append(k, v)
        a = self.cache.attention(q, DIM ** -0.5, one_row=one_row)
        codes, scales = quantize_rows(a.view(-1, HEADS * DIM))
        residual = linear(codes, self.out[0], residual=n.residual, x_scale=scales, weight_scale=self.out[1],
                          out_dtype=torch.float32)
        y = add_rms_norm(residual, self.block_norm, unit_offset=False).y.bfloat16()
        return self.moe(y), residual


class Decoder:
    def __init__(self, batch, seed=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        w, s, b = synthetic.q4_projection(1, VOCAB, HIDDEN, seed=seed + 7, scale_std=0.05)
        self.embed = StreamingQuantizedEmbedding.from_arrays(w[0], s[0], b[0], HIDDEN)
        self.layers = [Layer(batch, seed + i, gen) for i in range(2)]
        self.norm = torch.ones(HIDDEN, dtype=torch.bfloat16, device="cuda")
        self.head = (torch.randn(VOCAB, HIDDEN, device="cuda", generator=gen) * 4 * HIDDEN ** -0.5).bfloat16()

    def __call__(self, tokens, new_lens, release, uniform, last=None):
        """The next token of every sequence from packed ``tokens``; ``last``: each sequence's last row among them."""
        x = self.embed(tokens)
        residual = torch.zeros(x.shape, device="cuda")
        for layer in self.layers:
            x, residual = layer(x, residual, new_lens, release, last is None)
        if last is not None:
            x, residual = x[last], residual[last]
        y = add_rms_norm(x, self.norm, residual).y
        logits = linear(y, self.head, out_dtype=torch.float32)
        return sample(logits, uniform, temperature=0.8, top_k=50, top_p=0.95, min_p=0.02)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--eager", action="store_true", help="launch every step from Python")
    a = ap.parse_args(argv)
    rng, i32 = random.Random(a.seed), torch.int32
    gen = torch.Generator(device="cuda")
    gen.manual_seed(a.seed)
    model = Decoder(a.batch, a.seed)
    lens = [rng.randint(1, PAGE) for _ in range(a.batch)]
    steps = min(a.tokens, PAGE * PAGES - max(lens)) // 2 * 2
    uniform = torch.rand(1 + steps, a.batch, device="cuda", generator=gen)
    none = torch.zeros(a.batch, dtype=i32, device="cuda")
    new = torch.tensor(lens, dtype=i32, device="cuda")
    prompt = torch.randint(VOCAB, (sum(lens),), device="cuda", generator=gen)
    token, logprob = model(prompt, new, none, uniform[0], last=new.cumsum(0) - 1)
    one, out, scores = torch.ones_like(none), [token], [logprob]

    def two(token, u):
        got = []
        for i in range(2):
            got.append(model(token, one, none, u[i]))
            token = got[-1][0]
        return [torch.stack(t) for t in zip(*got)]

    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    if a.eager:
        begin.record()
        for i in range(1, 1 + steps, 2):
            t, s = two(out[-1], uniform[i:i + 2])
            out += t.unbind()
            scores += s.unbind()
    else:
        held, u = token.clone(), uniform[1:3].clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):  # captured, not run: the caches stay as they are
            t, s = two(held, u)
        begin.record()
        for i in range(1, 1 + steps, 2):
            u.copy_(uniform[i:i + 2])
            graph.replay()
            held.copy_(t[1])
            out += t.clone().unbind()
            scores += s.clone().unbind()
    end.record()
    torch.cuda.synchronize()
    if steps:
        print(f"{a.batch} sequences, {steps} steps, {1e3 * begin.elapsed_time(end) / steps:.0f} us a step, "
              f"mean log-probability {float(torch.stack(scores).mean()):.3f}")
    return torch.stack(out), torch.stack(scores)


if __name__ == "__main__":
    main()
