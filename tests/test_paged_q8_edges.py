"""The paged 8-bit KV cache at its edges: value scales far apart, rows of no
sequence, scratch under graphs and threads, descriptors of cut work,
tensors of another device, arrays off their alignment,
positions near 2^31, steps in which a request is refused, large batches, the weights' low terms.

Attention is held to this: an output is the bfloat16 rounding of a number within
2^-13 mean|v| of the truth, with mean|v| the weighted mean of the magnitudes.
That covers the float32 arithmetic: a weight enters the second product as two
bfloat16 terms, together within 2^-16; a score of magnitude below 64 (in log2)
is a few float32 roundings of 2^-24 off, 2^-16 of its weight; ex2, lg2 and the
reciprocal are within 2^-21; and a float32 sum of up to 5,000 terms of the matrix
instructions, 16 at a time and two for each, is within 700 * 2^-23 < 2^-13.5 in
the worst case.
"""
from __future__ import annotations

import ctypes
import threading

import numpy as np
import pytest

from flashnext_b200 import _lib
from oracle import paged_q8 as oq8
from test_paged_q8 import KINDS, _attention_args, _bf16, _cache_struct, _empty_cache, _place, _plan_args, _set, _slots

C_MAG = 2.0 ** -13


def _outside(out, want, mag, c=C_MAG):
    """How many of the bfloat16 values `out` are not the rounding of a float32
    within c * mag of `want` (rounding is monotonic)."""
    low, high = (_bf16((want + s * c * mag).astype(np.float32)).float().numpy() for s in (-1, 1))
    return int(((out < low) | (out > high) | np.isnan(out)).sum())


def _dev(a):
    import torch

    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _cache_of(table, pages, page, block, kind, k, ks, v, vs):
    """Device cache whose slots hold the code values k, v [slots, heads, dim]
    and whose blocks have the scales ks, vs [blocks, heads]."""
    import torch

    cache = _empty_cache(pages, page, block, k.shape[1], k.shape[2], kind)
    for i, (c, s) in enumerate(((k, ks), (v, vs))):
        cache[i].copy_(torch.from_numpy(c).to(cache[i].dtype).view(cache[i].shape).cuda())
        cache[2 + i].copy_(torch.from_numpy(s).view(cache[2 + i].shape))
    return cache


def _wrong(out, q, table, held, new, host, page, block, scale):
    """Outputs of all rows that are outside the bound."""
    (k, ks), (v, vs) = host
    at = wrong = 0
    for b, (h, n) in enumerate(zip(held, new)):
        if n == 0:
            continue
        slot = _slots(table, b, 0, h, page)
        kk, vv = (c[slot].astype(np.float64) * s[slot // block][:, :, None] for c, s in ((k, ks), (v, vs)))
        seen = np.arange(h)[None] <= (h - n + np.arange(n))[:, None]
        want, mag = oq8.attention(q[at:at + n], kk, vv, seen, scale)
        wrong += _outside(out[at:at + n], want, mag)
        at += n
    return wrong


FORMS = [None, [1, 40, 30], [64, 60, 70]]  # one row each; packed; packed rows of the many-row kernel alone


# ---- value scales far apart ----


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", FORMS)
@pytest.mark.parametrize("big", [-5.0, 20.0, 60.0])
@pytest.mark.parametrize("zeros_first", [True, False])
def test_blocks_of_zero_values_keep_their_share_of_the_weights(cuda_lib, kind, dim, new, big, zeros_first):
    """Half the blocks hold values of scale 2^big, half hold zeros (whose scale
    is the least that an append makes); every token scores about the same, so
    the zeros take half of the softmax."""
    from flashnext_b200.paged_q8 import paged_attention_q8

    page, block, kv, group = 16, 16, 1, 8
    held = [64, 352, 1024]
    rng = np.random.default_rng(dim + int(big) + 100)
    table, pages = _place(rng, held, page)
    n = pages * page
    k = np.ones((n, kv, dim), np.float32)
    k[:, :, 1:] = 0
    ks = np.ones((pages, kv), np.float32)
    v = rng.integers(1, 100, (n, kv, dim)).astype(np.float32)
    if kind == "e4m3":
        v = oq8.e4m3_round(v)
    vs = np.full((pages, kv), 2.0 ** big, np.float32)
    for row, h in zip(table, held):
        mine = row[: h // page]
        none = mine[: len(mine) // 2] if zeros_first else mine[1::2]
        vs[none] = oq8.TINY / oq8.TOP[kind]
        v.reshape(pages, -1)[none] = 0
    cache = _cache_of(table, pages, page, block, kind, k, ks, v, vs)
    rows = new or [1] * 3
    q = _bf16(rng.standard_normal((sum(rows), kv * group, dim)))
    cu = None if new is None else _dev(np.concatenate([[0], np.cumsum(new)]))
    out = paged_attention_q8(q.cuda(), *cache, _dev(table), _dev(held), 0.25, cu_q=cu).float().cpu().numpy()
    assert _wrong(out, q.float().numpy(), table, held, rows, ((k, ks), (v, vs)), page, block, 0.25) == 0
    assert _lib.read_device_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [None, [33]])
def test_many_light_tokens_of_zero_values_add_up(cuda_lib, kind, new):
    """One block of values of scale 8, then 65,584 zeros of 2^-17 the weight of
    its tokens each: together they take 3% of the softmax."""
    from flashnext_b200.paged_q8 import paged_attention_q8

    page = block = 16
    dim, held = 64, [65600]
    rng = np.random.default_rng(3)
    table, pages = _place(rng, held, page)
    first = table[0, 0]
    k = np.zeros((pages * page, 1, dim), np.float32)
    k[:, 0, 0] = 48
    k.reshape(pages, page, dim)[first, :, 0] = 64
    ks = np.ones((pages, 1), np.float32)
    v = np.zeros_like(k)
    v.reshape(pages, page, dim)[first] = 96
    vs = np.full((pages, 1), oq8.TINY / oq8.TOP[kind], np.float32)
    vs[first] = 8.0
    cache = _cache_of(table, pages, page, block, kind, k, ks, v, vs)
    rows = new or [1]
    q = np.zeros((sum(rows), 2, dim), np.float32)
    q[:, :, 0] = 1.0
    scale = 17.0 / 16.0 / np.log2(np.e)
    cu = None if new is None else _dev([0, rows[0]])
    out = paged_attention_q8(_bf16(q).cuda(), *cache, _dev(table), _dev(held), scale, cu_q=cu).float().cpu().numpy()
    # float32 sums of 65,600 equal weights, 64 or 128 at a time: within 1,025 * 2^-24, inside the bound
    share = 16 / (16 + (held[0] - 16 - np.arange(rows[0])[::-1]) * 2.0 ** -17)
    want = 768.0 * share[:, None, None] * np.ones_like(out)
    assert _outside(out, want, want) == 0, (out[0, 0, 0], want[0, 0, 0])


# ---- rows of no sequence ----


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [[1, 0, 2], [0, 0, 0], [3, 90, 1], [64, 60, 70]])
@pytest.mark.parametrize("extra", [1, 13, 700])
def test_rows_of_no_sequence_are_zero(cuda_lib, dim, new, extra):
    """A padded batch: q has more rows than cu_q counts."""
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    page, block, kv, group, held = 32, 16, 2, 4, [70, 95, 128]
    rng = np.random.default_rng(dim + extra + sum(new))
    table, pages = _place(rng, held, page)
    n, blocks = pages * page, pages * page // block
    k, v = (rng.integers(-100, 100, (n, kv, dim)).astype(np.float32) for _ in range(2))
    ks, vs = (np.exp(rng.standard_normal((blocks, kv))).astype(np.float32) / 50 for _ in range(2))
    cache = _cache_of(table, pages, page, block, "int8", k, ks, v, vs)
    q = _bf16(rng.standard_normal((sum(new) + extra, kv * group, dim)))
    cu = _dev(np.concatenate([[0], np.cumsum(new)]))
    out = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device="cuda")
    paged_attention_q8(q.cuda(), *cache, _dev(table), _dev(held), dim ** -0.5, cu_q=cu, out=out)
    out = out.float().cpu().numpy()
    assert (out[sum(new):] == 0).all()
    assert _wrong(out, q.float().numpy(), table, held, new, ((k, ks), (v, vs)), page, block, dim ** -0.5) == 0
    cu += 5  # the first sequence begins at row 5
    out = torch.full((q.shape[0] + 5, *q.shape[1:]), float("nan"), dtype=torch.bfloat16, device="cuda")
    q5 = torch.cat([torch.ones_like(q[:1]).expand(5, -1, -1), q])
    paged_attention_q8(q5.cuda(), *cache, _dev(table), _dev(held), dim ** -0.5, cu_q=cu, out=out)
    out = out.float().cpu().numpy()
    assert (out[:5] == 0).all() and (out[5 + sum(new):] == 0).all()
    assert _wrong(out[5:], q.float().numpy(), table, held, new, ((k, ks), (v, vs)), page, block, dim ** -0.5) == 0


@pytest.mark.gpu
def test_a_padded_step_of_the_cache_class_has_zero_rows(cuda_lib):
    import torch
    from flashnext_b200.paged_q8 import PagedKVCacheQ8

    junk = torch.full((1 << 22,), float("nan"), device="cuda")  # what the allocator hands out next
    del junk
    cache = PagedKVCacheQ8(8, 32, 1, 64, 4, 3, 64)
    cache.plan(_dev([7, 0, 20]))
    x = torch.randn(64, 1, 64, device="cuda").bfloat16()  # 27 tokens, padded to 64
    cache.append(x, x)
    out = cache.attention(x.expand(-1, 4, -1).contiguous(), 0.125)
    assert torch.isfinite(out).all() and bool((out[27:] == 0).all()) and bool((out[:27] != 0).any())


# ---- scratch ----


class _Cuda:
    """A CPU tensor that says that it is on CUDA device `index`."""

    is_cuda = True

    def __init__(self, *shape, dtype, index=0):
        import torch

        self.real, self.index = torch.zeros(shape, dtype=dtype), index

    def get_device(self):
        return self.index

    def __getattr__(self, name):
        return getattr(self.real, name)


class _Library:
    """Stands in for the C library: says what scratch a call needs and sees what it was given."""

    def __init__(self, seen=lambda args: None):
        self.seen = seen

    def fnmoe_paged_attention_q8_workspace_size(self, ref, need):
        need._obj.value = 4096 * ref._obj.q_rows
        return _lib.OK

    def fnmoe_paged_attention_q8(self, ref, stream):
        a = ref._obj
        if not a.workspace or a.workspace_bytes < 4096 * a.q_rows:
            return _lib.ERR_WORKSPACE
        self.seen(a)
        return _lib.OK


def _fake_attention(rows):
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    cache = [_Cuda(4, 32, 2, 64, dtype=torch.int8) for _ in range(2)] + [_Cuda(4, 2, 2, dtype=torch.float32) for _ in range(2)]
    paged_attention_q8(_Cuda(rows, 4, 64, dtype=torch.bfloat16), *cache, _Cuda(rows, 2, dtype=torch.int32),
                       _Cuda(rows, dtype=torch.int32), 0.125)


def test_calls_of_two_threads_on_one_stream_have_scratch_of_their_own(monkeypatch):
    import torch
    from flashnext_b200 import paged_q8

    inside, given = threading.Barrier(2), []
    lib = _Library()
    monkeypatch.setattr(paged_q8, "_ready", lambda t: (lib, 7))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    _fake_attention(3)  # whatever an earlier call may leave behind

    def seen(a):
        given.append((a.workspace, a.workspace_bytes))
        inside.wait(10)  # both calls are in the library

    lib.seen = seen
    threads = [threading.Thread(target=_fake_attention, args=(rows,)) for rows in (2, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(20)
    (a, n), (b, m) = sorted(given)
    assert a + n <= b, "two calls in flight were given the same scratch"


def test_a_captured_call_has_scratch_of_the_graphs_own(monkeypatch):
    """Allocated in the capture, by each call, and neither kept nor given to another."""
    import torch
    from flashnext_b200 import paged_q8

    made, used, capturing = [], [], [False]
    empty, new_empty = torch.empty, torch.Tensor.new_empty

    def note(t):
        made.append((t.data_ptr(), t.numel() * t.element_size(), t))  # the graph's pool keeps it
        return t

    lib = _Library(lambda a: used.append((a.workspace, a.workspace_bytes)))
    monkeypatch.setattr(paged_q8, "_ready", lambda t: (lib, 7))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(torch, "empty", lambda *a, **k: note(empty(*a, **k)))
    monkeypatch.setattr(torch.Tensor, "new_empty", lambda *a, **k: note(new_empty(*a, **k)))
    of_graphs = []
    for captured, rows in ((False, 3), (True, 3), (False, 2), (True, 2), (False, 5), (True, 5), (False, 5)):
        before, capturing[0] = len(made), captured
        _fake_attention(rows)
        at, n = used[-1]
        assert n >= 4096 * rows
        assert all(at + n <= p or p + m <= at for p, m in of_graphs), "a graph's scratch was given to another call"
        if captured:
            assert any(p <= at and at + n <= p + m for p, m, _ in made[before:]), "not the graph's own"
            of_graphs.append((at, n))


def _served(batch, held, dim=256, kv=2, seed=1):
    """A cache holding `held` tokens a sequence of random rows, by its own append."""
    import torch
    from flashnext_b200.paged_q8 import PagedKVCacheQ8

    page = 64
    cache = PagedKVCacheQ8(batch * (held // page + 4), page, kv, dim, held // page + 4, batch, batch * held)
    cache.plan(_dev([held] * batch))
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = torch.randn(2, batch * held, kv, dim, device="cuda", generator=g).bfloat16()
    cache.append(r[0], r[1])
    return cache


@pytest.mark.gpu
def test_a_captured_step_outlives_larger_calls_on_its_stream(cuda_lib):
    """Capture a decode, run a prefill that needs more scratch on the same
    stream, fill new tensors, replay: the outputs are those of an eager call and
    the tensors keep their values."""
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    cache = _served(4, 2000)
    p = cache.last
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    q = torch.randn(4, 16, 256, device="cuda", generator=g).bfloat16()
    long = torch.randn(4 * 700, 16, 256, device="cuda", generator=g).bfloat16()
    cu = _dev(700 * np.arange(5))
    args = (*cache.tensors, p.block_table, p.seq_lens, 0.0625)
    want = paged_attention_q8(q, *args)
    want_long = paged_attention_q8(long, *args, cu_q=cu)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    out = torch.empty_like(q)
    with torch.cuda.stream(s):
        paged_attention_q8(q, *args, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            paged_attention_q8(q, *args, out=out)
        assert torch.equal(paged_attention_q8(long, *args, cu_q=cu), want_long)
        torch.cuda.synchronize()
        fresh = [torch.full((n,), 7, dtype=torch.uint8, device="cuda") for n in [1 << 20] * 16 + [1 << 22] * 8 + [1 << 25] * 4]
        for _ in range(3):
            out.zero_()
            graph.replay()
            assert torch.equal(out, want)
            assert torch.equal(paged_attention_q8(long, *args, cu_q=cu), want_long)
        torch.cuda.synchronize()
        assert all(bool((t == 7).all()) for t in fresh)


@pytest.mark.gpu
def test_two_graphs_of_one_stream_may_replay_at_once(cuda_lib):
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    cache = _served(4, 3000)
    p = cache.last
    args = (*cache.tensors, p.block_table, p.seq_lens, 0.0625)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    qs = [torch.randn(4, 16, 256, device="cuda", generator=g).bfloat16() for _ in range(2)]
    wants = [paged_attention_q8(q, *args) for q in qs]
    s, outs, graphs = torch.cuda.Stream(), [torch.empty_like(q) for q in qs], []
    torch.cuda.synchronize()
    for q, out in zip(qs, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            paged_attention_q8(q, *args, out=out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for t, graph in zip(streams, graphs):
            with torch.cuda.stream(t):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, wants))


@pytest.mark.gpu
def test_two_threads_on_one_stream(cuda_lib):
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    jobs = []
    for i, (batch, held, rows) in enumerate(((3, 900, 60), (7, 300, 21))):
        cache = _served(batch, held, seed=10 + i)
        q = torch.randn(batch * rows, 16, 256, device="cuda").bfloat16()
        args = (q, *cache.tensors, cache.last.block_table, cache.last.seq_lens, 0.0625)
        cu = _dev(rows * np.arange(batch + 1))
        jobs.append((args, cu, paged_attention_q8(*args, cu_q=cu)))
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(2)

    def work(args, cu, want):
        start.wait(10)
        got = [paged_attention_q8(*args, cu_q=cu) for _ in range(50)]
        torch.cuda.synchronize()
        wrong.append(sum(not torch.equal(o, want) for o in got))

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [0, 0] and _lib.read_device_errors() == 0


# ---- descriptors of cut work ----

RANGES_CHECK = r"""
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>
#include "q8_ranges.cuh"
using namespace fnmoe;
#define CHECK(x) if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; }
int main() {
  std::mt19937_64 rng(1);
  auto pick = [&](long long lo, long long hi) { return lo + static_cast<long long>(rng() % (hi - lo + 1)); };
  // Segments laid end to end (the last `real` units of each are work, as the join sees it),
  // dealt to CTAs: each segment that several CTAs share is described exactly once, rightly.
  for (int round = 0; round < 3000; ++round) {
    const int segs = pick(1, 40), ctas = pick(1, 60), cost = round & 1 ? 6 : 0;
    std::vector<long long> begin(segs + 1);
    for (int s = 0; s < segs; ++s) begin[s + 1] = begin[s] + pick(1, pick(1, 50)) + cost;
    const Ranges r(begin[segs], ctas);
    CHECK(r.begin(0) == 0 && r.begin(ctas) == begin[segs]);
    std::vector<int> said(segs);
    for (int c = 0; c < ctas; ++c) {
      const long long at = r.begin(c);
      CHECK(r.begin(c + 1) >= at);
      if (r.begin(c + 1) == at) continue;
      CHECK(r.owner(at) == c && r.owner(r.begin(c + 1) - 1) == c);
      int s = 0;
      while (begin[s + 1] <= at) ++s;
      if (at <= begin[s] + cost) continue;  // not inside the segment's work
      const int4 cut = cut_of(r, s, 0, 3, begin[s], begin[s] + cost, begin[s + 1] - 1, c);
      if (cut.x < 0) continue;
      ++said[s];
      CHECK(cut.x == s && cut.z == 3 && cut_fits(cut, c - 1, cut.y, segs, 1, ctas));
      CHECK(last_cta(cut) == r.owner(begin[s + 1] - 1) && r.owner(begin[s] + cost) == c - 1);
      CHECK((cut.w >> 30 & 1) == (r.begin(c - 1) < begin[s]));
    }
    for (int s = 0; s < segs; ++s) CHECK(said[s] == (r.owner(begin[s] + cost) != r.owner(begin[s + 1] - 1)));
  }
  // Anything else is refused, or stays inside the arrays.
  const int batch = 5, heads = 3, ctas = 148;
  const unsigned fills[] = {0u, ~0u, 0x5A5A5A5Au, 0x7FFFFFFFu, 0x80000000u, 0x3FFFFFFFu, 0x40000000u, 1u};
  for (unsigned f : fills) {
    int4 cut;
    const unsigned w[4] = {f, f, f, f};
    std::memcpy(&cut, w, 16);
    CHECK(!cut_fits(cut, cut.y, 0, batch, heads, ctas) && !cut_fits(cut, 0, cut.y, batch, heads, ctas) || f == 1u);
  }
  for (int i = 0; i < 2000000; ++i) {
    const int bits = pick(1, 32);
    auto any = [&] { return static_cast<int>(static_cast<unsigned>(rng()) >> (32 - bits)) * (rng() & 1 ? 1 : -1); };
    const int4 cut = make_int4(any(), any(), any(), any());
    const int c0 = any(), h = any();
    if (!cut_fits(cut, c0, h, batch, heads, ctas)) continue;
    CHECK(cut.x >= 0 && cut.x < batch && h >= 0 && h < heads && cut.z >= 0);
    CHECK(c0 >= 0 && c0 < last_cta(cut) && last_cta(cut) < ctas);
  }
  return 0;
}
"""


def _run_host_code(tmp_path, text):
    import shutil
    import subprocess
    from pathlib import Path

    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    csrc = Path(__file__).resolve().parents[1] / "macqwen-releases_b200" / "csrc"
    src, exe = tmp_path / "check.cu", tmp_path / "check"
    src.write_text(text)
    subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-I", str(csrc), str(src), "-o",
                    str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout + got.stderr


def test_descriptors_of_cut_work_are_right_and_wild_ones_are_refused(tmp_path):
    """Host code: every shared segment is described once, and memory that no
    kernel wrote (one that gave up a wait) is no descriptor that can be followed."""
    _run_host_code(tmp_path, RANGES_CHECK)


@pytest.mark.gpu
def test_every_descriptor_by_segment_is_set_before_the_join(cuda_lib):
    """Three tiles of work where the workspace has room for six: the other
    descriptors say "no cut", not what the workspace held."""
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    cache = _served(3, 512, dim=128)
    q = torch.randn(3 * 16, 16, 128, device="cuda").bfloat16()
    ws = torch.full((64 << 20,), 0x5A, dtype=torch.uint8, device="cuda")
    paged_attention_q8(q, *cache.tensors, cache.last.block_table, cache.last.seq_lens, 0.09, cu_q=_dev([0, 16, 32, 48]),
                       workspace=ws)
    none = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device="cuda")
    assert int((ws.view(torch.int32).view(-1, 4) == none).all(1).sum()) >= 6  # (6 - 3) tiles x 2 kv heads


# ---- tensors of another device ----


def _calls(place):
    """Every call of the module on stand-in tensors; place(name) says where the named one is."""
    import torch
    from flashnext_b200 import paged_q8 as m

    def t(name, *shape, dtype=torch.int32):
        index = place(name)
        real = torch.zeros(shape, dtype=dtype)
        return real if index < 0 else _Cuda(*shape, dtype=dtype, index=index)

    def cache():
        return [t(n, 4, 32, 2, 64, dtype=torch.int8) for n in ("k_cache", "v_cache")] + \
            [t(n, 4, 2, 2, dtype=torch.float32) for n in ("k_scale", "v_scale")]

    def rows(name, heads=2):
        return t(name, 3, heads, 64, dtype=torch.bfloat16)

    def plan(names=("seq_lens", "new_lens", "release", "block_table", "free_pages", "free_state")):
        shapes = {"block_table": (3, 5), "free_pages": (9,), "free_state": (2,)}
        seq, new, gone, table, ring, state = (t(n, *shapes.get(n, (3,))) for n in names)
        out = m.PagePlan(t("out.block_table", 3, 5), t("out.seq_lens", 3), ring, t("out.free_state", 2),
                         t("out.slot_map", 8, dtype=torch.int64), t("out.token_seq", 8), t("out.positions", 8),
                         t("out.cu_new", 4), t("out.admitted", 3))
        return m.page_plan(seq, new, table, ring, state, 32, 8, release=gone, out=out)

    return {
        "plan": plan,
        "append": lambda: m.kv_append_q8(rows("k"), rows("v"), t("slot_map", 3, dtype=torch.int64), *cache()),
        "read": lambda: m.kv_read_q8(t("slots", 3, dtype=torch.int64), *cache(), out=(rows("out[0]"), rows("out[1]"))),
        "attention": lambda: m.paged_attention_q8(
            rows("q", 4), *cache(), t("block_table", 2, 5), t("context_lens", 2), 0.1, cu_q=t("cu_q", 3),
            out=rows("out", 4), workspace=t("workspace", 1 << 16, dtype=torch.uint8)),
    }


CACHE = ("k_cache", "v_cache", "k_scale", "v_scale")
TENSORS = {
    "plan": ("seq_lens", "new_lens", "release", "block_table", "free_pages", "free_state", "out.block_table", "out.seq_lens",
             "out.free_state", "out.slot_map", "out.token_seq", "out.positions", "out.cu_new", "out.admitted"),
    "append": ("k", "v", "slot_map", *CACHE),
    "read": ("slots", "out[0]", "out[1]", *CACHE),
    "attention": ("q", "block_table", "context_lens", "cu_q", "out", "workspace", *CACHE),
}


class _Accepts:
    """A library that takes every call."""

    def __getattr__(self, name):
        return lambda *a: _lib.OK


@pytest.mark.parametrize("call", list(TENSORS))
def test_calls_refuse_tensors_of_another_device_or_the_host(monkeypatch, call):
    from flashnext_b200 import paged_q8

    started = []
    monkeypatch.setattr(paged_q8, "_ready", lambda t: started.append(t) or (_Accepts(), 7))
    _calls(lambda name: 0)[call]()
    assert len(started) == 1
    for name in TENSORS[call]:
        for index, error in ((1, ValueError), (-1, TypeError)):
            with pytest.raises(error):
                _calls(lambda n: index if n == name else 0)[call]()
    assert len(started) == 1, "a call with a misplaced tensor reached the library"


def test_a_workspace_is_checked(monkeypatch):
    import torch
    from flashnext_b200 import paged_q8

    monkeypatch.setattr(paged_q8, "_ready", lambda t: (_Accepts(), 7))
    cache = [_Cuda(4, 32, 2, 64, dtype=torch.int8) for _ in range(2)] + [_Cuda(4, 2, 2, dtype=torch.float32) for _ in range(2)]
    args = (_Cuda(3, 4, 64, dtype=torch.bfloat16), *cache, _Cuda(3, 2, dtype=torch.int32), _Cuda(3, dtype=torch.int32), 0.1)
    good = _Cuda(1 << 16, dtype=torch.uint8)
    paged_q8.paged_attention_q8(*args, workspace=good)
    with pytest.raises(TypeError):
        paged_q8.paged_attention_q8(*args, workspace=_Cuda(1 << 14, dtype=torch.float32))
    strided = _Cuda(1 << 16, dtype=torch.uint8)
    strided.real = strided.real[::2]
    with pytest.raises(ValueError):
        paged_q8.paged_attention_q8(*args, workspace=strided)


# ---- arrays off their alignment ----


@pytest.mark.parametrize("entry,make,names,off", [
    ("fnmoe_page_plan", _plan_args, TENSORS["plan"], 2), ("fnmoe_page_plan", _plan_args, ("out.slot_map",), 4),
    ("fnmoe_paged_attention_q8", _attention_args, ("block_table", "context_lens", "cu_q"), 2)])
def test_entry_points_refuse_arrays_off_their_alignment(entry, make, names, off):
    fields = {"out.block_table": "block_table_out", "out.seq_lens": "seq_lens_out", "out.free_state": "free_state_out"}
    fn = getattr(_lib.load(), entry)
    for name in names:
        field = fields.get(name, name.removeprefix("out."))
        args = make()
        args = _set(args, field, (getattr(args, field) or 0x90000) + off)
        assert fn(ctypes.byref(args), None) == _lib.ERR_VALUE, name
        assert "aligned" in _lib.last_error()


# ---- positions near 2^31 ----


@pytest.mark.parametrize("page", [16, 48, 128, 1 << 20, 786432])
def test_attention_refuses_table_rows_whose_lookahead_would_pass_2_31(page):
    """The kernels step and look ahead in ints past a row's end."""
    fn, most = _lib.load().fnmoe_paged_attention_q8, ((1 << 31) - 1024) // page
    for pages, code in ((most, _lib.ERR_WORKSPACE), (most + 1, _lib.ERR_SHAPE)):  # the first lacks a workspace only
        a = _set(_set(_attention_args(), "cache", _cache_struct(page_size=page, block=16)), "max_pages", pages)
        assert fn(ctypes.byref(a), None) == code


@pytest.mark.gpu
@pytest.mark.parametrize("page,held,new", [((1 << 30) - 1, (1 << 31) - 4, 2), ((1 << 30) - 1, (1 << 31) - 3, 0),
                                           (715827882, (1 << 31) - 4, 2), ((1 << 31) - 1, 9, 4), ((1 << 31) - 1, 0, 4)])
def test_page_plan_of_lengths_near_2_31(cuda_lib, page, held, new):
    from flashnext_b200.paged_q8 import page_plan

    width = ((1 << 31) - 1) // page
    lens, add = [held, 0], [new, 1]
    table = np.full((2, width), -1)
    table[0, : -(-held // page)] = 3 + np.arange(-(-held // page))
    ring = [8, 7, 6, 9, 10]
    want = oq8.page_plan(lens, add, None, table.tolist(), ring, 4, 3, page, 8)
    got = page_plan(_dev(lens), _dev(add), _dev(table), _dev(ring), _dev([4, 3]), page, 8)
    for name in want:
        np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), np.asarray(want[name]), err_msg=name)


# ---- steps in which a request is refused ----


@pytest.mark.gpu
@pytest.mark.parametrize("refused", ["pages", "columns", "tokens"])
def test_rows_of_a_step_with_a_refused_request_line_up(cuda_lib, refused):
    """The rows of all requests go in; those of the admitted ones are stored
    and attended as if the refused one had not been there."""
    import torch
    from flashnext_b200.paged_q8 import PagedKVCacheQ8

    # the sums that decide over pages and tokens count a refused request too, if it fits its row
    pages, columns, most, admitted = {"pages": (12, 12, 400, [1, 0, 0, 1]), "columns": (40, 5, 400, [1, 0, 1, 1]),
                                      "tokens": (40, 12, 150, [1, 0, 0, 0])}[refused]
    page, batch, kv, group, dim = 32, 4, 2, 4, 64
    cache = PagedKVCacheQ8(pages, page, kv, dim, columns, batch, most, block=32)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    held, rows = [0] * batch, [[] for _ in range(batch)]
    for step, new in enumerate(([20, 33, 7, 1], [3, 330, 60, 2], [1, 5, 1, 1])):
        k, v, q = (torch.randn(sum(new), h, dim, device="cuda", generator=g).bfloat16() for h in (kv, kv, kv * group))
        first = np.concatenate([[0], np.cumsum(new)])
        plan = cache.plan(_dev(new))
        cache.append(cache.pack(k, _dev(first[:-1])), cache.pack(v, _dev(first[:-1])))
        out = cache.attention(cache.pack(q, _dev(first[:-1])), 0.125).float().cpu().numpy()
        ok = plan.admitted.tolist()
        assert ok == (admitted if step == 1 else [1] * 4)
        at = 0
        for b in range(batch):
            if not ok[b]:
                continue
            n, span = new[b], slice(int(first[b]), int(first[b + 1]))
            held[b] += n
            rows[b].append((k[span], v[span]))
            # the cache holds the request's own rows, to within half a code of their block's largest
            slots = torch.from_numpy(_slots(plan.block_table.cpu().numpy(), b, 0, held[b], page)).cuda()
            back = cache.read(slots)
            for i in range(2):
                mine = torch.cat([r[i] for r in rows[b]]).float()
                assert float((back[i].float() - mine).abs().max()) <= float(mine.abs().max()) * (1.5 / 127 + 2.0 ** -8)
            kk, vv = (c.float().view(-1, kv, dim)[slots].cpu().numpy() * s.view(-1, kv)[slots // 32].cpu().numpy()[:, :, None]
                      for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            seen = np.arange(held[b])[None] <= (held[b] - n + np.arange(n))[:, None]
            want, mag = oq8.attention(q[span].float().cpu().numpy(), kk, vv, seen, 0.125)
            assert _outside(out[at:at + n], want, mag) == 0
            at += n
        assert (out[at:] == 0).all()


# ---- large batches ----


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,batch", [(256, 170), (128, 210), (64, 300)])
@pytest.mark.parametrize("rows", [None, (0, 3), (9, 20), (0, 30)])
def test_large_batches_are_scanned_and_joined_by_cuts(cuda_lib, kind, dim, batch, rows):
    """More sequences than a CTA has threads, and more segments (sequence, kv
    head, tile) than CTAs to cut them, so that the join goes by the cuts: rows of
    the few-row kernel, of the many-row kernel and of both."""
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    page, block, kv, group = 32, 32, 4, 2
    rng = np.random.default_rng(dim + batch + (rows or (7, 7))[1])
    held = rng.integers(0, 200, batch)
    held[rng.integers(0, batch, 12)] = rng.integers(700, 3000, 12)
    held[[0, 5, batch - 1]] = 0, 1, 0
    new = [1] * batch if rows is None else rng.integers(rows[0], rows[1] + 1, batch).tolist()
    held = held.tolist()
    table, pages = _place(rng, held, page)
    n = pages * page
    k, v = (np.clip(np.rint(rng.standard_normal((n, kv, dim)) * 40), -127, 127).astype(np.float32) for _ in range(2))
    if kind == "e4m3":
        k, v = oq8.e4m3_round(k), oq8.e4m3_round(v)
    ks, vs = ((np.exp(0.5 * rng.standard_normal((n // block, kv))) / 40).astype(np.float32) for _ in range(2))
    cache = _cache_of(table, pages, page, block, kind, k, ks, v, vs)
    q = _bf16(rng.standard_normal((sum(new), kv * group, dim)))
    cu = None if rows is None else _dev(np.concatenate([[0], np.cumsum(new)]))
    args = (q.cuda(), *cache, _dev(table), _dev(held), dim ** -0.5)
    out = paged_attention_q8(*args, cu_q=cu)
    assert torch.equal(out, paged_attention_q8(*args, cu_q=cu))
    out = out.float().cpu().numpy()
    assert _wrong(out, q.float().numpy(), table, held, new, ((k, ks), (v, vs)), page, block, dim ** -0.5) == 0
    assert _lib.read_device_errors() == 0


# ---- the weights' low terms ----


def _opposed(dim, lengths, kind, page=16, seed=7):
    """Even tokens hold values +v with one score, odd ones -v with another a
    little lower, so an output is a small difference of large sums: (1 - w) / (1 + w)
    of v for w near 1, while mean|v| is v.  A weight that is off by 2^-10 shows."""
    rng = np.random.default_rng(seed + dim)
    table, pages = _place(rng, lengths, page)
    n = pages * page
    k, sign = np.zeros((n, 1, dim), np.float32), np.ones((n, 1, 1), np.float32)
    k[:, :, 1:] = np.rint(rng.standard_normal(dim - 1) * 3)  # alike for all tokens
    for b, length in enumerate(lengths):
        slot = _slots(table, b, 0, length, page)
        k[slot, 0, 0] = np.where(np.arange(length) % 2, 60, 64)
        sign[slot, 0, 0] = np.where(np.arange(length) % 2, -1, 1)
    v = (sign * 96 * rng.choice([-1, 1], (1, 1, dim))).astype(np.float32)
    one = np.ones((pages, 1), np.float32)
    return table, pages, ((k, one), (v, one / 32)), rng


def _queries(rng, rows, group, dim):
    q = np.zeros((rows, group, dim), np.float32)
    q[:, :, 0] = rng.uniform(0.5, 4.0, (rows, group))
    return _bf16(q)


def _bf16_of(x, up):
    """float32 to bfloat16 and back: to nearest, or (up False) toward zero."""
    return _bf16(x).float().numpy() if up else (np.ascontiguousarray(x, np.float32).view(np.uint32) & 0xFFFF0000).view(np.float32)


@pytest.mark.parametrize("up", [True, False])
def test_the_bound_on_opposed_values_tells_one_term_of_a_weight_from_two(up):
    """The test below, with the weights' rounding planted in the oracle: with
    both terms every output is inside the bound, with the high term alone some
    rows of every length have outputs outside."""
    dim, lengths, scale = 64, [2, 17, 64, 333, 1000, 5000], 1 / 64
    table, _, ((k, _), (v, vs)), rng = _opposed(dim, lengths, "int8")
    q = _queries(rng, len(lengths), 16, dim).float().numpy()
    for b, length in enumerate(lengths):
        slot = _slots(table, b, 0, length, 16)
        kk, vv = k[slot].astype(np.float64), v[slot].astype(np.float64) * vs[0, 0]
        want, mag = oq8.attention(q[b:b + 1], kk, vv, np.ones((1, length), bool), scale)
        t = (q[b].astype(np.float64) @ kk[:, 0].T) * scale * np.log2(np.e)
        u = np.exp2(t - t.max(1, keepdims=True)).astype(np.float32)
        hi = _bf16_of(u, up)
        for terms, w in ((2, hi.astype(np.float64) + _bf16_of(u - hi, True)), (1, hi.astype(np.float64))):
            out = _bf16((w @ vv[:, 0] / u.sum(1, dtype=np.float64, keepdims=True)).astype(np.float32)).float().numpy()
            off = [_outside(out[h], want[0, h], mag[0, h]) > 0 for h in range(16)]
            assert (sum(off) == 0) if terms == 2 else (sum(off) > 0), (length, terms, sum(off))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [None, 1, 2, 9])
def test_small_differences_of_large_sums(cuda_lib, kind, dim, rows):
    from flashnext_b200.paged_q8 import paged_attention_q8

    lengths, group, page = [2, 17, 64, 333, 1000, 5000], 16, 16
    table, pages, host, rng = _opposed(dim, lengths, kind)
    (k, ks), (v, vs) = host
    cache = _cache_of(table, pages, page, page, kind, k, ks, v, vs)
    new = [min(rows or 1, h) for h in lengths]
    q = _queries(rng, sum(new), group, dim)
    cu = None if rows is None else _dev(np.concatenate([[0], np.cumsum(new)]))
    out = paged_attention_q8(q.cuda(), *cache, _dev(table), _dev(lengths), 1 / 64, cu_q=cu).float().cpu().numpy()
    assert _wrong(out, q.float().numpy(), table, lengths, new, host, page, page, 1 / 64) == 0
