"""The paged 8-bit KV cache: page plan, quantising append, read, attention.

CPU: the oracle's own rounding, and every refusal of the C entry points.
GPU: the plan's integers and the append's codes and scales bit for bit, the
read bit for bit, and the attention against float64.

Attention bound, per output: the kernels round the softmax weight of each
token to float16 (2^-11 relative) and the result once to bfloat16 (2^-9);
float32 scores of magnitude below 64 with up to 256-term sums move a weight by
less than 2^-11 relative.  So |out - truth| <= 2^-8 |truth| + 2^-10 mean|v|,
with mean|v| the weighted mean of the magnitudes, covers them with a factor of
two on the final rounding.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from flashnext_b200 import _lib
from oracle import paged_q8 as oq8

KINDS = ("int8", "e4m3")


# ---- CPU: oracle and refusals ----


def test_oracle_e4m3_rounding_matches_the_type():
    import torch

    x = np.concatenate([np.linspace(-448, 448, 4001), np.geomspace(2.0 ** -12, 448, 3000)]).astype(np.float32)
    ties = np.float32(2.0 ** -6) * (1 + (np.arange(0, 64) * 2 + 1) / np.float32(16.0)) / 8  # midpoints among them
    x = np.concatenate([x, ties.astype(np.float32)])
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(oq8.e4m3_round(x), want)


def _cache_struct(**kw):
    c = _lib.FnQ8Cache(0x10000, 0x20000, 0x30000, 0x40000, 8, 64, 32, 2, 128, _lib.Q8_INT8)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = (({"k_codes": None}, _lib.ERR_NULL), ({"v_scale": None}, _lib.ERR_NULL),
              ({"code_type": 2}, _lib.ERR_UNSUPPORTED), ({"block": 8}, _lib.ERR_UNSUPPORTED),
              ({"block": 48}, _lib.ERR_UNSUPPORTED), ({"head_dim": 96}, _lib.ERR_UNSUPPORTED),
              ({"page_size": 48}, _lib.ERR_SHAPE), ({"num_pages": 0}, _lib.ERR_SHAPE),
              ({"kv_heads": 0}, _lib.ERR_SHAPE), ({"v_codes": 0x20008}, _lib.ERR_VALUE),
              ({"k_scale": 0x30002}, _lib.ERR_VALUE))


def _set(a, field, value):
    b = type(a).from_buffer_copy(a)
    setattr(b, field, value)
    return b


def _append_args():
    return _lib.FnQ8AppendArgs(_lib.ABI_VERSION, 3, _cache_struct(), 0x50000, 0x60000, 256, 256, 0x70000)


def _read_args():
    return _lib.FnQ8ReadArgs(_lib.ABI_VERSION, 3, _cache_struct(), 0x50000, 0x60000, 0x70000)


def _attention_args():
    return _lib.FnQ8AttentionArgs(_lib.ABI_VERSION, 2, 2, 16, 4, 0.125, _cache_struct(), 0x50000, 16 * 128, 0x60000,
                                  0x70000, None, 0x80000, None, 0)


def _plan_args():
    return _lib.FnPagePlanArgs(_lib.ABI_VERSION, 4, 64, 8, 32, 16, 0x1000, 0x2000, None, 0x3000, 0x4000, 0x5000, 0x6000,
                               0x7000, 0x8000, 0x9000, 0xA000, 0xB000, 0xC000, 0xD000)


ENTRY_CASES = [
    ("fnmoe_page_plan", _plan_args, (
        ("abi_version", 3, _lib.ERR_ABI), ("seq_lens", None, _lib.ERR_NULL), ("admitted", None, _lib.ERR_NULL),
        ("batch", 0, _lib.ERR_SHAPE), ("batch", 8193, _lib.ERR_SHAPE), ("page_size", 0, _lib.ERR_SHAPE),
        ("max_pages", 1 << 26, _lib.ERR_SHAPE), ("max_tokens", 0, _lib.ERR_SHAPE),
        ("seq_lens_out", 0x1000, _lib.ERR_VALUE), ("free_state_out", 0x5000, _lib.ERR_VALUE))),
    ("fnmoe_kv_append_q8", _append_args, (
        ("abi_version", 3, _lib.ERR_ABI), ("k", None, _lib.ERR_NULL), ("slot_map", None, _lib.ERR_NULL),
        ("k_stride", 248, _lib.ERR_SHAPE), ("v_stride", 260, _lib.ERR_VALUE), ("v", 0x60008, _lib.ERR_VALUE))),
    ("fnmoe_kv_read_q8", _read_args, (
        ("abi_version", 3, _lib.ERR_ABI), ("slots", None, _lib.ERR_NULL), ("k_out", 0x60008, _lib.ERR_VALUE),
        ("slots", 0x50004, _lib.ERR_VALUE))),
    ("fnmoe_paged_attention_q8", _attention_args, (
        ("abi_version", 3, _lib.ERR_ABI), ("q", None, _lib.ERR_NULL), ("out", None, _lib.ERR_NULL),
        ("batch", 0, _lib.ERR_SHAPE), ("q_rows", 3, _lib.ERR_SHAPE), ("q_heads", 15, _lib.ERR_SHAPE),
        ("q_heads", 66, _lib.ERR_UNSUPPORTED), ("max_pages", 1 << 26, _lib.ERR_SHAPE),
        ("scale", 0.0, _lib.ERR_VALUE), ("scale", -1.0, _lib.ERR_VALUE), ("scale", math.inf, _lib.ERR_VALUE),
        ("scale", math.nan, _lib.ERR_VALUE), ("q_stride", 8, _lib.ERR_SHAPE), ("q", 0x50008, _lib.ERR_VALUE),
        ("workspace", None, _lib.ERR_WORKSPACE))),
]


@pytest.mark.parametrize("entry,make,cases", ENTRY_CASES, ids=[e[0] for e in ENTRY_CASES])
def test_entry_points_refuse_before_any_device_call(entry, make, cases):
    fn = getattr(_lib.load(), entry)
    assert fn(None, None) == _lib.ERR_NULL
    for field, value, code in cases:
        assert fn(ctypes.byref(_set(make(), field, value)), None) == code, (field, value)
        assert _lib.last_error()
    if entry != "fnmoe_page_plan":
        for kw, code in BAD_CACHES:
            assert fn(ctypes.byref(_set(make(), "cache", _cache_struct(**kw))), None) == code, kw


def test_empty_calls_do_nothing_and_the_workspace_is_sized_on_the_host():
    lib = _lib.load()
    assert lib.fnmoe_kv_append_q8(ctypes.byref(_set(_append_args(), "tokens", 0)), None) == _lib.OK
    assert lib.fnmoe_kv_read_q8(ctypes.byref(_set(_read_args(), "count", 0)), None) == _lib.OK
    a = _set(_set(_attention_args(), "cu_q", 0x90000), "q_rows", 0)
    assert lib.fnmoe_paged_attention_q8(ctypes.byref(a), None) == _lib.OK
    need = ctypes.c_uint64(0)
    size = lib.fnmoe_paged_attention_q8_workspace_size
    assert size(ctypes.byref(_attention_args()), ctypes.byref(need)) == _lib.OK and need.value > 0
    assert size(ctypes.byref(_attention_args()), None) == _lib.ERR_NULL
    short = _set(_set(_attention_args(), "workspace", 0x100000), "workspace_bytes", need.value - 1)
    assert lib.fnmoe_paged_attention_q8(ctypes.byref(short), None) == _lib.ERR_WORKSPACE
    assert str(need.value) in _lib.last_error()


def test_struct_layout_matches_c_compiler(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    names = ("FnQ8Cache", "FnPagePlanArgs", "FnQ8AppendArgs", "FnQ8ReadArgs", "FnQ8AttentionArgs")
    lines = []
    for n in names:
        for f, _ in getattr(_lib, n)._fields_:
            lines.append(f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));')
        lines.append(f'printf("{n} %zu\\n", sizeof({n}));')
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fnmoe.h"\nint main(void) {' + "\n".join(lines) + "return 0;}")
    exe = tmp_path / "probe"
    root = Path(__file__).resolve().parents[1]
    subprocess.run(["gcc", "-I", str(root / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n") if x)
    for n in names:
        t = getattr(_lib, n)
        assert int(got[n]) == ctypes.sizeof(t)
        for f, _ in t._fields_:
            assert int(got[f"{n}.{f}"]) == getattr(t, f).offset, (n, f)


# ---- GPU ----


def _plan_case(rng, batch, page, width, num, cap, lo, hi, tight=False):
    """A consistent serving state: held pages, the ring's free ones, mixed requests."""
    lens = rng.integers(lo, hi + 1, batch)
    lens = np.minimum(lens, width * page)
    need = -(-lens // page)
    perm = rng.permutation(num)
    table = np.full((batch, width), -1, np.int32)
    at = 0
    for b in range(batch):
        table[b, : need[b]] = perm[at:at + need[b]]
        at += need[b]
    assert at <= num
    count = num - at
    head = int(rng.integers(0, num))
    ring = np.full(num, -7, np.int32)
    ring[(head + np.arange(count)) % num] = perm[at:]
    if tight:
        count = min(count, max(1, batch // 3))
    new = rng.choice([0, 1, 1, 1, 2, page, 3 * page + 1], batch)
    gone = (rng.random(batch) < 0.25).astype(np.int32)
    return lens.astype(np.int32), new.astype(np.int32), gone, table, ring, head, count


@pytest.mark.gpu
@pytest.mark.parametrize("batch,page,width,num,cap,lo,hi,tight", [
    (1, 64, 4, 8, 300, 0, 0, False), (1, 16, 3, 3, 1, 48, 48, False), (5, 16, 8, 64, 400, 0, 100, False),
    (33, 64, 7, 300, 7000, 0, 448, False), (40, 16, 6, 240, 2000, 0, 90, True), (257, 32, 9, 2400, 26000, 0, 250, False),
    (300, 128, 3, 900, 500, 0, 380, False), (1000, 16, 20, 21000, 60000, 0, 300, False)])
@pytest.mark.parametrize("with_release", [True, False])
def test_page_plan_matches_the_loop(cuda_lib, batch, page, width, num, cap, lo, hi, tight, with_release):
    import torch
    from flashnext_b200.paged_q8 import page_plan

    rng = np.random.default_rng(batch * 7 + page + num + cap)
    lens, new, gone, table, ring, head, count = _plan_case(rng, batch, page, width, num, cap, lo, hi, tight)
    release = gone if with_release else None
    want = oq8.page_plan(lens.tolist(), new.tolist(), release, table.tolist(), ring.tolist(), head, count, page, cap)
    dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    ring_t, table_t = dev(ring), dev(table)
    rel_t = None if release is None else dev(release)
    args = (dev(lens), dev(new), table_t, ring_t.clone(), dev([head, count]), page, cap)
    got = page_plan(*args, release=rel_t)
    for name in want:
        np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), np.asarray(want[name]), err_msg=name)
    assert got.free_pages is args[3]
    # into given buffers, the table in place
    got.block_table = table_t
    again = page_plan(args[0], args[1], table_t, ring_t, args[4], page, cap, release=rel_t, out=got)
    assert again is got
    for name in want:
        np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), np.asarray(want[name]), err_msg=name)


@pytest.mark.gpu
def test_page_plan_refuses(cuda_lib):
    import torch
    from flashnext_b200.paged_q8 import page_plan

    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    with pytest.raises(TypeError):
        page_plan(z(4).long(), z(4), z(4, 2), z(8), z(2), 16, 8)
    with pytest.raises(TypeError):
        page_plan(z(4).cpu(), z(4), z(4, 2), z(8), z(2), 16, 8)
    with pytest.raises(ValueError):
        page_plan(z(4), z(3), z(4, 2), z(8), z(2), 16, 8)
    with pytest.raises(ValueError):
        page_plan(z(4), z(4), z(2, 4).t(), z(8), z(2), 16, 8)
    with pytest.raises(ValueError):
        page_plan(z(4), z(4), z(4, 2), z(8), z(2), 16, 0)


def _empty_cache(pages, page, block, heads, dim, kind, fill=True):
    import torch

    dt = torch.int8 if kind == "int8" else torch.float8_e4m3fn
    shape = (pages, page, heads, dim)
    caches = []
    for _ in range(2):
        c = torch.empty(shape, dtype=torch.uint8, device="cuda")
        if fill:
            c.fill_(0x7F)  # unwritten slots: the largest int8, NaN in e4m3
        caches.append(c.view(dt))
    scales = [torch.full((pages, page // block, heads), float("nan"), device="cuda") for _ in range(2)]
    return caches[0], caches[1], scales[0], scales[1]


def _values(codes, scales, block):
    """float32 code values [slots, H, D] and scales [slots / block, H] on the host."""
    c = codes.float().cpu().numpy()
    return c.reshape(-1, *c.shape[2:]), scales.cpu().numpy().reshape(-1, scales.shape[-1])


def _place(rng, held, page, spare=2):
    """Random pages for sequences of these lengths -> table, pages."""
    need = [-(-h // page) for h in held]
    pages = sum(need) + spare
    perm = rng.permutation(pages)
    table = np.full((len(held), max(need + [1]) + 1), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, pages


def _slots(table, b, lo, hi, page):
    p = np.arange(lo, hi)
    return table[b, p // page].astype(np.int64) * page + p % page


def _bf16(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page,block,heads,dim,steps", [
    (16, 16, 1, 64, [(0, 1), (1, 2), (2, 40)]), (64, 64, 2, 256, [(0, 100), (100, 101), (101, 102), (102, 260)]),
    (64, 16, 3, 128, [(0, 17), (17, 17), (17, 64), (64, 65)]), (256, 128, 2, 256, [(0, 127), (127, 129), (129, 700)]),
    (128, 128, 5, 64, [(0, 5), (5, 300)]), (32, 32, 8, 128, [(0, 33), (33, 500)])])
@pytest.mark.parametrize("fused", [False, True])
def test_append_codes_and_scales_bit_for_bit(cuda_lib, kind, page, block, heads, dim, steps, fused):
    """Several sequences grow by ragged steps; after each step every written
    slot's code and every touched scale equal the loop's, and the read-back
    is the rounded product."""
    import torch
    from flashnext_b200.paged_q8 import kv_append_q8, kv_read_q8

    rng = np.random.default_rng(page + block + heads + dim + len(steps))
    seqs = 3
    ends = [max(0, steps[-1][1] - 3 * b) for b in range(seqs)]
    table, pages = _place(rng, ends, page)
    cache = _empty_cache(pages, page, block, heads, dim, kind)
    state = [_values(cache[0], cache[2], block), _values(cache[1], cache[3], block)]
    state = [(c.copy(), s.copy()) for c, s in state]
    for lo, hi in steps:
        spans = [(b, min(lo, ends[b]), min(hi, ends[b])) for b in range(seqs)]
        slots = np.concatenate([_slots(table, b, a, z, page) for b, a, z in spans] + [np.zeros(0, np.int64)])
        t = len(slots)
        x = rng.standard_normal((2, t, heads, dim)) * np.exp(rng.standard_normal((2, t, heads, 1)))
        rows = [_bf16(x[i]) for i in range(2)]
        if fused and t:
            wide = torch.zeros(t, heads * dim * 2 + 64, dtype=torch.bfloat16, device="cuda")
            wide[:, 64:] = torch.cat([r.reshape(t, -1) for r in rows], 1).cuda()
            k, v = wide[:, 64:].view(t, 2, heads, dim).unbind(1)
        else:
            k, v = (r.cuda() for r in rows)
        kv_append_q8(k, v, torch.from_numpy(slots).cuda(), *cache)
        for i in range(2):
            codes, scales = state[i]
            with np.errstate(invalid="ignore"):
                oq8.append(rows[i].float().numpy(), slots, codes, scales, block, kind)
            got_c, got_s = _values(cache[i], cache[2 + i], block)
            written = np.concatenate([_slots(table, b, 0, z, page) for b, _, z in spans] + [np.zeros(0, np.int64)])
            np.testing.assert_array_equal(got_c[written], codes[written])
            np.testing.assert_array_equal(got_s, scales)  # untouched blocks keep their NaN
            back = kv_read_q8(torch.from_numpy(written).cuda(), *cache)[i]
            want = _bf16(codes[written] * scales[written // block][:, :, None])
            assert torch.equal(back.cpu().view(torch.int16), want.view(torch.int16)) or \
                torch.equal(back.cpu().float(), want.float())  # +0 and -0 codes


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_append_of_zeros_infinities_nan_and_tiny_rows(cuda_lib, kind):
    import torch
    from flashnext_b200.paged_q8 import kv_append_q8, kv_read_q8

    page = block = 16
    cache = _empty_cache(4, page, block, 1, 64, kind)
    x = np.zeros((4, 16, 1, 64), np.float32)
    x[1, 3, 0, 5], x[1, 4, 0, 6], x[1, 5, 0, 7], x[1, 6, 0, 8] = np.inf, -np.inf, np.nan, 2.0
    x[2] = 1e-38
    x[3] = 3e38
    rows = _bf16(x.reshape(64, 1, 64))
    slots = np.arange(64)
    kv_append_q8(rows.cuda(), rows.cuda(), torch.from_numpy(slots).cuda(), *cache)
    codes, scales = (a.copy() for a in _values(cache[0], cache[2], block))
    want_c, want_s = np.zeros_like(codes), np.zeros_like(scales)
    oq8.append(rows.float().numpy(), slots, want_c, want_s, block, kind)
    np.testing.assert_array_equal(codes, want_c)
    np.testing.assert_array_equal(scales, want_s)
    top = float(oq8.TOP[kind])
    assert codes[16 + 3, 0, 5] == top and codes[16 + 4, 0, 6] == -top and codes[16 + 5, 0, 7] == 0
    assert codes[16 + 6, 0, 8] == top and (codes[:16] == 0).all() and (codes[48:] == top).all()
    out = kv_read_q8(torch.from_numpy(slots).cuda(), *cache)[0].float().cpu()
    assert torch.isfinite(out).all()


@pytest.mark.gpu
def test_append_skips_slots_outside_and_read_gives_zeros_there(cuda_lib):
    import torch
    from flashnext_b200.paged_q8 import kv_append_q8, kv_read_q8

    cache = _empty_cache(3, 32, 16, 2, 64, "int8")
    before = [c.clone() for c in cache]
    slots = torch.tensor([-1, 96, 1 << 40, -(1 << 40), 5, -1, 17], device="cuda")
    k = torch.ones(7, 2, 64, dtype=torch.bfloat16, device="cuda")
    kv_append_q8(k, 2 * k, slots, *cache)
    a, b = kv_read_q8(slots, *cache)
    want = torch.tensor([0, 0, 0, 0, 1.0, 0, 1.0], device="cuda").view(7, 1, 1).expand(7, 2, 64)
    assert torch.equal(a.float(), want) and torch.equal(b.float(), 2 * want)
    touched = torch.zeros(96, dtype=torch.bool, device="cuda")
    touched[[5, 17]] = True
    touched[0:5] = True  # earlier slots of a block that starts at 5 hold nothing: not compared
    touched[16] = True
    same = (cache[0].view(96, -1) == before[0].view(96, -1)).all(1)
    assert bool((same | touched).all())
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    kv_append_q8(k[:0], k[:0], none, *cache)
    assert kv_read_q8(none, *cache)[0].shape == (0, 2, 64)


@pytest.mark.gpu
def test_cache_calls_refuse(cuda_lib):
    import torch
    from flashnext_b200.paged_q8 import kv_append_q8, kv_read_q8, paged_attention_q8

    cache = _empty_cache(3, 32, 16, 2, 64, "int8")
    k = torch.ones(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(4, device="cuda")
    table, ctx = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda")
    cu = torch.arange(5, dtype=torch.int32, device="cuda")
    for bad in (k.float(), k.cpu()):
        with pytest.raises(TypeError):
            kv_append_q8(bad, k, slots, *cache)
        with pytest.raises(TypeError):
            paged_attention_q8(bad, *cache, table, ctx, 1.0)
    with pytest.raises(TypeError):
        kv_append_q8(k, k, slots.int(), *cache)
    with pytest.raises(TypeError):
        kv_read_q8(slots, cache[0].view(torch.uint8), *cache[1:])
    with pytest.raises(TypeError):
        kv_read_q8(slots, cache[0], cache[1].view(torch.uint8), *cache[2:])
    with pytest.raises(ValueError):
        kv_append_q8(k, k[:3], slots, *cache)
    with pytest.raises(ValueError):
        kv_append_q8(k.transpose(1, 2).contiguous().transpose(1, 2), k, slots, *cache)
    with pytest.raises(ValueError):
        kv_read_q8(slots, *cache[:2], cache[2][:, :1], cache[3])
    with pytest.raises(ValueError):
        paged_attention_q8(k[:3], *cache, table, ctx, 1.0)
    with pytest.raises(ValueError):
        paged_attention_q8(k, *cache, table, ctx, 0.0)
    with pytest.raises(ValueError):
        paged_attention_q8(k, *cache, table, ctx, 1.0, cu_q=cu[:4])
    with pytest.raises(RuntimeError):
        paged_attention_q8(k, *cache, table, ctx, 1.0, workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))


def _filled(rng, held, page, block, heads, dim, kind, big=None):
    """A cache holding these sequences: normal codes with uneven scales; unwritten slots keep 0x7F."""
    import torch

    table, pages = _place(rng, held, page)
    cache = _empty_cache(pages, page, block, heads, dim, kind)
    host = []
    for i in range(2):
        codes = np.clip(np.rint(rng.standard_normal((pages * page, heads, dim)) * 40), -127, 127).astype(np.float32)
        if kind == "e4m3":
            codes = oq8.e4m3_round((codes * 3).astype(np.float32))
        scales = (np.exp(0.7 * rng.standard_normal((pages * page // block, heads))) / 40).astype(np.float32)
        if kind == "e4m3":
            scales = (scales / 3).astype(np.float32)
        live = np.zeros(pages * page, bool)
        for b, h in enumerate(held):
            live[_slots(table, b, 0, h, page)] = True
        dt = cache[i].dtype
        enc = torch.from_numpy(codes).to(dt).view(torch.uint8)
        enc[torch.from_numpy(~live)] = 0x7F
        cache[i].view(torch.uint8).copy_(enc.view(cache[i].shape).cuda())
        cache[2 + i].copy_(torch.from_numpy(scales).view(cache[2 + i].shape))
        host.append((codes, scales))
    return table, cache, host


def _check_attention(out, q, table, held, new, host, page, block, scale, num_pages):
    """Every row of `out` against float64, within the derived bound."""
    at = 0
    for b, (h, n) in enumerate(zip(held, new)):
        if n == 0:
            continue
        cap = min(h, table.shape[1] * page)
        p = np.arange(cap)
        pg = table[b, p // page].astype(np.int64)
        ok = (pg >= 0) & (pg < num_pages)
        slot = np.where(ok, pg * page + p % page, 0)
        k, v = (c[slot] * s[slot // block][:, :, None] for c, s in host)
        seen = (p[None] <= (h - n + np.arange(n))[:, None]) & ok[None]
        want, mag = oq8.attention(q[at:at + n], k, v, seen, scale)
        got = out[at:at + n].astype(np.float64)
        bound = 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * mag + 1e-30
        off = np.abs(got - want)
        assert (off <= bound).all(), (b, h, n, float((off / bound).max()))
        at += n


ATTENTION_CASES = [
    # heads kv, group, dim, page, block, held, new (None: one row each, without cu_q)
    (2, 8, 256, 64, 64, [1, 64, 65, 1000, 0, 333], None),
    (4, 6, 256, 256, 64, [1000, 17], None),
    (1, 1, 64, 16, 16, [0, 1, 2, 15, 16, 17, 200], None),
    (8, 4, 128, 16, 16, [700, 3, 0, 129, 64], None),
    (1, 16, 128, 32, 32, [500, 31, 33], None),
    (2, 12, 64, 128, 128, [300, 128], None),
    (1, 32, 64, 64, 16, [90, 1], None),
    (2, 8, 256, 64, 64, [600, 64, 70, 9, 8], [8, 8, 1, 5, 8]),
    (3, 1, 128, 64, 32, [300, 20, 5, 1], [3, 0, 5, 1]),
    (2, 4, 64, 16, 16, [100, 47, 3], [4, 2, 3]),
    (2, 8, 256, 64, 64, [300], [300]),
    (2, 8, 256, 64, 64, [500, 77, 129], [131, 77, 2]),
    (1, 3, 128, 128, 64, [1000, 260, 1, 40], [257, 130, 1, 17]),
    (4, 2, 64, 32, 16, [411, 65], [200, 64]),
    (1, 16, 64, 16, 16, [150, 33], [60, 33]),
    (1, 12, 256, 32, 32, [200, 90], [45, 90]),
    (1, 32, 128, 64, 64, [100, 64], [33, 64]),
    # a context shorter than its rows: the first rows see nothing
    (2, 8, 256, 64, 64, [5, 0, 70], [9, 4, 3]),
    (1, 8, 128, 64, 64, [20, 0], [50, 30]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("kv,group,dim,page,block,held,new", ATTENTION_CASES)
def test_attention_against_float64(cuda_lib, kind, kv, group, dim, page, block, held, new):
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    rng = np.random.default_rng(kv * 31 + group + dim + page + sum(held))
    table, cache, host = _filled(rng, held, page, block, kv, dim, kind)
    rows = len(held) if new is None else sum(new)
    q = _bf16(rng.standard_normal((rows, kv * group, dim)) * 1.5)
    dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    cu = None if new is None else dev(np.concatenate([[0], np.cumsum(new)]))
    scale = dim ** -0.5
    out = torch.full((rows, kv * group, dim), float("nan"), dtype=torch.bfloat16, device="cuda")
    got = paged_attention_q8(q.cuda(), *cache, dev(table), dev(held), scale, cu_q=cu, out=out)
    assert got is out
    _check_attention(out.float().cpu().numpy(), q.float().numpy(), table, held, new or [1] * len(held), host, page,
                     block, scale, cache[0].shape[0])
    again = paged_attention_q8(q.cuda(), *cache, dev(table), dev(held), scale, cu_q=cu)
    assert torch.equal(again.view(torch.int16), out.view(torch.int16))  # no order that changes from call to call
    assert _lib.read_device_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("new", [None, [1, 1, 60, 200]])
def test_attention_long_contexts_are_split_and_joined(cuda_lib, new):
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    held, page, block, kv, group, dim = [20000, 1, 9001, 16384], 64, 64, 2, 8, 256
    rng = np.random.default_rng(5)
    table, cache, host = _filled(rng, held, page, block, kv, dim, "int8")
    n = new or [1] * 4
    q = _bf16(rng.standard_normal((sum(n), kv * group, dim)))
    dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    cu = None if new is None else dev(np.concatenate([[0], np.cumsum(new)]))
    out = paged_attention_q8(q.cuda(), *cache, dev(table), dev(held), 0.0625, cu_q=cu)
    _check_attention(out.float().cpu().numpy(), q.float().numpy(), table, held, n, host, page, block, 0.0625,
                     cache[0].shape[0])


@pytest.mark.gpu
@pytest.mark.parametrize("new", [None, [2, 150, 1]])
def test_attention_skips_pages_outside_the_cache_and_past_the_row(cuda_lib, new):
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    held, page, block, kv, group, dim = [300, 416, 200], 32, 32, 1, 8, 128  # whole pages where the context runs on
    rng = np.random.default_rng(6)
    table, cache, host = _filled(rng, held, page, block, kv, dim, "e4m3")
    table[0, 2], table[1, 0], table[1, 5], table[2, :] = -1, cache[0].shape[0], -5, -1
    held = [300, 100000, 200]  # past the row's end; the last sequence has no page at all
    n = new or [1] * 3
    q = _bf16(rng.standard_normal((sum(n), group, dim)))
    dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    cu = None if new is None else dev(np.concatenate([[0], np.cumsum(new)]))
    out = paged_attention_q8(q.cuda(), *cache, dev(table), dev(held), 0.09, cu_q=cu)
    _check_attention(out.float().cpu().numpy(), q.float().numpy(), table, held, n, host, page, block, 0.09,
                     cache[0].shape[0])
    assert bool((out[-1] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [None, [3, 90]])
def test_attention_of_uneven_magnitudes(cuda_lib, new):
    """Query rows of magnitudes from 1e-30 to 1e30 (with keys scaled against
    them), value scales from 2^-100 to 2^80 side by side, and all-zero blocks:
    the weights and sums stay in range."""
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    held, page, block, kv, group, dim = [200, 150], 32, 16, 1, 4, 128
    rng = np.random.default_rng(8)
    table, cache, host = _filled(rng, held, page, block, kv, dim, "int8")
    n = new or [1] * 2
    for gain, vlo, vhi in ((1e30, -100, -90), (1e-30, 70, 80), (1.0, -107, 20)):
        ks = (host[0][1] / np.float32(gain)).astype(np.float32)
        vs = np.exp2(rng.uniform(vlo, vhi, host[1][1].shape)).astype(np.float32)
        h2 = [(host[0][0], ks), (host[1][0], vs)]
        cache[2].copy_(torch.from_numpy(ks).view(cache[2].shape))
        cache[3].copy_(torch.from_numpy(vs).view(cache[3].shape))
        q = _bf16(rng.standard_normal((sum(n), group, dim)) * gain)
        dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
        cu = None if new is None else dev(np.concatenate([[0], np.cumsum(new)]))
        out = paged_attention_q8(q.cuda(), *cache, dev(table), dev(held), 0.088, cu_q=cu)
        _check_attention(out.float().cpu().numpy(), q.float().numpy(), table, held, n, h2, page, block, 0.088,
                         cache[0].shape[0])


@pytest.mark.gpu
@pytest.mark.parametrize("new", [None, [2, 100, 40]])
def test_attention_takes_strided_rows_and_another_stream(cuda_lib, new):
    import torch
    from flashnext_b200.paged_q8 import paged_attention_q8

    held, page, block, kv, group, dim = [130, 300, 64], 64, 32, 2, 4, 64
    rng = np.random.default_rng(9)
    table, cache, host = _filled(rng, held, page, block, kv, dim, "e4m3")
    n = new or [1] * 3
    wide = _bf16(rng.standard_normal((sum(n), (kv * group + 2 * kv) * dim))).cuda()
    q = wide[:, : kv * group * dim].view(sum(n), kv * group, dim)
    assert sum(n) == 1 or not q.is_contiguous()
    dev = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    cu = None if new is None else dev(np.concatenate([[0], np.cumsum(new)]))
    tt, hh = dev(table), dev(held)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:  # two calls in flight at once share no scratch
        with torch.cuda.stream(s):
            outs.append(paged_attention_q8(q, *cache, tt, hh, 0.125, cu_q=cu))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])
    _check_attention(outs[0].float().cpu().numpy(), q.float().cpu().numpy(), table, held, n, host, page, block, 0.125,
                     cache[0].shape[0])


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda_lib):
    """A cache of more than 2^32 bytes a side: a sequence in its last pages."""
    import torch
    from flashnext_b200.paged_q8 import kv_append_q8, kv_read_q8, paged_attention_q8

    page, block, kv, group, dim = 256, 128, 8, 2, 256
    pages = (1 << 32) // (page * kv * dim) + 5
    cache = _empty_cache(pages, page, block, kv, dim, "int8", fill=False)
    rng = np.random.default_rng(10)
    n = 300
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    slots = np.concatenate([(pages - 1) * page + np.arange(256), (pages - 3) * page + np.arange(n - 256)])
    x = [_bf16(rng.standard_normal((n, kv, dim))) for _ in range(2)]
    s = torch.from_numpy(slots).cuda()
    kv_append_q8(x[0].cuda(), x[1].cuda(), s, *cache)
    back = kv_read_q8(s, *cache)
    for i in range(2):
        assert float((back[i].float().cpu() - x[i].float()).abs().max()) < 0.5 * 6 / 127 + 6 * 2 ** -8
    ctx = torch.tensor([n], dtype=torch.int32, device="cuda")
    k, v = ((cache[i][[pages - 1, pages - 3]].float() * cache[2 + i][[pages - 1, pages - 3]].repeat_interleave(block, 1)[..., None])
            .reshape(-1, kv, dim)[:n].cpu().numpy() for i in range(2))
    for rows in (1, 100):
        q = _bf16(rng.standard_normal((rows, kv * group, dim)))
        cu = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        out = paged_attention_q8(q.cuda(), *cache, table, ctx, 0.0625, cu_q=cu).float().cpu().numpy()
        seen = np.arange(n)[None] <= (n - rows + np.arange(rows))[:, None]
        want, mag = oq8.attention(q.float().numpy(), k, v, seen, 0.0625)
        assert (np.abs(out - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * mag).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_serving_steps_match_attention_over_the_values_held(cuda_lib, kind):
    """Prompts, decodes, a verify step and a released row through
    PagedKVCacheQ8: after each step the attention equals float64 attention
    over the values that the cache then holds, read back by slot."""
    import torch
    from flashnext_b200.paged_q8 import PagedKVCacheQ8

    codes = torch.int8 if kind == "int8" else torch.float8_e4m3fn
    batch, kv, group, dim, page = 4, 2, 4, 64, 32
    cache = PagedKVCacheQ8(40, page, kv, dim, 10, batch, 512, block=16, codes=codes)
    rng = np.random.default_rng(12)
    lens = [0] * batch
    steps = [([70, 1, 0, 33], None), ([1, 1, 1, 1], None), ([4, 0, 7, 1], None), ([1, 1, 1, 50], [1, 0, 0, 0]),
             ([1, 1, 1, 1], None)]
    scale = 0.17
    for new, gone in steps:
        dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        plan = cache.plan(dev(new), None if gone is None else dev(gone))
        lens = [(0 if gone and gone[b] else lens[b]) + new[b] for b in range(batch)]
        n = sum(new)
        assert plan.seq_lens.tolist() == lens and plan.admitted.tolist() == [1] * batch
        x = [_bf16(rng.standard_normal((n, h, dim))).cuda() for h in (kv, kv, kv * group)]
        cache.append(x[0], x[1])
        out = cache.attention(x[2], scale, one_row=new == [1] * batch).float().cpu().numpy()
        q, table, at = x[2].float().cpu().numpy(), plan.block_table.cpu().numpy(), 0
        for b in range(batch):
            if new[b]:
                slots = torch.from_numpy(_slots(table, b, 0, lens[b], page)).cuda()
                c = [t.float().view(-1, kv, dim)[slots].cpu().numpy() for t in (cache.k, cache.v)]
                s = [t.view(-1, kv)[slots // 16].cpu().numpy()[:, :, None] for t in (cache.k_scale, cache.v_scale)]
                seen = np.arange(lens[b])[None] <= (lens[b] - new[b] + np.arange(new[b]))[:, None]
                want, mag = oq8.attention(q[at:at + new[b]], c[0] * s[0], c[1] * s[1], seen, scale)
                off = np.abs(out[at:at + new[b]] - want)
                assert (off <= 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * mag + 1e-30).all(), (b, new[b], lens[b])
                back = cache.read(slots)
                for i in range(2):
                    assert torch.equal(back[i].cpu().float(), _bf16(c[i] * s[i]).float())
            at += new[b]


@pytest.mark.gpu
def test_a_decode_step_replays_from_a_graph(cuda_lib):
    """Two steps (the two sets of buffers) captured and replayed: lengths grow
    on the device and the outputs equal those of eager calls."""
    import torch
    from flashnext_b200.paged_q8 import PagedKVCacheQ8

    def fresh():
        c = PagedKVCacheQ8(24, 32, 1, 128, 8, 3, 256)
        c.plan(torch.tensor([40, 7, 100], dtype=torch.int32, device="cuda"))
        g = torch.Generator(device="cuda")
        g.manual_seed(3)
        r = torch.randn(147, 1, 128, device="cuda", generator=g).bfloat16()
        c.append(r, 2 * r)
        return c

    one = torch.ones(3, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    k, q = torch.randn(3, 1, 128, device="cuda", generator=g).bfloat16(), torch.randn(3, 4, 128, device="cuda", generator=g).bfloat16()
    out = torch.empty(2, 3, 4, 128, dtype=torch.bfloat16, device="cuda")

    def two(c):
        for i in range(2):
            c.plan(one)
            c.append(k, k)
            c.attention(q, 0.09, one_row=True, out=out[i])

    eager = fresh()
    want = []
    for _ in range(3):
        two(eager)
        want.append(out.clone())
    c = fresh()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        two(c)  # warm-up: the stream's workspace
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        two(c)
    for i in (1, 2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
    assert c.last.seq_lens.tolist() == [46, 13, 106]


def test_cache_class_refuses_geometries():
    from flashnext_b200.paged_q8 import PagedKVCacheQ8

    import torch
    for kw, err in (({"page_size": 24}, ValueError), ({"block": 48}, ValueError), ({"head_dim": 96}, ValueError),
                    ({"codes": torch.uint8}, TypeError)):
        args = dict(num_pages=2, page_size=64, kv_heads=1, head_dim=64, max_pages_per_seq=1, batch=1, max_tokens=8,
                    device="cpu") | kw
        with pytest.raises(err):
            PagedKVCacheQ8(**args)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,most", [("int8", 0.03), ("e4m3", 0.08)])
def test_the_serving_example_stays_near_unquantised_attention(cuda_lib, kind, most):
    """The example's own comparison.  A code's rounding is uniform within half
    a code of the block's largest magnitude (about 4.5 of normal rows: 4.5 /
    127 / sqrt(12) = 1% of a value for int8; e4m3 keeps 4 bits, 2^-4 / sqrt(12)
    / 1.4 = 1.3% to 2.6% of each); keys and values each contribute, and the bound is
    about twice their sum."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "macqwen-releases_b200" / "examples" / "serve_q8.py"
    spec = importlib.util.spec_from_file_location("serve_q8", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(["--steps", "24", "--codes", kind]) < most
