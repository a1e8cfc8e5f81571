"""Paged KV cache in 8 bits: page planning, quantising append, attention.

Keys and values are codes of 8 bits (int8, or float8 e4m3) in HBM pages
``[pages, page_size, kv_heads, head_dim]`` with one float32 scale for each
``block`` consecutive tokens of a page and each kv head; a stored value is
``code * scale``.  Half the bytes of the bfloat16 cache of
:mod:`~flashnext_b200.paged_attention`, so about twice the contexts in a GPU's
memory and half the time of a decode step, which reads the cache once.

* :func:`page_plan` builds a serving step's block tables and slot map on the
  device from the requests' lengths (the bookkeeping of ``PagedKVCache``,
  ``models/qwen27b/paged_kv.py:54-400``, without a host read);
* :func:`kv_append_q8` quantises the step's K/V rows into their slots;
* :func:`paged_attention_q8` is ``paged_attention``'s computation
  (``paged_kv.py:417-495``) over such a cache, causal, for one query row per
  sequence or packed rows (multi-token verify, prefill chunks);
* :func:`kv_read_q8` takes values out as bfloat16;
* :class:`PagedKVCacheQ8` keeps the buffers and runs the four together.

Every call is ordered on torch's current stream and reads nothing on the
host, so a step can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes
import threading
from dataclasses import dataclass
from typing import Any

import torch

from . import _lib

BLOCKS = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)
_CODES = {torch.int8: _lib.Q8_INT8, torch.float8_e4m3fn: _lib.Q8_E4M3}


@dataclass(slots=True)
class PagePlan:
    """A serving step's pages and slots (:func:`page_plan`)."""

    block_table: Any  # [batch, max_pages] int32, -1 in unused cells
    seq_lens: Any     # [batch] int32, the admitted tokens included
    free_pages: Any   # [pages] int32 ring of free pages
    free_state: Any   # [2] int32: head of the ring, free pages
    slot_map: Any     # [max_tokens] int64 slot of each packed new token, -1 past the last
    token_seq: Any    # [max_tokens] int32 its sequence, or -1
    positions: Any    # [max_tokens] int32 its position, or -1
    cu_new: Any       # [batch + 1] int32 first packed token of each sequence
    admitted: Any     # [batch] int32: 0 where pages, tokens or table columns ran out


def _elsewhere(t, index, what):
    raise ValueError(f"{what} is on device {t.get_device()}, the call's other tensors are on device {index}")


def _refuse(t, dtype, shape, what, index):
    if t.dtype != dtype or not t.is_cuda:
        raise TypeError(f"{what} must be a {dtype} CUDA tensor")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, not {tuple(shape)}")
    if t.get_device() != index:
        _elsewhere(t, index, what)
    raise ValueError(f"{what} must be contiguous")


def _want(t, dtype, shape, what, index):
    """Pointer of a contiguous tensor of this type and shape on CUDA device ``index``."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == index >= 0 and t.is_contiguous():
        return t.data_ptr()
    _refuse(t, dtype, shape, what, index)


def _rows(t, heads, dim, what, index):
    """Pointer and token stride of bfloat16 rows [n, heads, dim]; a row is contiguous, rows may be apart."""
    if t.dtype is not torch.bfloat16 or not t.is_cuda:
        raise TypeError(f"{what} must be a bfloat16 CUDA tensor")
    if t.get_device() != index:
        _elsewhere(t, index, what)
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim:
        raise ValueError(f"{what} must be [tokens, {heads}, {dim}], not {tuple(shape)}")
    if shape[0] < 2 and t.is_contiguous():
        return t.data_ptr(), heads * dim
    s0, s1, s2 = t.stride()
    if (s2 != 1 and dim > 1) or (s1 != dim and heads > 1):
        raise ValueError(f"{what}'s heads must be contiguous within a token")
    return t.data_ptr(), s0 if shape[0] > 1 else heads * dim


def _cache(k_cache, v_cache, k_scale, v_scale):
    """FnQ8Cache of the four tensors, (kv_heads, head_dim) and their device."""
    dtype, shape, scales, index = k_cache.dtype, k_cache.shape, k_scale.shape, k_cache.get_device()
    if len(shape) != 4 or len(scales) != 3:
        raise ValueError("caches must be [pages, page_size, kv_heads, head_dim] and scales "
                         "[pages, page_size / block, kv_heads]")
    pages, page, heads, dim = shape
    blocks = scales[1]
    if (k_scale.dtype is v_scale.dtype is torch.float32 and v_cache.dtype is dtype and dtype in _CODES
            and v_cache.shape == shape and v_scale.shape == scales and scales[0] == pages and scales[2] == heads
            and blocks and page % blocks == 0 and 0 <= index == v_cache.get_device() == k_scale.get_device()
            and index == v_scale.get_device() and k_cache.is_contiguous() and v_cache.is_contiguous()
            and k_scale.is_contiguous() and v_scale.is_contiguous()):
        return _lib.FnQ8Cache(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                              pages, page, page // blocks, heads, dim, _CODES[dtype]), heads, dim, index
    # say which
    if dtype not in _CODES:
        raise TypeError("k_cache must be an int8 or float8_e4m3fn tensor")
    if blocks == 0 or page % blocks:
        raise ValueError("a page must hold a whole number of scale blocks")
    ss, f32 = (pages, blocks, heads), torch.float32
    for t, d, x, what in ((k_cache, dtype, shape, "k_cache"), (v_cache, dtype, shape, "v_cache"),
                          (k_scale, f32, ss, "k_scale"), (v_scale, f32, ss, "v_scale")):
        _want(t, d, x, what, index)
    raise AssertionError("unreachable")


def _ready(t):
    """The library and the current stream of the current device, which must be ``t``'s."""
    index = t.get_device()
    if torch._C._cuda_getDevice() != index or not _lib._available.get(index):
        _lib.ensure_device_of(index)  # refuses, or starts the library up
    return _lib._handle, torch._C._cuda_getCurrentRawStream(index)


def page_plan(seq_lens, new_lens, block_table, free_pages, free_state, page_size: int, max_tokens: int,
              release=None, out: PagePlan | None = None) -> PagePlan:
    """Pages and slots for ``new_lens[b]`` more tokens of every sequence.

    ``seq_lens`` / ``new_lens`` / ``release`` [batch], ``block_table``
    [batch, max_pages], ``free_pages`` [pages] (a ring) and ``free_state`` [2]
    (head, count) are int32.  A row with ``release`` set has ended: its pages
    join the ring's end (to be given from the next call on) and the row
    starts over with its ``new_lens``.  Sequences are served in order;
    one whose pages or tokens do not fit has ``admitted`` 0 and keeps what it
    had.  ``free_pages`` is updated in place; the rest is written to ``out``
    (a plan of the same sizes, whose ``block_table`` may be the input) or to
    new tensors.
    """
    i32, batch = torch.int32, seq_lens.shape[0]
    if block_table.dim() != 2:
        raise ValueError("block_table must be [batch, max_pages]")
    width, max_tokens = block_table.shape[1], int(max_tokens)
    if batch == 0 or width == 0 or max_tokens <= 0:
        raise ValueError("page_plan needs sequences, table columns and max_tokens > 0")
    one, cells, two, at = seq_lens.shape, block_table.shape, (2,), seq_lens.get_device()
    ins = (_want(seq_lens, i32, one, "seq_lens", at), _want(new_lens, i32, one, "new_lens", at),
           None if release is None else _want(release, i32, one, "release", at),
           _want(block_table, i32, cells, "block_table", at),
           _want(free_pages, i32, (free_pages.numel(),), "free_pages", at), _want(free_state, i32, two, "free_state", at))
    if out is None:
        dev = seq_lens.device
        words = torch.empty(batch * (width + 3) + 1 + 2 + 2 * max_tokens, dtype=i32, device=dev)
        t, lens, state, seq, pos, cu, ok = words.split((batch * width, batch, 2, max_tokens, max_tokens, batch + 1, batch))
        out = PagePlan(t.view(cells), lens, free_pages, state, torch.empty(max_tokens, dtype=torch.int64, device=dev),
                       seq, pos, cu, ok)
    tok = (max_tokens,)
    a = _lib.FnPagePlanArgs(
        _lib.ABI_VERSION, batch, int(page_size), width, free_pages.shape[0], max_tokens, *ins,
        _want(out.block_table, i32, cells, "out.block_table", at), _want(out.seq_lens, i32, one, "out.seq_lens", at),
        _want(out.free_state, i32, two, "out.free_state", at), _want(out.slot_map, torch.int64, tok, "out.slot_map", at),
        _want(out.token_seq, i32, tok, "out.token_seq", at), _want(out.positions, i32, tok, "out.positions", at),
        _want(out.cu_new, i32, (batch + 1,), "out.cu_new", at), _want(out.admitted, i32, one, "out.admitted", at))
    lib, stream = _ready(seq_lens)
    _lib.check(lib.fnmoe_page_plan(ctypes.byref(a), stream), "page_plan")
    out.free_pages = free_pages
    return out


def kv_append_q8(k, v, slot_map, k_cache, v_cache, k_scale, v_scale) -> None:
    """Quantise rows ``k``, ``v`` [tokens, kv_heads, head_dim] (bfloat16; rows
    may be slices of a wider row) into the slots ``slot_map`` [tokens] int64.

    A block's scale is the largest magnitude it holds over the code type's
    largest value; a row that raises it has the block's earlier codes rounded
    again to the new scale.  Rows of one block must be adjacent with
    ascending slots, as :func:`page_plan` maps them; slots outside the cache
    (-1) are skipped.  Infinities store the largest code, NaN stores 0.
    """
    c, heads, dim, index = _cache(k_cache, v_cache, k_scale, v_scale)
    kp, ks = _rows(k, heads, dim, "k", index)
    vp, vs = _rows(v, heads, dim, "v", index)
    tokens = k.shape[0]
    if v.shape[0] != tokens:
        raise ValueError("k and v must have the same number of rows")
    a = _lib.FnQ8AppendArgs(_lib.ABI_VERSION, tokens, c, kp, vp, ks, vs,
                            _want(slot_map, torch.int64, (tokens,), "slot_map", index))
    lib, stream = _ready(k)
    _lib.check(lib.fnmoe_kv_append_q8(ctypes.byref(a), stream), "kv_append_q8")


def kv_read_q8(slots, k_cache, v_cache, k_scale, v_scale, out=None):
    """The values ``(k, v)`` that ``slots`` [n] int64 hold, bfloat16
    [n, kv_heads, head_dim]; slots outside the cache (-1) read as zeros."""
    c, heads, dim, index = _cache(k_cache, v_cache, k_scale, v_scale)
    n = slots.shape[0]
    at = _want(slots, torch.int64, (n,), "slots", index)
    if out is None:
        both = k_scale.new_empty((2, n, heads, dim), dtype=torch.bfloat16)
        ko = both.data_ptr()
        vo = ko + 2 * n * heads * dim
        out = both.unbind()
    else:
        shape = (n, heads, dim)
        ko, vo = (_want(t, torch.bfloat16, shape, f"out[{i}]", index) for i, t in enumerate(out))
    a = _lib.FnQ8ReadArgs(_lib.ABI_VERSION, n, c, at, ko, vo)
    lib, stream = _ready(slots)
    _lib.check(lib.fnmoe_kv_read_q8(ctypes.byref(a), stream), "kv_read_q8")
    return out


class _Scratch(threading.local):
    """Attention scratch that a thread keeps for each (device, stream).

    A thread's calls on one stream follow one another there and may share it.
    Two threads may not (a call is several launches, which interleave), nor may
    graphs: a captured call gets memory of its own from the graph's pool, which
    lives as long as the graph, and never the kept one, which is dropped when a
    later call needs more.
    """

    def __init__(self):
        self.kept = {}


_scratch = _Scratch()


def paged_attention_q8(q, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, scale: float, cu_q=None,
                       out=None, workspace=None):
    """Causal attention of bfloat16 rows ``q`` [rows, q_heads, head_dim]
    (rows may be slices of a wider row) over the cache; -> like ``q``.

    With ``cu_q`` [batch + 1] int32, rows ``cu_q[b] .. cu_q[b + 1]`` are the
    last tokens of sequence b's ``context_lens[b]``, each seeing the positions
    up to its own; without it, row b sees all of sequence b's context.  A row
    that sees nothing is 0, as are rows past ``cu_q[batch]``.  ``workspace``:
    a uint8 tensor of as many bytes as
    ``fnmoe_paged_attention_q8_workspace_size`` reports, which no other call
    uses at the same time; or None for one that this module keeps for the
    calling thread and stream (in a CUDA graph's capture: one of the graph's own).
    """
    c, _, head_dim, index = _cache(k_cache, v_cache, k_scale, v_scale)
    shape, table = q.shape, block_table.shape
    if len(shape) != 3:
        raise ValueError("q must be [rows, q_heads, head_dim]")
    rows, heads, dim = shape
    if dim != head_dim:
        raise ValueError("cache head_dim differs from q")
    qp, qs = _rows(q, heads, dim, "q", index)
    if len(table) != 2:
        raise ValueError("block_table must be [batch, max_pages]")
    batch, width = table
    if out is None:
        out = k_scale.new_empty(shape, dtype=torch.bfloat16)
        op = out.data_ptr()
    else:
        op = _want(out, torch.bfloat16, shape, "out", index)
    if workspace is not None:
        _want(workspace, torch.uint8, workspace.shape, "workspace", index)
    i32 = torch.int32
    a = _lib.FnQ8AttentionArgs(
        _lib.ABI_VERSION, batch, rows, heads, width, float(scale), c, qp, qs,
        _want(block_table, i32, table, "block_table", index), _want(context_lens, i32, (batch,), "context_lens", index),
        None if cu_q is None else _want(cu_q, i32, (batch + 1,), "cu_q", index), op)
    lib, stream = _ready(q)
    ref = ctypes.byref(a)
    capturing = workspace is None and torch.cuda.is_current_stream_capturing()
    given = workspace
    if given is None and not capturing:
        given = _scratch.kept.get((index, stream))
    if given is not None:
        a.workspace, a.workspace_bytes = given.data_ptr(), given.numel()
    code = lib.fnmoe_paged_attention_q8(ref, stream)
    if code == _lib.ERR_WORKSPACE and workspace is None:  # none yet, or too small a one
        need = ctypes.c_uint64(0)
        _lib.check(lib.fnmoe_paged_attention_q8_workspace_size(ref, ctypes.byref(need)), "paged attention q8 workspace")
        given = k_scale.new_empty((need.value,), dtype=torch.uint8)
        if not capturing:
            _scratch.kept[(index, stream)] = given
        a.workspace, a.workspace_bytes = given.data_ptr(), given.numel()
        code = lib.fnmoe_paged_attention_q8(ref, stream)
    _lib.check(code, "paged_attention_q8")
    return out


class PagedKVCacheQ8:
    """Pages, scales, block tables and free ring of one attention layer's
    8-bit cache, and a serving step over them:

        plan = cache.plan(new_lens, release)   # tables and slots on the device
        cache.append(k, v)                     # the step's packed rows
        out = cache.attention(q, scale)        # causal, packed like k and v

    ``batch`` rows of at most ``max_pages_per_seq`` pages; ``max_tokens`` new
    tokens a step.  Nothing is read on the host: a sequence that does not fit
    has ``plan.admitted`` 0 and takes no part in the step, so its rows must not
    be among those packed (``plan.cu_new`` counts them as none): where that can
    happen, :meth:`pack` takes them out on the device.  Tables and
    lengths alternate between two sets of buffers; a captured CUDA graph
    therefore holds an even number of plans.
    """

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, max_pages_per_seq: int,
                 batch: int, max_tokens: int, block: int | None = None, codes=torch.int8, device="cuda"):
        if codes not in _CODES:
            raise TypeError("codes must be torch.int8 or torch.float8_e4m3fn")
        block = block or next((b for b in reversed(BLOCKS) if page_size % b == 0), 0)
        if block not in BLOCKS or page_size % block:
            raise ValueError(f"page_size must be a multiple of a block of {BLOCKS} tokens")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
        i32 = torch.int32
        # zeros: e4m3 slots that are never written stay finite
        self.k, self.v = (torch.zeros((num_pages, page_size, kv_heads, head_dim), dtype=torch.uint8, device=device).view(codes)
                          for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros((num_pages, page_size // block, kv_heads), device=device) for _ in range(2))
        self.free_pages = torch.arange(num_pages, dtype=i32, device=device)
        self.page_size, self.max_tokens = page_size, int(max_tokens)

        def buffers():
            return PagePlan(torch.full((batch, max_pages_per_seq), -1, dtype=i32, device=device),
                            torch.zeros(batch, dtype=i32, device=device), self.free_pages,
                            torch.tensor([0, num_pages], dtype=i32, device=device),
                            torch.full((self.max_tokens,), -1, dtype=torch.int64, device=device),
                            *(torch.full((self.max_tokens,), -1, dtype=i32, device=device) for _ in range(2)),
                            torch.zeros(batch + 1, dtype=i32, device=device),
                            torch.ones(batch, dtype=i32, device=device))

        self.last, self._other = buffers(), buffers()

    @property
    def tensors(self):
        """(k, v, k_scale, v_scale), as the functions of this module take them."""
        return self.k, self.v, self.k_scale, self.v_scale

    def plan(self, new_lens, release=None) -> PagePlan:
        """Give every row ``new_lens[b]`` more tokens (rows with ``release`` set start over)."""
        was = self.last
        self.last = page_plan(was.seq_lens, new_lens, was.block_table, self.free_pages, was.free_state, self.page_size,
                              self.max_tokens, release=release, out=self._other)
        self._other = was
        return self.last

    def pack(self, x, first):
        """The last plan's rows among ``x`` [n, ...], in which each row of the
        table has its ``new_lens[b]`` rows from ``first[b]`` on ([batch] int32),
        whether or not it was admitted.  -> [min(n, max_tokens), ...]: the
        admitted rows as :meth:`append` and :meth:`attention` want them; those
        past ``plan.cu_new[batch]`` repeat others, are stored nowhere and come
        back from the attention as zeros."""
        p, n = self.last, min(x.shape[0], self.max_tokens)
        seq = p.token_seq[:n].clamp(min=0).long()
        at = first[seq] + torch.arange(n, device=x.device) - p.cu_new[seq]
        return x[at.clamp(0, max(x.shape[0] - 1, 0))]

    def append(self, k, v) -> None:
        """Store the last plan's packed rows [tokens, kv_heads, head_dim]."""
        kv_append_q8(k, v, self.last.slot_map[: k.shape[0]], *self.tensors)

    def attention(self, q, scale: float, one_row: bool = False, out=None):
        """Attention of the last plan's packed rows [tokens, q_heads, head_dim];
        ``one_row``: every row of the table has exactly one (a decode step)."""
        p = self.last
        return paged_attention_q8(q, *self.tensors, p.block_table, p.seq_lens, scale,
                                  cu_q=None if one_row else p.cu_new, out=out)

    def read(self, slots):
        """The bfloat16 (k, v) that slots hold (:func:`kv_read_q8`)."""
        return kv_read_q8(slots, *self.tensors)
