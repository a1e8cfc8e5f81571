"""The draw of a token from logits (:func:`sample`)."""
from __future__ import annotations

import operator

import torch

from . import _lib
from .dense import _FLT_MAX, _float, _matrix, _ready_stream
from .paged_q8 import _want

MAX_VOCAB = _lib.SAMPLE_MAX_VOCAB


def _setting(v, dtype, rows, what, index):
    """(pointer of a [rows] tensor, or 0; value where it is a number)."""
    if isinstance(v, torch.Tensor):
        return _want(v, dtype, (rows,), what, index), 0
    return 0, v


def sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token a row of ``logits`` [rows, vocab] (bfloat16 or float32; rows may
    be slices of wider ones) from ``uniform`` [rows] float32 in [0, 1)
    -> ``(tokens [rows] int64, logprobs [rows] float32)``.

    Weights are ``exp((l - max l) / temperature)``.  Tokens are ranked by falling
    logit, equal ones by rising index, and kept while they are among the first
    ``top_k``, while the weight ranked before them is below ``top_p`` of the
    top-k's, and while their own weight is at least ``min_p`` (of the largest
    token's).  The token is the first, by index, at which the kept weights, it
    included, exceed ``uniform`` times their total; its log-probability is that
    among the kept.

    Each setting is a number or a [rows] tensor (float32; top_k int32), for
    requests with settings of their own.  ``top_k`` <= 0, ``top_p`` >= 1 and
    ``min_p`` <= 0 keep everything; ``temperature`` 0, ``top_k`` 1 or ``top_p``
    0 take the largest logit (log-probability 0).  Logits of -infinity and NaN
    are never taken; a row of nothing else has token -1.  The result does not
    depend on how the work is divided: weights are summed as exact integers,
    in units of 2^-44 of the largest token's.  So a log-probability is off by at
    most 2^-44 a kept token besides its rounding to float32: that of a token
    with almost all of the weight, itself near 0, has fewer significant digits.
    ``vocab`` is at most 262144.
    """
    index = logits.get_device()
    dtype = _float(logits, "logits")
    lp, rows, vocab, stride = _matrix(logits, "logits", index)
    f32 = torch.float32
    tp, t = _setting(temperature, f32, rows, "temperature", index)
    kp, k = _setting(top_k, torch.int32, rows, "top_k", index)
    pp, p = _setting(top_p, f32, rows, "top_p", index)
    mp, m = _setting(min_p, f32, rows, "min_p", index)
    if not tp and not 0.0 <= t <= _FLT_MAX:
        raise ValueError("temperature must be finite and not negative")
    if not kp and not -2 ** 31 <= operator.index(k) < 2 ** 31:
        raise ValueError("top_k must fit 32 bits")
    if not pp and not 0.0 <= p <= _FLT_MAX:
        raise ValueError("top_p must be finite and not negative")
    if not mp and not 0.0 <= m <= 1.0:
        raise ValueError("min_p must be between 0 and 1")
    up = _want(uniform, f32, (rows,), "uniform", index)
    stream = _ready_stream(index)
    device = logits.device
    tokens = torch.empty_strided((rows,), (1,), dtype=torch.int64, device=device)
    logprobs = torch.empty_strided((rows,), (1,), dtype=f32, device=device)
    code = _lib.packed["fnmoe_sample"](_lib.pack_sample(
        _lib.ABI_VERSION, rows, vocab, dtype, lp, stride, up, tp, kp, pp, mp, t, k, p, m, tokens.data_ptr(),
        logprobs.data_ptr()), stream)
    if code:
        _lib.check(code, "sample")
    return tokens, logprobs
