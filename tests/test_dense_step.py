"""The dense steps used together: a layer's chain of norm, 8-bit product, residual, norm, head and draw, and the
decoder example that runs them around the paged cache and the MoE block."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import numpy as np
import pytest

from oracle import dense as od

pytestmark = pytest.mark.gpu


def _np(t):
    return t.detach().float().double().cpu().numpy()


@pytest.mark.parametrize("rows", [1, 5, 64, 300])
def test_chain_against_the_oracle(cuda_lib, rows):
    """Each step against the oracle on the step's own inputs (bounds: tests/test_dense.py)."""
    import torch

    from flashnext_b200 import dense, sampling

    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    hidden, wide, vocab = 768, 1280, 5003
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, r, w = rand(rows, hidden).bfloat16(), rand(rows, hidden), 1 + 0.1 * rand(hidden)
    up, down = (dense.quantize_rows(rand(n, k) * k ** -0.5) for n, k in ((wide, hidden), (hidden, wide)))
    head = (rand(vocab, hidden) * hidden ** -0.5 * 3).bfloat16()
    n1 = dense.add_rms_norm(x, w, r, codes=torch.int8, keep=True)
    h = dense.linear(n1.codes, up[0], activation="silu", x_scale=n1.scales, weight_scale=up[1])
    hq, hs = dense.quantize_rows(h)
    stream = dense.linear(hq, down[0], residual=n1.residual, x_scale=hs, weight_scale=down[1], out_dtype=torch.float32)
    y = dense.add_rms_norm(stream, w).y
    logits = dense.linear(y.bfloat16(), head, out_dtype=torch.float32)
    u = torch.rand(rows, device="cuda", generator=g)
    tokens, logprobs = sampling.sample(logits, u, 0.7, 40, 0.9)

    want, s = od.add_rms_norm(_np(x), _np(w), _np(r))
    assert (np.abs(_np(n1.y) - want) <= np.abs(want) * (2.0 ** -8 + 2.0 ** -18)).all()
    assert (np.abs(_np(n1.residual) - s) <= np.abs(s) * 2.0 ** -23).all()
    want, _ = od.linear(_np(n1.codes), _np(up[0]), None, "silu", None, _np(n1.scales), _np(up[1]))
    a, _ = od.linear(_np(n1.codes), _np(up[0]), None, None, None, _np(n1.scales), _np(up[1]))
    assert (np.abs(_np(h) - want) <= np.abs(want) * 2.0 ** -8 + np.abs(a) * 2.0 ** -20 + 1e-30).all()
    want, _ = od.linear(_np(hq), _np(down[0]), None, None, _np(n1.residual), _np(hs), _np(down[1]))
    assert (np.abs(_np(stream) - want) <= (np.abs(want) + np.abs(_np(n1.residual))) * 2.0 ** -20).all()
    want, mag = od.linear(_np(y.bfloat16()), _np(head))
    assert (np.abs(_np(logits) - want) <= (hidden / 16 + 8) * 2.0 ** -22 * mag + np.abs(want) * 2.0 ** -20).all()
    z, us = logits.cpu().numpy(), u.cpu().numpy()
    for i in range(0, rows, max(1, rows // 32)):
        token, lp = od.sample(z[i], float(us[i]), float(np.float32(0.7)), 40, float(np.float32(0.9)))
        assert int(tokens[i]) == token and abs(float(logprobs[i]) - lp) <= 2.0 ** -23 * abs(lp) + 2.0 ** -28


def test_decoder_example_replays_what_it_runs(cuda_lib):
    """Replayed and launched steps draw the same tokens, and no device error is left."""
    import torch

    from flashnext_b200 import _lib

    path = Path(__file__).resolve().parents[1] / "macqwen-releases_b200" / "examples" / "decode_step.py"
    spec = importlib.util.spec_from_file_location("decode_step", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    _lib.read_device_errors()
    tokens, scores = mod.main(["--tokens", "12", "--batch", "5"])
    again, scores2 = mod.main(["--tokens", "12", "--batch", "5", "--eager"])
    assert tokens.shape == (13, 5) and torch.equal(tokens, again) and torch.equal(scores, scores2)
    assert (scores <= 0).all() and ((tokens >= 0) & (tokens < mod.VOCAB)).all()
    assert _lib.read_device_errors() == 0
