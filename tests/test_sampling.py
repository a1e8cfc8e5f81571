"""The draw of a token from logits.

CPU: refusals, and the oracle against hand-made cases.
GPU: tokens equal to the float64 oracle's -- integer sums of weights to 2^-45 of
the largest leave a border between two tokens uncertain by less than 2^-30 of
the total, and no input here lies that near one unless it is exactly on it by
construction -- and log-probabilities within their rounding to float32 and the
sums' 2^-30.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from flashnext_b200 import _lib
from oracle import dense as od

INF = math.inf


# ---- CPU ----


def test_oracle_on_small_rows():
    z = [1.0, 3.0, 3.0, -INF, math.nan, 2.0]
    assert od.sample(z, 0.5, temperature=0.0) == (1, 0.0)
    assert od.sample(z, 0.5, top_k=1)[0] == 1 and od.sample(z, 0.5, top_p=0.0)[0] == 1
    assert od.sample([-INF, math.nan], 0.1) == (-1, 0.0)
    # two equal tokens kept: a half each, the border belongs to the second
    assert od.sample(z, 0.49, top_k=2) == (1, -math.log(2)) and od.sample(z, 0.5, top_k=2) == (2, -math.log(2))
    assert od.sample([0.0] * 10, 0.999, top_p=0.5)[0] == 4  # five of ten
    assert od.sample([0.0, -1.0, -2.0], 0.999999, min_p=0.2)[0] == 1  # e^-1 = 0.37, e^-2 = 0.14
    assert od.sample([INF, 0.0, INF], 0.6) == (2, -math.log(2))


def test_sample_refuses_before_any_device_call():
    lib = _lib.load()
    a = _lib.FnSampleArgs(_lib.ABI_VERSION, 4, 100, 1, 0x1000, 100, 0x2000, None, None, None, None, 1.0, 0, 1.0, 0.0, 0x3000,
                          0x4000)

    def run(**kw):
        b = _lib.FnSampleArgs.from_buffer_copy(a)
        for k, v in kw.items():
            setattr(b, k, v)
        return lib.fnmoe_sample(ctypes.byref(b), None)

    for kw, code in (({"abi_version": 1}, _lib.ERR_ABI), ({"vocab": 0}, _lib.ERR_SHAPE), ({"vocab": 262145}, _lib.ERR_SHAPE),
                     ({"rows": 1 << 28}, _lib.ERR_SHAPE), ({"logits_dtype": 2}, _lib.ERR_UNSUPPORTED),
                     ({"logits": None}, _lib.ERR_NULL), ({"uniform": None}, _lib.ERR_NULL), ({"tokens": None}, _lib.ERR_NULL),
                     ({"logits_stride": 99}, _lib.ERR_SHAPE), ({"logits": 0x1002}, _lib.ERR_VALUE),
                     ({"uniform": 0x2001}, _lib.ERR_VALUE), ({"temperatures": 0x2002}, _lib.ERR_VALUE),
                     ({"top_ks": 0x2002}, _lib.ERR_VALUE), ({"top_ps": 0x2002}, _lib.ERR_VALUE),
                     ({"min_ps": 0x2002}, _lib.ERR_VALUE), ({"tokens": 0x3004}, _lib.ERR_VALUE),
                     ({"logprobs": 0x4002}, _lib.ERR_VALUE)):
        assert run(**kw) == code, kw
    assert run(rows=0) == _lib.OK
    assert lib.fnmoe_sample(None, None) == _lib.ERR_NULL


def test_python_refuses_cpu_tensors():
    import torch

    from flashnext_b200 import sampling

    with pytest.raises(TypeError):
        sampling.sample(torch.zeros(2, 5), torch.zeros(2))
    with pytest.raises(TypeError):
        sampling.sample(torch.zeros(2, 5).half(), torch.zeros(2))


# ---- GPU ----

gpu = pytest.mark.gpu


def _gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    import torch

    from flashnext_b200 import sampling

    tokens, logprobs = sampling.sample(logits, u, temperature, top_k, top_p, min_p)
    assert tokens.dtype is torch.int64 and logprobs.dtype is torch.float32
    z, us = logits.float().cpu().numpy(), u.cpu().numpy()
    at = lambda v, i: v[i].item() if isinstance(v, torch.Tensor) else (v if isinstance(v, int) else float(np.float32(v)))  # noqa: E731
    got, lps = tokens.cpu().tolist(), logprobs.cpu().tolist()
    for i in range(z.shape[0]):
        want, lp = od.sample(z[i], float(us[i]), *(at(v, i) for v in (temperature, top_k, top_p, min_p)))
        assert got[i] == want, (i, got[i], want)
        assert abs(lps[i] - lp) <= 2.0 ** -23 * abs(lp) + 2.0 ** -28, (i, lps[i], lp)
    return tokens


def _rows(rows, vocab, dtype, seed, scale=2.5):
    import torch

    g = _gen(seed)
    x = (scale * torch.randn(rows, vocab, device="cuda", generator=g)).to(dtype)
    return x, torch.rand(rows, device="cuda", generator=g)


FORMS = [{}, {"temperature": 0.7}, {"temperature": 0.0}, {"top_k": 1}, {"top_k": 7}, {"top_k": 1500}, {"top_p": 0.9},
         {"top_p": 0.01}, {"top_p": 0.0}, {"min_p": 0.05}, {"min_p": 1.0}, {"top_k": 50, "top_p": 0.95, "min_p": 0.02},
         {"temperature": 3.0, "top_k": 5000, "top_p": 0.8}, {"temperature": 0.05, "top_p": 0.99}]


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,vocab,pad", [(3, 1, 0), (4, 2, 1), (5, 33, 0), (3, 1000, 7), (2, 8191, 0), (3, 20011, 5),
                                            (2, 65536, 0)])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_sample(cuda_lib, dtype, rows, vocab, pad, form):
    import torch

    x, u = _rows(rows, vocab + pad, getattr(torch, dtype), vocab + form)
    _check(x[:, :vocab], u, **FORMS[form])


@gpu
@pytest.mark.parametrize("rows,vocab", [(1, 262144), (2, 131072), (160, 5001), (400, 700)])
def test_sample_cluster_sizes_and_settings_a_row(cuda_lib, rows, vocab):
    import torch

    g = _gen(rows)
    x, u = _rows(rows, vocab, torch.float32, vocab)
    i = torch.arange(rows, device="cuda")
    rand = lambda: torch.rand(rows, device="cuda", generator=g)  # noqa: E731
    _check(x, u, torch.where(i % 5 == 4, 0.0, 0.3 + rand()),
           torch.where(i % 3 == 0, 0, 1 + (300 * rand()).int()).to(torch.int32),
           torch.where(i % 4 == 0, 1.0, rand()), torch.where(i % 2 == 0, 0.0, 0.3 * rand()))
    _check(x, u)


@gpu
@pytest.mark.parametrize("vocab", [5, 1024, 3000, 40000])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_ties(cuda_lib, vocab, form):
    """Constant rows, rows of two values, and of a few: the boundary lies inside a run of equal logits."""
    import torch

    x = torch.zeros(4, vocab, device="cuda")
    x[1] = 3.25
    x[2, ::3] = 1.0
    x[3] = torch.randint(0, 4, (vocab,), device="cuda", generator=_gen(vocab)).float() - 2.0
    x[0, ::2] = -0.0  # equal to 0
    u = torch.tensor([0.0, 0.999, 0.4321, 0.77], device="cuda")
    _check(x, u, **FORMS[form])


@gpu
def test_exact_borders(cuda_lib):
    """u times the total exactly on a border takes the next token; the largest u the last one."""
    import torch

    n = 1024
    u = torch.arange(n, device="cuda", dtype=torch.float32) / n
    tokens = _check(torch.zeros(n, n, device="cuda"), u)
    assert torch.equal(tokens, torch.arange(n, device="cuda"))
    u = torch.tensor([1.0 - 2.0 ** -24, 0.0, 1.0, 2.0, -1.0, math.nan, math.inf], device="cuda")
    x = torch.zeros(7, 77, device="cuda")
    x[:, -5:] = -INF
    x[:, :2] = -INF
    from flashnext_b200 import sampling

    assert sampling.sample(x, u)[0].tolist() == [71, 2, 71, 71, 2, 2, 71]


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_masked_infinite_and_missing(cuda_lib, dtype, form):
    import torch

    from flashnext_b200 import sampling

    x, u = _rows(9, 9001, getattr(torch, dtype), form)
    low = torch.finfo(x.dtype).min
    x[0, 10:] = -INF          # few left
    x[1, :] = -INF
    x[1, 8123] = -3.0         # one left
    x[2, ::2] = math.nan
    x[3, 77] = INF            # infinite logits share everything
    x[3, 5000] = INF
    x[4, 3:] = low            # masked with the type's lowest value
    x[5, :] = low             # all of them
    x[6, 100] = 60000.0       # an outlier far above
    x[7, 5] = -1e30           # and one far below
    x[8, :] = -INF            # nothing left
    tokens = _check(x, u, **FORMS[form])
    assert tokens[8] == -1 and tokens[1] == 8123 and tokens[3] in (77, 5000)
    x[:, :] = math.nan
    assert (sampling.sample(x, u, **FORMS[form])[0] == -1).all()


@gpu
def test_settings_out_of_range_a_row(cuda_lib):
    """What the tensors of settings may hold although numbers are refused: not a number, negative, beyond 1, infinite."""
    import torch

    from flashnext_b200 import sampling

    x, u = _rows(8, 500, torch.float32, 3)
    f = lambda *v: torch.tensor(v, device="cuda", dtype=torch.float32)  # noqa: E731
    one = f(*[1.0] * 8)
    t = f(-1.0, math.nan, INF, 1e-45, 1e38, 1.0, 1.0, 1.0)
    got = sampling.sample(x, u, t)[0]
    assert torch.equal(got[[0, 1, 3]], x.argmax(1)[[0, 1, 3]])
    flat = [int(v * 500) for v in u[[2, 4]].tolist()]  # every token the same weight
    assert got[[2, 4]].tolist() == flat
    p = f(-1.0, math.nan, INF, 5.0, 1.0, 0.5, 0.5, 0.5)
    got = sampling.sample(x, u, one, 0, p)[0]
    assert torch.equal(got[:2], x.argmax(1)[:2]) and torch.equal(got[2:5], sampling.sample(x, u)[0][2:5])
    m = f(-1.0, math.nan, 2.0, INF, 1.0, 0.0, 0.0, 0.0)
    got = sampling.sample(x, u, one, 0, one, m)[0]
    assert torch.equal(got[:2], sampling.sample(x, u)[0][:2]) and torch.equal(got[2:5], x.argmax(1)[2:5])
    k = torch.tensor([-2 ** 31, -1, 0, 500, 501, 2 ** 31 - 1, 499, 1], device="cuda", dtype=torch.int32)
    got = sampling.sample(x, u, one, k)[0]
    assert torch.equal(got[:6], sampling.sample(x, u)[0][:6]) and got[7] == x[7].argmax()


@gpu
def test_draws_follow_the_weights(cuda_lib):
    """Evenly spaced u take each token as often as its probability says, to within one."""
    import torch

    from flashnext_b200 import sampling

    n, vocab = 4000, 300
    x = _rows(1, vocab, torch.float32, 8)[0].expand(n, vocab)
    x = x.contiguous()
    u = (torch.arange(n, device="cuda", dtype=torch.float32) + 0.5) / n
    for kw in ({}, {"top_k": 40}, {"temperature": 0.5, "top_p": 0.9}):
        count = torch.bincount(sampling.sample(x, u, **kw)[0], minlength=vocab).double()
        w = torch.exp(x[0].double() / kw.get("temperature", 1.0))
        order = w.argsort(descending=True)
        keep = torch.zeros(vocab, dtype=torch.bool, device="cuda")
        if "top_k" in kw:
            keep[order[:40]] = True
        elif "top_p" in kw:
            c = w[order].cumsum(0)
            keep[order[c - w[order] < float(np.float32(0.9)) * c[-1]]] = True
        else:
            keep[:] = True
        p = torch.where(keep, w, 0.0)
        assert ((count - n * p / p.sum()).abs() <= 1.0 + 1e-6).all()


@gpu
def test_streams_graphs_and_refusals(cuda_lib):
    import torch

    from flashnext_b200 import sampling

    x, u = _rows(5, 30000, torch.float32, 11)
    t = torch.full((5,), 0.8, device="cuda")
    want = sampling.sample(x, u, t, 40, 0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = sampling.sample(x, u, t, 40, 0.9)
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = sampling.sample(x, u, t, 40, 0.9)
    graph.replay()
    assert torch.equal(held[0], want[0])
    t.zero_()
    graph.replay()
    assert torch.equal(held[0], x.argmax(1))
    assert sampling.sample(x[:0], u[:0])[0].shape == (0,)
    for call in (lambda: sampling.sample(x[0], u), lambda: sampling.sample(x, u[:4]), lambda: sampling.sample(x, u, t[:4]),
                 lambda: sampling.sample(x, u, -1.0), lambda: sampling.sample(x, u, math.nan), lambda: sampling.sample(x, u, min_p=1.5),
                 lambda: sampling.sample(x, u, top_p=-0.1), lambda: sampling.sample(x, u, top_k=2 ** 31),
                 lambda: sampling.sample(x.t(), u), lambda: sampling.sample(torch.zeros(1, 262145, device="cuda"), u[:1])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: sampling.sample(x, u.double()), lambda: sampling.sample(x, u, t.double()),
                 lambda: sampling.sample(x, u, top_k=t), lambda: sampling.sample(x.half(), u), lambda: sampling.sample(x, u.cpu())):
        with pytest.raises(TypeError):
            call()


@gpu
@pytest.mark.parametrize("sign", [1, -1])
def test_min_p_whose_logit_lies_next_to_zero(cuda_lib, sign):
    """The least kept logit, max l + T ln(min_p), within 1e-9 of 0: floats lie 1e-16 apart there and less, closer than
    any sum of the larger terms, and what lies well above it has to stay."""
    import torch

    temps = np.float32(0.9) + np.arange(2000, dtype=np.float32) * np.float32(2.0 ** -24)
    mins = np.float32(0.01) + np.arange(2000, dtype=np.float32) * np.float32(2.0 ** -30)
    hi = np.float32(-np.log(np.float64(mins[0])) * np.float64(temps[0]))
    least = np.float64(hi) + np.outer(temps.astype(np.float64), np.log(mins.astype(np.float64)))
    least = np.where(sign * least > 0, np.abs(least), np.inf)
    order = np.argsort(least, axis=None)[:48]
    i, j = np.unravel_index(order, least.shape)
    assert least[i, j].max() < 1e-8  # 1e-10 for the nearest
    x = torch.tensor([[float(hi), 3.0, 2.0, 1.0, 0.5, 0.0, -0.5, -1.0, 1e-20, -1e-20] * 400], device="cuda").repeat(48, 1)
    u = (torch.arange(48, device="cuda", dtype=torch.float32) + 0.5) / 48
    _check(x.contiguous(), u, torch.from_numpy(temps[i]).cuda(), 0, 1.0, torch.from_numpy(mins[j]).cuda())


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_many_infinite_and_far_apart_logits(cuda_lib, dtype, form):
    """More infinities than a list holds, and logits whose distance from the largest is past float32's range."""
    import torch

    x, u = _rows(4, 7001, getattr(torch, dtype), 50 + form)
    x[0, ::15] = INF                      # 467 of them
    x[1, ::3] = INF                       # 2334
    x[2, 4000:] = torch.finfo(x.dtype).min
    x[2, ::11] = torch.finfo(x.dtype).max
    x[3] *= 1e37
    _check(x, u, **FORMS[form])


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("vocab", [300, 500, 3000, 20000])
@pytest.mark.parametrize("spread", [1e-45, 1e-41, 1e-38, 2.9e-36, 1e-35, 1e-30])
def test_close_logits(cuda_lib, dtype, vocab, spread):
    """Logits that differ by so little that a range of them, or the ranges in one of their differences, is no float."""
    import torch

    step = max(spread, 2.0 ** -133) if dtype == "bfloat16" else spread  # the least bfloat16
    x = torch.zeros(6, vocab, device="cuda")
    x[0, ::2] = step
    x[1, vocab // 3] = step
    x[2] = torch.randint(0, 8, (vocab,), device="cuda", generator=_gen(vocab)).float() * step
    x[3, : 2 * vocab // 3] = -step
    x[4] = 1.0
    x[5, 1::3] = -step
    x[5, ::400] = -INF
    x = x.to(getattr(torch, dtype))
    u = torch.tensor([0.0, 0.999, 0.4321, 0.77, 0.5, 0.123], device="cuda")
    for form in ({"top_k": 250}, {"top_k": 300, "top_p": 0.7}, {"top_p": 0.5}, {"top_p": 0.99, "min_p": 0.5},
                 {"temperature": 1e-38, "top_p": 0.6}, {"temperature": 1e-38, "top_k": 280}):
        _check(x, u, **form)


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("ties", [100, 385, 450, 512, 600, 2500])
@pytest.mark.parametrize("temperature", [1e-45, 1e-40, 1e-38, 9e-38, 1e-37, 1e-30])
def test_small_temperatures(cuda_lib, dtype, ties, temperature):
    """The largest logit, 0, many times over: it alone weighs something, however far below the others lie."""
    import torch

    x = torch.full((3, 3000), -1.0, device="cuda")
    x[:, 7:7 + ties] = 0.0
    x[1, 2700:] = -1e-38
    x[2, ::5] = -2e-38
    u = torch.tensor([0.999, 0.3, 0.65], device="cuda")
    for form in ({"top_p": 0.5}, {"top_p": 0.97}, {"top_k": 400, "top_p": 0.8}, {"top_k": 2000}):
        _check(x.to(getattr(torch, dtype)), u, temperature=temperature, **form)


@gpu
def test_two_threads_with_rows_of_different_widths(cuda_lib):
    """A call's shared memory depends on its rows: what one thread sets for its own must not refuse another's."""
    import threading

    import torch

    from flashnext_b200 import dense, sampling

    def draw(rows, vocab):
        x, u = _rows(rows, vocab, torch.float32, vocab)
        return lambda: sampling.sample(x, u, 0.8, 50, 0.9)

    def norm(dim):
        x, w = torch.randn(3, dim, device="cuda"), torch.ones(dim, device="cuda")
        return lambda: dense.add_rms_norm(x, w)[:1]

    for jobs in ((draw(1, 1000), draw(64, 131072), draw(3, 40000)), (norm(13001), norm(16375), norm(14003))):
        want = [job() for job in jobs]
        torch.cuda.synchronize()
        start, wrong = threading.Barrier(len(jobs)), []

        def work(job, out):
            try:
                with torch.cuda.stream(torch.cuda.Stream()):
                    start.wait()
                    for _ in range(3000):
                        got = job()
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, out)):
                        wrong.append("another result")
            except Exception as e:  # noqa: BLE001
                wrong.append(str(e))

        threads = [threading.Thread(target=work, args=j) for j in zip(jobs, want)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong


def test_outputs_that_overlap_are_refused():
    """Rows of a call are drawn side by side: a token written over another row's inputs would change that row's draw."""
    lib = _lib.load()
    a = _lib.FnSampleArgs(_lib.ABI_VERSION, 4, 100, 1, 0x10000, 128, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, 1.0, 0, 1.0, 0.0,
                          0x7000, 0x8000)

    def run(**kw):
        b = _lib.FnSampleArgs.from_buffer_copy(a)
        for k, v in kw.items():
            setattr(b, k, v)
        return lib.fnmoe_sample(ctypes.byref(b), None)

    # 4 rows: 32 bytes of tokens, 16 of log-probabilities and of each setting, 1936 of logits (float32)
    for kw in ({"tokens": 0x10000}, {"tokens": 0x10788}, {"tokens": 0xFFE8}, {"logprobs": 0x1078C}, {"logprobs": 0xFFF4},
               {"tokens": 0x2008}, {"logprobs": 0x200C}, {"tokens": 0x2FE8}, {"logprobs": 0x3000}, {"tokens": 0x4000},
               {"logprobs": 0x4004}, {"tokens": 0x5008}, {"logprobs": 0x4FF4}, {"tokens": 0x5FE8}, {"logprobs": 0x6008},
               {"logprobs": 0x701C}, {"tokens": 0x8008}):
        assert run(**kw) == _lib.ERR_VALUE, kw
        assert "overlap" in _lib.last_error(lib)
